"""What a call into the library uses lives until the call returns: seen from inside the call, with the library's entry points replaced (no GPU)."""
import weakref

import pytest
import torch

import kudnn_amd as K
import kudnn_amd.torch_moe as km

F8 = torch.float8_e4m3fn


class Entries:
    """The library, with `inside(name, handle)` in place of what would launch."""

    def __init__(self, real, inside):
        self.real, self.inside = real, inside

    def __getattr__(self, name):
        if not name.endswith(("_run", "_backward", "_backward_input", "_backward_weight")):
            return getattr(self.real, name)
        return lambda handle, *args: self.inside(name, handle) or 0


@pytest.fixture
def calls(monkeypatch):
    """Host tensors pass for the GPU's, and no plan stays in the cache, as after 256 others. -> what to do inside a call, and which there were."""
    seen, inside = [], []

    def enter(name, handle):
        seen.append(name)
        for f in inside:
            f(handle)

    entries = Entries(K.lib(), enter)
    monkeypatch.setattr(K, "lib", lambda: entries)
    monkeypatch.setattr(km, "lib", lambda: entries)
    monkeypatch.setattr(km, "_gpu", lambda *a: None)
    monkeypatch.setattr(km, "_current", lambda: None)
    monkeypatch.setattr(km, "_stream", lambda index: 0)
    monkeypatch.setattr(km, "MAX_CACHED_PLANS", 0)
    return inside, seen


def run_everything():
    order = torch.zeros(3, dtype=torch.int32)
    rows, slots = torch.zeros(200, dtype=torch.int32), torch.zeros(100, 2, dtype=torch.int32)
    for normalize in (True, False):
        logits = torch.randn(100, 2, requires_grad=True)
        km.route(logits, 2, normalize).weights.sum().backward()
    x, w = torch.randn(100, 9).bfloat16().requires_grad_(True), torch.randn(2, 11, 9).bfloat16().requires_grad_(True)
    km.grouped_linear(x, w, order, rows, slots).sum().backward()
    y, weights = torch.randn(200, 8, requires_grad=True), torch.rand(100, 2, requires_grad=True)
    km.combine(y, weights, slots).sum().backward()
    km.grouped_linear_fp8(torch.randn(100, 9).bfloat16(), torch.zeros(2, 11, 9).to(F8), torch.ones(2, 1, 1), order, rows)


def test_plans_outlive_their_calls(calls, monkeypatch):
    inside, seen = calls
    made = []
    plan_of = km._plan

    def plan(key, make):
        p = plan_of(key, make)
        made.append(weakref.ref(p))
        return p

    monkeypatch.setattr(km, "_plan", plan)

    def alive(handle):
        assert any(p() is not None and p().handle is handle for p in made), f"{seen[-1]}: its plan was destroyed before it"

    inside.append(alive)
    run_everything()
    assert {n.replace("kudnn_", "") for n in seen} == {"moe_route_run", "moe_route_backward", "grouped_linear_run", "grouped_linear_backward_input",
                                                       "grouped_linear_backward_weight", "moe_combine_run", "moe_combine_backward", "linear_fp8_run"}


def test_workspaces_outlive_their_calls(calls, monkeypatch):
    inside, seen = calls
    given, had = [], set()
    workspace_of = km._workspace

    def workspace(plan, device):
        w = workspace_of(plan, device)
        given.append((plan.handle, None if w is None else weakref.ref(w)))
        return w

    monkeypatch.setattr(km, "_workspace", workspace)

    def alive(handle):
        for of, w in given:
            if of is handle and w is not None:
                had.add(seen[-1])
                assert w() is not None, f"{seen[-1]}: its workspace went back to the allocator before it"

    inside.append(alive)
    run_everything()
    assert {"kudnn_moe_route_run", "kudnn_grouped_linear_backward_input", "kudnn_grouped_linear_backward_weight", "kudnn_linear_fp8_run"} <= had
