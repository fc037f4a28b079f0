"""Sizes that plans of the mixture-of-experts operators accept can be launched: a grid has fewer than 2^32 threads (no GPU)."""
import random
import re

import pytest

import kudnn_amd as K


def accepted(make):
    try:
        return make()
    except K.KudnnError as e:
        assert e.status == K.UNSUPPORTED
        return None


def test_router_tokens():
    d = lambda t, e: K.desc([t, e], K.BF16)
    most = ((1 << 23) - 1) * 64                     # workgroups of 512 threads for 64 tokens each
    assert accepted(lambda: K.MoeRoute(d(most, 2), 1)) and not accepted(lambda: K.MoeRoute(d(most + 1, 2), 1))
    assert accepted(lambda: K.MoeRoute(d(1 << 27, 1024), 8)) and not accepted(lambda: K.MoeRoute(d(1 << 28, 1024), 8))   # T k < 2^31
    assert not accepted(lambda: K.MoeRoute(d(1 << 60, 8), 8))


def test_router_launches():
    """The counts of many workgroups are summed in launches of their own, so that a call's work grows as its tokens."""
    d = lambda t: K.desc([t, 9], K.F32)
    few, many = K.MoeRoute(d(768 * 64), 3), K.MoeRoute(d(768 * 64 + 1), 3)
    assert "launches=2" in few.describe() and few.workspace_bytes == 768 * 12
    assert "launches=4" in many.describe() and many.workspace_bytes == 769 * 12 + (7 + 1) * 12 * 4


def test_weighted_sum_tokens():
    d = lambda t: K.desc([t, 8], K.F32)
    assert accepted(lambda: K.MoeCombine(d(1 << 24), d((1 << 31) - 1), 64)) and not accepted(lambda: K.MoeCombine(d(1 << 24), d(1 << 31), 2))


def grouped(R, E, N, K_, f8, c=K.BF16):
    if f8:
        return K.LinearFp8(K.desc([R, K_], K.F8E4M3), K.desc([E, K_, N], K.F8E4M3, "ACB"), K.desc([R, N], c), None, True)
    return K.GroupedLinear(K.desc([R, K_], K.BF16), K.desc([E, K_, N], K.BF16, "ACB"), K.desc([R, N], K.BF16))


def threads(plan, R, E, N):
    """Of the launch that the plan describes, from its tile."""
    m = re.search(r"tile=(stream|ring|pingpong)(\d+)x(\d+)(?:/(\d+))?", plan.describe())
    kind, bm, bn, form = m.group(1), int(m.group(2)), int(m.group(3)), m.group(4)
    groups = min(E + 1, R)
    rows = groups + (R - groups) // bm
    return rows * -(-N // bn) * {"stream": 64 * int(form or 0), "ring": 256 if bm == 64 else 512, "pingpong": 512}[kind]


@pytest.mark.parametrize("f8", [False, True])
def test_grouped_products(f8):
    assert accepted(lambda: grouped(1 << 22, 8, 4096, 256, f8)) and not accepted(lambda: grouped(1 << 22, 8, 1 << 18, 256, f8))
    assert f8 or not accepted(lambda: grouped(16, 1 << 20, 960, 128, f8))      # the weight gradient's tiles of every expert
    rng = random.Random(5)
    size = lambda lo, hi: int(2 ** rng.uniform(lo, hi))
    some = 0
    for _ in range(3000):
        R, E, N, K_ = size(0, 30), size(0, 20), size(0, 24), size(4, 14)
        plan = accepted(lambda: grouped(R, E, N, K_, f8, rng.choice([K.BF16, K.F32])))
        if plan is not None:
            assert threads(plan, R, E, N) < 1 << 32, (R, E, N, K_, plan.describe())
            some += threads(plan, R, E, N) > 1 << 30
    assert some > 20                                                           # the limit was near


def test_gradient_of_gathered_rows_refuses_in_the_forward_pass(monkeypatch):
    """The sum over a token's slots takes 64 of them: more are refused before the product, not in its backward pass."""
    import torch

    import kudnn_amd.torch_moe as km
    monkeypatch.setattr(km, "_gpu", lambda *a: None)
    x, w = torch.zeros(2, 8).bfloat16().requires_grad_(True), torch.zeros(2, 8, 8).bfloat16()
    with pytest.raises(ValueError, match="k up to 64"):
        km.grouped_linear(x, w, torch.zeros(3, dtype=torch.int32), torch.zeros(130, dtype=torch.int32), torch.zeros(2, 65, dtype=torch.int32))
