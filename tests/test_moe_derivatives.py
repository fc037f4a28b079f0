"""Derivatives that the mixture-of-experts operators do not have are refused, not dropped (no GPU: the launches are replaced)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import kudnn_amd.torch_moe as km
from test_moe_lifetimes import F8, calls  # noqa: F401 (a fixture)

ORDER = torch.zeros(3, dtype=torch.int32)
SLOTS = torch.zeros(4, 2, dtype=torch.int32)


def dual(*shape, dtype=torch.bfloat16):
    return forward_ad.make_dual(torch.randn(*shape).to(dtype), torch.ones(*shape, dtype=dtype))


FORWARD = {
    "route": lambda t: km.route(t(5, 4), 2),
    "grouped_linear x": lambda t: km.grouped_linear(t(4, 8), torch.zeros(2, 8, 8).bfloat16(), ORDER),
    "grouped_linear weight": lambda t: km.grouped_linear(torch.zeros(4, 8).bfloat16(), t(2, 8, 8), ORDER),
    "combine y": lambda t: km.combine(t(8, 8), None, SLOTS),
    "combine weights": lambda t: km.combine(torch.zeros(8, 8), t(4, 2, dtype=torch.float32), SLOTS),
    "linear_fp8": lambda t: km.linear_fp8(t(4, 8), torch.zeros(8, 8).to(F8), torch.ones(1, 1)),
    "linear_fp8 bias": lambda t: km.linear_fp8(torch.zeros(4, 8).bfloat16(), torch.zeros(8, 8).to(F8), torch.ones(1, 1), t(8)),
    "grouped_linear_fp8": lambda t: km.grouped_linear_fp8(t(4, 8), torch.zeros(2, 8, 8).to(F8), torch.ones(2, 1, 1), ORDER),
}


@pytest.mark.parametrize("name", list(FORWARD))
def test_forward_mode_is_refused(calls, name):  # noqa: F811
    with forward_ad.dual_level():
        FORWARD[name](lambda *s, dtype=torch.bfloat16: torch.randn(*s).to(dtype))     # no tangent: an ordinary call
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                FORWARD[name](dual)


@pytest.mark.parametrize("name", [n for n in FORWARD if "fp8" in n])
def test_8_bit_products_refuse_a_gradient(calls, name):  # noqa: F811
    given = lambda *s, dtype=torch.bfloat16: torch.randn(*s).to(dtype).requires_grad_(True)
    y = FORWARD[name](given)                    # serving without no_grad: the result is there
    with pytest.raises(RuntimeError, match="forward only"):
        y.float().sum().backward()
    with torch.no_grad():
        assert not FORWARD[name](given).requires_grad
    assert not FORWARD[name](lambda *s, dtype=torch.bfloat16: torch.randn(*s).to(dtype)).requires_grad


def test_8_bit_layer_refuses_a_gradient(calls, monkeypatch):  # noqa: F811
    monkeypatch.setattr(km, "quantize_blocks", lambda w: (w.to(F8), torch.ones(w.shape[0], 1, 1)))
    layer = km.MoEMlp(8, 16, 4, 2).quantized()
    x = torch.randn(3, 8).bfloat16().requires_grad_(True)
    with pytest.raises(RuntimeError, match="forward only"):
        layer(x).float().sum().backward()
    with torch.no_grad():
        assert not layer(x).requires_grad
    assert not layer(x.detach()).requires_grad


@pytest.mark.parametrize("tokens", [3, 0])
def test_layers_make_no_library_products(calls, monkeypatch, tokens):  # noqa: F811
    """The router's logits and their gradients come from the framework's own products."""
    def library(*a, **kw):
        raise AssertionError("a library product")

    for name in ("linear", "bilinear"):
        monkeypatch.setattr(torch.nn.functional, name, library)
    for name in ("matmul", "mm", "bmm", "addmm", "einsum"):
        monkeypatch.setattr(torch, name, library)
        if hasattr(torch.Tensor, name):
            monkeypatch.setattr(torch.Tensor, name, library)
    monkeypatch.setattr(torch.Tensor, "__matmul__", library)
    monkeypatch.setattr(km, "quantize_blocks", lambda w: (w.to(F8), torch.ones(w.shape[0], 1, 1)))
    _, seen = calls
    layer = km.MoEMlp(8, 16, 4, 2)
    x = torch.randn(tokens, 8).bfloat16().requires_grad_(True)
    layer(x).float().sum().backward()
    assert layer.router.grad.shape == (4, 8) and x.grad.shape == (tokens, 8)
    assert seen.count("kudnn_grouped_linear_run") == 3 and seen.count("kudnn_grouped_linear_backward_weight") == 3
    with torch.no_grad():
        layer(x), layer.quantized()(x)
