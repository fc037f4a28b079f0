"""PyTorch-ROCm interface of the mixture-of-experts operators: the router, the experts' Linear products over ragged groups
of rows, the 8-bit products with a scale for each block of 128, and the weighted sum of a token's experts.

    r = route(logits, top_k)                                    # [T, E] -> weights, experts and the order by expert
    h = grouped_linear(x, w1, r.offsets, r.rows, r.slots)       # row r of the order: x[rows[r]] times its expert's weight
    y = grouped_linear(act(h), w2, r.offsets)
    out = combine(y, r.weights, r.slots)                        # back to the tokens

``route``, ``grouped_linear`` and ``combine`` are differentiable. ``linear_fp8`` and ``grouped_linear_fp8`` are the serving
forms with e4m3 weights; they are forward only. :class:`MoEMlp` puts them together. Everything runs through the C ABI
(``include/kudnn_hip.h``) on torch's current stream, on the device of its arguments; nothing falls back to another path.

Nothing here waits for the device: the sizes of the groups stay on it, and outputs have room for every row that the
router could choose. Plans hold sizes only and are cached (at most ``MAX_CACHED_PLANS``); workspaces come from torch's
allocator for the length of a call.
"""
from __future__ import annotations

import threading
from collections import OrderedDict
from typing import NamedTuple, Optional, Tuple

import torch

from . import (BF16, F16, F32, F8E4M3, U8, GroupedLinear, LinearFp8, MoeCombine, MoeRoute, desc)
from . import quantize_blocks as _quantize_blocks
from . import quantize_rows as _quantize_rows

_FLOAT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_HALF = {torch.bfloat16: BF16, torch.float16: F16}
_F8 = torch.float8_e4m3fn

MAX_CACHED_PLANS = 256
_plans: "OrderedDict[Tuple, object]" = OrderedDict()
_plans_lock = threading.Lock()


def _plan(key, make):
    with _plans_lock:
        plan = _plans.get(key)
        if plan is not None:
            _plans.move_to_end(key)
            return plan
        plan = _plans[key] = make()
        while len(_plans) > MAX_CACHED_PLANS:
            _plans.popitem(last=False)  # destroyed once no caller holds it
        return plan


class Routing(NamedTuple):
    """What the router gives. T tokens, k experts a token, E experts.

    weights f32 [T, k] and experts int32 [T, k], by falling logit (expert -1 and weight 0 where a token has none left);
    offsets int32 [E + 1], rows int32 [T * k], slots int32 [T, k]: the order by expert. Expert e has the rows offsets[e] up
    to offsets[e + 1]; rows gives the token of each (-1 past the last), slots the row of each of a token's experts (-1: none).
    """

    weights: torch.Tensor
    experts: torch.Tensor
    offsets: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class _on:
    """Makes the tensors' device the current one where it is not (launches go to the current device)."""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.device.index:
            torch._C._cuda_setDevice(self.device.index)

    def __exit__(self, *exc):
        if self.before != self.device.index:
            torch._C._cuda_setDevice(self.before)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _gpu(name: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != device):
            raise ValueError(f"kudnn {name} takes GPU tensors of one device")
    return device


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous rows: itself where its rows are apart by at least their length, else a copy."""
    if x.is_contiguous() or (x.stride(1) == 1 and x.stride(0) >= x.shape[1]):
        return x
    return x.contiguous()


def _matrix_desc(x: torch.Tensor, dt: int):
    return desc(x.shape, dt) if x.is_contiguous() else desc(x.shape, dt, "AB", x.stride())


def _weight(w: torch.Tensor) -> torch.Tensor:
    """[E, N, K] with contiguous rows that do not overlap."""
    e, n, k = w.shape
    if w.is_contiguous() or (w.stride(2) == 1 and w.stride(1) >= k and w.stride(0) >= w.stride(1) * n):
        return w
    return w.contiguous()


def _weight_desc(w: torch.Tensor, dt: int):
    e, n, k = w.shape
    if w.is_contiguous():
        return desc([e, k, n], dt, "ACB")
    return desc([e, k, n], dt, "ACB", [w.stride(0), 1, w.stride(1)])


def _order(name: str, offsets: torch.Tensor, experts: int, rows: Optional[torch.Tensor]) -> None:
    _need(offsets.dtype == torch.int32 and offsets.shape == (experts + 1,) and offsets.is_contiguous(),
          f"kudnn {name}: offsets must be int32 [{experts + 1}]")
    if rows is not None:
        _need(rows.dtype == torch.int32 and rows.dim() == 1 and rows.is_contiguous(), f"kudnn {name}: rows must be int32 [R]")


# ---- router

def _route_plan(logits, mask, top_k, normalize) -> MoeRoute:
    key = ("route", logits.shape, logits.stride(), logits.dtype, None if mask is None else (mask.shape, mask.stride()), top_k,
           normalize)
    return _plan(key, lambda: MoeRoute(_matrix_desc(logits, _FLOAT[logits.dtype]), top_k, normalize,
                                       None if mask is None else desc(mask.shape, U8)))


def _route(logits, mask, top_k, normalize):
    tokens, experts = logits.shape
    plan = _route_plan(logits, mask, top_k, normalize)
    device = logits.device
    with _on(device):
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
        chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
        rows = torch.empty(tokens * top_k, dtype=torch.int32, device=device)
        slots = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device) if plan.workspace_bytes else None
        plan.run(logits, mask, weights, chosen, offsets, rows, slots, ws, _stream(device))
    return weights, chosen, offsets, rows, slots


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, top_k, normalize):
        outs = _route(logits, mask, top_k, normalize)
        # the logits are needed again only for the whole softmax
        ctx.save_for_backward(logits, mask, outs[0], outs[1])
        ctx.top_k, ctx.normalize = top_k, normalize
        ctx.mark_non_differentiable(*outs[1:])
        return outs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, *_):
        logits, mask, weights, experts = ctx.saved_tensors
        plan = _route_plan(logits, mask, ctx.top_k, ctx.normalize)
        with _on(logits.device):
            dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            plan.backward(logits, mask, weights, experts, dweights.contiguous(), dlogits, _stream(logits.device))
        return dlogits, None, None, None


def route(logits: torch.Tensor, top_k: int, normalize: bool = True, mask: Optional[torch.Tensor] = None) -> Routing:
    """The top_k experts of each token by the softmax of its logits, and the rows in the experts' order.

    logits: [T, E], float32, bfloat16 or float16, E up to 1024. mask: bool or uint8, [T, E], [T, 1], [1, E] or [E]; an expert
    is open to a token where the mask is true and its logit is not -inf, whatever the logits hold elsewhere. Ties go to the lowest
    index. weights are the softmax's values, over the sum of the chosen ones if normalize. A token without open experts
    has none and adds no rows. Differentiable in the weights.
    """
    _need(logits.dim() == 2, "kudnn route: logits must be [tokens, experts]")
    _gpu("route", logits, mask)
    _need(logits.dtype in _FLOAT, f"kudnn route: logits of {logits.dtype}")
    if mask is not None:
        _need(mask.dtype in (torch.bool, torch.uint8), "kudnn route: mask must be bool or uint8")
        if mask.dim() == 1:
            mask = mask[None, :]
        _need(mask.dim() == 2 and mask.shape[0] in (1, logits.shape[0]) and mask.shape[1] in (1, logits.shape[1]),
              "kudnn route: mask must be [tokens or 1, experts or 1]")
        mask = mask.contiguous()
    logits = _matrix(logits)
    normalize = bool(normalize)
    if torch.is_grad_enabled() and logits.requires_grad:
        return Routing(*_Route.apply(logits, mask, top_k, normalize))
    return Routing(*_route(logits, mask, top_k, normalize))


# ---- grouped Linear

def _grouped_plan(x, w, rows_out, gather) -> GroupedLinear:
    key = ("grouped", x.shape, x.stride(), w.shape, w.stride(), w.dtype, rows_out, gather)
    dt = _HALF[w.dtype]
    return _plan(key, lambda: GroupedLinear(_matrix_desc(x, dt), _weight_desc(w, dt), desc([rows_out, w.shape[1]], dt), gather))


def _grouped(x, w, offsets, rows):
    count = x.shape[0] if rows is None else rows.shape[0]
    device = x.device
    with _on(device):
        y = torch.empty((count, w.shape[1]), dtype=x.dtype, device=device)
        _grouped_plan(x, w, count, rows is not None).run(x, w, offsets, rows, y, _stream(device))
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, rows, slots):
        ctx.save_for_backward(x, w, offsets, rows, slots)
        return _grouped(x, w, offsets, rows)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, offsets, rows, slots = ctx.saved_tensors
        dy = dy.contiguous()
        device = x.device
        plan = _grouped_plan(x, w, dy.shape[0], rows is not None)
        dx = dw = None
        with _on(device):
            stream = _stream(device)
            if ctx.needs_input_grad[0]:
                dx = torch.empty((dy.shape[0], x.shape[1]), dtype=x.dtype, device=device)
                plan.backward_input(dy, w, offsets, dx, stream)
                if rows is not None:
                    dx = _combine(dx, None, slots)
            if ctx.needs_input_grad[1]:
                dw = torch.empty(w.shape, dtype=w.dtype, device=device)
                plan.backward_weight(dy, x, offsets, rows, dw, stream)
        return dx, dw, None, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                   slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = x[rows[r]] @ weight[e].T (x[r] without rows) for the rows offsets[e] <= r < offsets[e + 1]; zero past the last.

    x: [T, K] with rows, [R, K] without, bfloat16 or float16; weight: [E, N, K], an nn.Linear weight for each expert, of x's type;
    offsets, rows, slots as ``route`` gives them. Differentiable in x and weight; with rows, the gradient of x is a sum over
    each token's slots and needs them.
    """
    _need(x.dim() == 2 and weight.dim() == 3 and x.shape[1] == weight.shape[2],
          f"kudnn grouped_linear: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    _gpu("grouped_linear", x, weight, offsets, rows, slots)
    _need(x.dtype in _HALF and weight.dtype == x.dtype, f"kudnn grouped_linear: {x.dtype} x {weight.dtype}")
    _order("grouped_linear", offsets, weight.shape[0], rows)
    xm, w = _matrix(x), _weight(weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        if rows is not None and x.requires_grad:
            _need(slots is not None and slots.dtype == torch.int32 and slots.dim() == 2 and slots.shape[0] == x.shape[0]
                  and slots.numel() == rows.numel() and slots.is_contiguous(),
                  "kudnn grouped_linear: the gradient of gathered rows needs slots, int32 [T, k]")
        return _GroupedLinear.apply(xm, w, offsets, rows, slots)
    return _grouped(xm, w, offsets, rows)


# ---- 8-bit Linear

def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[M, K] -> e4m3 values [M, K] and the f32 scale [M, ceil(K / 128)] of each row's block of 128: amax / 448."""
    _need(x.dim() == 2 and x.dtype in _FLOAT, "kudnn quantize_rows: a matrix of float32, bfloat16 or float16")
    device = _gpu("quantize_rows", x)
    x = _matrix(x)
    m, k = x.shape
    with _on(device):
        q = torch.empty((m, k), dtype=_F8, device=device)
        scale = torch.empty((m, (k + 127) // 128), dtype=torch.float32, device=device)
        _quantize_rows(_matrix_desc(x, _FLOAT[x.dtype]), x, q, k, scale, _stream(device))
    return q, scale


def quantize_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[N, K] or [E, N, K] -> e4m3 values and the f32 scale [.., ceil(N / 128), ceil(K / 128)] of each 128 x 128 block."""
    _need(weight.dim() in (2, 3) and weight.dtype in _FLOAT, "kudnn quantize_blocks: float32, bfloat16 or float16 weights")
    device = _gpu("quantize_blocks", weight)
    w = _weight(weight if weight.dim() == 3 else weight[None])
    e, n, k = w.shape
    with _on(device):
        q = torch.empty((e, n, k), dtype=_F8, device=device)
        scale = torch.empty((e, (n + 127) // 128, (k + 127) // 128), dtype=torch.float32, device=device)
        _quantize_blocks(_weight_desc(w, _FLOAT[w.dtype]), w, q, scale, _stream(device))
    return (q, scale) if weight.dim() == 3 else (q[0], scale[0])


def _fp8(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype):
    device = _gpu(name, x, w, w_scale, bias, offsets, rows, x_scale)
    e, n, k = w.shape
    _need(w.dtype == _F8, f"kudnn {name}: weight must be float8_e4m3fn")
    _need(w_scale.dtype == torch.float32 and w_scale.shape == (e, (n + 127) // 128, (k + 127) // 128),
          f"kudnn {name}: weight_scale must be float32, one for each block of 128 x 128")
    quantized = x.dtype == _F8
    if quantized:
        _need(x_scale is not None and x_scale.dtype == torch.float32 and x_scale.shape == (x.shape[0], (k + 127) // 128),
              f"kudnn {name}: x_scale must be float32, one for each row's block of 128")
        x_scale = x_scale.contiguous()
    else:
        _need(x.dtype in _HALF and x_scale is None, f"kudnn {name}: x must be bfloat16 or float16, or e4m3 with its x_scale")
    dtype = out_dtype or (torch.bfloat16 if quantized else x.dtype)
    _need(dtype in _FLOAT, f"kudnn {name}: output of {dtype}")
    x, w, w_scale = _matrix(x), _weight(w), w_scale.contiguous()
    grouped = offsets is not None
    count = x.shape[0] if rows is None else rows.shape[0]
    key = ("fp8", x.shape, x.stride(), x.dtype, w.shape, w.stride(), dtype, bias is None, grouped, count, rows is None)
    plan = _plan(key, lambda: LinearFp8(_matrix_desc(x, F8E4M3 if quantized else _HALF[x.dtype]), _weight_desc(w, F8E4M3),
                                        desc([count, n], _FLOAT[dtype]),
                                        None if bias is None else desc([1, n], _FLOAT[dtype]), grouped, rows is not None))
    with _on(device):
        y = torch.empty((count, n), dtype=dtype, device=device)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device) if plan.workspace_bytes else None
        plan.run(x, x_scale, w, w_scale, y, bias, offsets, rows, ws, _stream(device))
    return y


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
               x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ weight.T + bias with e4m3 operands and a scale for each block of 128, summed in f32, rounded once.

    x: [..., K], bfloat16 or float16 (quantised here as ``quantize_rows`` does), or e4m3 with x_scale; weight: [N, K] and
    weight_scale as ``quantize_blocks`` gives them; bias: [N] of the output's type. out_dtype: x's type, bfloat16 for e4m3 x.
    """
    _need(weight.dim() == 2 and weight_scale.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1],
          f"kudnn linear_fp8: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if bias is not None:
        dtype = out_dtype or (torch.bfloat16 if x.dtype == _F8 else x.dtype)
        _need(bias.shape == (weight.shape[0],) and bias.dtype == dtype, "kudnn linear_fp8: bias must be [N] of the output's type")
        bias = bias.contiguous()
    if x_scale is not None and x_scale.dim() != 2:
        x_scale = x_scale.reshape(-1, x_scale.shape[-1])
    y = _fp8("linear_fp8", x2, weight[None], weight_scale[None], bias, None, None, x_scale, out_dtype)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.shape[0])


def grouped_linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, offsets: torch.Tensor,
                       rows: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
                       out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``grouped_linear`` with e4m3 operands and a scale for each block of 128. x as for ``linear_fp8``; weight: [E, N, K]."""
    _need(x.dim() == 2 and weight.dim() == 3 and x.shape[1] == weight.shape[2],
          f"kudnn grouped_linear_fp8: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    _order("grouped_linear_fp8", offsets, weight.shape[0], rows)
    return _fp8("grouped_linear_fp8", x, weight, weight_scale, None, offsets, rows, x_scale, out_dtype)


# ---- weighted sum

def _combine_plan(y, tokens, k) -> MoeCombine:
    dt = _FLOAT[y.dtype]
    return _plan(("combine", y.shape, y.stride(), y.dtype, tokens, k),
                 lambda: MoeCombine(_matrix_desc(y, dt), desc([tokens, y.shape[1]], dt), k))


def _combine(y, weights, slots):
    device = y.device
    tokens, k = slots.shape
    with _on(device):
        out = torch.empty((tokens, y.shape[1]), dtype=y.dtype, device=device)
        _combine_plan(y, tokens, k).run(y, weights, slots, out, _stream(device))
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots):
        ctx.save_for_backward(y, weights, slots)
        return _combine(y, weights, slots)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights, slots = ctx.saved_tensors
        device = y.device
        dout = dout.contiguous()
        with _on(device):
            dy = torch.empty(y.shape, dtype=y.dtype, device=device) if ctx.needs_input_grad[0] else None
            dw = torch.empty(slots.shape, dtype=torch.float32, device=device) if ctx.needs_input_grad[1] else None
            _combine_plan(y, *slots.shape).backward(y, weights, slots, dout, dy, dw, _stream(device))
        return dy, dw, None


def combine(y: torch.Tensor, weights: Optional[torch.Tensor], slots: torch.Tensor) -> torch.Tensor:
    """out[t] = sum over j of weights[t, j] * y[slots[t, j]], summed in f32, rounded once to y's type.

    y: [R, N], float32, bfloat16 or float16; weights: float32 [T, k], or None for ones; slots: int32 [T, k] as ``route`` gives
    them, -1 adds nothing. Differentiable in y and weights; the rows of y that no slot takes are the last ones, and get a
    gradient of zero.
    """
    _need(y.dim() == 2 and y.dtype in _FLOAT, "kudnn combine: y must be a matrix of float32, bfloat16 or float16")
    _gpu("combine", y, weights, slots)
    _need(slots.dtype == torch.int32 and slots.dim() == 2 and slots.is_contiguous() and slots.shape[1] > 0,
          "kudnn combine: slots must be int32 [T, k]")
    _need(weights is None or (weights.dtype == torch.float32 and weights.shape == slots.shape),
          "kudnn combine: weights must be float32 of slots' shape")
    ym = _matrix(y)
    w = None if weights is None else weights.contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or (w is not None and w.requires_grad)):
        return _Combine.apply(ym, w, slots)
    return _combine(ym, w, slots)


# ---- the operators together

class MoEMlp(torch.nn.Module):
    """A transformer's gated MLP with experts: out = sum over a token's experts of p_e W2_e (silu(G_e x) * U_e x).

    The first product's weight holds G above U, [E, 2 * hidden, width]; the second's is [E, width, hidden]. Trains in
    bfloat16 or float16; ``quantized()`` gives the serving form, whose experts are kept in 8 bits.
    """

    def __init__(self, width: int, hidden: int, experts: int, top_k: int, normalize: bool = True, device=None,
                 dtype=torch.bfloat16):
        super().__init__()
        self.top_k, self.normalize = top_k, normalize
        self.router = torch.nn.Parameter(torch.randn(experts, width, device=device, dtype=dtype) * width ** -0.5)
        self.up = torch.nn.Parameter(torch.randn(experts, 2 * hidden, width, device=device, dtype=dtype) * width ** -0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, width, hidden, device=device, dtype=dtype) * hidden ** -0.5)

    def forward(self, x: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: [..., width]; mask: bool, x's leading shape: False for padding, which no expert takes."""
        tokens = x.reshape(-1, x.shape[-1])
        r = route(torch.nn.functional.linear(tokens, self.router), self.top_k, self.normalize,
                  None if mask is None else mask.reshape(-1, 1))
        gate, up = grouped_linear(tokens, self.up, r.offsets, r.rows, r.slots).chunk(2, 1)
        y = grouped_linear(torch.nn.functional.silu(gate) * up, self.down, r.offsets)
        return combine(y, r.weights, r.slots).reshape(x.shape)

    def quantized(self) -> "QuantizedMoEMlp":
        return QuantizedMoEMlp(self)


class QuantizedMoEMlp(torch.nn.Module):
    """The serving form of :class:`MoEMlp`: the experts' weights as e4m3 values with block scales. Forward only."""

    def __init__(self, source: MoEMlp):
        super().__init__()
        self.top_k, self.normalize = source.top_k, source.normalize
        with torch.no_grad():
            self.register_buffer("router", source.router.detach().clone())
            for name in ("up", "down"):
                q, scale = quantize_blocks(getattr(source, name).detach())
                self.register_buffer(name, q)
                self.register_buffer(name + "_scale", scale)

    def forward(self, x: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        with torch.no_grad():
            tokens = x.reshape(-1, x.shape[-1])
            r = route(torch.nn.functional.linear(tokens, self.router), self.top_k, self.normalize,
                      None if mask is None else mask.reshape(-1, 1))
            gate, up = grouped_linear_fp8(tokens, self.up, self.up_scale, r.offsets, r.rows).chunk(2, 1)
            y = grouped_linear_fp8(torch.nn.functional.silu(gate) * up, self.down, self.down_scale, r.offsets)
            return combine(y, r.weights, r.slots).reshape(x.shape)
