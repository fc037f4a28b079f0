"""PyTorch-ROCm interface of the mixture-of-experts operators: the router, the experts' Linear products over ragged groups
of rows, the 8-bit products with a scale for each block of 128, and the weighted sum of a token's experts.

    r = route(logits, top_k)                                    # [T, E] -> weights, experts and the order by expert
    h = grouped_linear(x, w1, r.offsets, r.rows, r.slots)       # row r of the order: x[rows[r]] times its expert's weight
    y = grouped_linear(act(h), w2, r.offsets)
    out = combine(y, r.weights, r.slots)                        # back to the tokens

``route``, ``grouped_linear`` and ``combine`` are differentiable. ``linear_fp8`` and ``grouped_linear_fp8`` are the serving
forms with e4m3 weights; they are forward only, and a backward pass that comes to them raises. No operator has a forward-mode
derivative: dual tensors are refused. :class:`MoEMlp` puts them together. Everything runs through the C ABI
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
from torch.autograd import forward_ad as _forward_ad

from . import BF16, F16, F32, F8E4M3, U8, GroupedLinear, LinearFp8, MoeCombine, MoeRoute, check, desc, lib
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
            _plans.popitem(last=False)  # destroyed once no caller holds it: callers keep the plan, not its handle alone
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


# The calls of one token are bound by the time these functions take (a launch is some 3 us of a call's 8 to 10), so the common
# path makes no views, context managers or messages that it does not need, and hands pointers to the C ABI as numbers.
_current = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _gpu(name: str, *tensors: Optional[torch.Tensor]) -> None:
    device = tensors[0].device
    for t in tensors:
        if t is not None and not (t.is_cuda and t.device == device):
            raise ValueError(f"kudnn {name} takes GPU tensors of one device")


def _at(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _first_order(backward):
    """A backward that is not differentiable itself: as torch's own wrapper, which is only taken where a graph is being made."""
    again = torch.autograd.function.once_differentiable(backward)

    def run(ctx, grad):
        return again(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)

    return run


def _tracked(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a derivative may be taken through one of them. Dual tensors do not say so in requires_grad: while there can be any, calls go
    through the autograd functions, which have no forward-mode derivative and refuse a tensor with a tangent."""
    if _forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _ForwardOnly(torch.autograd.Function):
    """A forward-only call: its result, and an error where a derivative through it is asked for."""

    @staticmethod
    def forward(ctx, name, call, *tensors):
        ctx.name = name
        return call(*tensors)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"kudnn {ctx.name} is forward only: it has no gradient")


def _workspace(plan, device: torch.device) -> Optional[torch.Tensor]:
    n = plan.workspace_bytes
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


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
    if not (offsets.dtype == torch.int32 and offsets.shape == (experts + 1,) and offsets.is_contiguous()):
        raise ValueError(f"kudnn {name}: offsets must be int32 [{experts + 1}]")
    if rows is not None and not (rows.dtype == torch.int32 and rows.dim() == 1 and rows.is_contiguous()):
        raise ValueError(f"kudnn {name}: rows must be int32 [R]")


# ---- router

def _route_plan(logits, mask, top_k, normalize) -> MoeRoute:
    key = ("route", logits.shape, logits.stride(), logits.dtype, None if mask is None else (mask.shape, mask.stride()), top_k,
           normalize)
    return _plan(key, lambda: MoeRoute(_matrix_desc(logits, _FLOAT[logits.dtype]), top_k, normalize,
                                       None if mask is None else desc(mask.shape, U8)))


def _route(logits, mask, top_k, normalize):
    device = logits.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _route(logits, mask, top_k, normalize)
    tokens, experts = logits.shape
    plan = _route_plan(logits, mask, top_k, normalize)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    rows = torch.empty(tokens * top_k, dtype=torch.int32, device=device)
    slots = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    ws = _workspace(plan, device)   # held until the call returns
    rc = lib().kudnn_moe_route_run(plan.handle, logits.data_ptr(), _at(mask), weights.data_ptr(), chosen.data_ptr(), offsets.data_ptr(),
                                   rows.data_ptr(), slots.data_ptr(), _at(ws), _stream(device.index))
    if rc:
        check(rc)
    return weights, chosen, offsets, rows, slots


def _route_backward(logits, mask, top_k, normalize, weights, experts, dweights):
    device = logits.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _route_backward(logits, mask, top_k, normalize, weights, experts, dweights)
    plan = _route_plan(logits, mask, top_k, normalize)
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    rc = lib().kudnn_moe_route_backward(plan.handle, logits.data_ptr(), _at(mask), weights.data_ptr(), experts.data_ptr(),
                                        dweights.data_ptr(), dlogits.data_ptr(), _stream(device.index))
    if rc:
        check(rc)
    return dlogits


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, top_k, normalize, rest):
        weights, *order = _route(logits, mask, top_k, normalize)
        rest += order           # whole numbers: nothing for autograd to follow
        ctx.save_for_backward(logits, mask, weights, order[0])
        ctx.top_k, ctx.normalize = top_k, normalize
        return weights

    @staticmethod
    @_first_order
    def backward(ctx, dweights):
        logits, mask, weights, experts = ctx.saved_tensors
        return _route_backward(logits, mask, ctx.top_k, ctx.normalize, weights, experts, dweights.contiguous()), None, None, None, None


def route(logits: torch.Tensor, top_k: int, normalize: bool = True, mask: Optional[torch.Tensor] = None) -> Routing:
    """The top_k experts of each token by the softmax of its logits, and the rows in the experts' order.

    logits: [T, E], float32, bfloat16 or float16, E up to 1024. mask: bool or uint8, [T, E], [T, 1], [1, E] or [E]; an expert
    is open to a token where the mask is true and its logit is not -inf, whatever the logits hold elsewhere. Ties go to the lowest
    index. weights are the softmax's values, over the sum of the chosen ones if normalize. A token without open experts
    has none and adds no rows. Differentiable in the weights.
    """
    if logits.dim() != 2 or logits.dtype not in _FLOAT:
        raise ValueError(f"kudnn route: logits must be [tokens, experts], float32, bfloat16 or float16, got {logits.dtype} {tuple(logits.shape)}")
    _gpu("route", logits, mask)
    if mask is not None:
        if mask.dim() == 1:
            mask = mask[None, :]
        if (mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 or mask.shape[0] not in (1, logits.shape[0])
                or mask.shape[1] not in (1, logits.shape[1])):
            raise ValueError("kudnn route: mask must be bool or uint8 of [tokens or 1, experts or 1]")
        mask = mask.contiguous()
    logits = _matrix(logits)
    normalize = bool(normalize)
    if _tracked(logits):
        rest = []
        return Routing(_Route.apply(logits, mask, top_k, normalize, rest), *rest)
    return Routing(*_route(logits, mask, top_k, normalize))


# ---- grouped Linear

def _grouped_plan(x, w, rows_out, gather) -> GroupedLinear:
    key = ("grouped", x.shape, x.stride(), w.shape, w.stride(), w.dtype, rows_out, gather)
    dt = _HALF[w.dtype]
    return _plan(key, lambda: GroupedLinear(_matrix_desc(x, dt), _weight_desc(w, dt), desc([rows_out, w.shape[1]], dt), gather))


def _grouped(x, w, offsets, rows):
    device = x.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _grouped(x, w, offsets, rows)
    count = x.shape[0] if rows is None else rows.shape[0]
    plan = _grouped_plan(x, w, count, rows is not None)
    y = torch.empty((count, w.shape[1]), dtype=x.dtype, device=device)
    rc = lib().kudnn_grouped_linear_run(plan.handle, x.data_ptr(), w.data_ptr(), offsets.data_ptr(), _at(rows), y.data_ptr(),
                                        _stream(device.index))
    if rc:
        check(rc)
    return y


def _grouped_backward(x, w, offsets, rows, slots, dy, wants_dx, wants_dw):
    device = x.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _grouped_backward(x, w, offsets, rows, slots, dy, wants_dx, wants_dw)
    plan = _grouped_plan(x, w, dy.shape[0], rows is not None)
    stream, ws = _stream(device.index), _workspace(plan, device)
    dx = dw = None
    if wants_dx and rows is None:
        dx = torch.empty((dy.shape[0], x.shape[1]), dtype=x.dtype, device=device)
        plan.backward_input(dy, w, offsets, dx, stream, ws)
    elif wants_dx:
        # a token's gradient is one sum over its slots: f32 rows until it is whole. Rows of 16 bits save 1 to 2 % of forward and
        # backward (8192 tokens, 2 of 8 experts, 4096 x 4096: 1520 against 1537 us) and leave 1.4 times the error.
        dx = torch.empty((dy.shape[0], x.shape[1]), dtype=torch.float32, device=device)
        plan.backward_input(dy, w, offsets, dx, stream, ws, F32)
        dx = _combine(dx, None, slots, x.dtype)
    if wants_dw:
        dw = torch.empty(w.shape, dtype=w.dtype, device=device)
        plan.backward_weight(dy, x, offsets, rows, dw, stream, ws)
    return dx, dw


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, rows, slots):
        ctx.save_for_backward(x, w, offsets, rows, slots)
        return _grouped(x, w, offsets, rows)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        return *_grouped_backward(*ctx.saved_tensors, dy.contiguous(), *ctx.needs_input_grad[:2]), None, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                   slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = x[rows[r]] @ weight[e].T (x[r] without rows) for the rows offsets[e] <= r < offsets[e + 1]; zero before the first and past
    the last (offsets[i:j + 1] with weight[i:j] are the products of some of the experts).

    x: [T, K] with rows, [R, K] without, bfloat16 or float16; weight: [E, N, K], an nn.Linear weight for each expert, of x's type;
    offsets, rows, slots as ``route`` gives them. Differentiable in x and weight; with rows, the gradient of x is a sum over
    each token's slots and needs them.
    """
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2] or x.dtype not in _HALF or weight.dtype != x.dtype:
        raise ValueError(f"kudnn grouped_linear: x {x.dtype} {tuple(x.shape)}, weight {weight.dtype} {tuple(weight.shape)}")
    _gpu("grouped_linear", x, weight, offsets, rows, slots)
    _order("grouped_linear", offsets, weight.shape[0], rows)
    xm, w = _matrix(x), _weight(weight)
    if _tracked(x, weight):
        if rows is not None and x.requires_grad and not (
                slots is not None and slots.dtype == torch.int32 and slots.dim() == 2 and slots.shape[0] == x.shape[0]
                and slots.numel() == rows.numel() and slots.is_contiguous() and slots.shape[1] <= 64):
            raise ValueError("kudnn grouped_linear: the gradient of gathered rows needs slots, int32 [T, k], k up to 64")
        return _GroupedLinear.apply(xm, w, offsets, rows, slots)
    return _grouped(xm, w, offsets, rows)


# ---- 8-bit Linear

def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[M, K] -> e4m3 values [M, K] and the f32 scale [M, ceil(K / 128)] of each row's block of 128: amax / 448."""
    if x.dim() != 2 or x.dtype not in _FLOAT:
        raise ValueError("kudnn quantize_rows: a matrix of float32, bfloat16 or float16")
    _gpu("quantize_rows", x)
    x = _matrix(x)
    m, k = x.shape
    with torch.cuda.device(x.device):
        q = torch.empty((m, k), dtype=_F8, device=x.device)
        scale = torch.empty((m, (k + 127) // 128), dtype=torch.float32, device=x.device)
        _quantize_rows(_matrix_desc(x, _FLOAT[x.dtype]), x, q, k, scale, _stream(x.device.index))
    return q, scale


def quantize_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[N, K] or [E, N, K] -> e4m3 values and the f32 scale [.., ceil(N / 128), ceil(K / 128)] of each 128 x 128 block."""
    if weight.dim() not in (2, 3) or weight.dtype not in _FLOAT:
        raise ValueError("kudnn quantize_blocks: float32, bfloat16 or float16 weights of [N, K] or [E, N, K]")
    _gpu("quantize_blocks", weight)
    w = _weight(weight if weight.dim() == 3 else weight[None])
    e, n, k = w.shape
    with torch.cuda.device(w.device):
        q = torch.empty((e, n, k), dtype=_F8, device=w.device)
        scale = torch.empty((e, (n + 127) // 128, (k + 127) // 128), dtype=torch.float32, device=w.device)
        _quantize_blocks(_weight_desc(w, _FLOAT[w.dtype]), w, q, scale, _stream(w.device.index))
    return (q, scale) if weight.dim() == 3 else (q[0], scale[0])


def _fp8_plan(x, w, dtype, bias, grouped, count, gather) -> LinearFp8:
    """A weight of [N, K] or [E, N, K]."""
    def make():
        n, k = w.shape[-2:]
        wd = _weight_desc(w if w.dim() == 3 else w[None], F8E4M3)
        return LinearFp8(_matrix_desc(x, F8E4M3 if x.dtype == _F8 else _HALF[x.dtype]), wd, desc([count, n], _FLOAT[dtype]),
                         desc([1, n], _FLOAT[dtype]) if bias else None, grouped, gather)

    return _plan(("fp8", x.shape, x.stride(), x.dtype, w.shape, w.stride(), dtype, bias, grouped, count, gather), make)


def _fp8(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype):
    if _tracked(x, w, w_scale, bias, x_scale):
        return _ForwardOnly.apply(name, lambda x, w, w_scale, bias, x_scale: _fp8_run(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype),
                                  x, w, w_scale, bias, x_scale)
    return _fp8_run(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype)


def _fp8_run(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype):
    _gpu(name, x, w, w_scale, bias, offsets, rows, x_scale)
    device = x.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _fp8_run(name, x, w, w_scale, bias, offsets, rows, x_scale, out_dtype)
    n, k = w.shape[-2:]
    blocks = ((n + 127) // 128, (k + 127) // 128)
    if w.dtype != _F8 or w_scale.dtype != torch.float32 or w_scale.shape != (*w.shape[:-2], *blocks):
        raise ValueError(f"kudnn {name}: weight must be float8_e4m3fn and weight_scale float32, one for each block of 128 x 128")
    if x.dtype == _F8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != (x.shape[0], blocks[1]):
            raise ValueError(f"kudnn {name}: x_scale must be float32, one for each row's block of 128")
        x_scale = x_scale.contiguous()
        dtype = out_dtype or torch.bfloat16
    else:
        if x.dtype not in _HALF or x_scale is not None:
            raise ValueError(f"kudnn {name}: x must be bfloat16 or float16, or e4m3 with its x_scale")
        dtype = out_dtype or x.dtype
    if dtype not in _FLOAT:
        raise ValueError(f"kudnn {name}: output of {dtype}")
    x, w_scale = _matrix(x), w_scale.contiguous()
    w = w if w.is_contiguous() else (_weight(w) if w.dim() == 3 else _matrix(w))
    count = x.shape[0] if rows is None else rows.shape[0]
    plan = _fp8_plan(x, w, dtype, bias is not None, offsets is not None, count, rows is not None)
    y = torch.empty((count, n), dtype=dtype, device=device)
    ws = _workspace(plan, device)
    rc = lib().kudnn_linear_fp8_run(plan.handle, x.data_ptr(), _at(x_scale), w.data_ptr(), w_scale.data_ptr(), _at(bias), _at(offsets),
                                    _at(rows), y.data_ptr(), _at(ws), _stream(device.index))
    if rc:
        check(rc)
    return y


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
               x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ weight.T + bias with e4m3 operands and a scale for each block of 128, summed in f32, rounded once.

    The products of a block are exact in f32, except that bfloat16 results of 2**33 operations or more come from the e4m3 matrix
    instruction, which drops what lies more than 13 bits below the largest of 8 products, some 32 times below bfloat16's rounding.
    out_dtype=torch.float32 has exact products at every size.

    x: [..., K], bfloat16 or float16 (quantised here as ``quantize_rows`` does), or e4m3 with x_scale; weight: [N, K] and
    weight_scale as ``quantize_blocks`` gives them; bias: [N] of the output's type. out_dtype: x's type, bfloat16 for e4m3 x.
    """
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"kudnn linear_fp8: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if bias is not None:
        dtype = out_dtype or (torch.bfloat16 if x.dtype == _F8 else x.dtype)
        if bias.shape != (weight.shape[0],) or bias.dtype != dtype:
            raise ValueError("kudnn linear_fp8: bias must be [N] of the output's type")
        bias = bias.contiguous()
    if x.dim() == 2:
        return _fp8("linear_fp8", x, weight, weight_scale, bias, None, None, x_scale, out_dtype)
    if x_scale is not None:
        x_scale = x_scale.reshape(-1, x_scale.shape[-1])
    y = _fp8("linear_fp8", x.reshape(-1, x.shape[-1]), weight, weight_scale, bias, None, None, x_scale, out_dtype)
    return y.reshape(*x.shape[:-1], weight.shape[0])


def grouped_linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, offsets: torch.Tensor,
                       rows: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
                       out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``grouped_linear`` with e4m3 operands and a scale for each block of 128. x as for ``linear_fp8``; weight: [E, N, K]."""
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"kudnn grouped_linear_fp8: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    _order("grouped_linear_fp8", offsets, weight.shape[0], rows)
    return _fp8("grouped_linear_fp8", x, weight, weight_scale, None, offsets, rows, x_scale, out_dtype)


# ---- weighted sum

def _combine_plan(y, tokens, k, dtype) -> MoeCombine:
    return _plan(("combine", y.shape, y.stride(), y.dtype, tokens, k, dtype),
                 lambda: MoeCombine(_matrix_desc(y, _FLOAT[y.dtype]), desc([tokens, y.shape[1]], _FLOAT[dtype]), k))


def _combine(y, weights, slots, dtype):
    device = y.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _combine(y, weights, slots, dtype)
    tokens, k = slots.shape
    plan = _combine_plan(y, tokens, k, dtype)
    out = torch.empty((tokens, y.shape[1]), dtype=dtype, device=device)
    rc = lib().kudnn_moe_combine_run(plan.handle, y.data_ptr(), _at(weights), slots.data_ptr(), out.data_ptr(), _stream(device.index))
    if rc:
        check(rc)
    return out


def _combine_backward(y, weights, slots, dout, wants_dy, wants_dw):
    device = y.device
    if _current() != device.index:
        with torch.cuda.device(device):
            return _combine_backward(y, weights, slots, dout, wants_dy, wants_dw)
    plan = _combine_plan(y, *slots.shape, y.dtype)
    dy = torch.empty(y.shape, dtype=y.dtype, device=device) if wants_dy else None
    dw = torch.empty(slots.shape, dtype=torch.float32, device=device) if wants_dw else None
    rc = lib().kudnn_moe_combine_backward(plan.handle, y.data_ptr(), _at(weights), slots.data_ptr(), dout.data_ptr(), _at(dy), _at(dw),
                                          _stream(device.index))
    if rc:
        check(rc)
    return dy, dw


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots):
        ctx.save_for_backward(y, weights, slots)
        return _combine(y, weights, slots, y.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        return *_combine_backward(*ctx.saved_tensors, dout.contiguous(), *ctx.needs_input_grad[:2]), None


def combine(y: torch.Tensor, weights: Optional[torch.Tensor], slots: torch.Tensor) -> torch.Tensor:
    """out[t] = sum over j of weights[t, j] * y[slots[t, j]], summed in f32, rounded once to y's type.

    y: [R, N], float32, bfloat16 or float16; weights: float32 [T, k], or None for ones; slots: int32 [T, k] as ``route`` gives
    them, no row twice; any of them may be set to -1 (as may what names no row of y), which adds nothing. Differentiable in y and
    weights; the rows of y that no slot names get a gradient of zero.
    """
    if y.dim() != 2 or y.dtype not in _FLOAT:
        raise ValueError("kudnn combine: y must be a matrix of float32, bfloat16 or float16")
    _gpu("combine", y, weights, slots)
    if slots.dtype != torch.int32 or slots.dim() != 2 or not slots.is_contiguous() or slots.shape[1] == 0:
        raise ValueError("kudnn combine: slots must be int32 [T, k]")
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != slots.shape):
        raise ValueError("kudnn combine: weights must be float32 of slots' shape")
    ym = _matrix(y)
    w = None if weights is None else weights.contiguous()
    if _tracked(y, w):
        return _Combine.apply(ym, w, slots)
    return _combine(ym, w, slots, y.dtype)


# ---- the operators together

def _one_group(x: torch.Tensor) -> torch.Tensor:
    """Offsets of one group of all rows of x, made on the device (a copy from the host would wait)."""
    rows = x.shape[0]
    if rows == 0:
        return torch.zeros(2, dtype=torch.int32, device=x.device)
    return torch.arange(0, rows + 1, rows, dtype=torch.int32, device=x.device)


def _project(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """The router's logits, x @ w.T: the grouped product of one group, which keeps no memory between calls. (Its weight gradient has few tiles for a
    long sum: 16384 tokens, 64 experts, width 2048 take 265 us, 1.5 % of the layer's training pass.)"""
    return grouped_linear(x, w[None], _one_group(x))


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
        r = route(_project(tokens, self.router), self.top_k, self.normalize,
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
        if _tracked(x):
            return _ForwardOnly.apply("QuantizedMoEMlp", lambda x: self._run(x, mask), x)
        with torch.no_grad():
            return self._run(x, mask)

    def _run(self, x, mask):
        tokens = x.reshape(-1, x.shape[-1])
        r = route(_project(tokens, self.router), self.top_k, self.normalize,
                  None if mask is None else mask.reshape(-1, 1))
        gate, up = grouped_linear_fp8(tokens, self.up, self.up_scale, r.offsets, r.rows).chunk(2, 1)
        y = grouped_linear_fp8(torch.nn.functional.silu(gate) * up, self.down, self.down_scale, r.offsets)
        return combine(y, r.weights, r.slots).reshape(x.shape)
