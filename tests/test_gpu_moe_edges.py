"""Edges of the mixture-of-experts operators on the GPU: precision by type, odd choices, wide operands, large orders.

Bounds as in test_gpu_moe.py: half a unit of the result's type, and n 2^-23 of the terms' magnitudes for a sum of n terms.
"""
import math

import pytest
import torch

import kudnn_amd as K

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import kudnn_amd.torch_moe as km

from test_gpu_moe import DEV, HALF, dequant, gen, grouped_plain, make_fp8, make_order, near, randn


@pytest.mark.parametrize("counts,width,out", [([40, 0, 100] + [41] * 61, 2064, 1032), ([1500, 77, 3000, 0], 1040, 2056), ([2500], 2048, 4096)])
def test_large_fp8_products_into_f16_are_rounded_once(counts, width, out):
    """In norm an f16 result is as far from the 64-bit one as that result rounded to f16: the f32 sums' error, some 1e-6 in norm, adds
    less than 1e-4 of the rounding's 2e-4, taken at 1.003 times. (Products by the e4m3 instruction are 1.012 times as far.)"""
    g = gen(width + out)
    count = sum(counts)
    offsets, _ = make_order(counts, 0, 1, g)
    x = randn(g, count, width).half()
    w, ws = make_fp8(g, len(counts), out, width)
    xq, xs = km.quantize_rows(x)
    if len(counts) > 1:
        y = km.grouped_linear_fp8(x, w, ws, offsets)
    else:
        y = km.linear_fp8(x, w[0], ws[0])
    want, mag, *_ = grouped_plain(dequant(xq, xs), dequant(w, ws, 128), offsets, None, count)
    near(y, want, mag, width + 3 * (width // 128 + 1), "y")
    off = lambda v: float((v.double() - want).norm() / want.norm())
    assert off(y) <= 1.003 * off(want.half())


def combine_gradients(slots, rows, width, dtype, g, weighted=True):
    """Gradients of the weighted sum, written over NaN, against the formula."""
    tokens, k = slots.shape
    y = randn(g, rows, width).to(dtype)
    w = randn(g, tokens, k) if weighted else None
    dout = randn(g, tokens, width).to(dtype)
    kind = {torch.float32: K.F32, torch.bfloat16: K.BF16, torch.float16: K.F16}[dtype]
    dy, dw = torch.full((rows, width), math.nan, dtype=dtype, device=DEV), torch.full((tokens, k), math.nan, device=DEV)
    K.MoeCombine(K.desc([rows, width], kind), K.desc([tokens, width], kind), k).backward(y, w, slots, dout, dy, dw, torch.cuda.current_stream())
    named = (slots >= 0) & (slots < rows)
    want = torch.zeros(rows, width, dtype=torch.float64, device=DEV)
    scale = torch.ones(tokens, k, device=DEV) if w is None else w
    for j in range(k):
        at = named[:, j].nonzero()[:, 0]
        want[slots[at, j].long()] = scale[at, j, None].double() * dout[at].double()
    near(dy, want, want.abs(), 1, "dy")
    for j in range(k):
        picked = torch.where(named[:, j, None], y.double()[torch.where(named[:, j], slots[:, j], 0).long()], 0.0) * dout.double()
        near(dw[:, j], picked.sum(1), picked.abs().sum(1), width, "dweights")
    return dy


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,k,width,rows", [(1, 1, 8, 1), (1, 2, 7, 300), (40, 3, 1000, 120), (40, 3, 129, 63), (300, 8, 64, 2400), (3000, 4, 16, 9000),
                                                 (5000, 2, 3, 40000)])
def test_combine_gradients_of_any_slots(tokens, k, width, rows, dtype):
    """Slots taken out anywhere, more rows than slots and fewer, slots past the last row: the rows that none names are zero."""
    g = gen(rows + width)
    for out in (0.0, 0.3, 0.97):
        order = torch.randperm(max(rows, tokens * k) + 50, generator=g, device=DEV)[:tokens * k].int().reshape(tokens, k)   # some past the last
        slots = torch.where(torch.rand(tokens, k, generator=g, device=DEV) < out, torch.full_like(order, -1), order)
        combine_gradients(slots, rows, width, dtype, g, out == 0.3)
    combine_gradients(torch.full((tokens, k), -1, dtype=torch.int32, device=DEV), rows, width, dtype, g)
    odd = torch.empty(tokens * k + 1, dtype=torch.int32, device=DEV)[1:].reshape(tokens, k)      # off 16 bytes
    odd.copy_(order)
    combine_gradients(odd, rows, width, dtype, g)


def test_combine_gradient_of_more_rows_than_one_reading_marks():
    rows = (1 << 25) + 777
    g = gen(7)
    slots = torch.randint(0, rows, (900, 2), generator=g, device=DEV, dtype=torch.int32)
    slots[0], slots[1, 0] = torch.tensor([rows - 1, rows - 2]), 0
    slots = torch.unique(slots.flatten())[-1700:].reshape(850, 2).contiguous()
    combine_gradients(slots, rows, 1, torch.float16, g)


def test_combine_after_choices_are_dropped():
    """Choices over an expert's capacity set to -1 by the caller: gradients through torch, against differences of the output's formula."""
    g = gen(17)
    tokens, experts, k, width = 50, 6, 2, 40
    r = km.route(randn(g, tokens, experts), k)
    place = r.slots - r.offsets[:-1][r.experts.long()]
    slots = torch.where(place < 8, r.slots, -1).int()
    assert int((slots < 0).sum()) > 0
    y = randn(g, tokens * k, width).requires_grad_(True)
    dout = randn(g, tokens, width)
    dy, = torch.autograd.grad(km.combine(y, r.weights, slots), y, dout)
    want = torch.zeros(tokens * k, width, dtype=torch.float64, device=DEV)
    keep = slots >= 0
    want[slots[keep].long()] = (r.weights.double()[:, :, None] * dout.double()[:, None, :])[keep]
    near(dy, want, want.abs(), 1, "dy")


@pytest.mark.parametrize("tokens", [(1 << 23) + 101])
def test_weighted_sum_of_more_tokens_than_a_grid(tokens):
    g = gen(3)
    y = randn(g, 1000, 8).bfloat16()
    slots = torch.full((tokens, 1), -1, dtype=torch.int32, device=DEV)
    last = torch.arange(tokens - 900, tokens, device=DEV)
    slots[last, 0] = torch.randperm(1000, generator=g, device=DEV)[:900].int()
    out = km.combine(y, None, slots)
    assert torch.equal(out[last], y[slots[last, 0].long()]) and float(out[:-900].abs().sum()) == 0.0
    dout = randn(g, tokens, 8).bfloat16()
    dy, dw = torch.full_like(y, math.nan), torch.full((tokens, 1), math.nan, device=DEV)
    K.MoeCombine(K.desc([1000, 8], K.BF16), K.desc([tokens, 8], K.BF16), 1).backward(y, None, slots, dout, dy, dw, torch.cuda.current_stream())
    want = torch.zeros_like(y)
    want[slots[last, 0].long()] = dout[last]
    assert torch.equal(dy, want) and float(dw[:-900].abs().sum()) == 0.0
    products = dout[last].double() * y[slots[last, 0].long()].double()
    near(dw[last, 0], products.sum(1), products.abs().sum(1), 8, "dweights")


def test_router_gradient_of_more_tokens_than_a_grid():
    tokens = (1 << 28) + 77
    g = gen(4)
    logits = torch.zeros(tokens, 2, dtype=torch.float16, device=DEV)
    ends = torch.cat([torch.arange(500, device=DEV), torch.arange(tokens - 500, tokens, device=DEV)])
    logits[ends] = randn(g, 1000, 2).half()
    experts = torch.zeros(tokens, 1, dtype=torch.int32, device=DEV)
    p = torch.softmax(logits[ends].double(), 1)
    weights, d = torch.full((tokens, 1), 0.5, device=DEV), torch.ones(tokens, 1, device=DEV)
    weights[ends, 0], d[ends, 0] = p[:, 0].float(), randn(g, 1000)
    dlogits = torch.full_like(logits, math.nan)
    K.MoeRoute(K.desc([tokens, 2], K.F16), 1, False).backward(logits, None, weights, experts, d, dlogits, torch.cuda.current_stream())
    assert bool((dlogits[500:-500] == torch.tensor([0.25, -0.25], device=DEV).half()).all())
    dx = d[ends].double() * p[:, :1] * torch.stack([1 - p[:, 0], -p[:, 1]], 1)
    near(dlogits[ends], dx, 2.0 ** 7 * d[ends].double().abs(), 1, "dlogits")


@pytest.mark.parametrize("tokens,experts,k", [(65, 60, 4), (768 * 64, 9, 3), (768 * 64 + 1, 9, 3), (70001, 130, 2), (140007, 1024, 1), (1 << 20, 8, 2)])
def test_order_of_many_tokens(tokens, experts, k):
    """The order by expert against a stable sort, around and far above the count of workgroups from which their counts are scanned."""
    g = gen(experts)
    logits = randn(g, tokens, experts) + 2 * randn(g, 1, experts)
    mask = torch.rand(tokens, 1, generator=g, device=DEV) > 0.1
    r = km.route(logits, k, True, mask)
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    assert torch.equal(r.experts, torch.where(mask, top.indices[:, :k], -1).int())
    key = torch.where(r.experts < 0, experts, r.experts).reshape(-1)
    order = torch.sort(key, stable=True).indices
    assert torch.equal(r.offsets, torch.searchsorted(key[order], torch.arange(experts + 1, device=DEV, dtype=torch.int32)).int())
    count = int(r.offsets[-1])
    assert torch.equal(r.rows, torch.where(torch.arange(tokens * k, device=DEV) < count, order // k, -1).int())
    slots = torch.full((tokens * k,), -1, dtype=torch.int32, device=DEV)
    slots[order[:count]] = torch.arange(count, dtype=torch.int32, device=DEV)
    assert torch.equal(r.slots.reshape(-1), slots)
    want = torch.softmax(top.values[:, :k].double(), 1) * mask
    torch.testing.assert_close(r.weights.double(), want, rtol=2.0 ** -16, atol=1e-30)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("tokens,width,experts,pad", [(1, 256, 8, 0), (7, 40, 5, 3), (130, 33, 9, 0), (3001, 1024, 60, 0), (600, 264, 128, 8)])
def test_router_projection(tokens, width, experts, pad, dtype):
    g = gen(tokens + width)
    wide = randn(g, tokens, width + pad).to(HALF[dtype])
    x = wide[:, pad:].detach().requires_grad_(True)
    w = (randn(g, experts, width) * width ** -0.5).to(HALF[dtype]).requires_grad_(True)
    y = km._project(x, w)
    xd, wd, dy = x.detach().double(), w.detach().double(), randn(g, tokens, experts).to(HALF[dtype])
    near(y.detach(), xd @ wd.t(), xd.abs() @ wd.abs().t(), width + 1, "logits")
    assert torch.equal(km._project(x.detach(), w.detach()), y.detach())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    d = dy.double()
    near(dx, d @ wd, d.abs() @ wd.abs(), experts + 1, "dx")
    near(dw, d.t() @ xd, d.abs().t() @ xd.abs(), tokens + 1, "dw")


def part_of_the_experts(counts, skip, width, out, dtype, f8=False, gather=True):
    """Products and gradients of the experts from `skip` on, over NaN: equal to the whole's in their rows, zero in the others."""
    g = gen(width + out + skip)
    offsets, rows = make_order(counts, 3, 50, g)
    count, first = sum(counts) + 3, sum(counts[:skip])
    part, e = offsets[skip:], len(counts) - skip
    kind = K.BF16 if dtype == torch.bfloat16 else K.F16
    x = randn(g, 50 if gather else count, width).to(dtype)
    stream = torch.cuda.current_stream()
    r = rows if gather else None
    y = torch.full((count, out), math.nan, dtype=dtype, device=DEV)
    if f8:
        w, ws = make_fp8(g, len(counts), out, width)
        plan = K.LinearFp8(K.desc(x.shape, kind), K.desc([e, width, out], K.F8E4M3, "ACB"), K.desc(y.shape, kind), None, True, gather)
        room = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=DEV)
        plan.run(x, None, w[skip:], ws[skip:].contiguous(), y, None, part, r, room, stream)
        want = km.grouped_linear_fp8(x, w, ws, offsets, r).double()
        assert float(y[:first].abs().sum()) == 0.0 and float(y[sum(counts):].abs().sum()) == 0.0
        near(y[first:], want[first:], want[first:].abs(), width + 3 * (width // 128 + 1) + 2.0 ** 13, "y")
        return plan.describe()
    w = (randn(g, len(counts), out, width) * width ** -0.5).to(dtype)
    dy = randn(g, count, out).to(dtype)
    plan = K.GroupedLinear(K.desc(x.shape, kind), K.desc([e, width, out], kind, "ACB"), K.desc(y.shape, kind), gather)
    room = torch.full((plan.workspace_bytes,), 255, dtype=torch.uint8, device=DEV)
    dx, dw = torch.full((count, width), math.nan, dtype=dtype, device=DEV), torch.full((e, out, width), math.nan, dtype=dtype, device=DEV)
    plan.run(x, w[skip:], part, r, y, stream)
    plan.backward_input(dy, w[skip:], part, dx, stream, room)
    plan.backward_weight(dy, x, part, r, dw, stream, room)
    want, my, dxs, mx, dws, mw = grouped_plain(x, w[skip:], part, r, count, dy)
    near(y, want, my, width + 1, "y")
    near(dx, dxs, mx, out + 1, "dx")
    near(dw, dws, mw, max(counts) + 1, "dw")
    assert float(y[:first].abs().sum()) == 0.0 and float(dx[:first].abs().sum()) == 0.0
    return plan.describe()


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("counts,skip,width,out", [
    ([5, 3, 0, 9], 1, 64, 128), ([0, 17, 64, 1, 130], 2, 128, 96), ([70, 33, 5], 1, 8, 8), ([300, 5, 70], 1, 33, 7), ([700, 260, 1, 515], 1, 320, 512),
    ([257, 700, 30], 1, 1000, 520), ([1] * 80, 9, 192, 320), ([2, 1, 5] * 50, 100, 64, 72), ([4, 0, 0], 1, 64, 64), ([90, 0], 2, 64, 64)])
def test_part_of_the_experts(counts, skip, width, out, gather):
    if skip == len(counts):
        counts = counts + [0]               # an expert without rows behind all rows
    part_of_the_experts(counts, skip, width, out, torch.bfloat16, gather=gather)
    part_of_the_experts(counts, skip, width, out, torch.float16, f8=True, gather=gather)


@pytest.mark.parametrize("counts,skip,width,out,tile", [
    ([9] + [1] * 8, 1, 2048, 520, "stream16x32"), ([3, 3] + [1, 2, 0, 1] * 16, 2, 1024, 1032, "stream16x64"), ([35] + [20, 31, 0, 26, 22, 24, 30, 28], 1, 1024, 4096, "stream64x64"),
    ([200] + [30] * 60 + [0, 90, 5, 1], 1, 520, 2056, "ring64x128"), ([300] + [70] * 60 + [0, 290, 5, 1], 1, 520, 2056, "ring128x128"),
    ([300, 500, 1, 700, 900], 1, 2056, 4104, "pingpong256x256")])
def test_part_of_the_experts_by_each_kernel(counts, skip, width, out, tile):
    assert "tile=" + tile in part_of_the_experts(counts, skip, width, out, torch.bfloat16)


@pytest.mark.parametrize("counts,skip,width,out,tile", [([128, 40, 0, 100] + [41] * 61, 1, 2064, 1032, "ring64x128/2 e4m3"),
                                                        ([500, 1500, 77, 3000, 0], 1, 1040, 2056, "pingpong256x256 e4m3")])
def test_part_of_the_experts_by_the_e4m3_instruction(counts, skip, width, out, tile):
    assert "tile=" + tile in part_of_the_experts(counts, skip, width, out, torch.bfloat16, f8=True)


@pytest.mark.parametrize("t,e,k,width,out", [(300, 12, 3, 256, 128), (64, 6, 6, 72, 200), (500, 20, 4, 33, 17)])
def test_gradient_of_gathered_rows_is_rounded_once(t, e, k, width, out):
    g = gen(t)
    mask = torch.rand(t, e, generator=g, device=DEV) > 0.2
    r = km.route(randn(g, t, e), k, True, mask)
    x = randn(g, t, width).bfloat16().requires_grad_(True)
    w = (randn(g, e, out, width) * width ** -0.5).bfloat16()
    dy = randn(g, t * k, out).bfloat16()
    dx, = torch.autograd.grad(km.grouped_linear(x, w, r.offsets, r.rows, r.slots), x, dy)
    _, _, dxs, mx, *_ = grouped_plain(x.detach(), w, r.offsets, r.rows, t * k, dy)
    took = (r.slots >= 0)[:, :, None]
    pick = lambda v: torch.where(took, v[r.slots.long().clamp_min(0)], 0.0)
    want, terms = pick(dxs).sum(1), out + 1 + k
    near(dx, want, pick(mx).sum(1), terms, "dx")
    with pytest.raises(AssertionError):         # rows of 16 bits before the sum would not pass
        near(pick(dxs).bfloat16().double().sum(1).bfloat16(), want, pick(mx).sum(1), terms, "rows rounded first")


@pytest.mark.parametrize("counts,width,out,tile", [
    ([40, 0, 100] + [41] * 61, 2063, 1032, "ring64x128/2 any e4m3"), ([90] * 14 + [3, 300], 2050, 2056, "ring128x128/2 any e4m3"),
    ([2500], 2047, 4096, "ring128x128/2 any e4m3"), ([1030], 2063, 2056, "ring64x128/2 any e4m3"), ([1500, 77, 3000, 0], 1041, 2056, "ring128x128/2 any e4m3")])
def test_e4m3_instruction_on_rows_off_16_bytes(counts, width, out, tile):
    """Bounds as for whole rows: the instruction drops at most 8 x 2^-13 of the largest of 8 products, on top of the f32 sums' rounding."""
    g = gen(width + out)
    count = sum(counts) + 3
    offsets, rows = make_order(counts, 3, 777, g)
    grouped = len(counts) > 1
    x = (randn(g, 777 if grouped else count, width) * torch.exp(randn(g, 1, width))).bfloat16()
    w, ws = make_fp8(g, len(counts), out, width)
    xq, xs = km.quantize_rows(x)
    plan = K.LinearFp8(K.desc(x.shape, K.BF16), K.desc([len(counts), width, out], K.F8E4M3, "ACB"), K.desc([count, out], K.BF16), None, grouped, grouped)
    assert plan.describe().endswith("tile=" + tile), plan.describe()
    terms = width + 3 * (width // 128 + 1) + 2.0 ** 13
    if grouped:
        want, mag, *_ = grouped_plain(dequant(xq, xs), dequant(w, ws, 128), offsets, rows, count)
        ys = [km.grouped_linear_fp8(x, w, ws, offsets, rows), km.grouped_linear_fp8(xq, w, ws, offsets, rows, x_scale=xs)]
        assert float(ys[0][sum(counts):].abs().sum()) == 0.0
    else:
        xd, wd = dequant(xq, xs), dequant(w[0], ws[0], 128)
        want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
        ys = [km.linear_fp8(x, w[0], ws[0]), km.linear_fp8(xq, w[0], ws[0], x_scale=xs)]
    assert torch.equal(*ys)
    near(ys[0], want, mag, terms, "y")
    assert float((ys[0].double() - want).norm() / want.norm()) < 2.0 ** -9


WIDE = 1 << 20      # a row pitch of which some 4000 rows of 16 bits span 8 GB


@pytest.fixture(scope="module")
def room():
    """10 GB that operands with wide pitches lie in; what lies between their elements holds anything."""
    buffer = torch.empty(5 << 30, dtype=torch.bfloat16, device=DEV)
    yield buffer
    buffer.untyped_storage().resize_(0)
    torch.cuda.empty_cache()


def spread(room, values, *pitches):
    v = room.view(values.dtype) if values.element_size() == 2 else room.view(torch.uint8).view(values.dtype)
    at = torch.as_strided(v, values.shape, (*pitches, 1), 8)
    at.copy_(values)
    return at


@pytest.mark.parametrize("count", [200, 2100])
def test_offsets_past_32_bits_in_x_and_y(room, count):
    g = gen(count)
    x = spread(room, randn(g, 4200, 64).bfloat16(), WIDE + 8)
    counts = [count // 3, 0, count // 2]
    offsets, rows = make_order(counts, 5, 4200, g)
    rows[:3] = torch.tensor([4199, 0, 4198], dtype=torch.int32)
    total = sum(counts) + 5
    w = (randn(g, 3, 96, 64) / 8).bfloat16()
    dy = randn(g, total, 96).bfloat16()
    want, my, _, _, dw, mw = grouped_plain(x.contiguous(), w, offsets, rows, total, dy)
    near(km.grouped_linear(x, w, offsets, rows), want, my, 65, "y")
    wr = w.detach().requires_grad_(True)
    near(torch.autograd.grad(km.grouped_linear(x, wr, offsets, rows), wr, dy)[0], dw, mw, total, "dw")
    # rows of x in order, and of y: each tile's base is past 32 bits
    xs = spread(room, randn(g, total, 64).bfloat16(), 2 * WIDE + 8)
    near(km.grouped_linear(xs, w, offsets), *grouped_plain(xs.contiguous(), w, offsets, None, total)[:2], 65)
    y = spread(room, torch.zeros(total, 96).bfloat16(), 2 * WIDE + 8)
    dense = randn(g, total, 64).bfloat16()
    K.GroupedLinear(K.desc(dense.shape, K.BF16), K.desc([3, 64, 96], K.BF16, "ACB"), K.desc(y.shape, K.BF16, "AB", y.stride())).run(
        dense, w, offsets, None, y, torch.cuda.current_stream())
    near(y, *grouped_plain(dense, w, offsets, None, total)[:2], 65)


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 0, 50], [300, 500, 200]])
def test_offsets_past_32_bits_in_weights(room, counts):
    g = gen(sum(counts))
    offsets, _ = make_order(counts, 0, 1, g)
    total = sum(counts)
    x, dy = randn(g, total, 64).bfloat16(), randn(g, total, 300).bfloat16()
    for pitches, e in (((300 * (1 << 23), 1 << 23), 2), (((5 << 30) // 3 // 8 * 8 - 64 * 300, 64), 3)):     # far rows, far experts
        w = spread(room, (randn(g, e, 300, 64) / 8).bfloat16(), *pitches)
        mine = torch.cat([offsets[:e], offsets[-1:]]) if e == 3 else torch.cat([offsets[:2], offsets[-1:]])
        xr, wr = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = km.grouped_linear(xr, wr, mine)
        want, my, dxs, mx, dw, mw = grouped_plain(x, w.contiguous(), mine, None, total, dy)
        near(y.detach(), want, my, 65, "y")
        dx, = torch.autograd.grad(y, xr, dy)
        near(dx, dxs, mx, 301, "dx")
    w, ws = make_fp8(g, 3, 300, 128)
    far = spread(room, w, (10 << 30) // 3 // 16 * 16 - 128 * 300, 128)
    x = randn(g, total, 128).bfloat16()
    assert torch.equal(km.grouped_linear_fp8(x, far, ws, offsets), km.grouped_linear_fp8(x, w, ws, offsets))


def test_offsets_past_32_bits_in_8_bit_rows_logits_and_sums(room):
    g = gen(5)
    x = randn(g, 4200, 128).bfloat16()
    w, ws = make_fp8(g, 1, 264, 128)
    xq, xs = km.quantize_rows(x)
    for m in (4200, 40):                       # of one weight: the last rows alone as well
        far = spread(room, xq, 2 * WIDE + 16)[4200 - m:]
        want = km.linear_fp8(xq[4200 - m:].contiguous(), w[0], ws[0], x_scale=xs[4200 - m:], out_dtype=torch.float32)
        mag = dequant(xq, xs)[4200 - m:].abs() @ dequant(w[0], ws[0], 128).abs().t()
        near(km.linear_fp8(far, w[0], ws[0], x_scale=xs[4200 - m:], out_dtype=torch.float32), want.double(), 2 * mag, 140)
    far = spread(room, x, WIDE + 8)
    q, s = km.quantize_rows(far)
    assert torch.equal(q.view(torch.uint8), xq.view(torch.uint8)) and torch.equal(s, xs)
    rows = torch.randint(0, 4200, (500,), generator=g, device=DEV, dtype=torch.int32)
    offsets = torch.tensor([0, 500], dtype=torch.int32, device=DEV)
    far8 = spread(room, xq, 2 * WIDE + 16)
    xd, wd = dequant(xq, xs)[rows.long()], dequant(w[0], ws[0], 128)
    near(km.grouped_linear_fp8(far8, w, ws, offsets, rows, xs, torch.float32), xd @ wd.t(), xd.abs() @ wd.abs().t(), 140, "gathered")
    logits = randn(g, 4200, 60).bfloat16()
    a, b = km.route(spread(room, logits, WIDE + 8), 4, False), km.route(logits, 4, False)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    slots = torch.randperm(4200, generator=g, device=DEV).int().reshape(2100, 2)
    weights, dout = randn(g, 2100, 2), randn(g, 2100, 128).bfloat16()
    y = spread(room, x, WIDE + 8)
    assert torch.equal(km.combine(y, weights, slots), km.combine(x, weights, slots))
    wr = weights.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(km.combine(y, wr, slots), wr, dout)[0], torch.autograd.grad(km.combine(x, wr, slots), wr, dout)[0])


def test_layers_in_graphs():
    """Whole layers, captured at a size that no call had before and replayed between eager calls on other values."""
    g = gen(23)
    layer = km.MoEMlp(264, 200, 10, 3, device=DEV)
    served = layer.quantized()
    static = randn(g, 90, 264).bfloat16()
    mask = torch.ones(90, dtype=torch.bool, device=DEV)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = layer(static, mask), served(static, mask)
        for i in range(3):
            x, m = randn(g, 90, 264).bfloat16(), torch.rand(90, generator=g, device=DEV) > 0.3
            eager = layer(x, m), served(x, m)
            torch.cuda.synchronize()
            static.copy_(x)
            mask.copy_(m)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, captured))
