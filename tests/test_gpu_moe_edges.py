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
