"""Refusals and plans of the mixture-of-experts operators that need no GPU (plan creation makes no HIP calls)."""
import ctypes

import pytest

import kudnn_amd as K


def refused(status, make):
    with pytest.raises(K.KudnnError) as e:
        make()
    assert e.value.status == status and str(e.value)


def test_route_refusals():
    d = lambda *s, dt=K.F32, **kw: K.desc(list(s), dt, **kw)
    assert "launches=1" in K.MoeRoute(d(64, 8), 2).describe() and "launches=2" in K.MoeRoute(d(65, 8), 2).describe()
    assert K.MoeRoute(d(64, 8), 2).workspace_bytes == 0 and K.MoeRoute(d(65, 9), 2).workspace_bytes == 2 * 12
    K.MoeRoute(d(0, 8), 2), K.MoeRoute(d(7, 1024, dt=K.BF16), 32)
    for mask in (d(5, 8, dt=K.U8), d(1, 8, dt=K.U8), d(5, 1, dt=K.U8), d(1, 1, dt=K.U8)):
        K.MoeRoute(d(5, 8), 2, True, mask)
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(d(5, 8), 0))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(d(5, 8), 9))
    refused(K.UNSUPPORTED, lambda: K.MoeRoute(d(5, 64), 33))
    refused(K.UNSUPPORTED, lambda: K.MoeRoute(d(5, 1025), 2))
    refused(K.UNSUPPORTED, lambda: K.MoeRoute(d(5, 8, dt=K.S32), 2))
    refused(K.UNSUPPORTED, lambda: K.MoeRoute(d(1 << 29, 64), 8))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(d(2, 3, 8), 2))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(K.desc([5, 8], K.F32, "BA"), 2))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(d(5, 8), 2, True, d(4, 8, dt=K.U8)))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeRoute(d(5, 8), 2, True, d(5, 8)))


def test_grouped_linear_refusals():
    x, w, y = K.desc([6, 32], K.BF16), K.desc([3, 32, 24], K.BF16, "ACB"), K.desc([6, 24], K.BF16)
    assert "E=3" in K.GroupedLinear(x, w, y).describe()
    K.GroupedLinear(K.desc([4, 32], K.BF16), w, y, True)                                    # gathered: other row counts
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(K.desc([4, 32], K.BF16), w, y))
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(x, K.desc([3, 32, 24], K.BF16), y))    # K not contiguous
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(x, K.desc([32, 24], K.BF16, "BA"), y))
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(x, K.desc([3, 31, 24], K.BF16, "ACB"), y))
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(x, w, K.desc([6, 23], K.BF16)))
    refused(K.BAD_ARGUMENTS, lambda: K.GroupedLinear(x, K.desc([0, 32, 24], K.BF16, "ACB"), y))
    refused(K.UNSUPPORTED, lambda: K.GroupedLinear(x, K.desc([3, 32, 24], K.F16, "ACB"), y))
    refused(K.UNSUPPORTED, lambda: K.GroupedLinear(K.desc([6, 32], K.F32), K.desc([3, 32, 24], K.F32, "ACB"), K.desc([6, 24], K.F32)))
    refused(K.UNSUPPORTED, lambda: K.GroupedLinear(K.desc([1 << 24, 64], K.BF16), K.desc([3, 64, 1 << 20], K.BF16, "ACB"), K.desc([1 << 24, 1 << 20], K.BF16)))


def test_linear_fp8_refusals():
    f8 = K.F8E4M3
    x, w, y = K.desc([6, 200], K.BF16), K.desc([200, 24], f8, "BA"), K.desc([6, 24], K.F32)
    p = K.LinearFp8(x, w, y)
    assert p.workspace_bytes == 0 and " fused" in p.describe()                              # few rows: quantised by the product
    p = K.LinearFp8(K.desc([60, 200], K.BF16), w, K.desc([60, 24], K.F32))
    assert p.workspace_bytes == 60 * 256 + 60 * 2 * 4 and " fused" not in p.describe()
    assert K.LinearFp8(K.desc([6, 200], f8), w, y, K.desc([1, 24], K.F32)).workspace_bytes == 0
    wg = K.desc([3, 200, 24], f8, "ACB")
    K.LinearFp8(x, wg, y, None, True), K.LinearFp8(x, wg, K.desc([12, 24], K.F16), None, True, True)
    refused(K.BAD_ARGUMENTS, lambda: K.LinearFp8(x, wg, y))                                  # experts without groups
    refused(K.BAD_ARGUMENTS, lambda: K.LinearFp8(x, w, K.desc([12, 24], K.F16), None, False, True))
    refused(K.BAD_ARGUMENTS, lambda: K.LinearFp8(x, w, K.desc([5, 24], K.F32)))
    refused(K.BAD_ARGUMENTS, lambda: K.LinearFp8(x, K.desc([200, 24], f8), y))
    refused(K.UNSUPPORTED, lambda: K.LinearFp8(x, K.desc([200, 24], K.S8, "BA"), y))
    refused(K.UNSUPPORTED, lambda: K.LinearFp8(K.desc([6, 200], K.F32), w, y))
    refused(K.UNSUPPORTED, lambda: K.LinearFp8(x, w, K.desc([6, 24], K.S32)))
    refused(K.UNSUPPORTED, lambda: K.LinearFp8(x, w, y, K.desc([1, 24], K.BF16)))
    refused(K.UNSUPPORTED, lambda: K.LinearFp8(x, wg, y, K.desc([1, 24], K.F32), True))
    refused(K.BAD_ARGUMENTS, lambda: K.LinearFp8(x, w, y, K.desc([1, 23], K.F32)))


def test_combine_refusals():
    y, out = K.desc([12, 40], K.F16), K.desc([5, 40], K.F16)
    assert "k=2" in K.MoeCombine(y, out, 2).describe()
    refused(K.BAD_ARGUMENTS, lambda: K.MoeCombine(y, out, 0))
    refused(K.UNSUPPORTED, lambda: K.MoeCombine(y, out, 65))
    refused(K.BAD_ARGUMENTS, lambda: K.MoeCombine(y, K.desc([5, 41], K.F16), 2))
    refused(K.UNSUPPORTED, lambda: K.MoeCombine(y, K.desc([5, 40], K.F32), 2))
    refused(K.UNSUPPORTED, lambda: K.MoeCombine(K.desc([12, 40], K.S32), K.desc([5, 40], K.S32), 2))


def test_runs_refuse_missing_and_host_buffers():
    host = (ctypes.c_char * 4096)()
    at = ctypes.addressof(host) // 64 * 64 + 64
    r = K.MoeRoute(K.desc([4, 8], K.F32), 2)
    refused(K.NULL_POINTER, lambda: r.run(None, None, at, at, at, at, at))
    refused(K.NULL_POINTER, lambda: r.run(at, None, at, at, at, at, None))
    refused(K.BAD_ARGUMENTS, lambda: r.run(at, at, at, at, at, at, at))                      # a mask the plan has not
    refused(K.BAD_ARGUMENTS, lambda: r.run(at, None, at, at, at, at, at))                    # host memory
    refused(K.NULL_POINTER, lambda: r.backward(None, None, None, at, at, at))
    g = K.GroupedLinear(K.desc([4, 8], K.BF16), K.desc([2, 8, 8], K.BF16, "ACB"), K.desc([4, 8], K.BF16))
    refused(K.NULL_POINTER, lambda: g.run(at, at, None, None, at))
    refused(K.BAD_ARGUMENTS, lambda: g.run(at, at, at, at, at))                              # rows without gather
    refused(K.BAD_ARGUMENTS, lambda: g.run(at, at, at, None, at))
    refused(K.NULL_POINTER, lambda: g.backward_input(at, None, at, at))
    refused(K.NULL_POINTER, lambda: g.backward_weight(at, at, at, None, None))
    odd = K.GroupedLinear(K.desc([4, 9], K.BF16), K.desc([2, 9, 11], K.BF16, "ACB"), K.desc([4, 11], K.BF16))
    assert g.workspace_bytes == 0 and odd.workspace_bytes == 256 + 2 * 11 * 16 * 2
    refused(K.NULL_POINTER, lambda: odd.backward_input(at, at, at, at))                      # no workspace
    refused(K.NULL_POINTER, lambda: odd.backward_weight(at, at, at, None, at))
    f = K.LinearFp8(K.desc([40, 8], K.BF16), K.desc([8, 8], K.F8E4M3, "BA"), K.desc([40, 8], K.BF16))
    refused(K.NULL_POINTER, lambda: f.run(at, None, at, at, at))                             # no workspace
    refused(K.BAD_ARGUMENTS, lambda: f.run(at, at, at, at, at, workspace=at))                # a scale for bf16 x
    refused(K.BAD_ARGUMENTS, lambda: f.run(at, None, at, at, at, workspace=at))
    c = K.MoeCombine(K.desc([4, 8], K.BF16), K.desc([2, 8], K.BF16), 2)
    refused(K.NULL_POINTER, lambda: c.run(at, None, None, at))
    refused(K.BAD_ARGUMENTS, lambda: c.run(at, None, at, at))
    c.backward(None, None, None, None)                                                       # nothing asked for
    refused(K.BAD_ARGUMENTS, lambda: K.quantize_rows(K.desc([4, 8], K.BF16), at, at, 7, at))
    refused(K.BAD_ARGUMENTS, lambda: K.quantize_rows(K.desc([4, 8], K.BF16), at, at, 8, at))
    refused(K.UNSUPPORTED, lambda: K.quantize_rows(K.desc([4, 8], K.S8), at, at, 8, at))
    refused(K.NULL_POINTER, lambda: K.quantize_blocks(K.desc([1, 4, 8], K.BF16, "ACB"), at, None, at))
    for name in ("kudnn_moe_route_run", "kudnn_grouped_linear_run", "kudnn_linear_fp8_run", "kudnn_moe_combine_run"):
        fn = getattr(K.lib(), name)
        assert fn(*([None] * len(fn.argtypes))) == K.NULL_POINTER


def test_empty_calls_do_nothing():
    K.GroupedLinear(K.desc([0, 8], K.BF16), K.desc([2, 8, 8], K.BF16, "ACB"), K.desc([0, 8], K.BF16)).run(None, None, None, None, None)
    K.LinearFp8(K.desc([0, 8], K.BF16), K.desc([8, 8], K.F8E4M3, "BA"), K.desc([0, 8], K.BF16)).run(None, None, None, None, None)
    K.MoeCombine(K.desc([0, 8], K.BF16), K.desc([0, 8], K.BF16), 2).run(None, None, None, None)
    K.quantize_rows(K.desc([0, 8], K.BF16), None, None, 8, None)


def test_8_bit_floats_stay_out_of_the_other_operators():
    f8 = K.desc([8, 8], K.F8E4M3)
    b = K.desc([8, 8], K.BF16)
    for a in ((f8, b, b), (b, f8, b), (b, b, f8)):
        refused(K.UNSUPPORTED, lambda: K.Gemm(*a))
        refused(K.UNSUPPORTED, lambda: K.LinearPostOps(*a))
    refused(K.UNSUPPORTED, lambda: K.Gemm(b, b, b, K.desc([1, 8], K.F8E4M3)))


def test_torch_entry_points_refuse_host_tensors():
    import torch

    import kudnn_amd.torch_moe as km

    x, w, o = torch.randn(4, 8).bfloat16(), torch.randn(2, 8, 8).bfloat16(), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: km.route(torch.randn(4, 8), 2), lambda: km.grouped_linear(x, w, o), lambda: km.quantize_rows(x),
                 lambda: km.combine(x, None, torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: km.linear_fp8(x, w[0].to(torch.float8_e4m3fn), torch.ones(1, 1))):
        with pytest.raises(ValueError):
            call()


def test_types_of_the_input_gradient_and_of_f32_rows():
    host = (ctypes.c_char * 4096)()
    at = ctypes.addressof(host) // 64 * 64 + 64
    g = K.GroupedLinear(K.desc([4, 8], K.BF16), K.desc([2, 8, 8], K.BF16, "ACB"), K.desc([4, 8], K.BF16))
    refused(K.UNSUPPORTED, lambda: g.backward_input(at, at, at, at, dx_dtype=K.F16))
    refused(K.BAD_ARGUMENTS, lambda: g.backward_input(at, at, at, at, dx_dtype=K.F32))       # host memory
    c = K.MoeCombine(K.desc([12, 40], K.F32), K.desc([5, 40], K.F16), 2)
    refused(K.UNSUPPORTED, lambda: c.backward(at, at, at, at, at))
    refused(K.UNSUPPORTED, lambda: K.MoeCombine(K.desc([12, 40], K.BF16), K.desc([5, 40], K.F16), 2))
    refused(K.UNSUPPORTED, lambda: K.MoeCombine(K.desc([12, 40], K.F32), K.desc([5, 40], K.S32), 2))
