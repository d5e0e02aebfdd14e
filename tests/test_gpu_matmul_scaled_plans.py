"""Every kernel, tile and split of the product, on every pair of operand and output types, with the plan a call takes asserted.

The shapes have several tiles with ragged ends along M and N, and a ragged K. The CPU tests hold the list against the library's own
choice, so that a refit of the estimates that moves a shape to another plan shows here and not as lost coverage."""
import ctypes

import pytest
import torch

from dace_onnx_b200 import _lib, ops
from dace_onnx_b200._lib import GemmScaledDesc
from dace_onnx_b200.lowbit import FLOAT_TYPES, OPERAND_TYPES, _row_stride
from tests.test_gpu_matmul_scaled import TYPES, check, operands
from tests.test_gpu_rows_quant import U, make

PLANS = [(1, 128, 1), (1, 256, 1)] + [(0, rows, ctas) for rows in (16, 32, 64, 128, 256) for ctas in (1, 2, 4, 8)
                                      if (rows, ctas) != (256, 8)]
# plan: (M, N, K); the second ones where the first has a short K
CODES = {(1, 128, 1): (1192, 136, 1), (1, 256, 1): (3832, 552, 2221), (0, 16, 1): (17, 133, 2), (0, 16, 2): (18, 136, 907),
         (0, 16, 4): (17, 129, 2395), (0, 16, 8): (19, 129, 6092), (0, 32, 1): (2416, 134, 1), (0, 32, 2): (610, 144, 1423),
         (0, 32, 4): (313, 136, 2875), (0, 32, 8): (164, 136, 6688), (0, 64, 1): (4758, 137, 2), (0, 64, 2): (2425, 134, 651),
         (0, 64, 4): (611, 157, 2881), (0, 64, 8): (293, 135, 6698), (0, 128, 1): (6606, 261, 2), (0, 128, 2): (1739, 650, 643),
         (0, 128, 4): (2458, 134, 1448), (0, 128, 8): (595, 144, 6952), (0, 256, 1): (2920, 802, 3648), (0, 256, 2): (1075, 1037, 3648),
         (0, 256, 4): (942, 518, 3986)}
CODES_LONGER = {(1, 128, 1): (1192, 136, 625), (0, 16, 1): (22, 129, 614), (0, 32, 1): (1249, 131, 610), (0, 64, 1): (2448, 142, 778),
                (0, 128, 1): (1878, 1161, 629)}
HALVES = {(1, 128, 1): (1192, 136, 1), (1, 256, 1): (1538, 1416, 1098), (0, 16, 1): (17, 133, 2), (0, 16, 2): (24, 130, 473),
          (0, 16, 4): (20, 130, 1230), (0, 16, 8): (25, 136, 2835), (0, 32, 1): (2416, 134, 1), (0, 32, 2): (593, 168, 732),
          (0, 32, 4): (305, 136, 1493), (0, 32, 8): (154, 134, 3489), (0, 64, 1): (4758, 137, 2), (0, 64, 2): (2414, 138, 329),
          (0, 64, 4): (610, 144, 1423), (0, 64, 8): (291, 146, 3378), (0, 128, 1): (6606, 261, 2), (0, 128, 2): (1594, 675, 325),
          (0, 128, 4): (1242, 131, 1475), (0, 128, 8): (586, 157, 3459), (0, 256, 1): (3238, 645, 1957), (0, 256, 2): (1040, 1061, 1820),
          (0, 256, 4): (1714, 272, 1987)}
HALVES_LONGER = {(1, 128, 1): (1629, 264, 645), (0, 16, 1): (605, 136, 602), (0, 32, 1): (1192, 136, 625), (0, 64, 1): (1242, 385, 646),
                 (0, 128, 1): (1878, 1161, 629)}
CASES = [(t, p, s) for t, shapes in (("e4m3", CODES), ("e4m3", CODES_LONGER), ("bf16", HALVES), ("bf16", HALVES_LONGER), ("f16", HALVES),
                                     ("f16", HALVES_LONGER)) for p, s in shapes.items()]


def plan(m, n, k, t, out, lda, ldw, ldy, y=256):
    d = GemmScaledDesc(m, n, k, lda, ldw, ldy, ldy, 1, 1, OPERAND_TYPES[t], 0, FLOAT_TYPES[out], 0)
    p = (ctypes.c_int32 * 3)()
    _lib.check(_lib.load().b200_gemm_scaled_plan(ctypes.byref(d), None, ctypes.c_void_p(y), p))
    return tuple(p)


def test_the_lists_have_every_plan():
    assert set(CODES) == set(HALVES) == set(PLANS)


@pytest.mark.parametrize("t,want,shape", CASES)
def test_shapes_take_their_plans(t, want, shape):
    m, n, k = shape
    per = 16 // TYPES[t].itemsize
    pitch = -(-k // per) * per
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert plan(m, n, k, TYPES[t], out, pitch, pitch, n) == want


def test_query_refusals():
    lib, d = _lib.load(), GemmScaledDesc(4, 16, 32, 32, 32, 16, 16, 1, 1, 3, 0, 0, 0)
    p, y = (ctypes.c_int32 * 3)(), ctypes.c_void_p(256)
    assert lib.b200_gemm_scaled_plan(ctypes.byref(d), None, y, p) == _lib.OK
    assert lib.b200_gemm_scaled_plan(None, None, y, p) == _lib.EINVAL
    assert lib.b200_gemm_scaled_plan(ctypes.byref(d), None, y, None) == _lib.EINVAL
    for change in (dict(M=0), dict(N=-1), dict(K=0), dict(type=0), dict(y_type=3)):
        e = GemmScaledDesc(4, 16, 32, 32, 32, 16, 16, 1, 1, 3, 0, 0, 0)
        for key, v in change.items():
            setattr(e, key, v)
        assert lib.b200_gemm_scaled_plan(ctypes.byref(e), None, y, p) == _lib.EINVAL
    # rows that 16-byte accesses cannot address never take the kernel of many rows
    e = GemmScaledDesc(4096, 4096, 4096, 4096, 4096, 4096, 4096, 1, 1, 3, 0, 2, 0)
    assert lib.b200_gemm_scaled_plan(ctypes.byref(e), None, y, p) == _lib.OK and p[0] == 1
    for args in ((None, ctypes.c_void_p(258)), (ctypes.c_void_p(264), y)):
        assert lib.b200_gemm_scaled_plan(ctypes.byref(e), *args, p) == _lib.OK and p[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t,want,shape", CASES)
def test_products(t, want, shape, cuda):
    m, n, k = shape
    a, sa, w, sw = operands(m, n, k, TYPES[t])
    for out in (torch.float32, torch.bfloat16 if t != "f16" else torch.float16):
        y = torch.empty(m, n, device=cuda, dtype=out)
        assert plan(m, n, k, a.dtype, out, _row_stride(a), _row_stride(w), n, y.data_ptr()) == want
        bias, residual = make(5, n), make(6, m, n).to(out)
        ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, bias=bias, residual=residual, out=y)
        check(y, a, sa, w, sw, bias, None, residual)
    if t == "e4m3":
        check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=torch.float16), a, sa, w, sw)


# both kernels, K of a few and of many accumulators, split over CTAs and not
SUMS = [(1, 64, 16384), (40, 136, 16392), (300, 1001, 5536), (3055, 919, 2760), (3055, 920, 2760), (600, 2048, 16384), (1040, 1061, 1820)]


@pytest.mark.gpu
@pytest.mark.parametrize("one_sign", [True, False])
@pytest.mark.parametrize("t", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SUMS)
def test_sums_to_fp32(m, n, k, t, one_sign, cuda):
    """What the chunks of an fp32 sum are for. An addition in the tensor core truncates, so terms of one sign lose in one direction: with a
    single accumulator over all of K the sums fall short by about half of 2u an addition, 16392 / 16 of them 6e-5, far outside the bound
    of `check`. Chunks of c additions (32 of codes, 16 of 16-bit operands) lose at most 2u each at sums that grow evenly to the chunk's,
    so c u of it; their sums are added rounding to nearest, u each: in the 2-norm below (c + chunks + 11) u, with 8 for CTAs of a
    split and 3 for the scales. What the kernel's header states is measured: 1.5e-7 for codes, and 2.5e-6 (twice these chunks) for
    16-bit operands; twice the one and all of the other are asserted."""
    a, w = make(31, m, k), make(32, n, k, scale=k ** -0.5)
    if one_sign:
        a, w = a.abs(), w.abs()
    sa = sw = None
    if t == "e4m3":
        (a, sa), (w, sw) = ops.quantize_rows(a), ops.quantize_rows(w)
    else:
        a, w = a.to(TYPES[t]), w.to(TYPES[t])
    y = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=torch.float32)
    check(y, a, sa, w, sw)
    a64, w64 = (v.double() if s is None else v.double() * s.double()[:, None] for v, s in ((a, sa), (w, sw)))
    want = a64 @ w64.t()
    off = ((y.double() - want).norm() / want.norm()).item()
    print("2-norm error %.2e" % off)
    if one_sign:
        c, per = (32, 32) if t == "e4m3" else (16, 16)
        assert off < (c + -(-k // (c * per)) + 11) * U
    assert off < (3e-7 if t == "e4m3" else 2.5e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(3, 130, 28672), (600, 520, 28672)])
def test_long_sums_of_one_sign_to_16_bits(m, n, k, t, cuda):
    """One accumulator over all of K: 1792 truncating additions to sums that grow evenly lose at most 1792 u of the sum, 1.1e-4. That
    comes on top of the output's rounding, 4.9e-4 (fp16) or 3.9e-3 (bf16): `check` allows twice it."""
    a, w = make(41, m, k).abs().to(TYPES[t]), (make(42, n, k).abs() * k ** -0.5).to(TYPES[t])
    y = ops.matmul_scaled(a, w)
    check(y, a, None, w, None)
    want = a.double() @ w.double().t()
    assert ((y.double() - want).abs() <= (1792 * U + torch.finfo(TYPES[t]).eps / 2 * 1.001) * want).all()
