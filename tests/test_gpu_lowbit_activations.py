"""Gelu's tails on the 8-bit path, against 64 bits.

gelu(x) = max(x, 0) - |x| Q, Q = P(t) exp(-x^2 / 2). Relative error of Q in units of u = 2^-24: t = 1 / (1 + 0.35 w) one rounding and the
reciprocal's 2, which P takes at most 1.5 times over: 5; nine steps of P, whose terms partly cancel: 4; its fit 1; the exponent two
roundings and its constant's, 2.5 u of x^2 / 2: 1.25 x^2; the exponential 4, two products 2. So |error| <= (16 + 1.25 x^2) u |x| Phi(-|x|), and one
rounding of the result."""
import pytest
import torch

from dace_onnx_b200 import ops
from tests.test_gpu_rows_quant import U, check_codes, half_step, make

pytestmark = pytest.mark.gpu

# x < 0: only the tail; x > 0: what it takes off x
RANGES = [(-1, 0), (-4, -1), (-6, -4), (-8, -6), (-12, -8), (-0.01, 0.01), (0, 4), (4, 30), (-1e-6, 1e-6)]


def phi64(x):
    return 0.5 * torch.special.erfc(-x * 0.5 ** 0.5)   # (ndtr goes through 1 + erf, whose tail is lost below x = -6)


def gelu64(x):
    return x * phi64(x)


def gelu_error(x):
    return (16 + 1.25 * x * x) * U * x.abs() * phi64(-x.abs()) + 1.01 * U * gelu64(x).abs() + 1e-37


def spread(lo, hi, *shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (lo + (hi - lo) * torch.rand(*shape, generator=g, dtype=torch.float64)).float().cuda()


@pytest.mark.parametrize("lo,hi", RANGES)
@pytest.mark.parametrize("rows,length", [(3, 100), (1300, 64), (9, 4096), (400, 1001), (2, 40000)])
def test_rows_gated_in_one_range(lo, hi, rows, length, cuda):
    """The scale and the codes of a row are relative to its largest value, however small that is."""
    x, gate = make(2, rows, length), spread(lo, hi, rows, length)
    q, s = ops.quantize_rows(x, gate=gate, activation="gelu")
    y, err = gelu64(gate.double()) * x.double(), gelu_error(gate.double()) * x.double().abs()
    check_codes(q, s, y, 2 * U, err)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lo,hi", RANGES)
@pytest.mark.parametrize("m", [1, 5, 300])
def test_products(lo, hi, m, out, cuda):
    """Sums of one term (rows of a times the unit matrix): the activation's argument is exact."""
    a = spread(lo, hi, m, 64).bfloat16()
    w = torch.eye(64, device=cuda).bfloat16()
    y = ops.matmul_scaled(a, w, activation="gelu", out_dtype=out).double()
    x = a.double()
    want, err = gelu64(x), gelu_error(x)
    # the smallest normal number: the tail is flushed below it
    assert ((y - want).abs() <= err + half_step(out) * 1.0001 * (want.abs() + err) + 2.0 ** -126).all()


def test_infinities_and_nan(cuda):
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e30, -1e30, 3e38, -3e38, -20.0, 1e-38, -1e-38]], device=cuda)
    want = gelu64(x.double())
    w = torch.eye(16, device=cuda).bfloat16()
    for m in (1, 40):   # both kernels
        a = torch.zeros(m, 16, device=cuda, dtype=torch.bfloat16)
        for j in range(x.shape[1]):
            # one value a call: an infinity or a NaN spoils the sums of its row
            bias = torch.zeros(16, device=cuda)
            bias[j] = x[0, j]
            y = ops.matmul_scaled(a, w, bias=bias, activation="gelu", out_dtype=torch.float32)[:, j].double()
            assert torch.allclose(y, want[0, j].expand(m), rtol=1e-6, atol=2e-38, equal_nan=True), (j, y[0], want[0, j])
            q, s = ops.quantize_rows(torch.ones(1, 16, device=cuda), gate=bias[None], activation="gelu")
            top = want[0, j].abs()
            if torch.isnan(top):
                assert torch.isnan(s).all() and torch.isnan(q.float()).all()
            elif torch.isinf(top):
                assert torch.isinf(s).all()
            else:
                assert abs(s.item() - max(top.item(), 2.0 ** -100) / 448) <= 1e-6 * s.item()
