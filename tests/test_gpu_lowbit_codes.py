"""Codes and scales bit for bit: scale = max(max|y|, 2^-100) / 448 and code = y / scale, both quotients rounded to nearest in fp32, the
code then to nearest even in e4m3. IEEE division of tensors by tensors gives the same bits, so there is no tolerance."""
import pytest
import torch

from dace_onnx_b200 import ops
from tests.test_gpu_rows_quant import TINY, TYPES, make

pytestmark = pytest.mark.gpu


def expected(y):
    """y: fp32 rows."""
    scale = y.abs().amax(-1).clamp_min(TINY) / torch.full((), 448.0, device=y.device)
    return (y / scale[..., None]).to(torch.float8_e4m3fn), scale


def same(got, want):
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0].float(), want[0].float())


# a warp a row, a CTA a row, value by value, shifted, rows read twice
SHAPES = [(1, 1), (1300, 64), (1300, 100), (1300, 333), (103, 6622), (64, 4096), (7, 8191), (500, 1025), (3, 40000)]


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,length", SHAPES)
def test_rows(rows, length, t, cuda):
    """16-bit values over 16-bit maxima often lie at ties: the two roundings decide which way."""
    x = make(1, rows, length, t=TYPES[t])
    same(ops.quantize_rows(x), expected(x.float()))
    # every tie between two codes, and the fp32 values next to it
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    ties = (codes[1:] + codes[:-1]).cuda() / 2
    ties = torch.cat([ties, torch.nextafter(ties, ties + 1), torch.nextafter(ties, ties - 1), torch.full((1,), 448.0, device=cuda)])
    for top in (1.0, 3.0, 0.7):
        v = (ties * top).to(TYPES[t]).repeat(5, 1)
        same(ops.quantize_rows(v), expected(v.float()))


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,length", SHAPES)
def test_gated_rows(rows, length, t, cuda):
    x, gate = make(2, rows, length, t=TYPES[t]), make(3, rows, length, t=TYPES[t])
    same(ops.quantize_rows(x, gate=gate), expected(x.float() * gate.float()))
    same(ops.quantize_rows(x, gate=gate, activation="relu"), expected(x.float() * gate.float().clamp_min(0)))


@pytest.mark.parametrize("rows,length", [(1300, 64), (64, 4096), (5, 1024), (3, 40000)])
def test_normed_rows(rows, length, cuda):
    """The norm's codes are those of the values that the norm itself returns."""
    x, r = make(4, rows, length), make(5, rows, length)
    gamma = 1 + make(6, length, scale=0.2)
    for eps in (1e-5, 1e-12):
        y, _ = ops.rmsnorm(x, gamma, residual=r, eps=eps)
        same(ops.rmsnorm_quantize(x, gamma, residual=r, eps=eps), expected(y))


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("length", [1, 64, 333, 4096, 4097, 40000])
@pytest.mark.parametrize("eps", [1e-5, 1e-12, 1e-20, 1e-30])
def test_rows_of_zeros(length, eps, t, cuda):
    """Any eps: codes 0 and the floor's scale, whether the row, its sum with the residual or gamma is zero."""
    t = TYPES[t]
    zero, x, gamma = torch.zeros(3, length, device=cuda, dtype=t), make(7, 3, length, t=t), torch.ones(length, device=cuda, dtype=t)
    floor = expected(torch.zeros(3, 1, device=cuda))[1]
    for args in ((zero, gamma, None), (zero, None, zero), (x, gamma, -x), (x * 1e-4, gamma * 0, None)):
        q, s = ops.rmsnorm_quantize(args[0], args[1], residual=args[2], eps=eps)[:2]
        assert (q.float() == 0).all() and torch.equal(s, floor)


@pytest.mark.parametrize("length", [8, 100, 4096, 40000])
def test_small_rows_and_small_eps(length, cuda):
    """Values whose squares are lost beside eps: rho = 1 / sqrt(eps) alone, here a power of two."""
    x = make(8, 4, length) * 2.0 ** -80
    eps = 2.0 ** -60
    y = x * 2.0 ** 30
    same(ops.rmsnorm_quantize(x, eps=eps), expected(y))
    assert torch.equal(ops.rmsnorm(x, eps=eps), y)


@pytest.mark.parametrize("length", [64, 333, 4096, 40000])
def test_rows_of_any_magnitude(length, cuda):
    """A power of two moves to the scale: the codes stay, from values near the floor of a row's maximum to values near overflow."""
    x = make(9, 5, length).clamp(-7.9, 7.9)
    x[:, 0] = 2.0
    q, s = ops.quantize_rows(x)
    for k in (-99, -60, 60, 100, 125):
        same(ops.quantize_rows(x * 2.0 ** k), (q, s * 2.0 ** k))
