"""The product on e4m3 / 16-bit operands with scales and a fused epilogue, against the formula in 64 bits.

Tolerances, from the arithmetic (u = 2^-24; S = sum_k |a w| with its scales):
  sum    an addition into the tensor core's accumulator truncates: at most 2u of S each. One instruction takes 32 (codes) or
         16 values of K; fp32 outputs start a new accumulator every 32 (codes) or 16 instructions and add these rounding to
         nearest, and K may be split over 8 CTAs
  scales, bias: 3 roundings; activations: the bounds of act_error in test_gpu_rows_quant, slope at most 1.13
  result one rounding to its type: half a step
"""
import pytest
import torch

from dace_onnx_b200 import ops
from tests.test_gpu_rows_quant import U, act64, act_error, half_step, make

pytestmark = pytest.mark.gpu

TYPES = {"e4m3": torch.float8_e4m3fn, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def operands(m, n, k, t, seed=1):
    a, w = make(seed, m, k), make(seed + 1, n, k, scale=k ** -0.5)
    if t == torch.float8_e4m3fn:
        return ops.quantize_rows(a) + ops.quantize_rows(w)
    pitch = -(-k // 8) * 8
    rows = lambda x: torch.zeros(x.shape[0], pitch, device="cuda", dtype=t)[:, :k].copy_(x)  # noqa: E731
    return rows(a), None, rows(w), None


def check(y, a, sa, w, sw, bias=None, act=None, residual=None):
    k = a.shape[-1]
    wide = lambda v, s: v.double() if s is None else v.double() * s.double().reshape(-1, 1)  # noqa: E731
    a64, w64 = wide(a.reshape(-1, k), sa), wide(w, sw)
    pre, size = a64 @ w64.t(), a64.abs() @ w64.abs().t()
    codes = a.dtype == torch.float8_e4m3fn
    adds = -(-k // (32 if codes else 16))
    if y.dtype == torch.float32:
        adds = (32 if codes else 16) + 8 + -(-adds // (32 if codes else 16))
    err = (adds * 2 * U + 3 * U) * size
    if bias is not None:
        pre = pre + bias.double()
        err = err + U * pre.abs()
    want = act64(pre, act)
    err = 1.13 * err + act_error(pre, act)
    if residual is not None:
        want = want + residual.reshape(want.shape).double()
        err = err + U * want.abs()
    floor = torch.finfo(y.dtype).tiny * torch.finfo(y.dtype).eps
    bound = err + (half_step(y.dtype) * 1.0001 + U) * (want.abs() + err) + floor
    got = y.reshape(want.shape).double()
    off = (got - want).abs()
    assert (off <= bound).all(), "off by %.3g of the bound" % (off / bound).max().item()


# one row; the limits of each token tile; odd sizes; several row tiles with and without vector rows; K below, at and past
# a K-block, a stage, a chunk
SHAPES = [(1, 1, 1), (1, 128, 16), (1, 4096, 4096), (3, 31, 100), (16, 129, 128), (17, 200, 1000), (32, 512, 4096),
          (33, 1501, 333), (64, 64, 8192), (65, 96, 4112), (128, 1000, 257), (129, 256, 520), (256, 130, 1024),
          (257, 128, 128), (300, 136, 640), (333, 1501, 1000), (513, 768, 1040), (1000, 1032, 96), (2100, 640, 513)]


@pytest.mark.parametrize("t", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(m, n, k, t, cuda):
    t = TYPES[t]
    a, sa, w, sw = operands(m, n, k, t)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=out), a, sa, w, sw)
        bias, residual = make(5, n).to(out), make(6, m, n).to(out)
        y = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, bias=bias, activation="silu", residual=residual)
        assert y.dtype == out
        check(y, a, sa, w, sw, bias, "silu", residual)


# shapes that between them take every tile and split: 128 and 256 wide pairs, tiles of 16 to 256 rows on 1 to 8 CTAs
PLANS = [(2371, 64, 68), (4455, 536, 2204), (4154, 515, 66), (4991, 132, 688), (4898, 73, 1535), (1, 64, 904), (10, 64, 2349),
         (1, 64, 5667), (4993, 401, 3709), (4780, 135, 3993), (4836, 67, 4006), (4739, 70, 64), (1208, 72, 1495), (657, 64, 2915),
         (4786, 133, 79), (4979, 68, 656), (1189, 64, 3000), (289, 64, 7192), (594, 64, 7511), (593, 136, 7051)]


@pytest.mark.parametrize("m,n,k", PLANS)
def test_every_plan(m, n, k, cuda):
    a, sa, w, sw = operands(m, n, k, torch.float8_e4m3fn)
    for out in (torch.bfloat16, torch.float32):
        bias, residual = make(5, n), make(6, m, n).to(out)
        check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, bias=bias, residual=residual), a, sa, w, sw, bias, None, residual)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(3055, 919, 5536), (3055, 920, 5536), (40, 1001, 16392)])
def test_long_sums_to_fp32(m, n, k, t, cuda):
    """Many accumulators one after the other, on rows that vector accesses can address and not."""
    a, _, w, _ = operands(m, n, k, TYPES[t])
    bias = make(5, n)
    check(ops.matmul_scaled(a, w, bias=bias, activation="gelu_tanh", out_dtype=torch.float32), a, None, w, None, bias, "gelu_tanh")


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,n", [(5, 333), (300, 512)])
def test_epilogues(m, n, act, cuda):
    a, sa, w, sw = operands(m, n, 256, torch.float8_e4m3fn)
    for out in (torch.float32, torch.bfloat16):
        for bias in (None, make(7, n, scale=2.0), make(7, n, scale=2.0).half()):
            for residual in (None, make(8, m, n).to(out)):
                y = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, bias=bias, activation=act, residual=residual, out_dtype=out)
                check(y, a, sa, w, sw, bias, act, residual)


@pytest.mark.parametrize("m,n,k", [(7, 300, 512), (400, 512, 512)])
def test_strides_scales_and_layouts(m, n, k, cuda):
    a, sa, w, sw = operands(m, n, k, torch.float8_e4m3fn)
    want = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw)
    # operands inside wider tensors, aligned and not (the latter are copied), and transposed storage
    for off, pitch in ((0, k + 32), (16, k + 48), (5, k + 7)):
        wide_a = torch.zeros(m, pitch, device="cuda").to(a.dtype)[:, min(off, pitch - k):][:, :k]
        wide_a.copy_(a)
        assert torch.equal(ops.matmul_scaled(wide_a, w, a_scale=sa, w_scale=sw), want)
    wt = torch.empty(k, n, device="cuda", dtype=w.dtype).t()
    wt.copy_(w)
    assert torch.equal(ops.matmul_scaled(a, wt, a_scale=sa, w_scale=sw), want)
    # one scale for all rows, on either side
    one = torch.tensor(0.25, device="cuda")
    check(ops.matmul_scaled(a, w, a_scale=one, w_scale=sw), a, one.expand(m), w, sw)
    check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=one.reshape(1)), a, sa, w, one.expand(n))
    check(ops.matmul_scaled(a, w), a, None, w, None)
    # outputs with row strides (dividing the vector width or not), what lies around them stays; residual is the output
    for pitch in (n + 16, n + 3):
        buf = torch.full((m + 2, pitch), 3.0, device="cuda", dtype=torch.bfloat16)
        y = buf[:m, :n]
        residual = make(9, m, n).bfloat16()
        y.copy_(residual)
        ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, residual=y, out=y)
        check(y, a, sa, w, sw, None, None, residual)
        assert (buf[m:] == 3).all() and (buf[:, n:] == 3).all()
    # a broadcast residual, leading axes, no rows
    row = make(10, n).bfloat16()
    check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, residual=row.expand(m, n)), a, sa, w, sw, None, None, row.expand(m, n))
    a3 = a.reshape(1, m, k)
    assert torch.equal(ops.matmul_scaled(a3, w, a_scale=sa.reshape(1, m), w_scale=sw)[0], want)
    assert ops.matmul_scaled(a[:0], w, a_scale=sa[:0], w_scale=sw).shape == (0, n)
    assert ops.matmul_scaled(a, w[:0], a_scale=sa, w_scale=sw[:0]).shape == (m, 0)


def test_special_values(cuda):
    """An infinity or a NaN reaches exactly the outputs whose sums contain it; infinite scales too."""
    for m in (4, 300):
        a, w = make(11, m, 64).bfloat16(), make(12, 96, 64).bfloat16()
        a[1, 3], w[5, 0], a[2, 7] = float("nan"), float("inf"), float("-inf")
        y = ops.matmul_scaled(a, w, out_dtype=torch.float32)
        want = a.double() @ w.double().t()
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(torch.isinf(y), torch.isinf(want)) and torch.equal(y.sign()[torch.isinf(y)].double(), want.sign()[torch.isinf(want)])


@pytest.mark.parametrize("m,n,k", [(1, 512, 8192), (40, 256, 4096), (300, 256, 1024)])
def test_the_same_call_gives_the_same_bits(m, n, k, cuda):
    a, sa, w, sw = operands(m, n, k, torch.float8_e4m3fn)
    first = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(first, ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=torch.float32))


def test_streams_and_graphs(cuda):
    """Two products at once on two streams, and two captured ones replayed after their inputs changed."""
    small, large = operands(8, 1024, 2048, torch.float8_e4m3fn, 20), operands(600, 512, 1024, torch.float8_e4m3fn, 30)
    run = lambda o: ops.matmul_scaled(o[0], o[2], a_scale=o[1], w_scale=o[3])  # noqa: E731
    want = run(small), run(large)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, o in zip(streams, (small, large)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([run(o) for _ in range(4)])
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)
    graphs = []
    for o in (small, large):
        a = torch.zeros_like(o[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.matmul_scaled(a, o[2], a_scale=o[1], w_scale=o[3])
        graphs.append((g, a, y))
    for (g, a, y), o in zip(graphs, (small, large)):
        a.copy_(o[0])
    for g, _, _ in graphs:
        g.replay()
    for (_, _, y), w in zip(graphs, want):
        assert torch.equal(y, w)


def test_prepared_linear(cuda):
    weight, bias = make(40, 200, 333, scale=0.05), make(41, 200)
    for t in ("e4m3", "f16", "bf16"):
        layer = ops.PreparedLinear(weight, bias, activation="gelu", dtype=TYPES[t])
        for x in (make(42, 3, 7, 333), make(43, 400, 333, t=torch.bfloat16)):
            y = layer(x)
            assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (200,)
            if t == "e4m3":
                q, s = ops.quantize_rows(x)
                check(y, q, s, layer.weight, layer.w_scale, bias, "gelu")
                assert torch.equal(layer(q, a_scale=s, out_dtype=x.dtype), y)
            else:
                check(y, x.to(TYPES[t]), None, layer.weight, None, bias, "gelu")
    with pytest.raises(ValueError, match="a_scale"):
        ops.PreparedLinear(weight)(q)


def test_checked_path_gives_the_same(cuda, monkeypatch):
    """Calls that the C++ entry declines take the path that checks and copies in Python: the same bits."""
    from dace_onnx_b200 import torch_calls
    for m, n, k in ((5, 100, 333), (300, 264, 512)):
        a, sa, w, sw = operands(m, n, k, torch.float8_e4m3fn)
        bias, residual = make(50, n).bfloat16(), make(51, m, n).bfloat16()
        args = dict(a_scale=sa, w_scale=sw, bias=bias, activation="relu", residual=residual)
        want = ops.matmul_scaled(a, w, **args)
        with monkeypatch.context() as p:
            p.setattr(torch_calls, "matmul_scaled", lambda *_: None)
            p.setattr(torch_calls, "quantize_rows", lambda *_: None)
            assert torch.equal(ops.matmul_scaled(a, w, **args), want)
            out = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
            assert ops.matmul_scaled(a, w, out=out, **args) is out and torch.equal(out, want)
            again = ops.quantize_rows(make(1, m, k))
            assert torch.equal(again[0].float(), a.float()) and torch.equal(again[1], sa)
            assert ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=torch.float32).dtype == torch.float32


def test_refusals(cuda):
    a, sa, w, sw = operands(4, 32, 64, torch.float8_e4m3fn)
    with pytest.raises(TypeError):
        ops.matmul_scaled(a.float(), w.float())
    with pytest.raises(TypeError):
        ops.matmul_scaled(a, w.to(torch.bfloat16))
    with pytest.raises(ValueError, match="A must be"):
        ops.matmul_scaled(a, w[:, :32])
    with pytest.raises(ValueError, match="K must be"):
        ops.matmul_scaled(a[:, :0], w[:, :0])
    with pytest.raises(ValueError, match="a_scale"):
        ops.matmul_scaled(a, w, a_scale=sa[:3])
    with pytest.raises(TypeError, match="w_scale"):
        ops.matmul_scaled(a, w, w_scale=sw.half())
    with pytest.raises(ValueError, match="bias"):
        ops.matmul_scaled(a, w, bias=torch.ones(31, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        ops.matmul_scaled(a, w, residual=torch.ones(4, 31, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        ops.matmul_scaled(a, w, residual=torch.ones(4, 32, device="cuda"), out=torch.empty(4, 32, device="cuda").half())
    with pytest.raises(ValueError, match="activation"):
        ops.matmul_scaled(a, w, activation="tanh")
    with pytest.raises(TypeError, match="output must be"):
        ops.matmul_scaled(a, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="shape"):
        ops.matmul_scaled(a, w, out=torch.empty(4, 31, device="cuda"))
