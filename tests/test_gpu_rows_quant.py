"""RMS norm with residual and 8-bit output, and the row quantiser, against the formulas in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32):
  h      one fp32 addition and one rounding to the type: (u + eps/2) |h|
  rho    the sum of squares is a tree of at most 32 (or len / 1024, long rows) + 10 additions a leaf, all terms positive,
         then a division, an addition, a square root: relative error below CHAIN(len) u
  y      rho, two products, one rounding
  codes  half a step of e4m3, 2^-4 of the value or 2^-10 below the smallest normal number, plus the error of y / scale
"""
import math

import pytest
import torch

from dace_onnx_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = 2.0 ** -100


def chain(length):
    return (48 + length / 1024) * U


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def make(seed, *shape, t=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(t).cuda()


def act64(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "gelu":
        return v * 0.5 * (1 + torch.erf(v / math.sqrt(2)))
    if act == "gelu_tanh":
        return v * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def act_error(v, act):
    """Bound of the fp32 activation's absolute error. exp: (2 + 1.173 |z|) ulp (z = the sigmoid's argument), the division 2 ulp,
    three roundings around them; gelu: the polynomial's erf is within 6e-7, times |v| / 2, four roundings."""
    a = v.abs()
    if act == "silu":
        return (7 + 1.173 * a) * 2 * U * act64(v, act).abs()
    if act == "gelu_tanh":
        z = (2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)).abs()
        return (7 + 1.173 * z + 4 * z) * 2 * U * act64(v, act).abs()
    if act == "gelu":
        return 3e-7 * a + 4 * U * a
    return 0 * a


def check_codes(q, s, y, rel, err=0.0):
    """q, s against y (64 bits), y known to `rel` relative and `err` absolute (a tensor like y, or 0)."""
    assert q.dtype == torch.float8_e4m3fn and q.shape == y.shape and s.dtype == torch.float32
    worst = err.amax(-1) if isinstance(err, torch.Tensor) else 0.0
    top = y.abs().amax(-1).clamp_min(TINY)
    assert ((s.double() - top / 448).abs() <= (rel + 4 * U) * top / 448 + worst / 448).all()
    v = y / s.double()[..., None]
    slack = (rel + 6 * U) * v.abs() + err / s.double()[..., None]
    # the largest code of a row may round up to at most 448
    bound = torch.maximum((v.abs() + slack) * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + slack
    assert ((q.double() - v).abs() <= bound).all()


def norm64(x, residual, gamma, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, y if gamma is None else y * gamma.double()


def check_norm(x, residual, gamma, eps=1e-5):
    length = x.shape[-1]
    h64, y64 = norm64(x, residual, gamma, eps)
    got = ops.rmsnorm(x, gamma, residual=residual, eps=eps)
    codes = ops.rmsnorm_quantize(x, gamma, residual=residual, eps=eps)
    y = got if residual is None else got[0]
    if residual is not None:
        for h in (got[1], codes[2]):
            assert h.dtype == x.dtype
            tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # half a step of the subnormal numbers
            assert ((h.double() - h64).abs() <= (U + half_step(x.dtype)) * 1.0001 * h64.abs() + tiny).all()
    assert y.dtype == x.dtype
    floor = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert ((y.double() - y64).abs() <= (chain(length) + 1.0001 * half_step(x.dtype)) * y64.abs() + floor).all()
    check_codes(codes[0], codes[1], y64, chain(length))


# one value, below and at a vector, odd, a warp's and a CTA's limits, rows read twice
SHAPES = [(1, 1), (3, 7), (5, 8), (9, 64), (130, 333), (17, 512), (3, 513), (64, 1000), (33, 1024), (2, 1028), (7, 2561),
          (1, 4096), (300, 4096), (2, 8192), (3, 8200), (2, 16384), (2, 16392), (1, 20001), (2, 40000)]


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,length", SHAPES)
def test_norm(rows, length, t, cuda):
    t = TYPES[t]
    x, r = make(1, rows, length, t=t), make(2, rows, length, t=t, scale=3.0)
    gamma = 1 + make(3, length, scale=0.2)
    check_norm(x, r, gamma.to(t))
    check_norm(x, None, gamma)      # gamma in fp32 whatever x's type
    check_norm(x, r, None)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,length", SHAPES)
def test_quantize(rows, length, t, cuda):
    t = TYPES[t]
    x, gate = make(4, rows, length, t=t), make(5, rows, length, t=t, scale=2.0)
    q, s = ops.quantize_rows(x)
    check_codes(q, s, x.double(), 0.0)
    for act in (None, "relu", "gelu", "gelu_tanh", "silu"):
        q, s = ops.quantize_rows(x, gate=gate, activation=act)
        y = act64(gate.double(), act) * x.double()
        check_codes(q, s, y, 2 * U, act_error(gate.double(), act) * x.double().abs())


def test_rows_of_zeros_and_tiny_values(cuda):
    x = torch.zeros(3, 40, device="cuda")
    x[1] = 1e-38          # below the floor of a row's maximum
    x[2, 5] = 2.0 ** -90
    q, s = ops.quantize_rows(x)
    assert (q[0].float() == 0).all() and (q[1].float() == 0).all()
    assert s[0].item() == s[1].item() == torch.tensor(TINY / 448, dtype=torch.float32).item()
    assert q[2, 5].float().item() == 448
    z = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    q, s, h = ops.rmsnorm_quantize(z, residual=z, eps=1e-6)
    assert (q.float() == 0).all() and torch.isfinite(s).all() and (h == 0).all()
    assert torch.isnan(ops.rmsnorm(z, eps=0.0)).all()  # 0 / 0, as the formula says


@pytest.mark.parametrize("length", [40, 333, 4096, 20000])
def test_nan_and_infinity_stay_in_their_row(length, cuda):
    x = make(6, 4, length)
    x[1, length // 2] = float("nan")
    x[2, 3] = float("inf")
    q, s = ops.quantize_rows(x)
    assert torch.isnan(s[1]) and torch.isnan(q[1].float()).all()
    assert s[2].item() == float("inf") and torch.isnan(q[2, 3].float())
    clean = [0, 3]
    check_codes(q[clean], s[clean], x[clean].double(), 0.0)
    y = ops.rmsnorm(x)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[clean]).all()
    qn, sn = ops.rmsnorm_quantize(x)
    assert torch.isnan(sn[1]) and torch.isnan(qn[1].float()).all()
    check_codes(qn[clean], sn[clean], norm64(x, None, None, 1e-6)[1][clean], chain(length))


def test_strides_and_broadcast_rows(cuda):
    wide = make(7, 12, 300, t=torch.bfloat16)
    for x, g in ((wide[:, :128], wide[:, 128:256]), (wide[:, 3:131], wide[:, 150:278]), (wide[::2, :128], wide[1::2, 8:136])):
        q, s = ops.quantize_rows(x, gate=g, activation="silu")
        check_codes(q, s, act64(g.double(), "silu") * x.double(), 2 * U, act_error(g.double(), "silu") * x.double().abs())
        check_norm(x, g, None)
    row = make(8, 128, t=torch.bfloat16)
    check_norm(wide[:, :128], row.expand(12, 128), None)                    # row stride 0
    windows = make(17, 400).as_strided((12, 64), (24, 1))                   # rows that overlap
    check_norm(windows, windows, None)
    q, s = ops.quantize_rows(windows)
    check_codes(q, s, windows.double(), 0.0)
    x3 = make(9, 2, 3, 5, 64)
    check_norm(x3, x3 * 2, None)
    check_norm(x3.permute(1, 0, 2, 3), None, None)                          # leading axes that do not merge: copied
    check_norm(x3.transpose(2, 3), None, None)                              # elements of a row apart: copied
    check_norm(make(10, 77), None, None)                                    # one row without a leading axis
    for shape in ((0, 64), (2, 0, 64)):
        q, s, h = ops.rmsnorm_quantize(torch.empty(shape, device="cuda"), residual=torch.empty(shape, device="cuda"))
        assert q.shape == shape and s.shape == shape[:-1] and h.shape == shape


# a warp's and a CTA's limits; rows behind multiples of 16 bytes by every distance, all tensors by the same
@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("rows,length", [(1300, 9), (1300, 100), (1250, 249), (1200, 511), (1300, 1000), (40, 2305), (5, 4609),
                                         (3, 9217), (2, 18001)])
def test_rows_off_the_vector_grid(rows, length, t, cuda):
    t = TYPES[t]
    pitch = length | 1
    for off in (0, 1, 6):
        place = lambda seed: make(seed, rows * pitch + 16, t=t)[off:off + rows * pitch].view(rows, pitch)[:, :length]  # noqa: E731
        x, r, gamma = place(30), place(31), 1 + make(32, length, scale=0.1)
        check_norm(x, r, gamma.to(t))
        q, s = ops.quantize_rows(x, gate=r, activation="silu")
        check_codes(q, s, act64(r.double(), "silu") * x.double(), 2 * U, act_error(r.double(), "silu") * x.double().abs())
        # outputs at the same distance, in place and inside a larger buffer whose other values stay
        want = ops.rmsnorm(x, gamma, residual=r)
        y, h = ops.rmsnorm(x, gamma, residual=r, out=torch.empty_like(want[0]), residual_out=r)
        assert torch.equal(y, want[0]) and torch.equal(r, want[1])
        buf = torch.full((rows * pitch + 16,), 7.0, device="cuda", dtype=t)
        out = buf[off:off + rows * pitch].view(rows, pitch)[:, :length]
        ops.rmsnorm(x, gamma, out=out)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[off:off + rows * pitch].view(rows, pitch)[:, :length] = False
        # not the bits of an output that lies elsewhere: another kernel may add the squares in another order, so each is within
        # the bound of check_norm of the exact value
        y64 = norm64(x, None, gamma, 1e-6)[1]
        floor = torch.finfo(t).tiny * torch.finfo(t).eps
        assert ((out.double() - y64).abs() <= (chain(length) + 1.0001 * half_step(t)) * y64.abs() + floor).all()
        assert (buf[keep] == 7).all()


@pytest.mark.parametrize("length", [100, 4096, 20000])
def test_in_place_and_what_lies_behind_the_rows(length, cuda):
    x, r = make(11, 6, length, t=torch.float16), make(12, 6, length, t=torch.float16)
    h64, y64 = norm64(x, r, None, 1e-6)
    stream = r.clone()
    y, h = ops.rmsnorm(x, residual=stream, residual_out=stream)
    want = ops.rmsnorm(x, residual=r)
    assert h is stream and torch.equal(h, want[1]) and torch.equal(y, want[0])
    both = x.clone()
    y, h = ops.rmsnorm(both, residual=r, out=both, residual_out=torch.empty_like(r))
    assert y is both and torch.equal(y, want[0])
    # outputs inside larger buffers: what lies behind the last row and between the rows stays
    pitch = length + 24
    codes = torch.full((8, pitch), 1.0, device="cuda").to(torch.float8_e4m3fn)
    scale = torch.full((8,), 7.0, device="cuda")
    ops.quantize_rows(x, out=codes[:6, :length], scale=scale[:6])
    check_codes(codes[:6, :length], scale[:6], x.double(), 0.0)
    assert (codes[6:].float() == 1).all() and (codes[:, length:].float() == 1).all() and (scale[6:] == 7).all()


def test_other_stream_and_graph(cuda):
    x, r = make(13, 40, 1000, t=torch.bfloat16), make(14, 40, 1000, t=torch.bfloat16)
    want = ops.rmsnorm_quantize(x, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rmsnorm_quantize(x, residual=r)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.float(), b.float())
    sx, sr = torch.zeros_like(x), torch.zeros_like(r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s, h = ops.rmsnorm_quantize(sx, residual=sr)
        q2, s2 = ops.quantize_rows(h)
    for k in range(2):
        sx.copy_(x), sr.copy_(r * (k + 1))
        graph.replay()
        want = ops.rmsnorm_quantize(x, residual=r * (k + 1))
        again = ops.quantize_rows(want[2])
        for a, b in zip((q, s, h, q2, s2), want + again):
            assert torch.equal(a.float(), b.float())


def test_the_same_call_gives_the_same_bits(cuda):
    x = make(15, 64, 4096, t=torch.bfloat16)
    first = ops.rmsnorm_quantize(x)
    for _ in range(3):
        again = ops.rmsnorm_quantize(x)
        assert torch.equal(first[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(first[1], again[1])


def test_checked_path_gives_the_same(cuda, monkeypatch):
    """Calls that the C++ entry declines take the path that checks and copies in Python: the same bits."""
    from dace_onnx_b200 import torch_calls
    x, r, g = make(20, 5, 333, t=torch.bfloat16), make(21, 5, 333, t=torch.bfloat16), 1 + make(22, 333, scale=0.1)
    want = ops.rmsnorm_quantize(x, g, residual=r), ops.rmsnorm(x, g, residual=r), ops.quantize_rows(x, gate=r, activation="gelu")
    with monkeypatch.context() as p:
        for name in ("rmsnorm", "quantize_rows"):
            p.setattr(torch_calls, name, lambda *_: None)
        got = ops.rmsnorm_quantize(x, g, residual=r), ops.rmsnorm(x, g, residual=r), ops.quantize_rows(x, gate=r, activation="gelu")
        h, s, q = torch.empty_like(x), torch.empty(5, device="cuda"), ops.empty_codes((5, 333), "cuda")
        given = ops.rmsnorm_quantize(x, g, residual=r, out=q, scale=s, residual_out=h)
        assert given[0] is q and given[1] is s and given[2] is h
    for a, b in zip(want + (want[0],), got + (given,)):
        for u, v in zip(a, b):
            assert u.shape == v.shape and u.stride() == v.stride() and torch.equal(u.float(), v.float())
    given = ops.rmsnorm_quantize(x, g, residual=r, out=q, scale=s, residual_out=h)
    assert given[0] is q and given[1] is s and given[2] is h


def test_refusals(cuda):
    x = make(16, 4, 64)
    with pytest.raises(TypeError):
        ops.rmsnorm(x.double())
    with pytest.raises(ValueError, match="residual"):
        ops.rmsnorm(x, residual=x[:, :32])
    with pytest.raises(ValueError, match="residual"):
        ops.rmsnorm(x, residual=x.half())
    with pytest.raises(ValueError, match="needs a residual"):
        ops.rmsnorm(x, residual_out=x)
    with pytest.raises(ValueError, match="gamma"):
        ops.rmsnorm(x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError, match="gamma"):
        ops.rmsnorm(x, torch.ones(64, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="no CPU path"):
        ops.rmsnorm(x, torch.ones(64))
    with pytest.raises(ValueError, match="at least one value"):
        ops.quantize_rows(x[:, :0])
    with pytest.raises(ValueError, match="activation"):
        ops.quantize_rows(x, gate=x, activation="tanh")
    with pytest.raises(ValueError, match="belongs to a gate"):
        ops.quantize_rows(x, activation="silu")
    with pytest.raises(TypeError, match="out must be"):
        ops.quantize_rows(x, out=torch.empty(4, 64, device="cuda"))
    with pytest.raises(ValueError, match="without overlap"):
        ops.rmsnorm(x, out=torch.empty(64, device="cuda").expand(4, 64))
    with pytest.raises(ValueError, match="scale"):
        ops.quantize_rows(x, scale=torch.empty(3, device="cuda"))
