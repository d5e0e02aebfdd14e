"""Calls of the 8-bit path at the edges of what it takes: offsets past 2^31 elements, narrow outputs, rows at 8 bytes, copies and fills
around the kernels inside a captured graph."""
import pytest
import torch

from dace_onnx_b200 import ops
from tests.test_gpu_lowbit_codes import expected, same
from tests.test_gpu_matmul_scaled import check, operands
from tests.test_gpu_rows_quant import chain, half_step, make, norm64

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def noise(rows, length, t=torch.bfloat16, seed=1):
    """Random rows made on the GPU (a shifted block a row would do, but every row differs)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(rows, length, device="cuda", dtype=t)
    for i in range(0, rows, 16384):
        out[i:i + 16384] = torch.randn(out[i:i + 16384].shape, generator=g, device="cuda")
    return out


def around(rows, length):
    """The first rows, those where offsets pass 2^31 elements and 2^32 bytes of a 16-bit type, and the last."""
    middle = 2 ** 31 // length
    return [i for i in (0, 1, 2, middle - 1, middle, middle + 1, rows - 2, rows - 1) if i < rows]


def test_rows_past_32_bits(cuda):
    rows, length = 140000, 16384
    x = noise(rows, length)
    q, s = ops.quantize_rows(x)
    pick = around(rows, length)
    same((q[pick], s[pick]), expected(x[pick].float()))
    # the codes as an operand: rows of A past 2^31 elements
    w, sw = ops.quantize_rows(make(2, 24, length, scale=length ** -0.5))
    y = ops.matmul_scaled(q, w, a_scale=s, w_scale=sw)
    check(y[pick], q[pick], s[pick], w, sw)


@pytest.mark.parametrize("rows,length", [(70000, 32776), (280000, 8191)])
def test_norm_past_32_bits(rows, length, cuda):
    """Rows read twice, and rows off the 16-byte grid."""
    x = noise(rows, length)
    y = ops.rmsnorm(x)
    pick = around(rows, length)
    want = norm64(x[pick], None, None, 1e-6)[1]
    assert ((y[pick].double() - want).abs() <= (chain(length) + 1.0001 * half_step(x.dtype)) * want.abs() + 1e-38).all()


@pytest.mark.parametrize("n", [8192, 8191])
def test_outputs_past_32_bits(n, cuda):
    m, k = 270000, 64
    a, w = noise(m, k), make(3, n, k, scale=0.125).bfloat16()
    y = ops.matmul_scaled(a, w)
    pick = around(m, n)
    check(y[pick], a[pick], None, w, None)


@pytest.mark.parametrize("t", ["e4m3", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2388, 8, 1), (2500, 8, 40), (2370, 4, 1), (4000, 12, 100), (3000, 16, 64), (5000, 24, 33)])
def test_narrow_outputs(m, n, k, t, cuda):
    """Fewer columns than a block of outputs, and what lies around them."""
    from tests.test_gpu_matmul_scaled import TYPES
    a, sa, w, sw = operands(m, n, k, TYPES[t])
    for out in (torch.float32, torch.bfloat16):
        bias, residual = make(5, n), make(6, m, n).to(out)
        check(ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, bias=bias, activation="silu", residual=residual), a, sa, w, sw, bias, "silu",
              residual)
        buf = torch.full((m + 3, 32), 5.0, device=cuda, dtype=out)
        ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out=buf[1:m + 1, 0:n])
        check(buf[1:m + 1, :n], a, sa, w, sw)
        assert (buf[0] == 5).all() and (buf[m + 1:] == 5).all() and (buf[:, n:] == 5).all()


@pytest.mark.parametrize("t", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1200, 136, 40), (700, 517, 300), (300, 1003, 1000), (1100, 259, 1024), (3832, 549, 2221), (20, 77, 333)])
def test_ragged_outputs_inside_wider_rows(m, n, k, t, cuda):
    """Rows of Y at multiples of 16 bytes that end inside 16 bytes: nothing behind the end of a row is written, in either kernel."""
    from tests.test_gpu_matmul_scaled import TYPES
    a, sa, w, sw = operands(m, n, k, TYPES[t])
    for out in (torch.float32, torch.bfloat16, torch.float16):
        for cols in (n, n - 1, n - 2):
            pitch = -(-n // 8) * 8 + 8
            buf = torch.full((m + 1, pitch), 7.0, device=cuda, dtype=out)
            residual, bias = make(6, m, cols).to(out), make(7, cols)
            wc, swc = w[:cols], None if sw is None else sw[:cols]
            ops.matmul_scaled(a, wc, a_scale=sa, w_scale=swc, bias=bias, residual=residual, activation="relu", out=buf[:m, :cols])
            check(buf[:m, :cols], a, sa, wc, swc, bias, "relu", residual)
            assert (buf[:m, cols:] == 7).all() and (buf[m] == 7).all()
            buf[:m, :cols] = residual          # in place
            ops.matmul_scaled(a, wc, a_scale=sa, w_scale=swc, residual=buf[:m, :cols], out=buf[:m, :cols])
            check(buf[:m, :cols], a, sa, wc, swc, None, None, residual)
            assert (buf[:m, cols:] == 7).all() and (buf[m] == 7).all()


@pytest.mark.parametrize("t", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1200, 136, 1), (3, 40, 100), (17, 200, 1000), (300, 512, 333), (700, 520, 129), (40, 130, 2051)])
def test_what_lies_behind_the_rows_of_operands(m, n, k, t, cuda):
    """NaN behind the end of every row of A and W, and rows of NaN behind the last."""
    from tests.test_gpu_matmul_scaled import TYPES
    a, sa, w, sw = operands(m, n, k, TYPES[t])
    pitch = -(-k // 16) * 16 + 16

    def inside(v):
        buf = torch.full((v.shape[0] + 2, pitch), float("nan"), device=cuda).to(v.dtype)
        buf[1:-1, :k].copy_(v)
        return buf[1:-1, :k]

    for out in (torch.float32, torch.bfloat16):
        want = ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, out_dtype=out)
        assert torch.equal(ops.matmul_scaled(inside(a), inside(w), a_scale=sa, w_scale=sw, out_dtype=out), want)
        check(want, a, sa, w, sw)


@pytest.mark.parametrize("m,n,k", [(7, 300, 512), (400, 512, 512)])
@pytest.mark.parametrize("extra", [4, 2, 8])
def test_output_rows_at_few_bytes(m, n, k, extra, cuda):
    a, sa, w, sw = operands(m, n, k, E4M3)
    for out in (torch.bfloat16, torch.float32):
        buf, res = (torch.full((m, n + extra), 3.0, device=cuda, dtype=out) for _ in range(2))
        res[:, :n] = make(9, m, n)
        ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, residual=res[:, :n], out=buf[:, :n])
        check(buf[:, :n], a, sa, w, sw, None, None, res[:, :n])
        assert (buf[:, n:] == 3).all()
        # an output and a residual that lie differently
        wide = torch.zeros(m, n + 16, device=cuda, dtype=out)[:, :n]
        ops.matmul_scaled(a, w, a_scale=sa, w_scale=sw, residual=res[:, :n], out=wide)
        check(wide, a, sa, w, sw, None, None, res[:, :n])


def test_copies_and_fills_inside_a_capture(cuda):
    """Behind memory copies, fills and other kernels, and before them: the graph's edges wait for whole operations."""
    x, w = make(11, 300, 1000).bfloat16(), ops.PreparedLinear(make(12, 512, 1000))
    src, total = torch.zeros_like(x), torch.empty(300, 512, device=cuda, dtype=torch.bfloat16)
    q, s = ops.empty_codes((300, 1000), cuda), torch.empty(300, device=cuda)
    y, host = torch.empty_like(total), torch.empty(300, 512, dtype=torch.bfloat16, pin_memory=True)

    def step():
        work = src.clone()
        total.zero_()
        for _ in range(3):
            ops.quantize_rows(work, out=q, scale=s)
            work.copy_(src).mul_(2)          # overwrites what the quantiser has read
            w(q, a_scale=s, out=y, residual=total)
            q.view(torch.uint8).zero_()      # overwrites what the product has read
            total.copy_(y)
            y.zero_()
        host.copy_(total, non_blocking=True)

    src.copy_(x)
    step()
    torch.cuda.synchronize()
    want = host.clone()
    parts = [ops.quantize_rows(v) for v in (x, x * 2)]
    first, other = (w(c, a_scale=f).double() for c, f in parts)
    assert ((want.to(cuda).double() - (first + 2 * other)).norm() / want.double().norm()).item() < 2.0 ** -7
    graph = torch.cuda.CUDAGraph()
    src.zero_()
    with torch.cuda.graph(graph):
        step()
    for _ in range(10):
        src.zero_()
        graph.replay()
        src.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(host, want)
