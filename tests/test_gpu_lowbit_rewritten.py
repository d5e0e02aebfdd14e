"""Everything a kernel of the 8-bit path reads, written by the kernel right before it in the stream, over and over with other values
in the same memory: gamma, biases, scales, residuals. The results are those of calls with a synchronisation in between."""
import pytest
import torch

from dace_onnx_b200 import ops
from tests.test_gpu_rows_quant import make

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def runs(write, call, sets, repeats=60):
    """write(i) writes set i of the values, call() launches what reads them."""
    want = []
    for i in range(sets):
        write(i)
        torch.cuda.synchronize()
        want.append([t.clone() for t in call()])
        torch.cuda.synchronize()
    got = []
    for i in range(repeats):
        write(i % sets)
        got.append([t.clone() for t in call()])
    for i, ts in enumerate(got):
        for a, b in zip(ts, want[i % sets]):
            assert torch.equal(a.float(), b.float())
    assert not torch.equal(want[0][0].float(), want[1][0].float())


# every form of the row kernels: a warp and a CTA a row, shifted rows, value by value, rows read twice
@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,length", [(1, 256), (1300, 256), (64, 4096), (400, 1001), (1300, 333), (2, 40000)])
@pytest.mark.parametrize("gamma_f32", [False, True])
def test_gamma(rows, length, t, gamma_f32, cuda):
    t = TYPES[t]
    x, r = make(1, rows, length, t=t), make(2, rows, length, t=t)
    source = [make(10 + i, 1, length, t=torch.float32 if gamma_f32 else t) for i in range(3)]
    gamma = torch.empty_like(source[0])
    runs(lambda i: ops.rmsnorm(source[i], out=gamma), lambda: ops.rmsnorm_quantize(x, gamma[0], residual=r), 3)


@pytest.mark.parametrize("bias_type", sorted(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (40, 1001, 512), (300, 512, 256)])
def test_bias_and_residual(m, n, k, bias_type, cuda):
    qa, sa = ops.quantize_rows(make(3, m, k))
    qw, sw = ops.quantize_rows(make(4, n, k))
    source = [make(20 + i, 1, n, t=TYPES[bias_type]) for i in range(3)]
    bias = torch.empty_like(source[0])
    runs(lambda i: ops.rmsnorm(source[i], out=bias),
         lambda: [ops.matmul_scaled(qa, qw, a_scale=sa, w_scale=sw, bias=bias[0], activation="silu")], 3)
    source_r = [make(30 + i, m, n).bfloat16() for i in range(3)]
    residual = torch.empty_like(source_r[0])
    runs(lambda i: ops.rmsnorm(source_r[i], out=residual),
         lambda: [ops.matmul_scaled(qa, qw, a_scale=sa, w_scale=sw, residual=residual)], 3)


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (6, 1001, 512), (40, 512, 4096), (300, 512, 256)])
def test_scales(m, n, k, cuda):
    """The same codes (rows scaled by powers of two quantise to them) with other scales."""
    a, w = make(5, m, k), make(6, n, k)
    qa, sa = ops.quantize_rows(a)
    qw, sw = ops.quantize_rows(w)
    rows = [a * 2.0 ** i for i in range(3)]
    cols = [w * 2.0 ** -i for i in range(3)]
    runs(lambda i: ops.quantize_rows(rows[i], out=qa, scale=sa), lambda: [ops.matmul_scaled(qa, qw, a_scale=sa, w_scale=sw)], 3)
    runs(lambda i: ops.quantize_rows(cols[i], out=qw, scale=sw), lambda: [ops.matmul_scaled(qa, qw, a_scale=sa, w_scale=sw)], 3)
