"""The operators of the 8-bit path one after the other, as a model runs them, with buffers that the next step reuses."""
import os
import subprocess
import sys

import pytest
import torch

from dace_onnx_b200 import donnx, graphs, ops
from dace_onnx_b200.encoder import BertEncoderB200
from oracle import pure_oracle as po
from tests.test_gpu_rows_quant import make

pytestmark = pytest.mark.gpu


def layer(rows, hidden, ffn, seed):
    t = torch.bfloat16
    up, down = make(seed, 2 * ffn, hidden, scale=hidden ** -0.5), make(seed + 1, hidden, ffn, scale=ffn ** -0.5)
    return dict(gamma=(1 + make(seed + 2, hidden, scale=0.1)).to(t), up=ops.PreparedLinear(up), down=ops.PreparedLinear(down),
                h=torch.empty(rows, hidden, device="cuda", dtype=t), q=ops.empty_codes((rows, hidden), "cuda"),
                s=torch.empty(rows, device="cuda"), both=torch.empty(rows, 2 * ffn, device="cuda", dtype=t),
                qa=ops.empty_codes((rows, ffn), "cuda"), sa=torch.empty(rows, device="cuda"),
                y=torch.empty(rows, hidden, device="cuda", dtype=t), ffn=ffn)


def step(x, stream, w, wait):
    """h = stream + x; y = down(silu(gate) * up) of norm(h), all through w's buffers; the stream is updated in place."""
    pause = torch.cuda.synchronize if wait else (lambda: None)
    ops.rmsnorm_quantize(x, w["gamma"], residual=stream, out=w["q"], scale=w["s"], residual_out=stream)
    pause()
    w["up"](w["q"], a_scale=w["s"], out=w["both"])
    pause()
    ops.quantize_rows(w["both"][:, w["ffn"]:], gate=w["both"][:, :w["ffn"]], activation="silu", out=w["qa"], scale=w["sa"])
    pause()
    w["down"](w["qa"], a_scale=w["sa"], out=w["y"])
    pause()
    return w["y"]


@pytest.mark.parametrize("rows,hidden,ffn", [(1, 512, 1024), (5, 1000, 700), (200, 512, 1536), (1500, 768, 2048)])
def test_overlapped_launches_give_the_results_of_separate_ones(rows, hidden, ffn, cuda):
    w = layer(rows, hidden, ffn, 60)
    x, stream0 = make(61, rows, hidden).bfloat16(), make(62, rows, hidden).bfloat16()
    want, stream = x, stream0.clone()
    for _ in range(12):
        want = step(want, stream, w, True)
    want, want_stream = want.clone(), stream.clone()
    for _ in range(3):
        y, stream = x, stream0.clone()
        for _ in range(12):
            y = step(y, stream, w, False)
        assert torch.equal(y, want) and torch.equal(stream, want_stream)
    # the same captured
    static, stream = x.clone(), stream0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = static
        for _ in range(12):
            y = step(y, stream, w, False)
    for _ in range(2):
        stream.copy_(stream0)
        graph.replay()
        assert torch.equal(y, want) and torch.equal(stream, want_stream)


def test_chain_against_64_bits(cuda):
    """One pass against the formula. Both quantisations and the weights' round by at most 2^-4 of a value; in a dot product of
    n random terms these errors add like their squares: relative to the result's own size about 2^-4 / sqrt(3) per
    quantised operand, so sqrt(4) of them stay below 4 * 2^-4 / sqrt(3) * 0.5 < 0.075 in the 2-norm (uniform rounding errors
    have a mean square of a twelfth of the step's, steps lie between 2^-4 and 2^-3 of the value)."""
    rows, hidden, ffn = 64, 1024, 2048
    w = layer(rows, hidden, ffn, 70)
    up, down = make(70, 2 * ffn, hidden, scale=hidden ** -0.5).double(), make(71, hidden, ffn, scale=ffn ** -0.5).double()
    x, r = make(73, rows, hidden).bfloat16(), make(74, rows, hidden).bfloat16()
    stream = r.clone()
    y = step(x, stream, w, False).double()
    h = x.double() + r.double()
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * w["gamma"].double()
    both = n @ up.t()
    want = (both[:, :ffn] * torch.sigmoid(both[:, :ffn]) * both[:, ffn:]) @ down.t()
    assert ((y - want).norm() / want.norm()).item() < 0.075


def test_gated_mlp_forward(cuda):
    """The runner makes the calls of the chain above (same bits), on any leading shape; its error as derived there."""
    hidden, ffn = 520, 776
    gate, up, down = (make(80 + i, *s, scale=s[1] ** -0.5) for i, s in enumerate([(ffn, hidden), (ffn, hidden), (hidden, ffn)]))
    gamma = 1 + make(83, hidden, scale=0.1)
    for act, f in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu)):
        mlp = graphs.GatedMlp(gamma, gate, up, down, activation=act)
        for shape in ((3, 7, hidden), (130, hidden)):
            x, r = make(84, *shape).half(), make(85, *shape).half()
            y, h = graphs.gated_mlp_forward(x, r, mlp)
            assert y.shape == h.shape == x.shape and y.dtype == h.dtype == torch.float16
            h64 = x.double() + r.double()
            n = h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6) * gamma.double()
            want = (f(n @ gate.double().t()) * (n @ up.double().t())) @ down.double().t()
            assert ((y.double() - want).norm() / want.norm()).item() < 0.075
            q, s, h2 = ops.rmsnorm_quantize(x, gamma, residual=r)
            both = mlp.gate_up(q, a_scale=s, out_dtype=torch.float16)
            q, s = ops.quantize_rows(both[..., ffn:].contiguous(), gate=both[..., :ffn].contiguous(), activation=act)
            assert torch.equal(mlp.down(q, a_scale=s, out_dtype=torch.float16), y) and torch.equal(h, h2)
    with pytest.raises(ValueError, match="expected gamma"):
        graphs.GatedMlp(gamma, gate, up, down.t())


@pytest.mark.parametrize("hidden,heads,ffn,shape", [(256, 4, 1024, (3, 64)), (96, 2, 200, (2, 19))])
def test_encoder_on_8_bit_weights(hidden, heads, ffn, shape, cuda):
    """Two layers against the oracle in fp32. Four operands are quantised on the way through each half of a layer, each adding a
    relative error of at most 2^-3 / sqrt(12) = 0.036 in the 2-norm: 0.072 together, 1.13 times that through the Gelu. The residual
    is added in fp32, so a half whose branch is at most as large as its stream keeps below 0.072 * 1.13 / sqrt(2) = 0.058, and
    four halves below 2 * 0.058 (the errors are independent)."""
    layers = [po.make_bert_layer_params(hidden, ffn, seed=90 + i, std=0.05) for i in range(2)]
    x = torch.randn(*shape, hidden, generator=torch.Generator().manual_seed(92))
    ref = po.bert_encoder_forward(x, layers, heads=heads)
    enc = BertEncoderB200(layers, heads=heads, device=cuda, math_mode="fp8")
    y = enc.forward_device(x.to(cuda))
    assert ((y.cpu() - ref).norm() / ref.norm()).item() < 2 * 0.058
    assert torch.equal(enc(x.pin_memory()), y.cpu())
    pieces = BertEncoderB200(layers, heads=heads, device=cuda, math_mode="fp8", micro_batch=1)
    assert ((pieces(x) - ref).norm() / ref.norm()).item() < 2 * 0.058


def test_norm_nodes(cuda):
    x, skip, gamma = make(95, 4, 6, 100), make(96, 4, 6, 100), 1 + make(97, 100, scale=0.1)
    y = torch.empty_like(x)
    assert donnx.ONNXRMSNormalization(X=x, scale=gamma, Y=y, epsilon=1e-5) is y
    assert torch.equal(y, ops.rmsnorm(x, gamma, eps=1e-5))
    wide = torch.empty(4, 6, 200, device="cuda")[..., ::2]        # an output whose elements lie apart
    donnx.ONNXRMSNormalization(X=x, scale=gamma, Y=wide, epsilon=1e-5)
    assert torch.equal(wide, y)
    out, total = torch.empty_like(x), torch.empty_like(x)
    donnx.ONNXSkipSimplifiedLayerNormalization(input=x, skip=skip, gamma=gamma, output=out, input_skip_bias_sum=total)
    want = ops.rmsnorm(x, gamma, residual=skip, eps=1e-5)
    assert torch.equal(out, want[0]) and torch.equal(total, want[1])
    out.zero_()
    donnx.ONNXSkipSimplifiedLayerNormalization(input=x, skip=skip, gamma=gamma, output=out)
    assert torch.equal(out, want[0])
    with pytest.raises(NotImplementedError, match="last axis"):
        donnx.ONNXRMSNormalization(X=x, scale=gamma, Y=y, axis=1)
    with pytest.raises(NotImplementedError, match="stash_type"):
        donnx.ONNXRMSNormalization(X=x, scale=gamma, Y=y, stash_type=0)
    with pytest.raises(ValueError, match="output connector"):
        donnx.ONNXRMSNormalization(X=x, scale=gamma, Y=y[:2])


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing that a first call sets up (attributes, addresses, modules) keeps it from being captured."""
    code = """
import torch
from dace_onnx_b200 import ops
x, w = torch.randn(300, 256, device="cuda"), torch.randn(512, 256, device="cuda")
wide, few = torch.randn(2, 256, 512, device="cuda").bfloat16()[0], torch.randn(3, 512, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s = ops.rmsnorm_quantize(x)
    qw, sw = ops.quantize_rows(w)
    y = ops.matmul_scaled(q, qw, a_scale=s, w_scale=sw, out_dtype=torch.float32)
    z = ops.matmul_scaled(few, wide)
graph.replay()
torch.cuda.synchronize()
q2, s2 = ops.rmsnorm_quantize(x)
assert torch.equal(ops.matmul_scaled(q2, qw, a_scale=s2, w_scale=sw, out_dtype=torch.float32), y)
assert torch.equal(ops.matmul_scaled(few, wide), z)
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_fork_and_join_inside_a_capture(cuda):
    """Two branches of a captured step on two streams, joined by a third call that reads both."""
    x, a, b = make(100, 40, 512).bfloat16(), ops.PreparedLinear(make(101, 512, 512)), ops.PreparedLinear(make(102, 512, 512))
    side = torch.cuda.Stream()

    def step():
        q, s = ops.quantize_rows(x)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            u = b(q, a_scale=s, out_dtype=torch.bfloat16)
        v = a(q, a_scale=s, out_dtype=torch.bfloat16)
        torch.cuda.current_stream().wait_stream(side)
        return ops.rmsnorm(v, residual=u)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(20):
        for t in got:
            t.zero_()
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_written_weights_are_seen_by_the_next_product(cuda):
    """A product right behind the kernels that write its operands, over and over with other values in the same memory."""
    q, s = ops.empty_codes((6, 4096), "cuda"), torch.empty(6, device="cuda")
    qw, sw = ops.empty_codes((512, 4096), "cuda"), torch.empty(512, device="cuda")
    xs, ws = [make(110 + i, 6, 4096) for i in range(4)], [make(120 + i, 512, 4096) for i in range(4)]
    want = []
    for x, w in zip(xs, ws):
        ops.quantize_rows(x, out=q, scale=s)
        ops.quantize_rows(w, out=qw, scale=sw)
        torch.cuda.synchronize()
        want.append(ops.matmul_scaled(q, qw, a_scale=s, w_scale=sw).clone())
        torch.cuda.synchronize()
    got = [torch.empty_like(want[0]) for _ in range(80)]
    for i, y in enumerate(got):
        ops.quantize_rows(xs[i % 4], out=q, scale=s)
        ops.quantize_rows(ws[i % 4], out=qw, scale=sw)
        ops.matmul_scaled(q, qw, a_scale=s, w_scale=sw, out=y)
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])
