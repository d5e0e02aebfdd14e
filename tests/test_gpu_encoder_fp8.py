"""The encoder on 8-bit weights: its scratch, and every step of a layer against the formula in 64 bits on the same codes."""
import math

import pytest
import torch

from dace_onnx_b200.encoder import BertEncoderB200
from oracle import pure_oracle as po
from tests.test_gpu_matmul_scaled import check

pytestmark = pytest.mark.gpu


def test_scratch_is_allocated_once(cuda):
    """Nothing is allocated and thrown away while the buffers are set up."""
    enc = BertEncoderB200([po.make_bert_layer_params(256, 1024, seed=1)], heads=4, device=cuda, math_mode="fp8")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    enc._buffers(16, 128)
    held = torch.cuda.memory_allocated() - before
    assert held >= sum(t.numel() * t.element_size() for t in enc._buf.values() if t.is_contiguous())
    assert torch.cuda.max_memory_allocated() - before == held


def codes(x):
    """Codes and scales as IEEE division gives them."""
    scale = x.abs().amax(-1).clamp_min(2.0 ** -100) / torch.full((), 448.0, device=x.device)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("hidden,heads,ffn,shape", [(256, 4, 1024, (3, 64)), (96, 2, 200, (2, 19)), (128, 2, 512, (1, 1))])
def test_every_step_of_a_layer(hidden, heads, ffn, shape, cuda):
    """Each step from the buffer that holds its input, so that roundings of one step do not turn into other codes in the next. The
    linear layers: the bound of a product in test_gpu_matmul_scaled, an fp32 sum's rounding, on the codes of input and weight.
    LayerNorm and attention: the tolerances of their own tests (fp32 parity; TF32 operands)."""
    params = po.make_bert_layer_params(hidden, ffn, seed=5, std=0.05)
    g = torch.Generator().manual_seed(7)
    for key in ("bq", "bk", "bv", "bo", "bi", "bo2", "ln1_b", "ln2_b"):   # biases that matter
        params[key] = torch.randn(params[key].shape, generator=g) * 0.3
    for key in ("ln1_g", "ln2_g"):
        params[key] = 1 + torch.randn(params[key].shape, generator=g) * 0.2
    p = {k: v.to(cuda) for k, v in params.items()}
    x = torch.randn(*shape, hidden, generator=torch.Generator().manual_seed(6)).to(cuda)
    enc = BertEncoderB200([params], heads=heads, device=cuda, math_mode="fp8")
    y = enc.forward_device(x)
    b = enc._buf
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731

    def linear(out, inp, w, bias, act=None, residual=None):
        qa, sa = codes(flat(inp).float())
        qw, sw = codes(w)
        check(flat(out), qa, sa, qw, sw, bias, act, None if residual is None else flat(residual))

    def norm(out, inp, gamma, beta):
        want = torch.nn.functional.layer_norm(inp.double(), (hidden,), gamma.double(), beta.double(), enc.eps)
        assert torch.allclose(out.double(), want, rtol=1e-4, atol=1e-5)

    linear(b["qkv"], x, torch.cat([p["wq"], p["wk"], p["wv"]]), torch.cat([p["bq"], p["bk"], p["bv"]]))
    q, k, v = (t.reshape(*shape, heads, -1).transpose(1, 2).double() for t in b["qkv"].split(hidden, -1))
    ctx = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(hidden // heads), -1) @ v
    ctx = ctx.transpose(1, 2).reshape(*shape, hidden)
    # operands of both products rounded to TF32, half a step 2^-11 each: scores off by 2^-10 of sum|q k|, and exp turns that into
    # a relative error of the probabilities (twice, numerator and sum); V and the probabilities another 2^-10
    size = (q.abs() @ k.abs().transpose(-1, -2) / math.sqrt(hidden // heads)).max().item()
    assert (b["ctx"].double() - ctx).abs().max().item() <= 2.0 ** -10 * (2 * size + 1.1) * v.abs().max().item()
    linear(b["attn"], b["ctx"], p["wo"], p["bo"], residual=x)
    norm(b["h1"], b["attn"], p["ln1_g"], p["ln1_b"])
    assert b["inter"].dtype == torch.bfloat16
    linear(b["inter"], b["h1"], p["wi"], p["bi"], act="gelu")
    linear(b["out"], b["inter"], p["wo2"], p["bo2"], residual=b["h1"])
    norm(y, b["out"], p["ln2_g"], p["ln2_b"])


def test_two_encoders_at_once(cuda):
    """Products, attention and norms of two models on two streams, TMEM and shared memory shared as the kernels meet: the same bits as
    one after the other."""
    encs = [BertEncoderB200([po.make_bert_layer_params(256, 1024, seed=s)] * 2, heads=4, device=cuda, math_mode=mode)
            for s, mode in ((8, "fp8"), (9, "fp8"), (10, "tf32"))]
    xs = [torch.randn(n, 128, 256, generator=torch.Generator().manual_seed(n)).to(cuda) for n in (2, 24, 12)]
    want = [e.forward_device(x).clone() for e, x in zip(encs, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in encs]
    got = [[] for _ in encs]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(encs[i].forward_device(xs[i]))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)
