"""The operators of the 8-bit path one after the other, as a model runs them, with buffers that the next step reuses."""
import pytest
import torch

from dace_onnx_b200 import ops
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
