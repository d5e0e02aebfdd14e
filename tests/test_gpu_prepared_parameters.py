"""Layers prepared from parameters that require gradients: the layer keeps their values and no autograd graph."""
import pytest
import torch

from dace_onnx_b200 import graphs, ops
from tests.test_gpu_rows_quant import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias_step", [1, 2])
def test_prepared_linear(dtype, bias_step, cuda):
    w, b = make(1, 96, 130), make(2, 96 * bias_step)
    x = make(3, 7, 130)
    plain = ops.PreparedLinear(w, b[::bias_step], dtype=dtype)
    wp, bp = torch.nn.Parameter(w), torch.nn.Parameter(b)
    layer = ops.PreparedLinear(wp, bp[::bias_step], dtype=dtype)
    for t in (layer.weight, layer.bias) + (() if layer.w_scale is None else (layer.w_scale,)):
        assert not t.requires_grad and t.grad_fn is None
    y = layer(x)
    assert not y.requires_grad and torch.equal(y, plain(x))


def test_gated_mlp(cuda):
    gate, up, down, gamma = make(4, 48, 64), make(5, 48, 64), make(6, 64, 48), make(7, 64)
    p = torch.nn.Parameter
    mlp, plain = graphs.GatedMlp(p(gamma), p(gate), p(up), p(down)), graphs.GatedMlp(gamma, gate, up, down)
    x, r = make(8, 5, 64), make(9, 5, 64)
    for a, b in zip(graphs.gated_mlp_forward(x, r, mlp), graphs.gated_mlp_forward(x, r, plain)):
        assert not a.requires_grad and torch.equal(a, b)
