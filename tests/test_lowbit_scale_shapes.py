"""Scales belong to rows: the shapes a product takes them in, and those it refuses although the number of entries fits."""
import pytest
import torch

from dace_onnx_b200 import ops
from dace_onnx_b200.lowbit import _scale_shape

GOOD = [((2, 3), (2, 3)), ((2, 3, 1), (2, 3)), ((1, 2, 3), (2, 3)), ((6,), (2, 3)), ((6, 1), (2, 3)), ((1, 6), (6,)), ((4,), (1, 4)),
        ((2, 1, 3), (2, 3)), ((2, 3), (2, 1, 3)), ((), ()), ((1,), ()), ((), (1,)), ((0,), (0,)), ((0,), (2, 0)), ((2, 0), (2, 0))]
BAD = [((3, 2), (2, 3)), ((2, 3), (6,)), ((2, 3), (3, 2)), ((5,), (2, 3)), ((2, 2, 3), (4, 3)), ((3, 1, 2), (2, 3)), ((2, 6), (3, 4)),
       ((3,), (2, 3)), ((2,), ())]


@pytest.mark.parametrize("shape,lead", GOOD)
def test_shapes(shape, lead):
    assert _scale_shape(torch.Size(shape), lead)


@pytest.mark.parametrize("shape,lead", BAD)
def test_shapes_in_another_order(shape, lead):
    assert not _scale_shape(torch.Size(shape), lead)


@pytest.mark.gpu
@pytest.mark.parametrize("direct", [True, False])
def test_products(direct, cuda, monkeypatch):
    """The C++ entry and the checked path agree."""
    from dace_onnx_b200 import torch_calls
    if not direct:
        monkeypatch.setattr(torch_calls, "matmul_scaled", lambda *_: None)
    w = torch.randn(6, 32, device=cuda).bfloat16()
    for shape, lead in GOOD + BAD:
        a = torch.randn(*lead, 32, device=cuda).bfloat16()
        scale = torch.rand(shape, device=cuda) + 0.5
        if (shape, lead) in GOOD:
            want = ops.matmul_scaled(a.reshape(-1, 32), w, a_scale=scale.reshape(-1))
            assert torch.equal(ops.matmul_scaled(a, w, a_scale=scale).reshape(want.shape), want)
        else:
            with pytest.raises(ValueError, match="a_scale must have one entry"):
                ops.matmul_scaled(a, w, a_scale=scale)
    a = torch.randn(5, 32, device=cuda).bfloat16()
    scale = torch.rand(6, device=cuda)
    want = ops.matmul_scaled(a, w, w_scale=scale)
    for shape in ((6, 1), (1, 6)):
        assert torch.equal(ops.matmul_scaled(a, w, w_scale=scale.reshape(shape)), want)
    with pytest.raises(ValueError, match="w_scale must have one entry"):
        ops.matmul_scaled(a, w, w_scale=scale.reshape(2, 3))
