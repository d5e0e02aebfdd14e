"""Refusals of the 8-bit linear path that need no GPU: argument checks come before any CUDA call."""
import ctypes

import pytest
import torch

from dace_onnx_b200 import _lib, ops
from dace_onnx_b200._lib import GemmScaledDesc, QuantizeDesc, RmsnormDesc
from dace_onnx_b200.lowbit import _row_stride

P = ctypes.c_void_p(256)  # never read: the calls below are refused


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 16)
    for call in (lambda: ops.rmsnorm(x), lambda: ops.rmsnorm_quantize(x), lambda: ops.quantize_rows(x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        ops.rmsnorm([1.0])


@pytest.mark.parametrize("change,args,code", [
    (dict(rows=-1), {}, _lib.EINVAL), (dict(len=0), {}, _lib.EINVAL), (dict(type=3), {}, _lib.EINVAL),
    (dict(gamma_type=2), {}, _lib.EINVAL), (dict(y_type=2), {}, _lib.EINVAL), (dict(eps=-1.0), {}, _lib.EINVAL),
    (dict(eps=float("nan")), {}, _lib.EINVAL), (dict(x_stride=-1), {}, _lib.EINVAL), (dict(y_stride=0), {}, _lib.EINVAL),
    (dict(h_stride=0), {}, _lib.EINVAL), (dict(rows=1 << 31), {}, _lib.EUNSUPPORTED), (dict(len=1 << 31), {}, _lib.EUNSUPPORTED),
    ({}, dict(x=None), _lib.EINVAL), ({}, dict(h=None), _lib.EINVAL), ({}, dict(residual=None), _lib.EINVAL),
    ({}, dict(y=None), _lib.EINVAL), (dict(y_type=3), dict(scale=None), _lib.EINVAL), (dict(rows=0), dict(x=None), _lib.OK)])
def test_rmsnorm_refusals(change, args, code):
    d = RmsnormDesc(4, 8, 8, 8, 8, 8, 0, 0, 0, 1e-6)
    for k, v in change.items():
        setattr(d, k, v)
    a = dict(x=P, residual=P, gamma=P, h=P, y=P, scale=P)
    a.update(args)
    assert _lib.load().b200_rmsnorm(None, ctypes.byref(d), a["x"], a["residual"], a["gamma"], a["h"], a["y"], a["scale"]) == code
    assert _lib.load().b200_rmsnorm(None, None, P, P, P, P, P, P) == _lib.EINVAL


@pytest.mark.parametrize("change,args,code", [
    (dict(rows=-1), {}, _lib.EINVAL), (dict(len=0), {}, _lib.EINVAL), (dict(type=3), {}, _lib.EINVAL),
    (dict(activation=5), {}, _lib.EINVAL), (dict(activation=-1), {}, _lib.EINVAL), (dict(gate_stride=-1), {}, _lib.EINVAL),
    (dict(q_stride=0), {}, _lib.EINVAL), (dict(rows=1 << 31), {}, _lib.EUNSUPPORTED), ({}, dict(x=None), _lib.EINVAL),
    ({}, dict(gate=None), _lib.EINVAL), ({}, dict(q=None), _lib.EINVAL), ({}, dict(scale=None), _lib.EINVAL),
    (dict(rows=0), dict(x=None), _lib.OK)])
def test_quantize_rows_refusals(change, args, code):
    d = QuantizeDesc(4, 8, 8, 8, 8, 0, 4)
    for k, v in change.items():
        setattr(d, k, v)
    a = dict(x=P, gate=P, q=P, scale=P)
    a.update(args)
    assert _lib.load().b200_quantize_rows(None, ctypes.byref(d), a["x"], a["gate"], a["q"], a["scale"]) == code
    assert _lib.load().b200_quantize_rows(None, None, P, P, P, P) == _lib.EINVAL


def test_row_strides():
    t = torch.zeros(4, 6, 8)
    assert _row_stride(t) == 8 and _row_stride(t[:, :, :5]) == 8 and _row_stride(t[:, ::2]) == 16
    assert _row_stride(t[:, :4]) is None            # the leading axes are not evenly spaced together
    assert _row_stride(t[:1, :4]) == 8 and _row_stride(t[:, :1]) == 48
    assert _row_stride(t.transpose(1, 2)) is None   # elements of a row apart
    assert _row_stride(t[0, 0].expand(3, 8)) == 0
    assert _row_stride(torch.zeros(5)) == 5 and _row_stride(torch.zeros(3, 1).t()) == 3


@pytest.mark.parametrize("change,args,code", [
    (dict(M=-1), {}, _lib.EINVAL), (dict(N=-1), {}, _lib.EINVAL), (dict(K=0), {}, _lib.EINVAL), (dict(type=0), {}, _lib.EINVAL),
    (dict(y_type=3), {}, _lib.EINVAL), (dict(bias_type=3), {}, _lib.EINVAL), (dict(activation=5), {}, _lib.EINVAL),
    (dict(a_scale_step=2), {}, _lib.EINVAL), (dict(w_scale_step=-1), {}, _lib.EINVAL), (dict(lda=16), {}, _lib.EINVAL),
    (dict(ldw=16), {}, _lib.EINVAL), (dict(ldy=8), {}, _lib.EINVAL), (dict(ldr=8), {}, _lib.EINVAL),
    (dict(lda=33), {}, _lib.EUNSUPPORTED), (dict(ldw=40), {}, _lib.EUNSUPPORTED), (dict(M=1 << 31), {}, _lib.EUNSUPPORTED),
    ({}, dict(A=ctypes.c_void_p(264)), _lib.EUNSUPPORTED), ({}, dict(W=ctypes.c_void_p(257)), _lib.EUNSUPPORTED),
    ({}, dict(A=None), _lib.EINVAL), ({}, dict(W=None), _lib.EINVAL), ({}, dict(Y=None), _lib.EINVAL),
    (dict(M=0), dict(A=None), _lib.OK), (dict(N=0), dict(W=None), _lib.OK)])
def test_gemm_scaled_refusals(change, args, code):
    d = GemmScaledDesc(4, 16, 32, 32, 32, 16, 16, 1, 1, 3, 0, 0, 0)
    for k, v in change.items():
        setattr(d, k, v)
    a = dict(A=P, W=P, a_scale=P, w_scale=P, bias=P, residual=P, Y=P)
    a.update(args)
    assert _lib.load().b200_gemm_scaled(None, ctypes.byref(d), *a.values()) == code
    assert _lib.load().b200_gemm_scaled(None, None, P, P, P, P, P, P, P) == _lib.EINVAL


def test_products_of_cpu_tensors_are_refused():
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.matmul_scaled(x, x)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.PreparedLinear(x)
