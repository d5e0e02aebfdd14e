"""The 8-bit linear path: RMS norm and row quantiser with e4m3 output, and the matrix product that consumes the codes.

Like `ops` (which re-exports these functions): CUDA tensors in, work launched on torch's current stream of the tensors'
device, nothing synchronised, no CPU path. Tensors are fp32, fp16 or bf16; sums and norms are computed in fp32.

8-bit rows are `torch.float8_e4m3fn` codes with one fp32 scale a row, value = code * scale. A new codes tensor has its rows
start at multiples of 16 bytes (`empty_codes`), the layout in which the product reads them without a copy.
"""
import ctypes

import torch

from . import _lib
from ._lib import ACTIVATIONS, TYPE_BF16, TYPE_E4M3, TYPE_F16, TYPE_F32, GemmScaledDesc, QuantizeDesc, RmsnormDesc, check

FLOAT_TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
E4M3 = torch.float8_e4m3fn
OPERAND_TYPES = {E4M3: TYPE_E4M3, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}


def _act(activation):
    code = ACTIVATIONS.get("none" if activation is None else activation)
    if code is None:
        raise ValueError("activation must be one of %s or None" % sorted(ACTIVATIONS))
    return code


def _tensor(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor" % name)
    if not t.is_cuda:
        raise ValueError("%s must live on a CUDA device (this library has no CPU path)" % name)
    if like is not None and t.get_device() != like.get_device():
        raise ValueError("%s must be on the same device as the first operand" % name)
    return t


def _float_type(t, name):
    code = FLOAT_TYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    return code


def _row_stride(t):
    """Elements from one row (last axis) to the next, or None when the rows are not evenly spaced or not adjacent."""
    shape, stride = t.shape, t.stride()
    n = len(shape)
    if stride[-1] != 1 and shape[-1] != 1:
        return None
    if n == 2:
        return stride[0] if shape[0] > 1 else shape[1]
    if t.numel() == 0:
        return shape[-1]
    step = None  # spacing of the merged leading axes, from the innermost that is not 1
    extent = 1
    for i in range(n - 2, -1, -1):
        if shape[i] == 1:
            continue
        if step is None:
            step, extent = stride[i], shape[i]
        elif stride[i] == step * extent:
            extent *= shape[i]
        else:
            return None
    return shape[-1] if step is None else step


def _input_rows(t):
    """(tensor, row stride): the tensor itself where its rows are evenly spaced, a contiguous copy elsewhere."""
    s = _row_stride(t)
    if s is None:
        t = t.contiguous()
        s = t.shape[-1]
    return t, s


def _output_rows(t, name, shape, dtype, like):
    _tensor(t, name, like)
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    s = _row_stride(t)
    if s is None or (s < shape[-1] and t.numel() > shape[-1]):
        raise ValueError("%s: the rows of an output must be evenly spaced, without overlap, their elements adjacent" % name)
    return s


def _scales(t, shape, like):
    if t is None:
        return torch.empty(shape, device=like.device, dtype=torch.float32)
    _tensor(t, "scale", like)
    if t.dtype != torch.float32:
        raise TypeError("scale must be float32, got %s" % t.dtype)
    if t.shape != shape or not t.is_contiguous():
        raise ValueError("scale must be contiguous with shape %s" % (tuple(shape),))
    return t


def _call(fn, device, *args):
    """Launch on the current stream of `device`, which need not be the current device."""
    if device == torch._C._cuda_getDevice():
        check(fn(torch._C._cuda_getCurrentRawStream(device), *args))
    else:
        with torch.cuda.device(device):
            check(fn(torch._C._cuda_getCurrentRawStream(device), *args))


def empty_codes(shape, device):
    """An uninitialised e4m3 tensor whose rows (last axis) start at multiples of 16 bytes."""
    shape = tuple(shape)
    pitch = -(-shape[-1] // 16) * 16
    t = torch.empty(shape[:-1] + (pitch,), device=device, dtype=E4M3)
    return t if pitch == shape[-1] else t[..., :shape[-1]]


def _rmsnorm(x, gamma, residual, eps, out, scale, residual_out, codes):
    _tensor(x, "x")
    code = _float_type(x, "x")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError("rmsnorm: rows need at least one value")
    length = shape[-1]
    rows = x.numel() // length
    xr, xs = _input_rows(x)
    rr, rs, hs = None, 0, 0
    if residual is not None:
        _tensor(residual, "residual", x)
        if residual.dtype != x.dtype or residual.shape != shape:
            raise ValueError("rmsnorm: residual must have the shape and type of x")
        rr, rs = _input_rows(residual)
        if residual_out is None:
            residual_out = torch.empty(shape, device=x.device, dtype=x.dtype)
        hs = _output_rows(residual_out, "residual_out", shape, x.dtype, x)
    elif residual_out is not None:
        raise ValueError("rmsnorm: residual_out needs a residual")
    gtype = code
    if gamma is not None:
        _tensor(gamma, "gamma", x)
        if gamma.dtype not in (x.dtype, torch.float32) or gamma.numel() != length or gamma.dim() != 1:
            raise ValueError("rmsnorm: gamma must be [%d], of the type of x or float32" % length)
        gamma = gamma.contiguous()
        gtype = FLOAT_TYPES[gamma.dtype]
    if out is None:
        out = empty_codes(shape, x.device) if codes else torch.empty(shape, device=x.device, dtype=x.dtype)
    ys = _output_rows(out, "out", shape, E4M3 if codes else x.dtype, x)
    if codes:
        scale = _scales(scale, shape[:-1], x)
    d = RmsnormDesc(rows, length, xs, rs, hs, ys, code, gtype, TYPE_E4M3 if codes else code, float(eps))
    _call(_lib.load().b200_rmsnorm, x.get_device(), ctypes.byref(d), xr.data_ptr(),
          None if rr is None else rr.data_ptr(), None if gamma is None else gamma.data_ptr(),
          None if rr is None else residual_out.data_ptr(), out.data_ptr(), scale.data_ptr() if codes else None)
    return out, scale, residual_out


def rmsnorm(x, gamma=None, *, residual=None, eps=1e-6, out=None, residual_out=None):
    """Root-mean-square norm over the last axis: y = h / sqrt(mean(h^2) + eps) * gamma with h = x + residual.

    Returns y (in x's type), or (y, h) with a residual; h is the updated residual stream, rounded to x's type after the norm
    has used it in fp32. `residual_out` may be `residual` or `x` itself (update in place)."""
    y, _, h = _rmsnorm(x, gamma, residual, eps, out, None, residual_out, False)
    return y if residual is None else (y, h)


def rmsnorm_quantize(x, gamma=None, *, residual=None, eps=1e-6, out=None, scale=None, residual_out=None):
    """`rmsnorm` with e4m3 output: (codes, scale), or (codes, scale, h) with a residual.

    scale = max(max|y|, 2^-100) / 448 of each row, codes = y / scale rounded to nearest even. A NaN in a row makes its scale
    and codes NaN."""
    q, s, h = _rmsnorm(x, gamma, residual, eps, out, scale, residual_out, True)
    return (q, s) if residual is None else (q, s, h)


def quantize_rows(x, *, gate=None, activation=None, out=None, scale=None):
    """Rows (last axis) of x, or of activation(gate) * x, to e4m3 codes: (codes, scale), as in `rmsnorm_quantize`.

    activation: None / "none", "relu", "gelu", "gelu_tanh" or "silu"; it belongs to the gate. x and gate may be halves of one
    tensor (rows further apart than they are long)."""
    _tensor(x, "x")
    code = _float_type(x, "x")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError("quantize_rows: rows need at least one value")
    act = _act(activation)
    length = shape[-1]
    rows = x.numel() // length
    xr, xs = _input_rows(x)
    gr, gs = None, 0
    if gate is not None:
        _tensor(gate, "gate", x)
        if gate.dtype != x.dtype or gate.shape != shape:
            raise ValueError("quantize_rows: gate must have the shape and type of x")
        gr, gs = _input_rows(gate)
    elif act:
        raise ValueError("quantize_rows: an activation belongs to a gate")
    if out is None:
        out = empty_codes(shape, x.device)
    qs = _output_rows(out, "out", shape, E4M3, x)
    scale = _scales(scale, shape[:-1], x)
    d = QuantizeDesc(rows, length, xs, gs, qs, code, act)
    _call(_lib.load().b200_quantize_rows, x.get_device(), ctypes.byref(d), xr.data_ptr(),
          None if gr is None else gr.data_ptr(), out.data_ptr(), scale.data_ptr())
    return out, scale


def _operand(t, name, code, like):
    """(tensor, row stride) as the product reads it: 16-byte aligned rows; a copy in that layout for any other."""
    s = _row_stride(t)
    size = 1 if code == TYPE_E4M3 else 2
    if s is None or t.data_ptr() % 16 or ((s * size) % 16 and t.numel() > t.shape[-1]) or (s == 0 and t.numel() > t.shape[-1]):
        k = t.shape[-1]
        pitch = -(-k * size // 16) * 16 // size
        padded = torch.empty(t.shape[:-1] + (pitch,), device=t.device, dtype=t.dtype)[..., :k]
        padded.copy_(t)
        return padded, pitch
    return t, s


def _scale_operand(t, name, rows, like):
    """(tensor, step) of a scale operand: one entry, or one a row."""
    if t is None:
        return None, 0
    _tensor(t, name, like)
    if t.dtype != torch.float32:
        raise TypeError("%s must be float32, got %s" % (name, t.dtype))
    if t.numel() == 1:
        return t, 0
    if t.numel() != rows:
        raise ValueError("%s must have one entry, or one for each of the %d rows" % (name, rows))
    return t.contiguous(), 1


def matmul_scaled(A, W, *, a_scale=None, w_scale=None, bias=None, activation=None, residual=None, out=None, out_dtype=None):
    """Y = activation((A W^T) * a_scale[:, None] * w_scale + bias) + residual, accumulated in fp32.

    A: [..., K], W: [N, K] (a Linear layer's layout), both e4m3 codes, float16 or bfloat16. a_scale: one fp32 entry a row of A
    (A's leading shape) or one in all; w_scale: [N] or one in all. bias: [N], float32, float16 or bfloat16. activation: as in
    `quantize_rows`. residual: the output's shape and type; it may be `out`. Output type: out's, or out_dtype, or the
    residual's, or A's (bfloat16 for codes).

    Operands whose rows do not start at multiples of 16 bytes are copied into such rows first: keep weights in a
    `PreparedLinear`, codes in tensors from `empty_codes` or the quantisers."""
    _tensor(A, "A")
    _tensor(W, "W", A)
    code = OPERAND_TYPES.get(A.dtype)
    if code is None or W.dtype != A.dtype:
        raise TypeError("A and W must both be float8_e4m3fn, float16 or bfloat16, got %s and %s" % (A.dtype, W.dtype))
    if A.dim() < 1 or W.dim() != 2 or A.shape[-1] != W.shape[1]:
        raise ValueError("matmul_scaled: A must be [..., K] and W [N, K], got %s and %s" % (tuple(A.shape), tuple(W.shape)))
    K, N = A.shape[-1], W.shape[0]
    if K == 0:
        raise ValueError("matmul_scaled: K must be at least 1")
    act = _act(activation)
    M = A.numel() // K
    shape = A.shape[:-1] + (N,)
    if out is None:
        dtype = out_dtype if out_dtype is not None else residual.dtype if residual is not None else \
            torch.bfloat16 if code == TYPE_E4M3 else A.dtype
        if dtype not in FLOAT_TYPES:
            raise TypeError("matmul_scaled: the output must be float32, float16 or bfloat16, not %s" % dtype)
        out = torch.empty(shape, device=A.device, dtype=dtype)
    elif out_dtype is not None and out_dtype != out.dtype:
        raise TypeError("matmul_scaled: out is %s, not %s" % (out.dtype, out_dtype))
    ytype = _float_type(out, "out")
    ldy = _output_rows(out, "out", shape, out.dtype, A)
    rr, ldr = None, 0
    if residual is not None:
        _tensor(residual, "residual", A)
        if residual.dtype != out.dtype or residual.shape != shape:
            raise ValueError("matmul_scaled: residual must have the output's shape and type")
        rr, ldr = _input_rows(residual)
        if ldr < N and M > 1:
            rr = residual.contiguous()
            ldr = N
    btype = 0
    if bias is not None:
        _tensor(bias, "bias", A)
        btype = _float_type(bias, "bias")
        if bias.shape != (N,):
            raise ValueError("matmul_scaled: bias must be [%d]" % N)
        bias = bias.contiguous()
    a_scale, sa = _scale_operand(a_scale, "a_scale", M, A)
    w_scale, sw = _scale_operand(w_scale, "w_scale", N, A)
    A, lda = _operand(A, "A", code, A)
    W, ldw = _operand(W, "W", code, A)
    d = GemmScaledDesc(M, N, K, lda, ldw, ldy, ldr, sa, sw, code, btype, ytype, act)
    _call(_lib.load().b200_gemm_scaled, A.get_device(), ctypes.byref(d), A.data_ptr(), W.data_ptr(),
          None if a_scale is None else a_scale.data_ptr(), None if w_scale is None else w_scale.data_ptr(),
          None if bias is None else bias.data_ptr(), None if rr is None else rr.data_ptr(), out.data_ptr())
    return out


class PreparedLinear:
    """A linear layer whose weight is brought into the product's layout once: e4m3 codes with one scale an output (the
    default), or float16 / bfloat16.

    weight: [N, K], float32, float16 or bfloat16, on a CUDA device. Calls take activations in any of these types and, for
    an e4m3 layer, quantise their rows; or e4m3 codes with `a_scale`, as the quantisers return them."""

    def __init__(self, weight, bias=None, *, activation=None, dtype=E4M3):
        _tensor(weight, "weight")
        _float_type(weight, "weight")
        if weight.dim() != 2 or 0 in weight.shape:
            raise ValueError("PreparedLinear: weight must be [N, K]")
        if dtype not in OPERAND_TYPES:
            raise TypeError("PreparedLinear: dtype must be float8_e4m3fn, float16 or bfloat16")
        _act(activation)
        self.N, self.K = weight.shape
        self.activation, self.dtype = activation, dtype
        if bias is not None:
            _tensor(bias, "bias", weight)
            _float_type(bias, "bias")
            if bias.shape != (self.N,):
                raise ValueError("PreparedLinear: bias must be [%d]" % self.N)
            bias = bias.contiguous()
        self.bias = bias
        if dtype == E4M3:
            self.weight, self.w_scale = quantize_rows(weight)
        else:
            pitch = -(-self.K // 8) * 8
            self.weight = torch.empty(self.N, pitch, device=weight.device, dtype=dtype)[:, :self.K]
            self.weight.copy_(weight)
            self.w_scale = None

    def __call__(self, x, *, a_scale=None, residual=None, out=None, out_dtype=None):
        """x: [..., K]. Returns activation(x W^T + bias) + residual in out's type, or out_dtype, or the residual's, or x's
        (bfloat16 for codes)."""
        if isinstance(x, torch.Tensor) and x.dtype in FLOAT_TYPES:
            if out is None and out_dtype is None and residual is None:
                out_dtype = x.dtype
            if self.dtype == E4M3:
                if a_scale is not None:
                    raise ValueError("PreparedLinear: a_scale belongs to e4m3 codes")
                x, a_scale = quantize_rows(x)
            elif x.dtype != self.dtype:
                x = x.to(self.dtype)
        elif self.dtype == E4M3 and isinstance(x, torch.Tensor) and x.dtype == E4M3 and a_scale is None:
            raise ValueError("PreparedLinear: e4m3 codes need their a_scale")
        return matmul_scaled(x, self.weight, a_scale=a_scale, w_scale=self.w_scale, bias=self.bias,
                             activation=self.activation, residual=residual, out=out, out_dtype=out_dtype)
