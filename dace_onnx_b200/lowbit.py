"""The 8-bit linear path: RMS norm and row quantiser with e4m3 output, and the matrix product that consumes the codes.

Like `ops` (which re-exports these functions): CUDA tensors in, work launched on torch's current stream of the tensors'
device, nothing synchronised, no CPU path. Tensors are fp32, fp16 or bf16; sums and norms are computed in fp32.

8-bit rows are `torch.float8_e4m3fn` codes with one fp32 scale a row, value = code * scale. A new codes tensor has its rows
start at multiples of 16 bytes (`empty_codes`), the layout in which the product reads them without a copy.

Ordinary calls go through `torch_calls`, which reads the tensors in C++; whatever it declines comes back here, where arguments
are checked, errors raised and operands in other layouts copied.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import ACTIVATIONS, TYPE_BF16, TYPE_E4M3, TYPE_F16, TYPE_F32, GemmScaledDesc, QuantizeDesc, RmsnormDesc, check

torch_calls = None  # the compiled module: opened by the first call, as libb200ops.so is

FLOAT_TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
E4M3 = torch.float8_e4m3fn
OPERAND_TYPES = {E4M3: TYPE_E4M3, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}


def _calls():
    global torch_calls
    try:
        from . import torch_calls as module
    except ImportError as e:
        raise ImportError("dace_onnx_b200/torch_calls.so is missing or does not fit this torch: build it with "
                          "`python -m dace_onnx_b200.build` (%s)" % e) from e
    torch_calls = module
    return module


def _act(activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        if activation is None:
            return 0
        raise ValueError("activation must be one of %s or None" % sorted(ACTIVATIONS))
    return code


def _device(t, name):
    """Index of the CUDA device of a tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor" % name)
    device = t.get_device()
    if device < 0:
        raise ValueError("%s must live on a CUDA device (this library has no CPU path)" % name)
    return device


def _on(device, t, name):
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        _device(t, name)
        raise ValueError("%s must be on the same device as the first operand" % name)


def _float_type(t, name):
    code = FLOAT_TYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    return code


def _row_stride(t):
    """Elements from one row (last axis) to the next, or None when the rows are not evenly spaced or not adjacent."""
    shape = t.shape
    if t.is_contiguous():
        return shape[-1]
    stride = t.stride()
    n = len(shape)
    if stride[-1] != 1 and shape[-1] != 1:
        return None
    if n == 2:
        return stride[0] if shape[0] > 1 else shape[1]
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
    if t.is_contiguous():
        return t, t.shape[-1]
    s = _row_stride(t)
    if s is None:
        t = t.contiguous()
        s = t.shape[-1]
    return t, s


def _output_rows(t, name, shape, dtype, device):
    """Row stride of an output. shape: a tuple."""
    _on(device, t, name)
    if t.dtype is not dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if t.is_contiguous():
        return shape[-1]
    s = _row_stride(t)
    if s is None or (s < shape[-1] and t.numel() > shape[-1]):
        raise ValueError("%s: the rows of an output must be evenly spaced, without overlap, their elements adjacent" % name)
    return s


def _scales(t, shape, device):
    _on(device, t, "scale")
    if t.dtype is not torch.float32:
        raise TypeError("scale must be float32, got %s" % t.dtype)
    if t.shape != shape or not t.is_contiguous():
        raise ValueError("scale must be contiguous with shape %s" % (tuple(shape),))


def _call(fn, device, *args):
    """Launch on the current stream of `device`, which need not be the current device."""
    if device == torch._C._cuda_getDevice():
        status = fn(torch._C._cuda_getCurrentRawStream(device), *args)
    else:
        with torch.cuda.device(device):
            status = fn(torch._C._cuda_getCurrentRawStream(device), *args)
    if status:
        check(status)


def empty_codes(shape, device):
    """An uninitialised e4m3 tensor whose rows (last axis) start at multiples of 16 bytes."""
    shape = tuple(shape)
    pitch = -(-shape[-1] // 16) * 16
    t = torch.empty(shape[:-1] + (pitch,), device=device, dtype=E4M3)
    return t if pitch == shape[-1] else t[..., :shape[-1]]


def _rmsnorm(x, gamma, residual, eps, out, scale, residual_out, codes):
    done = (torch_calls or _calls()).rmsnorm(x, gamma, residual, eps, out, scale, residual_out, codes)
    if done is not None:
        if type(done) is int:
            check(done)
        return done
    device = _device(x, "x")
    dtype = x.dtype
    code = FLOAT_TYPES.get(dtype)
    if code is None:
        code = _float_type(x, "x")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError("rmsnorm: rows need at least one value")
    length = shape[-1]
    xr, xs = _input_rows(x)
    rp, hp, rs, hs = None, None, 0, 0
    if residual is not None:
        _on(device, residual, "residual")
        if residual.dtype is not dtype or residual.shape != shape:
            raise ValueError("rmsnorm: residual must have the shape and type of x")
        rr, rs = _input_rows(residual)
        if residual_out is None:
            residual_out = torch.empty(shape, device=x.device, dtype=dtype)
        hs = _output_rows(residual_out, "residual_out", shape, dtype, device)
        rp, hp = rr.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("rmsnorm: residual_out needs a residual")
    gp, gtype = None, code
    if gamma is not None:
        _on(device, gamma, "gamma")
        if gamma.dtype is not dtype:
            if gamma.dtype is not torch.float32:
                raise ValueError("rmsnorm: gamma must be of the type of x or float32")
            gtype = TYPE_F32
        if gamma.dim() != 1 or gamma.shape[0] != length:
            raise ValueError("rmsnorm: gamma must be [%d]" % length)
        if not gamma.is_contiguous():
            gamma = gamma.contiguous()
        gp = gamma.data_ptr()
    ytype, ydtype = (TYPE_E4M3, E4M3) if codes else (code, dtype)
    if out is None:
        out = empty_codes(shape, x.device) if codes else torch.empty(shape, device=x.device, dtype=dtype)
    ys = _output_rows(out, "out", shape, ydtype, device)
    sp = None
    if codes:
        if scale is None:
            scale = torch.empty(shape[:-1], device=x.device, dtype=torch.float32)
        else:
            _scales(scale, shape[:-1], device)
        sp = scale.data_ptr()
    rows = shape[0] if len(shape) == 2 else x.numel() // length
    d = RmsnormDesc(rows, length, xs, rs, hs, ys, code, gtype, ytype, eps)
    _call(_lib.load().b200_rmsnorm, device, ctypes.byref(d), xr.data_ptr(), rp, gp, hp, out.data_ptr(), sp)
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
    act = _act(activation)
    done = (torch_calls or _calls()).quantize_rows(x, gate, act, out, scale)
    if done is not None:
        if type(done) is int:
            check(done)
        return done
    device = _device(x, "x")
    code = _float_type(x, "x")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError("quantize_rows: rows need at least one value")
    length = shape[-1]
    xr, xs = _input_rows(x)
    gp, gs = None, 0
    if gate is not None:
        _on(device, gate, "gate")
        if gate.dtype != x.dtype or gate.shape != shape:
            raise ValueError("quantize_rows: gate must have the shape and type of x")
        gr, gs = _input_rows(gate)
        gp = gr.data_ptr()
    elif act:
        raise ValueError("quantize_rows: an activation belongs to a gate")
    if out is None:
        out = empty_codes(shape, x.device)
    qs = _output_rows(out, "out", shape, E4M3, device)
    if scale is None:
        scale = torch.empty(shape[:-1], device=x.device, dtype=torch.float32)
    else:
        _scales(scale, shape[:-1], device)
    rows = shape[0] if len(shape) == 2 else x.numel() // length
    d = QuantizeDesc(rows, length, xs, gs, qs, code, act)
    _call(_lib.load().b200_quantize_rows, device, ctypes.byref(d), xr.data_ptr(), gp, out.data_ptr(), scale.data_ptr())
    return out, scale


def _operand(t, size):
    """(tensor, row stride) as the product reads it: rows that start at multiples of 16 bytes; any other is copied into such
    rows. size: bytes of an element."""
    k = t.shape[-1]
    s = k if t.is_contiguous() else _row_stride(t)
    if s is None or t.data_ptr() % 16 or ((s * size % 16 or s < k) and t.numel() > k):
        pitch = -(-k * size // 16) * 16 // size
        padded = torch.empty(t.shape[:-1] + (pitch,), device=t.device, dtype=t.dtype)[..., :k]
        padded.copy_(t)
        return padded, pitch
    return t, s


def _scale_shape(shape, lead):
    """Whether a tensor of `shape` has one entry for each row of a tensor with leading axes `lead`, in their order: the axes that
    are not 1 agree, or there is only one (all rows in order)."""
    longer = [n for n in shape if n != 1]
    return longer == [n for n in lead if n != 1] or (len(longer) <= 1 and math.prod(shape) == math.prod(lead))


def _scale_operand(t, name, lead, device):
    """(tensor, step) of a scale operand: one entry for all rows, or one a row."""
    _on(device, t, name)
    if t.dtype is not torch.float32:
        raise TypeError("%s must be float32, got %s" % (name, t.dtype))
    if _scale_shape(t.shape, lead):
        return t if t.is_contiguous() else t.contiguous(), 1
    if t.numel() != 1:
        raise ValueError("%s must have one entry, or one for each row: shape %s, got %s" % (name, tuple(lead), tuple(t.shape)))
    return t, 0


def matmul_scaled(A, W, *, a_scale=None, w_scale=None, bias=None, activation=None, residual=None, out=None, out_dtype=None):
    """Y = activation((A W^T) * a_scale[:, None] * w_scale + bias) + residual, accumulated in fp32.

    A: [..., K], W: [N, K] (a Linear layer's layout), both e4m3 codes, float16 or bfloat16. a_scale: one fp32 entry a row of A
    (A's leading shape, axes of 1 aside, or all rows along one axis) or one in all; w_scale: [N] or one in all. bias: [N],
    float32, float16 or bfloat16. activation: as in `quantize_rows`. residual: the output's shape and type; it may be `out`.
    Output type: out's, or out_dtype, or the residual's, or A's (bfloat16 for codes).

    Operands whose rows do not start at multiples of 16 bytes are copied into such rows first: keep weights in a
    `PreparedLinear`, codes in tensors from `empty_codes` or the quantisers."""
    act = _act(activation)
    done = (torch_calls or _calls()).matmul_scaled(A, W, a_scale, w_scale, bias, act, residual, out,
                                                   -1 if out_dtype is None else FLOAT_TYPES.get(out_dtype, TYPE_E4M3))
    if done is not None:
        if type(done) is int:
            check(done)
        return done
    device = _device(A, "A")
    _on(device, W, "W")
    code = OPERAND_TYPES.get(A.dtype)
    if code is None or W.dtype is not A.dtype:
        raise TypeError("A and W must both be float8_e4m3fn, float16 or bfloat16, got %s and %s" % (A.dtype, W.dtype))
    shape = A.shape
    if len(shape) < 1 or W.dim() != 2 or shape[-1] != W.shape[1]:
        raise ValueError("matmul_scaled: A must be [..., K] and W [N, K], got %s and %s" % (tuple(shape), tuple(W.shape)))
    N, K = W.shape
    if K == 0:
        raise ValueError("matmul_scaled: K must be at least 1")
    if len(shape) == 2:
        M = shape[0]
        shape = (M, N)
    else:
        M = A.numel() // K
        shape = tuple(shape[:-1]) + (N,)
    if out is None:
        dtype = out_dtype if out_dtype is not None else residual.dtype if residual is not None else \
            torch.bfloat16 if code == TYPE_E4M3 else A.dtype
        if dtype not in FLOAT_TYPES:
            raise TypeError("matmul_scaled: the output must be float32, float16 or bfloat16, not %s" % dtype)
        out = torch.empty(shape, device=A.device, dtype=dtype)
    else:
        dtype = out.dtype
        if out_dtype is not None and out_dtype != dtype:
            raise TypeError("matmul_scaled: out is %s, not %s" % (dtype, out_dtype))
    ytype = FLOAT_TYPES.get(dtype)
    if ytype is None:
        raise TypeError("out must be float32, float16 or bfloat16, got %s" % dtype)
    ldy = _output_rows(out, "out", shape, dtype, device)
    rp, ldr = None, 0
    if residual is not None:
        _on(device, residual, "residual")
        if residual.dtype is not dtype or residual.shape != shape:
            raise ValueError("matmul_scaled: residual must have the output's shape and type")
        rr, ldr = _input_rows(residual)
        if ldr < N and M > 1:
            rr, ldr = residual.contiguous(), N
        rp = rr.data_ptr()
    bp, btype = None, 0
    if bias is not None:
        _on(device, bias, "bias")
        btype = _float_type(bias, "bias")
        if bias.dim() != 1 or bias.shape[0] != N:
            raise ValueError("matmul_scaled: bias must be [%d]" % N)
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bp = bias.data_ptr()
    sap, sa, swp, sw = None, 0, None, 0
    if a_scale is not None:
        a_scale, sa = _scale_operand(a_scale, "a_scale", shape[:-1], device)
        sap = a_scale.data_ptr()
    if w_scale is not None:
        w_scale, sw = _scale_operand(w_scale, "w_scale", (N,), device)
        swp = w_scale.data_ptr()
    size = 1 if code == TYPE_E4M3 else 2
    A, lda = _operand(A, size)
    W, ldw = _operand(W, size)
    d = GemmScaledDesc(M, N, K, lda, ldw, ldy, ldr, sa, sw, code, btype, ytype, act)
    _call(_lib.load().b200_gemm_scaled, device, ctypes.byref(d), A.data_ptr(), W.data_ptr(), sap, swp, bp, rp, out.data_ptr())
    return out


class PreparedLinear:
    """A linear layer whose weight is brought into the product's layout once: e4m3 codes with one scale an output (the
    default), or float16 / bfloat16.

    weight: [N, K], float32, float16 or bfloat16, on a CUDA device. Calls take activations in any of these types and, for
    an e4m3 layer, quantise their rows; or e4m3 codes with `a_scale`, as the quantisers return them."""

    def __init__(self, weight, bias=None, *, activation=None, dtype=E4M3):
        device = _device(weight, "weight")
        _float_type(weight, "weight")
        if weight.dim() != 2 or 0 in weight.shape:
            raise ValueError("PreparedLinear: weight must be [N, K]")
        if dtype not in OPERAND_TYPES:
            raise TypeError("PreparedLinear: dtype must be float8_e4m3fn, float16 or bfloat16")
        _act(activation)
        weight = weight.detach()  # the layer keeps values, not the graph of a parameter
        self.N, self.K = weight.shape
        self.activation, self.dtype = activation, dtype
        if bias is not None:
            _on(device, bias, "bias")
            _float_type(bias, "bias")
            if bias.shape != (self.N,):
                raise ValueError("PreparedLinear: bias must be [%d]" % self.N)
            bias = bias.detach().contiguous()
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
