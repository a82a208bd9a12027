"""Linear layers on top of the CUDA backend, for training and for single tokens:

  y = act(x W^T + b) + r                      linear, linear_backward
  y[rows of expert g] = act(x W[g]^T + b[g])  grouped_linear, grouped_linear_backward

Weights are stored as the framework's GEMM stores its B, [out, in] (row n holds
the weights of output n), products accumulate in f32.  The reference's GEMM ends
at its accumulator (python/mlir/dialects/wave_matmul.py:11163-11241); there is no
counterpart of these there.

Like `wave_attention.attention` these are plain functions on CUDA tensors: they
run on the current stream, return without waiting, and take no part in
autograd -- the backward functions give the gradients.  There is no CPU
implementation.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import wave_cuda as wc

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_TYPES = {torch.bfloat16: wc.BF16, torch.float16: wc.F16, torch.float32: wc.F32}


class _Plan:
    """What a call makes of its tensors' shapes, strides and types: the
    descriptor, the bytes of workspace and the results' shapes and types.
    Everything here is a function of those alone and is checked once for each
    combination of them; addresses and contents are looked at in every call."""
    __slots__ = ("desc", "ref", "need", "device", "index", "outs")

    def __init__(self, device, backward: bool, fields, outs):
        self.desc = wc.LinearDesc(*fields)
        self.ref = C.byref(self.desc)
        self.device, self.index, self.outs = device, device.index, outs
        with torch.cuda.device(device):  # the workspace goes by the device's SMs
            try:
                wc.linear_validate(self.desc)
                self.need = wc.linear_workspace_bytes(self.desc, backward)
            except wc.WaveCudaError as err:
                raise _refusal(err) from None


def _refusal(err):
    """What the library refuses is a ValueError, like what is refused here."""
    return ValueError(err.message) if err.code in (wc.E_INVALID, wc.E_UNSUPPORTED) else err


def _check(code: int) -> None:
    if code != wc.OK:
        try:
            wc.check(code)
        except wc.WaveCudaError as err:
            raise _refusal(err) from None


_plans: dict = {}


def _remember(key, plan):
    if len(_plans) >= 4096:
        _plans.clear()
    _plans[key] = plan
    return plan


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _matrix(t, name: str, rows: int, cols: int, dtypes, device):
    """Checks a [rows, cols] tensor; returns the elements from row to row (0: no gaps)."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
        raise ValueError(f"{name} must have shape ({rows}, {cols}); got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}; got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}; got {t.device}")
    return _row_stride(t, name, rows, cols, 0)


def _row_stride(t, name: str, rows: int, cols: int, dim: int) -> int:
    if cols > 1 and t.stride(dim + 1) != 1:
        raise ValueError(f"{name} must have contiguous rows (stride 1 in its last dimension)")
    if rows <= 1:
        return 0
    ld = t.stride(dim)
    if ld < cols:
        raise ValueError(f"the rows of {name} must not overlap; got a row stride of {ld} for {cols} columns")
    return ld


def _layer(x, weight, offsets):
    """Checks x, weight (and offsets); returns sizes and strides."""
    if not x.is_cuda:
        raise ValueError("the tensors must be CUDA tensors: this backend has no CPU path")
    device = x.device
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must have dtype bf16 or f16; got {x.dtype}")
    grouped = offsets is not None
    if x.dim() != 2 or weight.dim() != (3 if grouped else 2):
        raise ValueError("x must be (tokens, in_features) and weight (out_features, in_features), "
                         "(experts, out_features, in_features) where it is grouped")
    tokens, k = x.shape
    experts = weight.shape[0] if grouped else 0
    n = weight.shape[-2]
    if weight.shape[-1] != k:
        raise ValueError(f"x has {k} features and weight takes {weight.shape[-1]}")
    if weight.dtype != x.dtype or weight.device != device:
        raise ValueError("weight must share dtype and device with x")
    if n < 1 or k < 1 or (grouped and experts < 1):
        raise ValueError("features and experts must not be empty")
    ldx = _row_stride(x, "x", tokens, k, 0)
    ldw = _row_stride(weight, "weight", n, k, 1 if grouped else 0)
    stride_w = 0
    if grouped:
        if (offsets.dim() != 1 or offsets.shape[0] != experts + 1 or offsets.dtype != torch.int32 or offsets.device != device
                or not offsets.is_contiguous()):
            raise ValueError(f"offsets must be a contiguous int32 tensor of {experts + 1} entries on {device}")
        if experts > 1:
            stride_w = weight.stride(0)
            if stride_w < (ldw or k) * (n - 1) + k:
                raise ValueError("the experts' weights must not overlap")
    return device, tokens, n, k, experts, ldx, ldw, stride_w


def _act(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}")
    return code


def _aligned(t):
    """TMA loads start on 16-byte boundaries: a view that does not is copied."""
    if t.data_ptr() % 16 == 0:
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _on_its_device(call, plan, *args):
    """`call` with the tensors' device current: the library launches on the current device."""
    with torch.cuda.device(plan.device):
        return call(*args)


def _workspace(plan):
    return torch.empty(plan.need, dtype=torch.uint8, device=plan.device) if plan.need else None


def _plan_forward(x, weight, offsets, bias, residual, activation, out, out_dtype):
    device, tokens, n, k, experts, ldx, ldw, stride_w = _layer(x, weight, offsets)
    io = x.dtype
    bias_type = io
    if bias is not None:
        shape = (experts, n) if offsets is not None else (n,)
        if tuple(bias.shape) != shape or not bias.is_contiguous() or bias.device != device:
            raise ValueError(f"bias must be a contiguous tensor of shape {shape} on {device}")
        if bias.dtype not in (io, torch.float32):
            raise ValueError(f"bias must have dtype {io} or f32; got {bias.dtype}")
        bias_type = bias.dtype
    ldr = 0
    if residual is not None:
        ldr = _matrix(residual, "residual", tokens, n, (io,), device)
    if out is None:
        y_type = io if out_dtype is None else out_dtype
        if y_type not in (io, torch.float32):
            raise ValueError(f"out_dtype must be {io} or f32; got {y_type}")
        zero_rest, ldy = int(offsets is not None), 0
    else:
        y_type, zero_rest = out.dtype, 0
        if out_dtype is not None and out_dtype != y_type:
            raise ValueError(f"out has dtype {y_type}, out_dtype says {out_dtype}")
        ldy = _matrix(out, "out", tokens, n, (io, torch.float32), device)
    fields = (tokens, n, k, experts, _TYPES[io], _TYPES[y_type], _TYPES[bias_type], _TYPES[io], wc.F32, _act(activation), zero_rest, 0,
              ldx, ldw, ldy, ldr, 0, 0, 0, stride_w, 0)
    return _Plan(device, False, fields, ((tokens, n), y_type))


def _forward(x, weight, offsets, bias, residual, activation, out, out_dtype, save):
    key = (x.shape, x.stride(), x.dtype, x.device, weight.shape, weight.stride(), weight.dtype, weight.device, _meta(offsets),
           _meta(bias), _meta(residual), activation, _meta(out), out_dtype)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _plan_forward(x, weight, offsets, bias, residual, activation, out, out_dtype))
    if torch.cuda.current_device() != plan.index:
        return _on_its_device(_forward, plan, x, weight, offsets, bias, residual, activation, out, out_dtype, save)
    px, pw = x.data_ptr(), weight.data_ptr()
    if (px | pw) & 15:
        return _forward(_aligned(x), _aligned(weight), offsets, bias, residual, activation, out, out_dtype, save)
    shape, y_type = plan.outs
    y = out
    if y is None:
        y = x.new_empty(shape) if y_type is x.dtype else torch.empty(shape, dtype=y_type, device=plan.device)
    z = None
    if save:  # rows that belong to no expert are left alone with `out`
        z = x.new_zeros(shape) if offsets is not None and out is not None else x.new_empty(shape)
    ws = _workspace(plan)
    _check(wc.lib().wave_cuda_linear_fwd(plan.ref, px, pw, _ptr(bias), _ptr(residual), _ptr(offsets), y.data_ptr(), _ptr(z),
                                         _ptr(ws), torch._C._cuda_getCurrentRawStream(plan.index)))
    return (y, z) if save else y


def _plan_backward(dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype):
    device, tokens, n, k, experts, ldx, ldw, stride_w = _layer(x, weight, offsets)
    io = x.dtype
    act = _act(activation)
    ldy = _matrix(dy, "dy", tokens, n, (io, torch.float32), device)
    ldz = 0
    if act:
        if pre_activation is None:
            raise ValueError(f"the gradient of {activation} needs the pre-activation")
        ldz = _matrix(pre_activation, "pre_activation", tokens, n, (io,), device)
    dweight_dtype = dweight_dtype or io
    dbias_dtype = dbias_dtype or torch.float32
    for name, t in (("dweight_dtype", dweight_dtype), ("dbias_dtype", dbias_dtype)):
        if t not in (io, torch.float32):
            raise ValueError(f"{name} must be {io} or f32; got {t}")
    lead = (experts,) if offsets is not None else ()
    fields = (tokens, n, k, experts, _TYPES[io], _TYPES[dy.dtype], _TYPES[io], _TYPES[dweight_dtype], _TYPES[dbias_dtype], act,
              int(offsets is not None), 0, ldx, ldw, ldy, 0, ldz, 0, 0, stride_w, 0)
    return _Plan(device, True, fields, (((tokens, k), io), ((*lead, n, k), dweight_dtype), ((*lead, n), dbias_dtype)))


def _backward(dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype, need_dx, need_dweight,
              need_dbias):
    key = (_meta(dy), _meta(x), _meta(weight), _meta(offsets), activation, _meta(pre_activation), dweight_dtype, dbias_dtype)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _plan_backward(dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype))
    if torch.cuda.current_device() != plan.index:
        return _on_its_device(_backward, plan, dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype,
                              need_dx, need_dweight, need_dbias)
    pdy, px, pw = dy.data_ptr(), x.data_ptr(), weight.data_ptr()
    if (pdy | px | pw) & 15:
        return _backward(_aligned(dy), _aligned(x), _aligned(weight), offsets, activation, pre_activation, dweight_dtype,
                         dbias_dtype, need_dx, need_dweight, need_dbias)
    (dx_shape, io), (dw_shape, dw_type), (db_shape, db_type) = plan.outs
    dx = x.new_empty(dx_shape) if need_dx else None
    dw = None
    if need_dweight:
        dw = x.new_empty(dw_shape) if dw_type is io else torch.empty(dw_shape, dtype=dw_type, device=plan.device)
    db = torch.empty(db_shape, dtype=db_type, device=plan.device) if need_dbias else None
    ws = _workspace(plan)
    z = _ptr(pre_activation) if plan.desc.activation else None
    _check(wc.lib().wave_cuda_linear_bwd(plan.ref, pdy, px, pw, z, _ptr(offsets), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                                         torch._C._cuda_getCurrentRawStream(plan.index)))
    return dx, dw, db


def linear(x, weight, bias=None, residual=None, *, activation: str = "none", out=None, out_dtype=None,
           save_pre_activation: bool = False):
    """act(x @ weight.T + bias) + residual in one kernel.

    x (tokens, in) and weight (out, in) in bf16 or f16, rows of any stride; bias
    (out,) in that type or f32; residual (tokens, out) in that type.
    `activation`: none, relu, gelu (erf), gelu_tanh or silu.  Returns y (tokens,
    out) in x's type, or f32 with `out_dtype`; `out` is written instead where it
    is given; it may be the residual and overlaps no other tensor.  With
    `save_pre_activation` returns (y, z), z = x @ weight.T + bias in x's type, which
    the backward pass wants.  Few tokens -- one, in decoding -- read the weights at
    memory speed."""
    return _forward(x, weight, None, bias, residual, activation, out, out_dtype, save_pre_activation)


def linear_backward(dy, x, weight, *, activation: str = "none", pre_activation=None, dweight_dtype=None, dbias_dtype=None,
                    need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """Gradients of `linear`: (dx, dweight, dbias), None for what is not needed.
    dz = dy * act'(pre_activation) is rounded to x's type for the two matrix
    products; dx has x's type, dweight that or f32 (its sums in 32 bits, of factors
    in 16), dbias f32 (default) or that, from the unrounded dz.  The residual's
    gradient is dy."""
    return _backward(dy, x, weight, None, activation, pre_activation, dweight_dtype, dbias_dtype, need_dx, need_dweight,
                     need_dbias)


def grouped_linear(x, weight, offsets, bias=None, *, activation: str = "none", out=None, out_dtype=None,
                   save_pre_activation: bool = False):
    """`linear` with a weight matrix for each expert: rows offsets[g] to
    offsets[g + 1] of x (tokens, in), sorted by expert, go through weight[g] of
    (experts, out, in) and bias[g] of (experts, out).  offsets is an int32 tensor
    of experts + 1 entries on the GPU; it stays there.  Weights of experts
    without rows are not read.  Rows that belong to no expert are zero in a new y and
    z and stay as they are in `out`."""
    if offsets is None:
        raise ValueError("offsets must be given")
    return _forward(x, weight, offsets, bias, None, activation, out, out_dtype, save_pre_activation)


def grouped_linear_backward(dy, x, weight, offsets, *, activation: str = "none", pre_activation=None, dweight_dtype=None,
                            dbias_dtype=None, need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """Gradients of `grouped_linear`, as `linear_backward`: dweight (experts, out,
    in) and dbias (experts, out) are zero for experts without rows, dx is zero in
    rows that belong to no expert."""
    if offsets is None:
        raise ValueError("offsets must be given")
    return _backward(dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype, need_dx, need_dweight,
                     need_dbias)
