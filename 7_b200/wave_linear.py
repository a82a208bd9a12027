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
import functools

from . import wave_cuda as wc

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


@functools.lru_cache(maxsize=None)
def _types():
    import torch
    return torch, {torch.bfloat16: wc.BF16, torch.float16: wc.F16, torch.float32: wc.F32}


@functools.lru_cache(maxsize=4096)
def _plan(device: int, backward: bool, *fields):
    """A descriptor (a pure function of sizes, strides and types) and the bytes
    of workspace a call with it takes on that device."""
    desc = wc.LinearDesc(*fields)
    try:
        wc.linear_validate(desc)
        need = wc.linear_workspace_bytes(desc, backward)
    except wc.WaveCudaError as err:
        if err.code in (wc.E_INVALID, wc.E_UNSUPPORTED):
            raise ValueError(err.message) from None
        raise
    return desc, C.byref(desc), need


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
    torch, types = _types()
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
    return torch, types, device, tokens, n, k, experts, ldx, ldw, stride_w


def _act(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}")
    return code


def _aligned(t):
    """TMA loads start on 16-byte boundaries: a view that does not is copied."""
    if t.data_ptr() % 16 == 0:
        return t
    torch, _ = _types()
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


class _On:
    """The tensors' device made current (its streams and the library's launches
    go by the current device), and its current stream."""

    def __init__(self, torch, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None
        self.torch, self.device = torch, device

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _forward(x, weight, offsets, bias, residual, activation, out, out_dtype, save):
    torch, types, device, tokens, n, k, experts, ldx, ldw, stride_w = _layer(x, weight, offsets)
    io = x.dtype
    x, weight = (t if t.data_ptr() % 16 == 0 else _aligned(t) for t in (x, weight))
    ldx = ldx if tokens <= 1 else x.stride(0)
    if weight.stride(-1) == 1 and n > 1:
        ldw = weight.stride(-2)
    if experts > 1:
        stride_w = weight.stride(0)
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
        y, zero_rest, ldy = torch.empty((tokens, n), dtype=y_type, device=device), int(offsets is not None), 0
    else:
        y_type, zero_rest = out.dtype, 0
        if out_dtype is not None and out_dtype != y_type:
            raise ValueError(f"out has dtype {y_type}, out_dtype says {out_dtype}")
        y, ldy = out, _matrix(out, "out", tokens, n, (io, torch.float32), device)
    z = None
    if save:
        z = (torch.zeros if offsets is not None and not zero_rest else torch.empty)((tokens, n), dtype=io, device=device)
    with _On(torch, device) as stream:
        _, ref, need = _plan(device.index, False, tokens, n, k, experts, types[io], types[y_type], types[bias_type], types[io],
                             wc.F32, _act(activation), zero_rest, 0, ldx, ldw, ldy, ldr, 0, 0, 0, stride_w, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        wc.check(wc.lib().wave_cuda_linear_fwd(
            ref, x.data_ptr(), weight.data_ptr(), bias.data_ptr() if bias is not None else None,
            residual.data_ptr() if residual is not None else None, offsets.data_ptr() if offsets is not None else None,
            y.data_ptr(), z.data_ptr() if save else None, ws.data_ptr() if need else None, stream))
    return (y, z) if save else y


def _backward(dy, x, weight, offsets, activation, pre_activation, dweight_dtype, dbias_dtype, need_dx, need_dweight,
              need_dbias):
    torch, types, device, tokens, n, k, experts, ldx, ldw, stride_w = _layer(x, weight, offsets)
    io = x.dtype
    act = _act(activation)
    _matrix(dy, "dy", tokens, n, (io, torch.float32), device)
    ldz = 0
    if act:
        if pre_activation is None:
            raise ValueError(f"the gradient of {activation} needs the pre-activation")
        ldz = _matrix(pre_activation, "pre_activation", tokens, n, (io,), device)
    dweight_dtype = io if dweight_dtype is None else dweight_dtype
    for name, t in (("dweight_dtype", dweight_dtype), ("dbias_dtype", dbias_dtype or torch.float32)):
        if t not in (io, torch.float32):
            raise ValueError(f"{name} must be {io} or f32; got {t}")
    dbias_dtype = dbias_dtype or torch.float32
    x, weight, dy = (t if t.data_ptr() % 16 == 0 else _aligned(t) for t in (x, weight, dy))
    ldx, ldy = (t.stride(0) if tokens > 1 else 0 for t in (x, dy))
    if n > 1:
        ldw = weight.stride(-2)
    if experts > 1:
        stride_w = weight.stride(0)
    lead = (experts,) if offsets is not None else ()
    dx = torch.empty((tokens, k), dtype=io, device=device) if need_dx else None
    dw = torch.empty((*lead, n, k), dtype=dweight_dtype, device=device) if need_dweight else None
    db = torch.empty((*lead, n), dtype=dbias_dtype, device=device) if need_dbias else None
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    with _On(torch, device) as stream:
        _, ref, need = _plan(device.index, True, tokens, n, k, experts, types[io], types[dy.dtype], types[io],
                             types[dweight_dtype], types[dbias_dtype], act, int(offsets is not None), 0, ldx, ldw, ldy, 0, ldz,
                             0, 0, stride_w, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        wc.check(wc.lib().wave_cuda_linear_bwd(ref, ptr(dy), ptr(x), ptr(weight), ptr(pre_activation) if act else None,
                                               ptr(offsets), ptr(dx), ptr(dw), ptr(db), ptr(ws), stream))
    return dx, dw, db


def linear(x, weight, bias=None, residual=None, *, activation: str = "none", out=None, out_dtype=None,
           save_pre_activation: bool = False):
    """act(x @ weight.T + bias) + residual in one kernel.

    x (tokens, in) and weight (out, in) in bf16 or f16, rows of any stride; bias
    (out,) in that type or f32; residual (tokens, out) in that type.
    `activation`: none, relu, gelu (erf), gelu_tanh or silu.  Returns y (tokens,
    out) in x's type, or f32 with `out_dtype`; `out` is written instead where it
    is given and may be the residual.  With `save_pre_activation` returns (y, z),
    z = x @ weight.T + bias in x's type, which the backward pass wants.  Few
    tokens -- one, in decoding -- read the weights at memory speed."""
    return _forward(x, weight, None, bias, residual, activation, out, out_dtype, save_pre_activation)


def linear_backward(dy, x, weight, *, activation: str = "none", pre_activation=None, dweight_dtype=None, dbias_dtype=None,
                    need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """Gradients of `linear`: (dx, dweight, dbias), None for what is not needed.
    dz = dy * act'(pre_activation) is rounded to x's type for the two matrix
    products; dx has x's type, dweight that or f32, dbias f32 (default) or that.
    The residual's gradient is dy."""
    return _backward(dy, x, weight, None, activation, pre_activation, dweight_dtype, dbias_dtype, need_dx, need_dweight,
                     need_dbias)


def grouped_linear(x, weight, offsets, bias=None, *, activation: str = "none", out=None, out_dtype=None,
                   save_pre_activation: bool = False):
    """`linear` with a weight matrix for each expert: rows offsets[g] to
    offsets[g + 1] of x (tokens, in), sorted by expert, go through weight[g] of
    (experts, out, in) and bias[g] of (experts, out).  offsets is an int32 tensor
    of experts + 1 entries on the GPU; it stays there.  Experts without rows cost
    nothing.  Rows that belong to no expert are zero in a new y and z and stay as
    they are in `out`."""
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
