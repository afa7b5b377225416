"""Layer norm of the policy's blocks on the B200 library (rl_norm_fwd / rl_norm_bwd), with the residual sum before it:

    y = layer_norm(x, weight, bias, eps)                             # as torch.nn.functional.layer_norm over the last axis
    y, stream = layer_norm(x, weight, bias, eps, residual=branch)    # stream = x + branch, y = its norm

A SimBa block (rl/model.py:64-72) is x + mlp(norm(x)): the sum and the next block's norm read the stream once here. x and
residual: [..., D] fp32, bf16 or fp16, any leading shape and row strides; weight and bias: [D] of any of the three types,
each may be None; out_dtype: x's type (default) or fp32. The stream is kept in x's type, and what is kept is what is
normalised. Statistics and sums are fp32, every output is rounded once. Differentiable (once) in x, residual, weight and
bias; the gradients of weight and bias are summed in a fixed order, so the same inputs give the same bits."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from rlenv import default_lib

_LIB = None
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_stream = torch._C._cuda_getCurrentRawStream   # the current stream's handle, without an object made for it


def _lib(path=None):
    global _LIB
    if _LIB is None or path is not None:
        lib = ctypes.CDLL(str(path or default_lib()))
        P, I, L, SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
        lib.rl_norm_fwd.argtypes = [P] * 7 + [L] * 4 + [I] * 3 + [ctypes.c_float, P]
        lib.rl_norm_bwd_work_bytes.argtypes = [L, L]
        lib.rl_norm_bwd_work_bytes.restype = SZ
        lib.rl_norm_bwd.argtypes = [P] * 8 + [L] * 5 + [I] * 3 + [P, SZ, P]
        lib.rl_norm_error.restype = ctypes.c_char_p
        _LIB = lib
    return _LIB


def _rows(t, width):
    """t as [rows, width] with adjacent columns (a view where its strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


def _check(x, weight, bias, residual, out_dtype):
    if not x.is_cuda:
        raise RuntimeError('layer_norm runs on the GPU only')
    if x.dtype not in _TYPES:
        raise RuntimeError(f'layer_norm: x must be fp32, bf16 or fp16, got {x.dtype}')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f'layer_norm: x needs a last axis of at least one value, got shape {tuple(x.shape)}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != x.shape[-1] or t.dtype not in _TYPES or t.device != x.device):
            raise RuntimeError(f'layer_norm: {name} must be [{x.shape[-1]}], fp32, bf16 or fp16, on {x.device}; got '
                               f'{list(t.shape)} {t.dtype} on {t.device}')
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f'layer_norm: weight ({weight.dtype}) and bias ({bias.dtype}) must have one type')
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise RuntimeError(f'layer_norm: the residual must be as x, {list(x.shape)} {x.dtype} on {x.device}; got '
                           f'{list(residual.shape)} {residual.dtype} on {residual.device}')
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise RuntimeError(f'layer_norm: out_dtype must be {x.dtype} or fp32, got {out_dtype}')


def _forward(x, weight, bias, eps, residual, out_dtype, lib_path, want_stats):
    """(y, stream or None, the rows that were normalised, their statistics or None)."""
    dev, width = x.device, x.shape[-1]
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _forward(x, weight, bias, eps, residual, out_dtype, lib_path, want_stats)
    x2 = _rows(x, width)
    rows = x2.shape[0]
    plain = x.is_contiguous()
    y = torch.empty_like(x) if plain and out_dtype == x.dtype else torch.empty(x.shape, dtype=out_dtype, device=dev)
    r2 = total = stats = None
    if residual is not None:
        r2 = _rows(residual, width)
        total = torch.empty_like(x) if plain else torch.empty(x.shape, dtype=x.dtype, device=dev)
    if want_stats:
        stats = torch.empty((rows, 2), dtype=torch.float32, device=dev)
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    param = bias if weight is None else weight
    lib = _lib(lib_path)
    rc = lib.rl_norm_fwd(x2.data_ptr(), None if r2 is None else r2.data_ptr(), None if weight is None else weight.data_ptr(),
                         None if bias is None else bias.data_ptr(), y.data_ptr(), None if total is None else total.data_ptr(),
                         None if stats is None else stats.data_ptr(), rows, width, x2.stride(0),
                         0 if r2 is None else r2.stride(0), _TYPES[x.dtype], _TYPES[out_dtype],
                         0 if param is None else _TYPES[param.dtype], eps, _stream(dev.index))
    if rc != 0:
        raise RuntimeError(f'rl_norm_fwd: {lib.rl_norm_error().decode()}')
    return y, total, x2 if total is None else total, stats


def _backward(gy, gsum, s, stats, weight, w_dtype, want_dx, want_dw, want_db, lib_path):
    """Gradients (dx, dweight, dbias) from gy [..., D] and gsum [..., D] or None."""
    dev, width = s.device, s.shape[-1]
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _backward(gy, gsum, s, stats, weight, w_dtype, want_dx, want_dw, want_db, lib_path)
    s = _rows(s, width)
    gy = _rows(gy, width)
    rows = s.shape[0]
    gsum = None if gsum is None else _rows(gsum, width)
    dx = dw = db = work = None
    nbytes = 0
    lib = _lib(lib_path)
    if want_dx:
        dx = torch.empty((rows, width), dtype=s.dtype, device=dev)
    if want_dw or want_db:
        nbytes = lib.rl_norm_bwd_work_bytes(rows, width)
        work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        if want_dw:
            dw = torch.empty(width, dtype=w_dtype, device=dev)
        if want_db:
            db = torch.empty(width, dtype=w_dtype, device=dev)
    rc = lib.rl_norm_bwd(gy.data_ptr(), None if gsum is None else gsum.data_ptr(), s.data_ptr(), stats.data_ptr(),
                         None if weight is None else weight.data_ptr(), None if dx is None else dx.data_ptr(),
                         None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), rows, width,
                         gy.stride(0), 0 if gsum is None else gsum.stride(0), s.stride(0), _TYPES[s.dtype],
                         _TYPES[gy.dtype], _TYPES[w_dtype], None if work is None else work.data_ptr(), nbytes,
                         _stream(dev.index))
    if rc != 0:
        raise RuntimeError(f'rl_norm_bwd: {lib.rl_norm_error().decode()}')
    return dx, dw, db


def _gradients(ctx, gy, gsum):
    s, stats, weight = ctx.saved_tensors
    shape, b_dtype, lib_path = ctx.opts
    need_x, need_w, need_b, need_r, *_ = ctx.needs_input_grad
    w_dtype = weight.dtype if weight is not None else b_dtype or torch.float32
    if gy is None or stats.shape[0] == 0:
        # nothing came through the norm: the stream's gradient passes as it is
        dx = torch.empty(shape, dtype=s.dtype, device=s.device) if stats.shape[0] == 0 else gsum
        dw = torch.zeros(shape[-1], dtype=w_dtype, device=s.device) if need_w else None
        db = torch.zeros(shape[-1], dtype=w_dtype, device=s.device) if need_b else None
    else:
        dx, dw, db = _backward(gy, gsum, s, stats, weight, w_dtype, need_x or need_r, need_w, need_b, lib_path)
        if dx is not None and len(shape) != 2:
            dx = dx.view(shape)
    return dx if need_x else None, dw, db, dx if need_r else None, None, None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, out_dtype, lib_path):
        ctx.set_materialize_grads(False)
        if weight is not None:
            weight = weight.contiguous()
        y, total, s, stats = _forward(x, weight, bias, eps, residual, out_dtype, lib_path, True)
        ctx.save_for_backward(s, stats, weight)
        ctx.opts = (x.shape, None if bias is None else bias.dtype, lib_path)
        return y if total is None else (y, total)

    @staticmethod
    def backward(ctx, gy, gsum=None):
        if torch.is_grad_enabled():   # the gradients' own graph is wanted: they have none, and say so when it is used
            return once_differentiable(_gradients)(ctx, gy, gsum)
        return _gradients(ctx, gy, gsum)


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None, out_dtype=None, lib_path=None):
    """The norm of x's last axis; with a residual, (norm of x + residual, x + residual)."""
    out_dtype = out_dtype or x.dtype
    _check(x, weight, bias, residual, out_dtype)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, residual, eps, out_dtype, lib_path)
    y, total, _, _ = _forward(x, weight, bias, eps, residual, out_dtype, lib_path, False)
    return y if total is None else (y, total)
