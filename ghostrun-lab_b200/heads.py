"""The policy's action heads on the B200 library: moves sampled from given random numbers, and the log-probability and
entropy of given moves (rl/model.py:176-194, ordered heads masked by the legal parts).

    ids, logp = sample_moves(logits, cond, masks, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    logp, entropy = moves_logp(logits, cond, masks, ids)                    # differentiable in logits and cond
    choice, logp = sample(logits, u, legal=masks, top_p=0.95)               # rows of any width up to 4096

logits: [B, 19] fp32, bf16 or fp16, the five heads side by side in the mask bytes' order (actions.PARTS); cond: the ten
tables [choices of part j, choices of part k] for k = 1..4, j < k (policy.Policy.tables()), or None; masks: [B, 19] bytes, as
RlEnv.masks; u: fp32 random numbers in [0, 1), [B, 5] (sample: [B]); ids: int16 packed moves, as RlEnv.actions. sample's
legal is [B, V], or the 19 mask bytes for a flat head over the 324 packed moves, or None.

temperature (0: the best choice), top_k (0: all), top_p and min_p are numbers, or tensors with one for each row. They apply
in this order: top-k of the logits / temperature, the shortest run of what is left that holds top_p of its probability,
those of it with at least min_p of the best one's. Equal logits rank by index. The log-probability returned is that of the
distribution drawn from. The same inputs give the same choice on any launch shape (csrc/heads.cu). A part (or row) with
nothing legal answers 0, the neutral choice, with log-probability and entropy 0 and no gradient."""
from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd.function import once_differentiable

from rlenv import default_lib

SIZES = (9, 3, 3, 2, 2)                                              # choices of each part
TABLES = [(SIZES[j], SIZES[k]) for k in range(5) for j in range(k)]   # shapes of the ten tables of cond
MOVES, BYTES, MAX_WIDTH = 324, 19, 4096

_LIB = None
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_Tables = ctypes.c_void_p * len(TABLES)
_TABLE_AT = [sum(a * b for a, b in TABLES[:t]) for t in range(len(TABLES) + 1)]   # where each table starts, laid end to end
_CUT = (('temperature', 1.0, torch.float32), ('top_k', 0, torch.int32), ('top_p', 1.0, torch.float32),
        ('min_p', 0.0, torch.float32))
_stream = torch._C._cuda_getCurrentRawStream   # the current stream's handle, without an object made for it
_HERE = contextlib.nullcontext()


def _on(dev):
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _lib(path=None):
    global _LIB
    if _LIB is None or path is not None:
        lib = ctypes.CDLL(str(path or default_lib()))
        P, I, L, SZ, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_float
        cut = [F, I, F, F, P, P, P, P]
        lib.rl_moves_sample.argtypes = [P, L, I, P, I, P, L, P, *cut, P, P, L, P]
        lib.rl_sample.argtypes = [P, L, I, I, P, L, I, P, *cut, P, P, L, P]
        lib.rl_moves_logp.argtypes = [P, L, I, P, I, P, L, P, P, P, L, P]
        lib.rl_moves_logp_bwd_work_bytes.restype = SZ
        lib.rl_moves_logp_bwd.argtypes = [P, L, P, L, P, L, I, P, I, P, L, P, P, P, L, P, SZ, P]
        lib.rl_heads_error.restype = ctypes.c_char_p
        _LIB = lib
    return _LIB


def _adjacent(t):
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_logits(what, logits, width=None):
    if not logits.is_cuda:
        raise RuntimeError(f'{what} runs on the GPU only')
    if logits.dim() != 2 or logits.dtype not in _TYPES or (width is not None and logits.shape[1] != width):
        raise RuntimeError(f'{what}: logits must be [B, {width or "V"}] fp32, bf16 or fp16, got {list(logits.shape)} '
                           f'{logits.dtype}')
    return _adjacent(logits)


def _check_bytes(what, name, t, rows, widths, dev):
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] not in widths or t.dtype not in (torch.uint8, torch.bool) \
            or t.device != dev:
        raise RuntimeError(f'{what}: {name} must be [{rows}, {" or ".join(map(str, widths))}] bytes (uint8 or bool) on '
                           f'{dev}, got {list(t.shape)} {t.dtype} on {t.device}')
    return _adjacent(t)


def _check_row(what, name, t, shape, dtype, dev):
    if t.shape != shape or t.dtype != dtype or t.device != dev:
        raise RuntimeError(f'{what}: {name} must be {list(shape)} {dtype} on {dev}, got {list(t.shape)} {t.dtype} on '
                           f'{t.device}')
    return t.contiguous()


def _check_cond(what, cond, dev):
    """The tables, each contiguous; () without tables."""
    if cond is None:
        return ()
    cond = [t.contiguous() for t in cond]
    if len(cond) != len(TABLES) or any([t.shape != s for t, s in zip(cond, TABLES)]):
        raise RuntimeError(f'{what}: cond must be ten tables of shapes {TABLES}, got {[tuple(t.shape) for t in cond]}')
    dtype = cond[0].dtype
    if dtype not in _TYPES or any([t.dtype != dtype or t.device != dev for t in cond]):
        raise RuntimeError(f'{what}: the tables of cond must be fp32, bf16 or fp16, all alike, on {dev}')
    return cond


def _pointers(cond):
    """The tables as the library takes them: an array of their pointers and their type."""
    return (_Tables(*[t.data_ptr() for t in cond]), _TYPES[cond[0].dtype]) if cond else (None, 0)


def _check_cut(what, rows, dev, temperature, top_k, top_p, min_p):
    """The four parameters as the library takes them (numbers, then pointers), and the tensors that the pointers are of."""
    values = [temperature, top_k, top_p, min_p]
    pointers, kept = [None] * 4, []
    for i, v in enumerate(values):
        if isinstance(v, torch.Tensor):
            name, off, dtype = _CUT[i]
            if v.dim() != 1 or v.shape[0] != rows or v.device != dev or v.dtype == torch.bool or v.is_complex() \
                    or (name == 'top_k' and v.is_floating_point()):
                raise RuntimeError(f'{what}: {name} must be a number or [{rows}] on {dev}, got {list(v.shape)} {v.dtype} '
                                   f'on {v.device}')
            v = v.to(dtype).contiguous()
            values[i], pointers[i] = off, v.data_ptr()
            kept.append(v)
    t, k, p, m = values
    if not (t >= 0 and p >= 0 and m <= 1 and 0 <= k < 2 ** 31 and int(k) == k):
        raise RuntimeError(f'{what}: temperature and top_p must be 0 or more, top_k a whole number of 0 or more, min_p at most '
                           f'1; got temperature {t}, top_k {k}, top_p {p}, min_p {m}')
    return (t, int(k), p, m, *pointers), kept


def _call(lib, name, *args):
    if getattr(lib, name)(*args) != 0:
        raise RuntimeError(f'{name}: {lib.rl_heads_error().decode()}')


def sample_moves(logits, cond, masks, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lib_path=None):
    """One move for each row, part by part: (packed ids int16 [B], log-probabilities fp32 [B])."""
    logits = _check_logits('sample_moves', logits, BYTES)
    rows, dev = logits.shape[0], logits.device
    cond = _check_cond('sample_moves', cond, dev)
    masks = _check_bytes('sample_moves', 'masks', masks, rows, (BYTES,), dev)
    u = _check_row('sample_moves', 'u', u, (rows, 5), torch.float32, dev)
    cut, kept = _check_cut('sample_moves', rows, dev, temperature, top_k, top_p, min_p)
    ids = torch.empty(rows, dtype=torch.int16, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        _call(_lib(lib_path), 'rl_moves_sample', logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], *_pointers(cond),
              masks.data_ptr(), masks.stride(0), u.data_ptr(), *cut, ids.data_ptr(), logp.data_ptr(), rows, _stream(dev.index))
    return ids, logp


def sample(logits, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lib_path=None):
    """One choice for each row of logits [B, V]: (choices int64 [B], log-probabilities fp32 [B])."""
    logits = _check_logits('sample', logits)
    (rows, width), dev = logits.shape, logits.device
    if not 1 <= width <= MAX_WIDTH:
        raise RuntimeError(f'sample: rows must have 1 to {MAX_WIDTH} choices, got {width}')
    if legal is not None:
        legal = _check_bytes('sample', 'legal', legal, rows, (width, BYTES) if width == MOVES else (width,), dev)
    u = _check_row('sample', 'u', u, (rows,), torch.float32, dev)
    cut, kept = _check_cut('sample', rows, dev, temperature, top_k, top_p, min_p)
    choice = torch.empty(rows, dtype=torch.int64, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        _call(_lib(lib_path), 'rl_sample', logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], width,
              None if legal is None else legal.data_ptr(), 0 if legal is None else legal.stride(0),
              0 if legal is None else legal.shape[1], u.data_ptr(), *cut, choice.data_ptr(), logp.data_ptr(), rows,
              _stream(dev.index))
    return choice, logp


def _logp_forward(logits, cond, masks, ids, lib_path):
    rows, dev = logits.shape[0], logits.device
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        _call(_lib(lib_path), 'rl_moves_logp', logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], *_pointers(cond),
              masks.data_ptr(), masks.stride(0), ids.data_ptr(), logp.data_ptr(), entropy.data_ptr(), rows,
              _stream(dev.index))
    return logp, entropy


def _logp_gradients(ctx, glp, gent):
    logits, masks, ids, *cond = ctx.saved_tensors
    rows, dev, need = logits.shape[0], logits.device, ctx.needs_input_grad
    dlogits = dcond = work = None
    if need[0]:
        dlogits = torch.empty((rows, BYTES), dtype=logits.dtype, device=dev)
    if any(need[4:]):
        dcond = torch.empty(_TABLE_AT[-1], dtype=torch.float32, device=dev)
    if rows == 0 or (glp is None and gent is None):
        for t in (dlogits, dcond):
            if t is not None:
                t.zero_()
    else:
        lib = _lib(ctx.lib_path)
        with _on(dev):
            nbytes = 0
            if dcond is not None:
                nbytes = lib.rl_moves_logp_bwd_work_bytes()
                work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
            _call(lib, 'rl_moves_logp_bwd', None if glp is None else glp.data_ptr(), 0 if glp is None else glp.stride(0),
                  None if gent is None else gent.data_ptr(), 0 if gent is None else gent.stride(0), logits.data_ptr(),
                  logits.stride(0), _TYPES[logits.dtype], *_pointers(cond), masks.data_ptr(), masks.stride(0),
                  ids.data_ptr(), None if dlogits is None else dlogits.data_ptr(),
                  None if dcond is None else dcond.data_ptr(), rows, None if work is None else work.data_ptr(), nbytes,
                  _stream(dev.index))
    if dcond is None:
        return (dlogits, None, None, None, *[None] * len(cond))
    if cond[0].dtype != torch.float32:
        dcond = dcond.to(cond[0].dtype)
    tables = [dcond.as_strided(s, (s[1], 1), at) if n else None for s, at, n in zip(TABLES, _TABLE_AT, need[4:])]
    return (dlogits, None, None, None, *tables)


class _MovesLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, masks, ids, lib_path, *cond):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, masks, ids, *cond)
        ctx.lib_path = lib_path
        return _logp_forward(logits, cond, masks, ids, lib_path)

    @staticmethod
    def backward(ctx, glp, gent):
        if torch.is_grad_enabled():   # the gradients' own graph is wanted: they have none, and say so when it is used
            return once_differentiable(_logp_gradients)(ctx, glp, gent)
        return _logp_gradients(ctx, glp, gent)


def moves_logp(logits, cond, masks, ids, lib_path=None):
    """(log-probability, entropy) fp32 [B] of the moves ids under the ordered heads, the entropy the sum of the parts'
    conditional entropies along the move. A move that the masks exclude has log-probability -inf, an id outside 0..323 NaN
    in both."""
    logits = _check_logits('moves_logp', logits, BYTES)
    rows, dev = logits.shape[0], logits.device
    masks = _check_bytes('moves_logp', 'masks', masks, rows, (BYTES,), dev)
    ids = _check_row('moves_logp', 'ids', ids, (rows,), torch.int16, dev)
    cond = _check_cond('moves_logp', cond, dev)
    if torch.is_grad_enabled() and (logits.requires_grad or any([t.requires_grad for t in cond])):
        return _MovesLogp.apply(logits, masks, ids, lib_path, *cond)
    return _logp_forward(logits, cond, masks, ids, lib_path)
