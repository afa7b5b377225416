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
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_logits(what, logits, width=None):
    if logits.device.type != 'cuda':
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
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != dev:
        raise RuntimeError(f'{what}: {name} must be {list(shape)} {dtype} on {dev}, got {list(t.shape)} {t.dtype} on '
                           f'{t.device}')
    return t.contiguous()


def _check_cond(what, cond, dev):
    """The tables' pointers (None without tables), their type, and the tensors that the pointers are of."""
    if cond is None:
        return None, 0, ()
    cond = [t.contiguous() for t in cond]
    if len(cond) != len(TABLES) or any(t.shape != s for t, s in zip(cond, TABLES)):
        raise RuntimeError(f'{what}: cond must be ten tables of shapes {TABLES}, got {[tuple(t.shape) for t in cond]}')
    dtype = cond[0].dtype
    if dtype not in _TYPES or any(t.dtype != dtype or t.device != dev for t in cond):
        raise RuntimeError(f'{what}: the tables of cond must be fp32, bf16 or fp16, all alike, on {dev}')
    return _Tables(*[t.data_ptr() for t in cond]), _TYPES[dtype], cond


def _check_cut(what, rows, dev, temperature, top_k, top_p, min_p):
    """The four parameters as rl_sample takes them (numbers, then pointers), and the tensors that the pointers are of."""
    numbers, pointers, kept = [], [], []
    for name, v, off, dtype in (('temperature', temperature, 1.0, torch.float32), ('top_k', top_k, 0, torch.int32),
                                ('top_p', top_p, 1.0, torch.float32), ('min_p', min_p, 0.0, torch.float32)):
        if torch.is_tensor(v):
            if v.dim() != 1 or v.shape[0] != rows or v.device != dev or v.dtype == torch.bool or v.is_complex() \
                    or (name == 'top_k' and v.is_floating_point()):
                raise RuntimeError(f'{what}: {name} must be a number or [{rows}] on {dev}, got {list(v.shape)} {v.dtype} '
                                   f'on {v.device}')
            v = v.to(dtype).contiguous()
            numbers.append(off)
            pointers.append(v.data_ptr())
            kept.append(v)
        else:
            numbers.append(v)
            pointers.append(None)
    t, k, p, m = numbers
    if not (t >= 0 and p >= 0 and m <= 1 and 0 <= k < 2 ** 31 and int(k) == k):
        raise RuntimeError(f'{what}: temperature and top_p must be 0 or more, top_k a whole number of 0 or more, min_p at most '
                           f'1; got temperature {t}, top_k {k}, top_p {p}, min_p {m}')
    return (t, int(k), p, m, *pointers), kept


def _call(lib, what, rc):
    if rc != 0:
        raise RuntimeError(f'{what}: {lib.rl_heads_error().decode()}')


def sample_moves(logits, cond, masks, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lib_path=None):
    """One move for each row, part by part: (packed ids int16 [B], log-probabilities fp32 [B])."""
    logits = _check_logits('sample_moves', logits, BYTES)
    rows, dev = logits.shape[0], logits.device
    tables, cond_type, kept = _check_cond('sample_moves', cond, dev)
    masks = _check_bytes('sample_moves', 'masks', masks, rows, (BYTES,), dev)
    u = _check_row('sample_moves', 'u', u, (rows, 5), torch.float32, dev)
    cut, cut_kept = _check_cut('sample_moves', rows, dev, temperature, top_k, top_p, min_p)
    ids = torch.empty(rows, dtype=torch.int16, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    lib = _lib(lib_path)
    with torch.cuda.device(dev):
        _call(lib, 'rl_moves_sample', lib.rl_moves_sample(
            logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], tables, cond_type, masks.data_ptr(), masks.stride(0),
            u.data_ptr(), *cut, ids.data_ptr(), logp.data_ptr(), rows, torch.cuda.current_stream(dev).cuda_stream))
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
    cut, cut_kept = _check_cut('sample', rows, dev, temperature, top_k, top_p, min_p)
    choice = torch.empty(rows, dtype=torch.int64, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    lib = _lib(lib_path)
    with torch.cuda.device(dev):
        _call(lib, 'rl_sample', lib.rl_sample(
            logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], width, None if legal is None else legal.data_ptr(),
            0 if legal is None else legal.stride(0), 0 if legal is None else legal.shape[1], u.data_ptr(), *cut,
            choice.data_ptr(), logp.data_ptr(), rows, torch.cuda.current_stream(dev).cuda_stream))
    return choice, logp


def _logp_forward(logits, cond, masks, ids, lib_path):
    rows, dev = logits.shape[0], logits.device
    tables, cond_type, kept = _check_cond('moves_logp', cond, dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    lib = _lib(lib_path)
    with torch.cuda.device(dev):
        _call(lib, 'rl_moves_logp', lib.rl_moves_logp(
            logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], tables, cond_type, masks.data_ptr(), masks.stride(0),
            ids.data_ptr(), logp.data_ptr(), entropy.data_ptr(), rows, torch.cuda.current_stream(dev).cuda_stream))
    return logp, entropy


class _MovesLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, masks, ids, lib_path, *cond):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, masks, ids, *cond)
        ctx.lib_path = lib_path
        return _logp_forward(logits, cond or None, masks, ids, lib_path)

    @staticmethod
    @once_differentiable
    def backward(ctx, glp, gent):
        logits, masks, ids, *cond = ctx.saved_tensors
        rows, dev = logits.shape[0], logits.device
        want_cond = any(ctx.needs_input_grad[4:])
        dlogits = torch.empty((rows, BYTES), dtype=logits.dtype, device=dev) if ctx.needs_input_grad[0] else None
        none = (glp is None and gent is None) or rows == 0
        dcond = (torch.zeros if none else torch.empty)(sum(a * b for a, b in TABLES), dtype=torch.float32,
                                                       device=dev) if want_cond else None
        if none:
            dlogits = None if dlogits is None else dlogits.zero_()
        else:
            tables, cond_type, kept = _check_cond('moves_logp', cond or None, dev)
            lib = _lib(ctx.lib_path)
            with torch.cuda.device(dev):
                nbytes = int(lib.rl_moves_logp_bwd_work_bytes()) if want_cond else 0
                work = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
                _call(lib, 'rl_moves_logp_bwd', lib.rl_moves_logp_bwd(
                    None if glp is None else glp.data_ptr(), 0 if glp is None else glp.stride(0),
                    None if gent is None else gent.data_ptr(), 0 if gent is None else gent.stride(0),
                    logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], tables, cond_type, masks.data_ptr(),
                    masks.stride(0), ids.data_ptr(), None if dlogits is None else dlogits.data_ptr(),
                    None if dcond is None else dcond.data_ptr(), rows, None if work is None else work.data_ptr(), nbytes,
                    torch.cuda.current_stream(dev).cuda_stream))
        grads, at = [], 0
        for need, t, (a, b) in zip(ctx.needs_input_grad[4:], cond, TABLES):
            grads.append(dcond[at:at + a * b].view(a, b).to(t.dtype) if need else None)
            at += a * b
        return (dlogits, None, None, None, *grads)


def moves_logp(logits, cond, masks, ids, lib_path=None):
    """(log-probability, entropy) fp32 [B] of the moves ids under the ordered heads, the entropy the sum of the parts'
    conditional entropies along the move. A move that the masks exclude has log-probability -inf, an id outside 0..323 NaN
    in both."""
    logits = _check_logits('moves_logp', logits, BYTES)
    rows, dev = logits.shape[0], logits.device
    masks = _check_bytes('moves_logp', 'masks', masks, rows, (BYTES,), dev)
    ids = _check_row('moves_logp', 'ids', ids, (rows,), torch.int16, dev)
    cond = () if cond is None else tuple(cond)
    if cond and len(cond) != len(TABLES):
        raise RuntimeError(f'moves_logp: cond must be ten tables, got {len(cond)}')
    if torch.is_grad_enabled() and (logits.requires_grad or any(t.requires_grad for t in cond)):
        return _MovesLogp.apply(logits, masks, ids, lib_path, *cond)
    return _logp_forward(logits, cond or None, masks, ids, lib_path)
