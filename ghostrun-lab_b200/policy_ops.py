"""Loads what norm.py and heads.py call: the GPU library (rl_norm_*, rl_sample, rl_moves_*) and policy_ops_b200, its PyTorch
binding, which is given the library's functions."""
from __future__ import annotations

import ctypes

import torch  # noqa: F401  (before the binding: it uses torch's libraries)

from rlenv import default_lib

ENTRIES = ('rl_norm_fwd', 'rl_norm_bwd_work_bytes', 'rl_norm_bwd', 'rl_norm_error', 'rl_moves_sample', 'rl_sample', 'rl_moves_logp',
           'rl_moves_logp_bwd_work_bytes', 'rl_moves_logp_bwd', 'rl_heads_error')

_LIB = None


def load(path=None):
    """The library, with the C-ABI's argument types, bound to policy_ops_b200; another path takes the place of the one
    before, for every later call in the process."""
    global _LIB
    if _LIB is None or path is not None:
        try:
            import policy_ops_b200
        except ImportError as e:
            raise RuntimeError(f'policy_ops_b200 cannot be loaded ({e}): build it with ghostrun-lab_b200/build.py') from e
        lib = ctypes.CDLL(str(path or default_lib()))
        P, I, L, SZ, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_float
        cut = [F, I, F, F, P, P, P, P]
        lib.rl_norm_fwd.argtypes = [P] * 7 + [L] * 4 + [I] * 3 + [F, P]
        lib.rl_norm_bwd_work_bytes.argtypes = [L, L]
        lib.rl_norm_bwd_work_bytes.restype = SZ
        lib.rl_norm_bwd.argtypes = [P] * 8 + [L] * 5 + [I] * 3 + [P, SZ, P]
        lib.rl_norm_error.restype = ctypes.c_char_p
        lib.rl_moves_sample.argtypes = [P, L, I, P, I, P, L, P, *cut, P, P, L, P]
        lib.rl_sample.argtypes = [P, L, I, I, P, L, I, P, *cut, P, P, L, P]
        lib.rl_moves_logp.argtypes = [P, L, I, P, I, P, L, P, P, P, L, P]
        lib.rl_moves_logp_bwd_work_bytes.restype = SZ
        lib.rl_moves_logp_bwd.argtypes = [P, L, P, L, P, L, I, P, I, P, L, P, P, P, L, P, SZ, P]
        lib.rl_heads_error.restype = ctypes.c_char_p
        policy_ops_b200.bind({n: ctypes.cast(getattr(lib, n), P).value for n in ENTRIES})
        _LIB = lib
    return _LIB
