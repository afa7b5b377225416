"""Each refusal of the policy operators' C entries, with the message of that refusal (no GPU needed: nothing is launched)."""
from __future__ import annotations

import ctypes
import math

import pytest

from norm import _lib

ONE, OFF = ctypes.c_void_p(16), ctypes.c_void_p(17)   # an address that is given, and one that no value starts at
NONE4 = [None] * 4


@pytest.fixture(scope='module')
def lib():
    import build
    return _lib(build.build())


def _fwd(lib, x=ONE, r=None, y=ONE, total=None, rows=1, width=8, xt=0, yt=0, wt=0, w=None, stats=None):
    return lib.rl_norm_fwd(x, r, w, None, y, total, stats, rows, width, 8, 8, xt, yt, wt, 1e-5, None)


def _bwd(lib, gy=ONE, s=ONE, stats=ONE, dx=ONE, dw=None, rows=1, width=8, xt=0, yt=0, work=None, nbytes=0):
    return lib.rl_norm_bwd(gy, None, s, stats, None, dx, dw, None, rows, width, 8, 8, 8, xt, yt, 0, work, nbytes, None)


@pytest.mark.parametrize('call, given, word', [
    (_fwd, dict(rows=-1), 'rows must not be negative'), (_fwd, dict(width=0), 'width must be'), (_fwd, dict(width=2 ** 31), 'width must be'),
    (_fwd, dict(xt=3), 'unknown type'), (_fwd, dict(wt=-1), 'unknown type'), (_fwd, dict(xt=1, yt=2), "y must have x's type"),
    (_fwd, dict(x=None), 'must be given'), (_fwd, dict(y=None), 'must be given'), (_fwd, dict(r=ONE), 'must be given'),
    (_fwd, dict(x=OFF), 'misaligned'), (_fwd, dict(w=OFF), 'misaligned'), (_fwd, dict(stats=ctypes.c_void_p(20)), 'misaligned'),
    (_bwd, dict(rows=0), 'rows must be positive'), (_bwd, dict(width=0), 'width must be'), (_bwd, dict(gy=None), 'gy, s and stats'),
    (_bwd, dict(stats=None), 'gy, s and stats'), (_bwd, dict(dx=OFF), 'misaligned'), (_bwd, dict(dw=ONE), 'work space smaller'),
    (_bwd, dict(dw=ONE, work=ONE, nbytes=4), 'work space smaller'), (_bwd, dict(xt=2, yt=1), "y must have x's type")])
def test_norm(lib, call, given, word):
    other = _fwd(lib, width=0) if 'width' not in word else _fwd(lib, rows=-1)   # another message first
    assert other != 0
    assert call(lib, **given) != 0 and word in lib.rl_norm_error().decode()


GAPS = (ctypes.c_void_p * 10)(*([16] * 9))


def _moves(lib, logits=ONE, type=0, rows=1, T=1.0, k=0, p=1.0, m=0.0, cond=None, ctype=0, masks=ONE, u=ONE, Ts=None):
    return lib.rl_moves_sample(logits, 19, type, cond, ctype, masks, 19, u, T, k, p, m, Ts, None, None, None, ONE, ONE, rows, None)


def _rows(lib, width=5, legal=None, lw=0, rows=1, logits=ONE, T=1.0, choice=ONE, p=1.0, m=0.0, type=0):
    return lib.rl_sample(logits, width, type, width, legal, width, lw, ONE, T, 0, p, m, *NONE4, choice, ONE, rows, None)


def _logp(lib, logits=ONE, ids=ONE, type=0, rows=1, cond=None):
    return lib.rl_moves_logp(logits, 19, type, cond, 0, ONE, 19, ids, ONE, ONE, rows, None)


def _logp_bwd(lib, logits=ONE, dcond=None, cond=None, rows=1, work=None, nbytes=0, glp=ONE):
    return lib.rl_moves_logp_bwd(glp, 1, ONE, 1, logits, 19, 0, cond, 0, ONE, 19, ONE, ONE, dcond, rows, work, nbytes, None)


ALL = (ctypes.c_void_p * 10)(*([16] * 10))


@pytest.mark.parametrize('call, given, word', [
    (_moves, dict(rows=-1), 'rows must not be negative'), (_moves, dict(logits=None), 'must be given'), (_moves, dict(u=None), 'must be given'),
    (_moves, dict(type=3), 'unknown type'), (_moves, dict(T=-1.0), 'temperature'), (_moves, dict(T=math.nan), 'temperature'),
    (_moves, dict(p=-1.0), 'top_p'), (_moves, dict(m=2.0), 'min_p'), (_moves, dict(Ts=OFF), 'misaligned parameters'),
    (_moves, dict(cond=GAPS), 'ten tables'), (_moves, dict(cond=ALL, ctype=5), 'ten tables'), (_moves, dict(logits=OFF), 'misaligned pointer'),
    (_rows, dict(width=0), 'width must be'), (_rows, dict(width=4097), 'width must be'), (_rows, dict(legal=ONE, lw=19), 'legal must have'),
    (_rows, dict(rows=-1), 'rows must not be negative'), (_rows, dict(logits=None), 'must be given'), (_rows, dict(T=-0.5), 'temperature'),
    (_rows, dict(p=math.nan), 'top_p'), (_rows, dict(m=1.5), 'min_p'), (_rows, dict(type=-1), 'unknown type'),
    (_rows, dict(choice=ctypes.c_void_p(20)), 'misaligned pointer'),
    (_logp, dict(rows=-1), 'rows must not be negative'), (_logp, dict(logits=None), 'must be given'), (_logp, dict(ids=OFF), 'misaligned pointer'),
    (_logp, dict(type=4), 'unknown type'), (_logp, dict(cond=GAPS), 'ten tables'),
    (_logp_bwd, dict(rows=0), 'rows must be positive'), (_logp_bwd, dict(logits=None), 'must be given'),
    (_logp_bwd, dict(dcond=ONE), 'dcond needs the tables'), (_logp_bwd, dict(dcond=ONE, cond=ALL), 'work space smaller'),
    (_logp_bwd, dict(glp=OFF), 'misaligned pointer')])
def test_heads(lib, call, given, word):
    other = _rows(lib, width=0) if 'width' not in word else _rows(lib, T=-1.0)   # another message first
    assert other != 0
    assert call(lib, **given) != 0 and word in lib.rl_heads_error().decode()
