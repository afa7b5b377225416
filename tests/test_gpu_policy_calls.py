"""What the policy operators' calls take and refuse beyond their values: forward-mode derivatives (norm.py, heads.py,
csrc/policy_ops.cpp)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from heads import SIZES, TABLES, _lib, moves_logp
from norm import layer_norm


@pytest.fixture
def lib(gpu_lib_path):
    return _lib(gpu_lib_path)


def _heads(rows, seed):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(rows, 19, generator=g).cuda()
    cond = [torch.randn(s, generator=g).cuda() for s in TABLES]
    parts = [torch.randint(0, n, (rows,), generator=g) for n in SIZES]
    ids = parts[0] + 9 * parts[1] + 27 * parts[2] + 81 * parts[3] + 162 * parts[4]
    return logits, cond, torch.ones(rows, 19, dtype=torch.uint8, device='cuda'), ids.to(torch.int16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
def test_tangents_are_refused_not_lost(lib, grad):
    """Forward-mode derivatives are not there: a call with one among its inputs says so."""
    x, r = torch.randn(2, 6, 32, device='cuda').unbind()
    w, b = torch.randn(2, 32, device='cuda').unbind()
    logits, cond, masks, ids = _heads(6, 1)
    for n in range(4):
        with fwAD.dual_level():
            t = [v.clone().requires_grad_(grad) for v in (x, w, b, r)]
            t[n] = fwAD.make_dual(t[n], torch.ones_like(t[n]))
            with pytest.raises(RuntimeError, match='layer_norm: .*forward-mode'):
                layer_norm(*t[:3], residual=t[3])
    for n in (0, 4):
        with fwAD.dual_level():
            t = [v.clone().requires_grad_(grad) for v in (logits, *cond)]
            t[n] = fwAD.make_dual(t[n], torch.ones_like(t[n]))
            with pytest.raises(RuntimeError, match='moves_logp: .*forward-mode'):
                moves_logp(t[0], t[1:], masks, ids)
    assert layer_norm(x, w, b).shape == x.shape   # without one, as before
