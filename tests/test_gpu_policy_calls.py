"""What the policy operators' calls take and refuse beyond their values: forward-mode derivatives, whole numbers of
more than 32 bits, and CUDA graphs that hold both directions (norm.py, heads.py, csrc/policy_ops.cpp)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from heads import SIZES, TABLES, _lib, moves_logp, sample, sample_moves
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


@pytest.mark.gpu
def test_top_k_of_each_row_in_64_bits(lib):
    """A whole number past 31 bits is as large as it says: more than any row has, not what its low bits are."""
    g = torch.Generator(device='cuda').manual_seed(3)
    l = torch.randn(8, 50, generator=g, device='cuda')
    u = torch.rand(8, generator=g, device='cuda')
    k = torch.tensor([2 ** 32 + 1, 2 ** 32 + 5, 2 ** 31, 2 ** 33, 2 ** 63 - 1, -2 ** 32 + 1, -2 ** 63, 3], device='cuda')
    want = torch.tensor([50, 50, 50, 50, 50, 0, 0, 3], dtype=torch.int32, device='cuda')   # below 0: all, as 0
    assert all(torch.equal(a, b) for a, b in zip(sample(l, u, top_k=k), sample(l, u, top_k=want)))
    logits, cond, masks, _ = _heads(8, 4)
    v = torch.rand(8, 5, generator=g, device='cuda')
    got, ref = (sample_moves(logits, cond, masks, v, top_k=n) for n in (k, want))
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.gpu
def test_both_directions_in_a_graph(lib):
    """A captured step of the norm and the log-probabilities with their gradients, played again on new inputs: the bits of the
    same step outside the graph."""
    g = torch.Generator(device='cuda').manual_seed(5)
    x = torch.randn(600, 512, generator=g, device='cuda').bfloat16().requires_grad_(True)
    r = torch.randn(600, 512, generator=g, device='cuda').bfloat16().requires_grad_(True)
    w, b = (torch.randn(512, generator=g, device='cuda').requires_grad_(True) for _ in range(2))
    gy, gs = (torch.randn(600, 512, generator=g, device='cuda').bfloat16() for _ in range(2))
    logits, cond, masks, ids = _heads(600, 6)
    leaves = [t.requires_grad_(True) for t in (logits, *cond)]
    ga = torch.randn(600, generator=g, device='cuda')

    def step():
        out = layer_norm(x, w, b, residual=r)
        lp = moves_logp(leaves[0], leaves[1:], masks, ids)
        return [t.detach() for t in (*out, *lp)] + [*torch.autograd.grad(out, (x, w, b, r), (gy, gs)),
                                                    *torch.autograd.grad(lp, leaves, (ga, ga))]

    q = torch.cuda.Stream()
    q.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(q):
        step()
    torch.cuda.current_stream().wait_stream(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        for t in (x, r, w, b, gy, logits):
            t.mul_(0.75)
    graph.replay()
    want = step()
    assert all(torch.equal(a, c) for a, c in zip(held, want))
