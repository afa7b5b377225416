"""Draws at the ends of fp32's range (heads.sample, heads.sample_moves; csrc/heads.cuh): temperatures down to 1e-30 and logits
up to the type's lowest value, where one unit in a logit's last place is worth many temperatures or none. Every row has to be
answered, with the choice of the definition in whole numbers, which a plain program repeats exactly: fp32 differences and
expf, the rest whole numbers and fp64 comparisons. Its log-probability d - log(total 2^-27) is off by d's 3 roundings and the
logarithm's 4: (3 |d| + 8) 2^-24, and its own rounding 2^-24 of its size."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from actions import PARTS, unpack
from heads import _lib, sample, sample_moves

U = 2.0 ** -24
LOWEST = float(torch.finfo(torch.float32).min)
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


@pytest.fixture
def lib(gpu_lib_path):
    return _lib(gpu_lib_path)


def _whole(l, ok, u, T, k, p, mp):
    """(choice, log-probability in fp64, d) of each row of fp32 logits, from the definition of a draw; T: [rows] fp32."""
    n, width = l.shape
    one = torch.ones((), dtype=torch.float32, device=l.device)
    scale = one / T
    greedy = ~(T > 0) | torch.isinf(scale)
    scale = torch.where(greedy, one, scale)[:, None]
    first = torch.where(greedy, 1, k if k > 0 else width)[:, None]
    p, mp = float(np.float32(p)), float(np.float32(mp))
    lm = torch.where(ok, l, -torch.inf)
    d = torch.where(lm == lm.max(1, keepdim=True).values, 0.0, (lm - lm.max(1, keepdim=True).values) * scale)
    w = torch.where(ok, torch.round(torch.exp(d) * 2.0 ** 27), 0.0).long()
    order = lm.sort(dim=1, descending=True, stable=True).indices
    rank = torch.arange(width, device=l.device)
    ranked = w.gather(1, order) * (rank < first)
    run = ranked.cumsum(1)
    keep = (rank < first) & ((rank == 0) | (((run - ranked).double() < p * run[:, -1:].double()) & (ranked.double() >= mp * 2.0 ** 27)))
    w = w * torch.zeros_like(w).scatter_(1, order, keep.long())
    run = w.cumsum(1)
    target = ((u * 2.0 ** 24).long()[:, None] * run[:, -1:]) >> 24
    some = ok.any(1)
    c = torch.where(some, (run <= target).sum(1), 0)
    d = d.double().gather(1, c[:, None]).squeeze(1)
    return c, torch.where(some, d - torch.log(run[:, -1].double() * 2.0 ** -27), 0.0), torch.where(some, d, 0.0)


def _rows(rows, width, base, T, seed):
    """Logits from `base` upwards in up to 30 steps of a temperature each, or of one unit in the base's last place where that is
    more: weights of every size where the type has values between, and many ties where it has not."""
    g = torch.Generator().manual_seed(seed)
    at = np.float32(base if base else 1.0)
    unit = abs(float(at) - float(np.nextafter(at, np.float32(0))))
    step = max(T, unit)
    l = (base + torch.randint(0, 31, (rows, width), generator=g).double() * step).float()
    ok = torch.rand(rows, width, generator=g) < 0.8
    ok[torch.arange(rows), torch.randint(0, width, (rows,), generator=g)] = True
    return l, ok, torch.rand(rows, generator=g)


def _entry(lib, l, ok, u, T, k, p, mp):
    """sample by its C entry, into outputs that hold a marker first."""
    l, ok, u = l.contiguous(), None if ok is None else ok.contiguous(), u.contiguous()
    choice = torch.full((len(l),), -7, dtype=torch.int64, device='cuda')
    logp = torch.full((len(l),), 777.0, device='cuda')
    P = ctypes.c_void_p
    rc = lib.rl_sample(P(l.data_ptr()), l.shape[1], {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[l.dtype], l.shape[1],
                       P(ok.data_ptr() if ok is not None else None), l.shape[1], l.shape[1], P(u.data_ptr()), 1.0, k, p, mp,
                       P(T.data_ptr()), None, None, None, P(choice.data_ptr()), P(logp.data_ptr()), len(l),
                       P(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.rl_heads_error()
    return choice, logp


def _check(got, want, what):
    (c, lp), (wc, wl, d) = got, want
    assert torch.equal(c, wc), (what, int((c != wc).sum()), c[c != wc][:3].tolist(), wc[c != wc][:3].tolist())
    err, tol = (lp.double() - wl).abs(), (3 * d.abs() + 8) * U + U * wl.abs()
    assert bool((err <= tol).all()), (what, float((err - tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize('width', [5, 130, 324, 500, 1000, 2000, 4001])
@pytest.mark.parametrize('base', [0.0, 5.0, 600.0, 1e6, -1e9, LOWEST])
def test_every_row_is_answered(lib, width, base):
    for T in (0.0, 1e-30, 1e-8, 1e-6, 1e-4, 1e-3, 0.01, 1.0):
        l, ok, u = (t.cuda() for t in _rows(24, width, base, T, width + 3))
        each = torch.full((24,), T, device='cuda')
        for p in (0.5, 0.9, 1 - U):
            for k, mp in ((0, 0.0), (0, 0.02), (3, 0.0), (100, 0.0), (width // 2 + 1, 0.0)):
                want = _whole(l, ok, u, each, k, p, mp)
                _check(_entry(lib, l, ok, u, each, k, p, mp), want, (T, k, p, mp))
            _check(sample(l, u, ok, temperature=T, top_p=p), _whole(l, ok, u, each, 0, p, 0.0), (T, p))


@pytest.mark.gpu
def test_temperatures_of_each_row(lib):
    """1e-30 to 1e30, 0 and infinity side by side."""
    T = torch.tensor([0.0, 1e-39, 1e-38, 1e-30, 1e-8, 1e-6, 1e-3, 1.0, 1e3, 1e9, 1e30, 3e38, float('inf')]).repeat(20)
    for width in (5, 324, 1000, 2000, 4001):
        for base in (0.0, 600.0, -1e9, LOWEST):
            l, ok, u = (t.cuda() for t in _rows(len(T), width, base, 1e-6, width))
            each = T.cuda()
            for k, p in ((0, 0.9), (7, 0.9), (0, 1.0)):
                _check(sample(l, u, ok, temperature=each, top_k=k, top_p=p), _whole(l, ok, u, each, k, p, 0.0), (width, base, k, p))


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
def test_rows_masked_softly(lib, kind):
    """Every choice at -1e9 or at the type's lowest value, or but one: the run of the first choices that hold top_p, or that one."""
    dt = DT[kind]
    for value in (-1e9, float(torch.finfo(dt).min)):
        if abs(value) > torch.finfo(dt).max:
            continue
        for width in (4, 324, 700, 2500):
            l = torch.full((16, width), value, dtype=dt, device='cuda')
            l[8:, width // 3] = torch.arange(8, device='cuda').to(dt)
            u = torch.linspace(0, 0.999, 16, device='cuda')
            ones = torch.ones(16, device='cuda')
            for p in (0.25, 0.9):
                got = _entry(lib, l, None, u, ones, 0, p, 0.0)
                _check(got, _whole(l.float(), torch.ones_like(l, dtype=torch.bool), u, ones, 0, p, 0.0), (value, width, p))
                assert bool((got[0][8:] == width // 3).all()) and bool((got[0][:8] < p * width + 1).all())


@pytest.mark.gpu
def test_moves_at_small_temperatures(lib):
    """The ordered heads by the same definition, part by part."""
    g = torch.Generator().manual_seed(2)
    for T in (0.0, 1e-30, 1e-8, 1e-6, 1e-4, 0.01):
        for base in (0.0, 5.0, 600.0, 1e6, -1e9, LOWEST):
            l = _rows(400, 19, base, T, 7)[0].cuda()
            masks = (torch.rand(400, 19, generator=g) < 0.7).to(torch.uint8).cuda()
            u = torch.rand(400, 5, generator=g).cuda()
            each = torch.full((400,), T, device='cuda')
            for k, p, mp in ((0, 0.5, 0.0), (0, 0.9, 0.0), (2, 0.9, 0.1)):
                ids, lp = sample_moves(l, None, masks, u, temperature=T, top_k=k, top_p=p, min_p=mp)
                total, tol = torch.zeros(400, dtype=torch.float64, device='cuda'), 0.0
                for (a, b), c, v in zip(PARTS, unpack(ids), u.t()):
                    wc, wl, d = _whole(l[:, a:b], masks[:, a:b] != 0, v, each, k, p, mp)
                    assert torch.equal(c.long(), wc), (T, base, k, p, mp)
                    total, tol = total + wl, tol + (3 * d.abs() + 8) * U + 2 * U * wl.abs()
                assert bool(((lp.double() - total).abs() <= tol).all()), (T, base, k, p, mp)
