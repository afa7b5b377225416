"""Moves sampled from given random numbers and the log-probability and entropy of given moves (heads.py, csrc/heads.cu)
against the distributions in fp64. Tolerances: a scaled difference d from the largest logit is off by 3 |d| 2^-24, and by 5 sums'
2^-24 |l| each where tables are added; exp and log by 4 2^-24 of their size, a weight by 2^-28; so a running sum is off by its
terms' share of that. A drawn choice has to be the one that the fp64 distribution gives, unless the random number, or a
truncation's threshold, lies within that distance of a boundary; fewer than 2 in 100 rows may."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from actions import PARTS, pack, unpack
from heads import SIZES, TABLES, _lib, moves_logp, sample, sample_moves

DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
U = 2.0 ** -24


@pytest.fixture
def lib(gpu_lib_path):
    return _lib(gpu_lib_path)


def _masks(rows, g, empty=0.0):
    m = (torch.rand(rows, 19, generator=g) < 0.6).to(torch.uint8)
    for a, b in PARTS:
        m[torch.arange(rows), a + torch.randint(0, b - a, (rows,), generator=g)] = 1
        m[torch.rand(rows, generator=g) < empty, a:b] = 0
    return m * torch.randint(1, 256, m.shape, generator=g, dtype=torch.int32).to(torch.uint8)


def _inputs(rows, seed, dt=torch.float32, empty=0.0, cond_dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, 19, generator=g) * 1.5).to(dt)
    cond = [(torch.randn(a, b, generator=g) * 0.5).to(cond_dt) for a, b in TABLES]
    return logits, cond, _masks(rows, g, empty), torch.rand(rows, 5, generator=g), g


def _draw64(l, legal, u, T=1.0, k=0, p=1.0, mp=0.0, sums=0):
    """(choice, log-probability, whether rounding could change it, tolerance) of one row, from the definition; sums: fp32
    additions that made a logit."""
    idx = np.flatnonzero(legal)
    if not len(idx):
        return 0, 0.0, False, 0.0
    T, p, mp = (float(np.float32(x)) for x in (T, p, mp))
    v = np.where(np.isnan(l), -np.inf, l)[idx].astype(np.float64)
    order = sorted(range(len(idx)), key=lambda i: (-v[i], i))
    if T <= 0:
        return int(idx[order[0]]), 0.0, False, 0.0
    with np.errstate(invalid='ignore'):
        d = np.where(v == v.max(), 0.0, (v - v.max()) / T)
    w = np.exp(d)
    finite = np.abs(v[np.isfinite(v)])
    add = sums * U * (float(finite.max()) if len(finite) else 0.0) / T
    off = w * ((3 * np.where(w > 0, -d, 0) + 4) * U + 2 * add) + 2.0 ** -28   # a weight's error
    near = False
    keep = order[:k] if k > 0 else order
    if sums and k > 0 and k < len(order):
        near |= abs(v[order[k - 1]] - v[order[k]]) < 4 * add * T
    total = w[keep].sum()
    tol = off[keep].sum() / total
    out, mass = [], 0.0
    for rank, i in enumerate(keep):
        near |= rank > 0 and p < 1 and abs(mass / total - p) < tol
        near |= rank > 0 and mp > 0 and abs(w[i] - mp) < off[i]
        if rank == 0 or (mass < p * total and w[i] >= mp):
            out.append(i)
        mass += w[i]
    out.sort()
    total, run, c = w[out].sum(), 0.0, None
    tol = off[out].sum() / total
    u = min(max(float(np.float32(u)), 0.0), 1 - U) if u == u else 0.0
    for n, i in enumerate(out):
        run += w[i]
        near |= n < len(out) - 1 and abs(run / total - u) < tol + U
        if c is None and run > u * total:
            c = i
    c = out[-1] if c is None else c
    return int(idx[c]), float(d[c] - math.log(total)), near, (3 * abs(d[c]) + 8) * U + 2 * add + tol


def _check_flat(logits, legal, u, choice, logp, cut=lambda row: {}):
    l, ok = logits.float().double().numpy(), legal.numpy()
    skipped = 0
    for row in range(len(l)):
        c, lp, near, tol = _draw64(l[row], ok[row], float(u[row]), **cut(row))
        if near:
            skipped += 1
            continue
        assert int(choice[row]) == c, (row, int(choice[row]), c)
        assert abs(float(logp[row]) - lp) <= tol + 2 * U * abs(lp), (row, float(logp[row]), lp, tol)
    assert skipped <= 0.02 * len(l) + 1, skipped


def _part_logits(logits, cond, parts, k):
    l = logits[:, PARTS[k][0]:PARTS[k][1]].float().double()
    for j in range(k):
        if cond is not None:
            l = l + cond[k * (k - 1) // 2 + j].float().double()[parts[j]]
    return l


def _check_moves(logits, cond, masks, u, ids, logp, cut=lambda row: {}):
    """Each part under the earlier parts as they were drawn."""
    parts = unpack(ids)
    assert torch.equal(pack(parts), ids)
    rows = len(ids)
    lp, tol, near = [0.0] * rows, [0.0] * rows, [False] * rows
    for k, (a, b) in enumerate(PARTS):
        l = _part_logits(logits, cond, parts, k).numpy()
        ok = masks[:, a:b].numpy() != 0
        for row in range(rows):
            c, one, close, t = _draw64(l[row], ok[row], float(u[row, k]), sums=5, **cut(row))
            near[row] |= close
            if not near[row]:
                assert int(parts[k][row]) == c, (row, k)
            lp[row] += one
            tol[row] += t + 2 * U * (abs(one) + abs(lp[row]))
    assert sum(near) <= 0.02 * rows + 1
    for row in range(rows):
        assert near[row] or abs(float(logp[row]) - lp[row]) <= tol[row], (row, float(logp[row]), lp[row])


CUTS = [dict(), dict(temperature=0.6), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.3),
        dict(temperature=1.7, top_k=3, top_p=0.8, min_p=0.1), dict(temperature=0.0), dict(top_p=0.0), dict(top_k=1),
        dict(top_k=100, top_p=2.0), dict(min_p=1.0)]
SHORT = {'temperature': 'T', 'top_k': 'k', 'top_p': 'p', 'min_p': 'mp'}


def _cut(c):
    short = {SHORT[n]: v for n, v in c.items()}
    return lambda row: short


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows', [1, 31, 129, 700])
def test_moves(lib, rows, kind):
    for n, c in enumerate(CUTS if rows == 129 else CUTS[:1] + CUTS[5:6]):
        logits, cond, masks, u, _ = _inputs(rows, rows * 31 + n, DT[kind], empty=0.05)
        ids, logp = sample_moves(logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda(), **c)
        assert ids.dtype == torch.int16 and logp.dtype == torch.float32
        _check_moves(logits, cond, masks, u, ids.cpu(), logp.cpu(), _cut(c))


@pytest.mark.gpu
def test_moves_without_tables_and_with_tables_of_other_types(lib):
    logits, cond, masks, u, _ = _inputs(200, 9, cond_dt=torch.bfloat16)
    ids, logp = sample_moves(logits.cuda(), None, masks.cuda(), u.cuda())
    _check_moves(logits, None, masks, u, ids.cpu(), logp.cpu())
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        c = [t.to(dt) for t in cond]
        ids, logp = sample_moves(logits.cuda(), [t.cuda() for t in c], masks.cuda(), u.cuda())
        _check_moves(logits, c, masks, u, ids.cpu(), logp.cpu())


@pytest.mark.gpu
def test_moves_parameters_of_each_row(lib):
    logits, cond, masks, u, g = _inputs(300, 10)
    T = torch.rand(300, generator=g) * 2
    T[::7] = 0
    k = torch.randint(0, 5, (300,), generator=g)
    p, mp = torch.rand(300, generator=g), torch.rand(300, generator=g) * 0.4
    ids, logp = sample_moves(logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda(), T.cuda(), k.cuda(), p.cuda(),
                             mp.cuda())
    _check_moves(logits, cond, masks, u, ids.cpu(), logp.cpu(),
                 lambda row: dict(T=float(T[row]), k=int(k[row]), p=float(p[row]), mp=float(mp[row])))
    f = torch.rand(300, generator=g)
    flat, ok = torch.randn(300, 50, generator=g), torch.ones(300, 50, dtype=torch.bool)
    c, lp = sample(flat.cuda(), f.cuda(), None, T.cuda(), k.cuda(), p.cuda(), mp.cuda())
    _check_flat(flat, ok, f, c.cpu(), lp.cpu(),
                lambda row: dict(T=float(T[row]), k=int(k[row]), p=float(p[row]), mp=float(mp[row])))


@pytest.mark.gpu
def test_moves_of_a_large_batch_are_those_of_its_pieces(lib):
    logits, cond, masks, u, _ = _inputs(70001, 11, torch.bfloat16)
    lc, cc, mc, uc = logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda()
    ids, logp = sample_moves(lc, cc, mc, uc)
    for a, b in ((0, 1), (1, 40), (40, 30000), (30000, 70001)):
        i, p = sample_moves(lc[a:b], cc, mc[a:b], uc[a:b])
        assert torch.equal(i, ids[a:b]) and torch.equal(p, logp[a:b])
    _check_moves(logits[-200:], cond, masks[-200:], u[-200:], ids[-200:].cpu(), logp[-200:].cpu())


@pytest.mark.gpu
def test_masked_places_hold_anything(lib):
    logits, cond, masks, u, g = _inputs(400, 12)
    want = sample_moves(logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda(), top_p=0.9)
    lw = moves_logp(logits.cuda(), [t.cuda() for t in cond], masks.cuda(), want[0])
    for bad in (float('nan'), float('inf'), float('-inf'), torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        l = torch.where(masks != 0, logits, torch.tensor(bad))
        got = sample_moves(l.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda(), top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a = l.cuda().requires_grad_(True)
        lp, ent = moves_logp(a, [t.cuda() for t in cond], masks.cuda(), want[0])
        assert torch.equal(lp, lw[0]) and torch.equal(ent, lw[1])
        d, = torch.autograd.grad(lp.sum() + ent.sum(), [a])
        assert bool(torch.isfinite(d).all()) and not d[(masks == 0).cuda()].any()
    flat = torch.randn(64, 70, generator=g)
    ok = torch.rand(64, 70, generator=g) < 0.5
    ok[:, 3] = True
    f = torch.rand(64, generator=g)
    want = sample(flat.cuda(), f.cuda(), ok.cuda(), top_k=9)
    for bad in (float('nan'), float('inf'), float('-inf')):
        got = sample(torch.where(ok, flat, torch.tensor(bad)).cuda(), f.cuda(), ok.cuda(), top_k=9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_infinite_and_nan_logits_among_the_legal(lib):
    inf = math.inf
    rows = torch.tensor([[-inf, -inf, -inf, -inf], [1.0, -inf, 2.0, -inf], [inf, 0.0, inf, 1.0], [-0.0, 0.0, -0.0, 0.0],
                         [math.nan, 1.0, 0.0, -inf], [math.nan] * 4, [5.0, 5.0, 5.0, 5.0]])
    u = torch.tensor([0.6, 0.5, 0.9, 0.3, 0.1, 0.6, 0.26])
    for k in (0, 1, 3):
        c, lp = sample(rows.cuda(), u.cuda(), top_k=k)
        c, lp = c.cpu(), lp.cpu()
        for i in range(7):
            want, one, _, _ = _draw64(rows[i].double().numpy(), np.ones(4, bool), float(u[i]), k=k)
            assert int(c[i]) == want, (i, k, int(c[i]), want)
            if i in (4, 5):
                assert math.isnan(float(lp[i]))
            else:
                assert abs(float(lp[i]) - one) < 4 * U * 4
    # the same through the parts: all choices of a part alike
    logits = torch.zeros(3, 19)
    logits[0], logits[1], logits[2, 4] = -inf, inf, math.nan
    ids, lp = sample_moves(logits.cuda(), None, torch.ones(3, 19, dtype=torch.uint8).cuda(), torch.full((3, 5), 0.5).cuda())
    parts = unpack(ids.cpu())
    assert [int(q[0]) for q in parts] == [4, 1, 1, 1, 1] == [int(q[1]) for q in parts]
    assert abs(float(lp[0]) + math.log(324)) < 1e-5 and math.isnan(float(lp[2]))


@pytest.mark.gpu
def test_random_numbers_at_the_ends(lib):
    logits = torch.zeros(6, 19)
    u = torch.tensor([0.0, 1 - U, 1.0, -3.0, math.nan, 7.0])[:, None].expand(6, 5).contiguous()
    ids, _ = sample_moves(logits.cuda(), None, torch.ones(6, 19, dtype=torch.uint8).cuda(), u.cuda())
    assert ids.cpu().tolist() == [0, 323, 323, 0, 0, 323]
    c, _ = sample(torch.zeros(6, 5).cuda(), u[:, 0].contiguous().cuda())
    assert c.cpu().tolist() == [0, 4, 4, 0, 0, 4]


WIDTHS = [1, 2, 3, 19, 31, 32, 33, 101, 128, 129, 255, 324, 511, 512, 513, 1000, 1024, 1025, 2047, 2049, 4095, 4096]


@pytest.mark.gpu
@pytest.mark.parametrize('width', WIDTHS)
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
def test_rows(lib, width, kind):
    rows = 40 if width > 600 else 90
    for n, c in enumerate([dict(), dict(temperature=0.8, top_k=7), dict(top_p=0.7), dict(top_k=20, top_p=0.9, min_p=0.05),
                           dict(temperature=0.0), dict(min_p=0.2)]):
        g = torch.Generator().manual_seed(width * 13 + n)
        logits = (torch.randn(rows, width, generator=g) * 2).to(DT[kind])
        ok = torch.rand(rows, width, generator=g) < 0.8
        ok[torch.rand(rows, generator=g) < 0.05] = False
        u = torch.rand(rows, generator=g)
        choice, logp = sample(logits.cuda(), u.cuda(), ok.cuda(), **c)
        assert choice.dtype == torch.int64 and logp.dtype == torch.float32
        _check_flat(logits, ok, u, choice.cpu(), logp.cpu(), _cut(c))


@pytest.mark.gpu
def test_rows_with_many_equal_logits(lib):
    """Ties decide: equal logits stay or go by their index."""
    g = torch.Generator().manual_seed(5)
    for width in (40, 324, 700, 2500):
        logits = torch.randint(0, 4, (60, width), generator=g).float()
        ok = torch.rand(60, width, generator=g) < 0.7
        u = torch.rand(60, generator=g)
        for c in (dict(top_k=3), dict(top_k=width // 3), dict(top_p=0.37), dict(top_k=width // 2, top_p=0.61)):
            choice, logp = sample(logits.cuda(), u.cuda(), ok.cuda(), **c)
            _check_flat(logits, ok, u, choice.cpu(), logp.cpu(), _cut(c))


@pytest.mark.gpu
def test_flat_moves_under_the_mask_bytes(lib):
    g = torch.Generator().manual_seed(21)
    logits = torch.randn(300, 324, generator=g).bfloat16()
    masks = _masks(300, g, empty=0.02)
    u = torch.rand(300, generator=g)
    parts = unpack(torch.arange(324))
    ok = torch.stack([masks[:, a:b][:, c] != 0 for (a, b), c in zip(PARTS, parts)]).all(0)
    choice, logp = sample(logits.cuda(), u.cuda(), masks.cuda(), top_p=0.9)
    _check_flat(logits, ok, u, choice.cpu(), logp.cpu(), _cut(dict(top_p=0.9)))
    again = sample(logits.cuda(), u.cuda(), ok.cuda(), top_p=0.9)
    assert torch.equal(again[0], choice) and torch.equal(again[1], logp)


@pytest.mark.gpu
def test_strides_and_empty_batches(lib):
    logits, cond, masks, u, g = _inputs(90, 14)
    cc = [t.cuda() for t in cond]
    want = sample_moves(logits.cuda(), cc, masks.cuda(), u.cuda())
    lw = moves_logp(logits.cuda(), cc, masks.cuda(), want[0])
    wide = torch.full((90, 40), math.nan, device='cuda')
    wide[:, 3:22] = logits.cuda()
    wm = torch.zeros(90, 23, dtype=torch.uint8, device='cuda')
    wm[:, 1:20] = masks.cuda()
    wu = torch.zeros(90, 8, device='cuda')
    wu[:, 2:7] = u.cuda()
    got = sample_moves(wide[:, 3:22], [t.t().contiguous().t() for t in cc], wm[:, 1:20], wu[:, 2:7])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = sample_moves(logits.cuda().t().contiguous().t(), cc, masks.cuda().t().contiguous().t(), u.cuda())
    assert torch.equal(got[0], want[0])
    lp, ent = moves_logp(wide[:, 3:22], cc, wm[:, 1:20].bool(), want[0])
    assert torch.equal(lp, lw[0]) and torch.equal(ent, lw[1])
    one = sample_moves(logits[:1].cuda().expand(90, 19), cc, masks[:1].cuda().expand(90, 19), u.cuda())
    assert torch.equal(one[0][0], want[0][0])
    f = torch.rand(30, generator=g).cuda()
    x = torch.randn(30, 101, generator=g).cuda()
    c, p = sample(x, f, top_k=11)
    w2 = torch.full((30, 150), math.nan, device='cuda')
    for off in (0, 1, 4):
        w2[:, off:off + 101] = x
        c2, p2 = sample(w2[:, off:off + 101], f, top_k=11)
        assert torch.equal(c, c2) and torch.equal(p, p2)
    ids, lp = sample_moves(logits[:0].cuda(), cc, masks[:0].cuda(), u[:0].cuda())
    assert ids.shape == lp.shape == (0,)
    assert sample(x[:0], f[:0])[0].shape == (0,)
    e = logits[:0].cuda().requires_grad_(True)
    t = [q.clone().requires_grad_(True) for q in cc]
    lp, ent = moves_logp(e, t, masks[:0].cuda(), ids)
    (lp.sum() + ent.sum()).backward()
    assert e.grad.shape == (0, 19) and not t[0].grad.any()


# ---------------------------------------------------------------- log-probability, entropy and gradients

def _logp64(logits, cond, masks, ids):
    chosen, lp, ent = unpack(ids), 0.0, 0.0
    for k, (a, b) in enumerate(PARTS):
        l = logits[:, a:b]
        for j in range(k):
            if cond is not None:
                l = l + cond[k * (k - 1) // 2 + j][chosen[j]]
        ok = masks[:, a:b] != 0
        some = ok.any(1)
        q = torch.log_softmax(l.masked_fill(~ok & some[:, None], -1e300), 1)
        lp = lp + torch.where(some, q.gather(1, chosen[k][:, None]).squeeze(1), 0.0)
        ent = ent - torch.where(some, (q.exp() * q.clamp(min=-1e4)).sum(1), 0.0)
    return lp, ent


def _legal_ids(masks, g):
    parts = [(torch.rand(len(masks), b - a, generator=g) * (masks[:, a:b] != 0)).argmax(1) for a, b in PARTS]
    return pack(parts)


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows', [1, 2, 33, 500, 3001])
def test_logp_and_gradients(lib, rows, kind):
    """fp32 softmax over at most 9 choices of logits up to 16: 12 (16 + 1) 2^-24 per part; the gradients the same of the
    incoming gradients' size, their rows' type's rounding, and (rows / 32 + 64) 2^-24 of the summed terms for the tables."""
    dt = DT[kind]
    logits, cond, masks, _, g = _inputs(rows, rows + 5, dt, empty=0.05)
    ids = _legal_ids(masks, g)
    ga, gb = torch.randn(rows, generator=g), torch.randn(rows, generator=g) * 0.1
    a = logits.cuda().requires_grad_(True)
    t = [q.cuda().requires_grad_(True) for q in cond]
    lp, ent = moves_logp(a, t, masks.cuda(), ids.cuda())
    grads = torch.autograd.grad((lp, ent), [a, *t], (ga.cuda(), gb.cuda()))
    a64 = logits.double().requires_grad_(True)
    t64 = [q.double().requires_grad_(True) for q in cond]
    lp64, ent64 = _logp64(a64, t64, masks, ids)
    refs = torch.autograd.grad((lp64, ent64), [a64, *t64], (ga.double(), gb.double()))
    part = 12 * 17 * U
    assert ((lp.cpu().double() - lp64).abs() <= 5 * part).all()
    assert ((ent.cpu().double() - ent64).abs() <= 5 * part).all()
    size = (ga.abs() + 20 * gb.abs()).double()
    unit = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dt]
    tol = unit * refs[0].abs() + (part * size)[:, None] + (2.0 ** -25 if dt == torch.float16 else 0)
    assert ((grads[0].cpu().double() - refs[0]).abs() <= tol).all()
    bound = float((size * (part + (rows / 32 + 64) * U)).sum())
    for got, ref in zip(grads[1:], refs[1:]):
        assert ((got.cpu().double() - ref).abs() <= bound).all()
    again = torch.autograd.grad(moves_logp(a, t, masks.cuda(), ids.cuda()), [a, *t], (ga.cuda(), gb.cuda()))
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.gpu
def test_logp_of_sampled_moves(lib):
    """Without truncation the sampler's log-probability is the one that is trained: both to (5 parts) 12 * 17 * 2^-24."""
    logits, cond, masks, u, _ = _inputs(4000, 31, empty=0.02)
    cc = [t.cuda() for t in cond]
    ids, lp = sample_moves(logits.cuda(), cc, masks.cuda(), u.cuda())
    again, _ = moves_logp(logits.cuda(), cc, masks.cuda(), ids)
    assert float((lp - again).abs().max()) <= 2 * 5 * 12 * 17 * U


@pytest.mark.gpu
def test_gradient_against_differences(lib):
    """Central differences of sum(a logp + b entropy) in fp32 with h = 2^-6: 2 x 200 values rounding to 12 * 17 * 2^-24 at random
    over 2 h, and h^2 / 6 of third derivatives below 2 per row and unit of direction."""
    rows, h = 200, 2.0 ** -6
    logits, cond, masks, _, g = _inputs(rows, 41)
    ids = _legal_ids(masks, g).cuda()
    ga, gb = torch.randn(rows, generator=g).double(), torch.randn(rows, generator=g).double()
    v = torch.randn(rows, 19, generator=g)
    vt = [torch.randn(s, generator=g) for s in TABLES]
    a = logits.cuda().requires_grad_(True)
    t = [q.cuda().requires_grad_(True) for q in cond]
    lp, ent = moves_logp(a, t, masks.cuda(), ids)
    grads = torch.autograd.grad((lp, ent), [a, *t], (ga.float().cuda(), gb.float().cuda()))

    def f(s):
        lp, ent = moves_logp((logits + s * v).cuda(), [(q + s * d).cuda() for q, d in zip(cond, vt)], masks.cuda(), ids)
        return float((lp.cpu().double() * ga + ent.cpu().double() * gb).sum())

    want = (f(h) - f(-h)) / (2 * h)
    got = sum(float((x.cpu().double() * d.double()).sum()) for x, d in zip(grads, [v, *vt]))
    # a direction moves a logit by up to 5 terms of size 1; a third derivative grows as its cube
    tol = (2 * rows) ** 0.5 * 12 * 17 * U / (2 * h) + h * h / 6 * 2 * 5 ** 1.5 * (5 * rows) ** 0.5 * 4
    assert abs(got - want) < tol, (got, want, tol)


@pytest.mark.gpu
def test_logp_edges(lib):
    logits, cond, masks, _, g = _inputs(6, 51)
    masks[:] = 1
    masks[1, 0] = 0           # the move's d-pad choice is not legal
    masks[2, 9:12] = 0        # nothing legal for A
    ids = torch.tensor([5, 9, 200, 324, -1, 323], dtype=torch.int16)
    a = logits.cuda().requires_grad_(True)
    t = [q.cuda().requires_grad_(True) for q in cond]
    lp, ent = moves_logp(a, t, masks.cuda(), ids.cuda())
    assert float(lp[1]) == -math.inf and bool(torch.isfinite(ent[:3]).all()) and bool(torch.isfinite(lp[[0, 2, 5]]).all())
    assert bool(lp[3:5].isnan().all()) and bool(ent[3:5].isnan().all())
    grads = torch.autograd.grad((lp, ent), [a, *t], (torch.ones(6, device='cuda'), torch.ones(6, device='cuda')))
    assert all(bool(torch.isfinite(q).all()) for q in grads)
    assert not grads[0][3:5].any() and not grads[0][2, 9:12].any() and float(grads[0][1, 0]) == 0
    # only one of the two outputs used; gradients that are one number repeated; leaves one at a time; no tables
    b = logits.cuda().requires_grad_(True)
    lp, ent = moves_logp(b, None, masks[:1].expand(6, 19).cuda(), torch.zeros(6, dtype=torch.int16).cuda())
    ent.mean().backward()
    ref = logits.double().requires_grad_(True)
    _logp64(ref, None, torch.ones(6, 19), torch.zeros(6, dtype=torch.int16))[1].mean().backward()
    assert torch.allclose(b.grad.cpu().double(), ref.grad, rtol=0, atol=1e-6)
    good = torch.zeros(6, dtype=torch.int16).cuda()
    ones = torch.ones(6, 19, dtype=torch.uint8).cuda()
    want = torch.autograd.grad(moves_logp(a, t, ones, good)[0].sum(), [a, *t])
    for n in (0, 3, 10):
        leaves = [q.detach().clone() for q in (a, *t)]
        leaves[n].requires_grad_(True)
        got, = torch.autograd.grad(moves_logp(leaves[0], leaves[1:], ones, good)[0].sum(), [leaves[n]])
        assert torch.equal(got, want[n])
    d, = torch.autograd.grad(moves_logp(a, t, ones, good)[0].sum(), [a], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph(lib):
    logits, cond, masks, u, g = _inputs(3000, 61)
    lc, cc, mc, uc = logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda()
    want = sample_moves(lc, cc, mc, uc, top_p=0.8)
    flat, f = torch.randn(3000, 324, generator=g).cuda(), torch.rand(3000, generator=g).cuda()
    wf = sample(flat, f, mc, top_k=40)
    q = torch.cuda.Stream()
    q.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(q):
        got = sample_moves(lc, cc, mc, uc, top_p=0.8)
        gf = sample(flat, f, mc, top_k=40)
    torch.cuda.current_stream().wait_stream(q)
    assert all(torch.equal(x, y) for x, y in zip((*want, *wf), (*got, *gf)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_moves(lc, cc, mc, uc, top_p=0.8)
        gf = sample(flat, f, mc, top_k=40)
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip((*want, *wf), (*got, *gf)))


@pytest.mark.gpu
def test_refusals(lib):
    logits, cond, masks, u, _ = _inputs(8, 71)
    l, c, m, v = logits.cuda(), [t.cuda() for t in cond], masks.cuda(), u.cuda()
    ids = torch.zeros(8, dtype=torch.int16, device='cuda')
    for args, kw in (((l[:, :18], c, m, v), {}), ((l.double(), c, m, v), {}), ((l, c[:9], m, v), {}), ((l, c[::-1], m, v), {}),
                     ((l, [*c[:9], c[9].half()], m, v), {}), ((l, c, m[:7], v), {}), ((l, c, m.float(), v), {}),
                     ((l, c, m, v.double()), {}), ((l, c, m, v[:, :4]), {}), ((l, c, m, v), dict(temperature=-1.0)),
                     ((l, c, m, v), dict(temperature=math.nan)), ((l, c, m, v), dict(top_k=-1)), ((l, c, m, v), dict(top_k=1.5)),
                     ((l, c, m, v), dict(min_p=1.5)), ((l, c, m, v), dict(top_p=-0.1)), ((l, c, m, v), dict(top_p=v[:7, 0])),
                     ((l, c, m, v), dict(top_k=v[:, 0])), ((l, c, m.cpu(), v), {}), ((l, c, m, v), dict(top_p=v[:, 0].cpu())),
                     ((l, [t.cpu() for t in c], m, v), {})):
        with pytest.raises(RuntimeError, match='sample_moves'):
            sample_moves(*args, **kw)
    for args in ((l[:, :18], c, m, ids), (l, c[:9], m, ids), (l, c, m[:7], ids), (l, c, m, ids.long()), (l, c, m, ids[:7]),
                 (l, c, m, ids.cpu())):
        with pytest.raises(RuntimeError, match='moves_logp'):
            moves_logp(*args)
    for args in ((torch.zeros(2, 4097, device='cuda'), v[:2, 0]), (torch.zeros(2, 0, device='cuda'), v[:2, 0]),
                 (l, v[:, 0], m[:, :18]), (l, v[:7, 0]), (torch.zeros(8, 320, device='cuda'), v[:, 0], m), (l[0], v[:, 0])):
        with pytest.raises(RuntimeError, match='sample'):
            sample(*args)


def test_refuses_the_cpu():
    logits, cond, masks, u, _ = _inputs(2, 81)
    with pytest.raises(RuntimeError, match='GPU only'):
        sample_moves(logits, cond, masks, u)
    with pytest.raises(RuntimeError, match='GPU only'):
        sample(logits, u[:, 0])
    with pytest.raises(RuntimeError, match='GPU only'):
        moves_logp(logits, cond, masks, torch.zeros(2, dtype=torch.int16))


def test_c_entry_refusals():
    """Bad arguments come back as an error and a message before anything is launched (no GPU needed)."""
    import build
    lib = _lib(build.build())
    one, none8 = ctypes.c_void_p(16), [None] * 4

    def moves(logits=one, type=0, rows=1, T=1.0, k=0, p=1.0, m=0.0, cond=None):
        return lib.rl_moves_sample(logits, 19, type, cond, 0, one, 19, one, T, k, p, m, *none8, one, one, rows, None)

    def rows_(width=5, legal=None, lw=0, rows=1, logits=one, T=1.0):
        return lib.rl_sample(logits, width, 0, width, legal, width, lw, one, T, 0, 1.0, 0.0, *none8, one, one, rows, None)

    gaps = (ctypes.c_void_p * 10)(*([16] * 9))
    for rc in (moves(logits=None), moves(type=3), moves(rows=-1), moves(T=-1.0), moves(T=math.nan), moves(p=-1.0), moves(m=2.0),
               moves(cond=gaps), rows_(width=0), rows_(width=4097), rows_(legal=one, lw=19), rows_(rows=-1), rows_(logits=None),
               rows_(T=-0.5),
               lib.rl_moves_logp(None, 19, 0, None, 0, one, 19, one, one, one, 1, None),
               lib.rl_moves_logp_bwd(one, 1, one, 1, one, 19, 0, None, 0, one, 19, one, one, one, 1, one, 0, None),
               lib.rl_moves_logp_bwd(one, 1, one, 1, one, 19, 0, None, 0, one, 19, one, one, None, 0, None, 0, None)):
        assert rc != 0 and lib.rl_heads_error()
    assert moves(rows=0) == 0 and rows_(rows=0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fp32', 'bf16'])
def test_gradients_of_a_large_batch(lib, kind):
    """More rows than one batch per block: the logits' gradients first without the tables', then with them, equal row by row
    to a small batch's; the tables' to (rows / 32 + 64) 2^-24 of the summed terms."""
    rows = 90001
    logits, cond, masks, _, g = _inputs(rows, 91, DT[kind], empty=0.01)
    ids = _legal_ids(masks, g)
    ga, gb = torch.randn(rows, generator=g), torch.randn(rows, generator=g) * 0.1
    mc, ic, gc = masks.cuda(), ids.cuda(), (ga.cuda(), gb.cuda())
    fixed = [q.cuda() for q in cond]
    a = logits.cuda().requires_grad_(True)
    alone, = torch.autograd.grad(moves_logp(a, fixed, mc, ic), [a], gc)
    t = [q.clone().requires_grad_(True) for q in fixed]
    grads = torch.autograd.grad(moves_logp(a, t, mc, ic), [a, *t], gc)
    assert torch.equal(grads[0], alone)
    for lo, hi in ((0, 300), (44000, 44511), (89800, rows)):
        b = logits[lo:hi].cuda().requires_grad_(True)
        part, = torch.autograd.grad(moves_logp(b, fixed, mc[lo:hi], ic[lo:hi]), [b], (gc[0][lo:hi], gc[1][lo:hi]))
        assert torch.equal(part, alone[lo:hi])
    a64, t64 = logits.double().requires_grad_(True), [q.double().requires_grad_(True) for q in cond]
    refs = torch.autograd.grad(_logp64(a64, t64, masks, ids), [a64, *t64], (ga.double(), gb.double()))
    bound = float(((ga.abs() + 20 * gb.abs()).double() * 12 * 17 * U).sum()) + (rows / 32 + 64) * U * rows ** 0.5 * 4
    for got, ref in zip(grads[1:], refs[1:]):
        assert float((got.cpu().double() - ref).abs().max()) <= bound


@pytest.mark.gpu
def test_offsets_past_32_bits(lib):
    """113,100,000 rows of 19 and 6,630,000 rows of 324 are more than 2^31 values: their last rows are those of a batch of their
    own, bit for bit, forward and backward."""
    g = torch.Generator(device='cuda').manual_seed(3)
    rows = 113_100_000
    cond = [torch.randn(s, generator=g, device='cuda') for s in TABLES]
    logits = torch.randn(rows, 19, generator=g, device='cuda', dtype=torch.bfloat16).requires_grad_(True)
    masks = torch.randint(0, 2, (rows, 19), generator=g, device='cuda', dtype=torch.uint8)
    u = torch.rand(rows, 5, generator=g, device='cuda')
    ids, logp = sample_moves(logits.detach(), cond, masks, u, top_k=4)
    cut = slice(rows - 2000, rows)
    few = sample_moves(logits.detach()[cut].clone(), cond, masks[cut].clone(), u[cut].clone(), top_k=4)
    assert torch.equal(ids[cut], few[0]) and torch.equal(logp[cut], few[1])
    lp, ent = moves_logp(logits, cond, masks, ids)
    one = torch.ones(1, device='cuda').expand(rows)
    d, = torch.autograd.grad((lp, ent), [logits], (one, one))
    t = logits.detach()[cut].clone().requires_grad_(True)
    lt, et = moves_logp(t, cond, masks[cut].clone(), ids[cut].clone())
    assert torch.equal(lp[cut], lt) and torch.equal(ent[cut], et)
    assert torch.equal(d[cut], torch.autograd.grad((lt, et), [t], (one[cut], one[cut]))[0])
    del logits, masks, u, ids, logp, lp, ent, d
    rows = 6_630_000
    cut = slice(rows - 2000, rows)
    logits = torch.randn(rows, 324, generator=g, device='cuda', dtype=torch.bfloat16)
    masks = torch.randint(0, 2, (rows, 19), generator=g, device='cuda', dtype=torch.uint8)
    u = torch.rand(rows, generator=g, device='cuda')
    c, p = sample(logits, u, masks, top_p=0.9)
    few = sample(logits[cut].clone(), u[cut].clone(), masks[cut].clone(), top_p=0.9)
    assert torch.equal(c[cut], few[0]) and torch.equal(p[cut], few[1])
