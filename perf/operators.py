"""The policy operators' measured cases: layer norm with its gradients, sampling of moves from given random numbers, and
the log-probability and entropy of given moves with their gradients.

Widths are the policy's (512 wide blocks, 19 mask bytes in five parts, 324 packed moves), counts are the rollout's (1
console, 64, 2,048 or 8,192 envs; 16 or 128 decisions per learner batch), and the other sizes are generic.

`run` computes the operators in plain torch operations (32 bits, rounded once), or, where `own` is true, by the calls a
user makes of ghostrun-lab_b200's norm.py and heads.py."""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

PARTS = [(0, 9), (9, 12), (12, 15), (15, 17), (17, 19)]   # the mask bytes of d-pad, A, B, Start, Select
RADIX = [9, 3, 3, 2, 2]
PAIRS = [(k, j) for k in range(5) for j in range(k)]      # a table of part k's logits for each choice of part j
SCALE = 2.0 ** 27                                         # a weight of 1 in the sampler's fixed point
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def norm(name, rows, width, dtype, *, train, residual, out=None):
    return dict(name=name, op='norm', rows=rows, width=width, dtype=dtype, train=train, residual=residual, out=out or dtype)


def moves(name, rows, dtype, temperature=1.0, per_row=False, top_k=0, top_p=1.0, min_p=0.0, empty=0.0):
    return dict(name=name, op='moves', rows=rows, dtype=dtype, temperature=temperature, per_row=per_row, top_k=top_k,
                top_p=top_p, min_p=min_p, empty=empty)


def flat(name, rows, width, dtype, temperature=1.0, per_row=False, top_k=0, top_p=1.0, min_p=0.0, empty=0.0):
    return dict(name=name, op='flat', rows=rows, width=width, dtype=dtype, temperature=temperature, per_row=per_row,
                top_k=top_k, top_p=top_p, min_p=min_p, empty=empty)


def logp(name, rows, dtype, empty=0.0):
    return dict(name=name, op='logp', rows=rows, dtype=dtype, empty=empty)


def listed():
    return [
        # one console played by the policy: the encoder's last norm, whose fp32 output feeds the GRU
        norm('norm, one console', 1, 512, 'bfloat16', train=False, residual=False, out='float32'),
        # a rollout decision of 8,192 envs: a block's output added to the stream and normed for the next block
        norm('norm, rollout', 8192, 512, 'bfloat16', train=False, residual=True),
        # a learner's minibatch, 256 envs x 16 decisions: forward and backward
        norm('norm, minibatch', 4096, 512, 'bfloat16', train=True, residual=True),
        # odd rows and an odd width in fp32, as a learner without mixed precision has them
        norm('norm, odd', 777, 1001, 'float32', train=True, residual=False),
        # a whole rollout of 8,192 envs x 128 decisions in one batch
        norm('norm, whole rollout', 8192 * 128, 512, 'bfloat16', train=True, residual=True),
        # the parity configuration's 64 envs choose their moves
        moves('moves, 64 envs', 64, 'float32'),
        # evaluation of 8,192 envs with every truncation on and a temperature of each env's own
        moves('moves, evaluation', 8191, 'float32', temperature=0.7, per_row=True, top_k=5, top_p=0.9, min_p=0.02),
        # moves of a whole rollout's decisions drawn again (8,192 envs x 128) from stored bf16 head outputs
        moves('moves, whole rollout', 8192 * 128, 'bfloat16'),
        # a learner's minibatch of the actions' log-probabilities and entropies, with gradients
        logp('logp, minibatch', 4096, 'float32'),
        logp('logp, whole rollout', 8192 * 128, 'float32'),
        # a flat head over the 324 packed moves, legal under the same 19 mask bytes, for 8,192 envs
        flat('flat, 324 moves', 8192, 324, 'bfloat16', temperature=0.9, top_p=0.95),
        # wide rows of an odd width with a mask byte for each choice
        flat('flat, wide', 2049, 4001, 'float32', top_k=50, top_p=0.9, min_p=0.001),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'moves', 'flat', 'logp'])
    dtype = rng.choice(sorted(TYPES))
    cut = dict(temperature=rng.choice([1.0, 0.5, 0.8, 1.3]), per_row=rng.random() < 0.3, top_k=rng.choice([0, 0, 2, 4]),
               top_p=rng.choice([1.0, 1.0, 0.5, 0.9]), min_p=rng.choice([0.0, 0.0, 0.01, 0.1]), empty=rng.choice([0.0, 0.02]))
    if op == 'norm':
        width = rng.choice([512, _log(rng, 33, 4096), 8 * _log(rng, 4, 512)])
        rows = _log(rng, 1, max(2, min(1 << 20, (1 << 28) // width)))
        case = norm('', rows, width, dtype, train=rng.random() < 0.6, residual=rng.random() < 0.5,
                    out=rng.choice([dtype, 'float32']))
    elif op == 'moves':
        case = moves('', _log(rng, 1, 1 << 20), dtype, **cut)
    elif op == 'logp':
        case = logp('', _log(rng, 1, 1 << 20), dtype, empty=cut['empty'])
    else:
        width = rng.choice([324, 324, _log(rng, 2, 4096)])
        cut['top_k'] = rng.choice([0, 0, 1, 20, 50])
        case = flat('', _log(rng, 1, min(1 << 18, (1 << 23) // width)), width, dtype, **cut)
    del case['name']
    return case


# ---------------------------------------------------------------- inputs

def _masks(rows, empty, g, dev):
    """Mask bytes as the env writes them: neutral always legal, a held button's part often down to one choice; a share
    `empty` of the rows has a part with nothing legal."""
    m = (torch.rand(rows, 19, generator=g, device=dev) < 0.65).to(torch.uint8)
    for a, b in PARTS:
        held = torch.rand(rows, generator=g, device=dev) < 0.2
        m[held, a + 1:b] = 0
        m[:, a] = 1
        m[torch.rand(rows, generator=g, device=dev) < empty, a:b] = 0
    return m


def _parts_of(ids):
    """The five choices of each packed id."""
    out, rest = [], ids.long()
    for n in RADIX:
        out.append(rest % n)
        rest = rest // n
    return out


def _cut(case, g, dev):
    """The sampling parameters: plain numbers, or a temperature for each row."""
    t = case['temperature']
    if case['per_row']:
        t = t * (0.5 + torch.rand(case['rows'], generator=g, device=dev))
    return dict(temperature=t, top_k=case['top_k'], top_p=case['top_p'], min_p=case['min_p'])


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    n, dt = case['rows'], TYPES[case['dtype']]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=dtype) * scale)

    if case['op'] == 'norm':
        d, out = case['width'], TYPES[case['out']]
        s = dict(case, x=normal(n, d, dtype=dt) + 0.25, weight=1 + normal(d, scale=0.1), bias=normal(d, scale=0.1),
                 r=normal(n, d, dtype=dt, scale=0.5) if case['residual'] else None)
        if case['train']:
            s['gy'] = normal(n, d, dtype=out)
            s['gs'] = normal(n, d, dtype=dt) if case['residual'] else None
        for k in ('x', 'weight', 'bias', 'r'):
            if s[k] is not None:
                s[k].requires_grad_(case['train'])
        return s
    if case['op'] == 'flat':
        w = case['width']
        s = dict(case, logits=normal(n, w, dtype=dt, scale=2.0), u=torch.rand(n, generator=g, device=dev))
        if w == 324:
            s['legal'] = _masks(n, case['empty'], g, dev)
        else:
            s['legal'] = (torch.rand(n, w, generator=g, device=dev) < 0.8).to(torch.uint8)
            s['legal'][torch.rand(n, generator=g, device=dev) < case['empty']] = 0
        s['cut'] = _cut(case, g, dev)
        return s
    s = dict(case, logits=normal(n, 19, dtype=dt, scale=1.5), masks=_masks(n, case['empty'], g, dev),
             cond=[normal(RADIX[j], RADIX[k], scale=0.5) for k, j in PAIRS])
    if case['op'] == 'moves':
        s['u'] = torch.rand(n, 5, generator=g, device=dev)
        s['cut'] = _cut(case, g, dev)
        return s
    # the moves that were made: a legal choice of each part (the neutral one where nothing is legal)
    ids, mult = torch.zeros(n, dtype=torch.int64, device=dev), 1
    for a, b in PARTS:
        pick = torch.rand(n, b - a, generator=g, device=dev) * s['masks'][:, a:b]
        ids += mult * pick.argmax(1)
        mult *= b - a
    s['ids'] = ids.to(torch.int16)
    s['glp'], s['gent'] = normal(n), torch.full((n,), -0.01, device=dev)
    s['logits'].requires_grad_(True)
    for t in s['cond']:
        t.requires_grad_(True)
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_norm(s):
    x = s['x'].detach()
    if s['r'] is not None:
        x = (x.float() + s['r'].detach().float()).to(x.dtype)   # the stream as it is kept
    x32, w, b = x.float(), s['weight'].detach(), s['bias'].detach()
    c = x32 - x32.mean(1, keepdim=True)
    r = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xh = c * r
    y = (xh * w + b).to(TYPES[s['out']])
    out = {'y': y} if s['r'] is None else {'y': y, 'sum': x}
    if s['train']:
        g = s['gy'].float()
        h = g * w
        dx = r * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
        if s['r'] is not None:
            dx = dx + s['gs'].float()
        out.update(dx=dx.to(x.dtype), dweight=(g * xh).sum(0), dbias=g.sum(0))
    return out


def _choose(l, legal, u, temperature, top_k, top_p, min_p):
    """One choice for each row of fp32 logits among its legal ones, and its log-probability. Weights are whole numbers
    (2^27 for the best choice), so their sums are the same in every order."""
    n, width = l.shape
    each = torch.is_tensor(temperature)                     # one for each row; else a number, in 32 bits as the rest
    by = (1.0 / temperature)[:, None] if each else float(np.float32(1) / np.float32(temperature))
    top_p, min_p = float(np.float32(top_p)), float(np.float32(min_p))
    lm = torch.where(legal, l, -math.inf)
    m = lm.max(1, keepdim=True).values
    d = torch.where(lm == m, 0.0, (lm - m) * by)
    w = torch.where(legal, torch.round(torch.exp(d) * SCALE), 0.0).long()
    if top_k > 0 or top_p < 1 or min_p > 0:
        order = lm.sort(dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        keep = (torch.arange(width, device=l.device) < (top_k if top_k > 0 else width)).expand(n, width)
        ws = ws * keep
        run = ws.cumsum(1)
        before, total = (run - ws).double(), run[:, -1:].double()
        first = torch.arange(width, device=l.device) == 0
        keep = keep & (first | (before < top_p * total)) & (first | (ws.double() >= min_p * SCALE))
        w = w * torch.zeros_like(legal).scatter_(1, order, keep)
    run = w.cumsum(1)
    total = run[:, -1:]
    target = ((u * 2.0 ** 24).long().reshape(-1, 1) * total) >> 24
    some = legal.any(1)
    c = torch.where(some, (run <= target).sum(1).clamp(max=width - 1), 0)
    lp = d.gather(1, c[:, None]).squeeze(1) - torch.log(total.squeeze(1).float() * 2.0 ** -27)
    return c, torch.where(some, lp, 0.0)


def _plain_moves(s):
    chosen, lp, ids, mult = [], None, 0, 1
    for k, (a, b) in enumerate(PARTS):
        l = s['logits'][:, a:b].float()
        for j in range(k):
            l = l + s['cond'][PAIRS.index((k, j))][chosen[j]]
        c, one = _choose(l, s['masks'][:, a:b] != 0, s['u'][:, k], **s['cut'])
        chosen.append(c)
        lp = one if lp is None else lp + one
        ids, mult = ids + c * mult, mult * (b - a)
    return {'ids': ids.to(torch.int16), 'logp': lp}


def _plain_flat(s):
    legal = s['legal'] != 0
    if s['width'] == 324:
        ids = torch.arange(324, device=legal.device)
        each = [legal[:, a:b][:, c] for (a, b), c in zip(PARTS, _parts_of(ids))]
        legal = each[0] & each[1] & each[2] & each[3] & each[4]
    c, lp = _choose(s['logits'].float(), legal, s['u'], **s['cut'])
    return {'choice': c, 'logp': lp}


def _plain_logp(s):
    logits, cond = s['logits'].detach().float(), [t.detach() for t in s['cond']]
    chosen = _parts_of(s['ids'])
    lp, ent, dl, dcond = 0.0, 0.0, [], []
    glp, gent = s['glp'][:, None], s['gent'][:, None]
    for k, (a, b) in enumerate(PARTS):
        l, legal, c = logits[:, a:b], s['masks'][:, a:b] != 0, chosen[k][:, None]
        for j in range(k):
            l = l + cond[PAIRS.index((k, j))][chosen[j]]
        some = legal.any(1, keepdim=True)
        lm = torch.where(legal, l, -math.inf)
        d = torch.where(legal, l - torch.where(some, lm.max(1, keepdim=True).values, 0.0), 0.0)
        w = torch.where(legal, torch.exp(d), 0.0)
        total = torch.where(some, w.sum(1, keepdim=True), 1.0)
        q = d - torch.log(total)                              # log p of the legal choices
        p = w / total
        h = -(p * q).sum(1, keepdim=True)
        lp = lp + torch.where(some, q.gather(1, c), 0.0)
        ent = ent + h
        hit = torch.arange(b - a, device=l.device) == c
        g = torch.where(legal, glp * (hit.float() - p) - gent * p * (q + h), 0.0)
        dl.append(g)
        for j in range(k):
            dcond.append(torch.nn.functional.one_hot(chosen[j], RADIX[j]).float().T @ g)
    return {'logp': lp.squeeze(1), 'entropy': ent.squeeze(1), 'dlogits': torch.cat(dl, 1).to(s['logits'].dtype),
            'dcond': dcond}


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    here = str(Path.cwd() / 'ghostrun-lab_b200')
    if here not in sys.path:
        sys.path.insert(0, here)
    if s['op'] == 'norm':
        from norm import layer_norm
        y = layer_norm(s['x'], s['weight'], s['bias'], eps=1e-5, residual=s['r'], out_dtype=TYPES[s['out']])
        if s['r'] is None:
            if not s['train']:
                return {'y': y}
            dx, dw, db = torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['gy'])
            return {'y': y, 'dx': dx, 'dweight': dw, 'dbias': db}
        y, total = y
        if not s['train']:
            return {'y': y, 'sum': total}
        dx, dr, dw, db = torch.autograd.grad((y, total), (s['x'], s['r'], s['weight'], s['bias']), (s['gy'], s['gs']))
        return {'y': y, 'sum': total, 'dx': dx, 'dweight': dw, 'dbias': db}
    from heads import moves_logp, sample, sample_moves
    if s['op'] == 'moves':
        ids, lp = sample_moves(s['logits'], s['cond'], s['masks'], s['u'], **s['cut'])
        return {'ids': ids, 'logp': lp}
    if s['op'] == 'flat':
        c, lp = sample(s['logits'], s['u'], legal=s['legal'], **s['cut'])
        return {'choice': c, 'logp': lp}
    lp, ent = moves_logp(s['logits'], s['cond'], s['masks'], s['ids'])
    grads = torch.autograd.grad((lp, ent), [s['logits'], *s['cond']], (s['glp'], s['gent']))
    return {'logp': lp, 'entropy': ent, 'dlogits': grads[0], 'dcond': list(grads[1:])}


def run(state):
    if own:
        return _own(state)
    return {'norm': _plain_norm, 'moves': _plain_moves, 'flat': _plain_flat, 'logp': _plain_logp}[state['op']](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    n, e = case['rows'], 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'norm':
        d, o = case['width'], 4 if case['out'] == 'float32' else 2
        streams = 2 if case['residual'] else 1
        b = n * d * (e * (1 + (2 if case['residual'] else 0)) + o) + 8 * d    # x (, r, sum), y, weight and bias
        f = 8 * n * d
        if case['train']:                                                   # gy (, gs), dx, dweight and dbias
            b += n * d * (o + e * streams) + 8 * d
            f += 14 * n * d
        return {'bytes': b, 'flops': f}
    if case['op'] == 'flat':
        mask = 19 if case['width'] == 324 else case['width']
        return {'bytes': n * (case['width'] * e + mask + 4 + 8 + 4 + (4 if case['per_row'] else 0)), 'flops': 10 * n * case['width']}
    if case['op'] == 'moves':
        return {'bytes': n * (19 * e + 19 + 20 + 2 + 4 + (4 if case['per_row'] else 0)), 'flops': 10 * 19 * n}
    return {'bytes': n * (2 * 19 * e + 19 + 2 + 8 + 8), 'flops': 25 * 19 * n}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'norm': _exact_norm, 'moves': _exact_moves, 'flat': _exact_flat, 'logp': _exact_logp}[case['op']](s)


def _exact_norm(s):
    x = s['x'].double()
    total = x if s['r'] is None else x + s['r'].double()
    x = total.to(s['x'].dtype).double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    std = (var + 1e-5).sqrt()
    z = (x - mean) / std
    out = {'y': torch.addcmul(s['bias'].double(), z, s['weight'].double())}
    if s['r'] is not None:
        out['sum'] = total
    if s['train']:
        # the row's Jacobian (I - 1/D - z z^T / D) / std applied to weight * gy
        gy = s['gy'].double()
        v = gy * s['weight'].double()
        along = torch.linalg.vecdot(v, z)[:, None] / x.shape[1]
        out['dx'] = (v - v.mean(1, keepdim=True) - z * along) / std + (0 if s['r'] is None else s['gs'].double())
        out['dweight'], out['dbias'] = torch.linalg.vecdot(gy, z, dim=0), gy.sum(0)
    return out


def _invert(l, legal, u, temperature, top_k, top_p, min_p):
    """The choice and its log-probability from the distribution's own definition: softmax, truncation of the ranked
    probabilities, inverse of the running sum."""
    t = torch.as_tensor(temperature, dtype=torch.float32, device=l.device).double().reshape(-1, 1)
    legal = legal | ~legal.any(1, keepdim=True)
    p = torch.softmax((l.masked_fill(~legal, -math.inf)) / t, 1)
    ranked, at = torch.sort(torch.where(legal, l, -math.inf), dim=1, descending=True, stable=True)
    q = p.gather(1, at)
    rank = torch.arange(l.shape[1], device=l.device)
    if top_k > 0:
        q = q.masked_fill(rank >= top_k, 0)
    q = q / q.sum(1, keepdim=True)
    mass = q.cumsum(1) - q
    q = q.masked_fill((mass >= top_p) & (rank > 0), 0)
    q = q.masked_fill(q < min_p * q[:, :1], 0)
    q = torch.zeros_like(q).scatter_(1, at, q / q.sum(1, keepdim=True))
    c = torch.searchsorted(q.cumsum(1), u.double()[:, None], right=True).clamp(max=l.shape[1] - 1)
    return c.squeeze(1), q.gather(1, c).log().squeeze(1)


def _exact_moves(s):
    lp, table, parts = 0.0, {kj: t.double() for kj, t in zip(PAIRS, s['cond'])}, []
    for k, (a, b) in enumerate(PARTS):
        legal = s['masks'][:, a:b].bool()
        l = s['logits'][:, a:b].double() + sum(table[k, j][c] for j, c in enumerate(parts))
        c, one = _invert(l, legal, s['u'][:, k], **s['cut'])
        some = legal.any(1)
        parts.append(c * some)
        lp = lp + torch.where(some, one, 0)
    return {'ids': None, 'logp': lp}


def _exact_flat(s):
    legal = s['legal'].bool()
    if s['width'] == 324:
        select, start, b, a, pad = (legal[:, lo:hi] for lo, hi in reversed(PARTS))
        legal = (select[:, :, None, None, None, None] & start[:, None, :, None, None, None] & b[:, None, None, :, None, None]
                 & a[:, None, None, None, :, None] & pad[:, None, None, None, None, :]).flatten(1)
    c, lp = _invert(s['logits'].double(), legal, s['u'], **s['cut'])
    return {'choice': None, 'logp': torch.where(legal.any(1), lp, 0)}


def _exact_logp(s):
    with torch.enable_grad():
        logits = s['logits'].detach().double().requires_grad_(True)
        cond = [t.detach().double().requires_grad_(True) for t in s['cond']]
        chosen, lp, ent = _parts_of(s['ids']), 0.0, 0.0
        for k, (a, b) in enumerate(PARTS):
            l = logits[:, a:b] + sum(cond[PAIRS.index((k, j))][chosen[j]] for j in range(k))
            legal = s['masks'][:, a:b].bool()
            some = legal.any(1)
            q = torch.log_softmax(l.masked_fill(~(legal | ~some[:, None]), -1e30), 1)
            lp = lp + torch.where(some, q.gather(1, chosen[k][:, None]).squeeze(1), 0)
            ent = ent - torch.where(some, (q.exp() * q.clamp(min=-1e3)).sum(1), 0)
        grads = torch.autograd.grad((lp, ent), [logits, *cond], (s['glp'].double(), s['gent'].double()))
    return {'logp': lp.detach(), 'entropy': ent.detach(), 'dlogits': grads[0], 'dcond': list(grads[1:])}
