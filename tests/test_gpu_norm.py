"""Layer norm with its residual sum and gradients (norm.layer_norm, csrc/norm.cu) against the formulas in fp64, and its
gradients against differences. Tolerances: a value summed over D fp32 terms, D / 32 of them in a row in one lane, is off by at
most (D / 32 + 40) 2^-24 of the terms' mean size; a row whose mean is many deviations away loses as many times more; an
output rounds once to its type (2^-24 fp32, 2^-11 fp16, 2^-8 bf16 of its size)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from norm import _lib, layer_norm

DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EPS = 1e-5


@pytest.fixture
def lib(gpu_lib_path):
    return _lib(gpu_lib_path)


def _inputs(rows, width, dt, seed, residual=True, w_dt=torch.float32, mean=0.25):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=g) + mean).to(dt)
    r = (torch.randn(rows, width, generator=g) * 0.5).to(dt) if residual else None
    w = (1 + 0.2 * torch.randn(width, generator=g)).to(w_dt)
    b = (0.2 * torch.randn(width, generator=g)).to(w_dt)
    return x, r, w, b, g


def _stream(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def _stats(s):
    s = s.double()
    mu = s.mean(1, keepdim=True)
    sd = ((s - mu).square().mean(1, keepdim=True) + EPS).sqrt()
    return s, mu, sd, (s - mu) / sd


def _k(width):
    return (width / 32 + 40) * 2.0 ** -24


def _check_y(y, s, w, b, width):
    _, mu, sd, xh = _stats(s)
    w = torch.ones(width) if w is None else w.cpu()
    b = torch.zeros(width) if b is None else b.cpu()
    ref = xh * w.double() + b.double()
    tol = UNIT[y.dtype] * ref.abs() + _k(width) * (1 + mu.abs() / sd + xh.abs()) * w.double().abs() + 2.0 ** -24 * b.double().abs()
    tol = tol + (2.0 ** -25 if y.dtype == torch.float16 else 0)   # fp16's smallest numbers
    err = (y.double().cpu() - ref).abs()
    assert not (err > tol).any(), f'worst {float((err / tol).max()):.3g} of its tolerance'


WIDTHS = [1, 2, 7, 32, 33, 64, 200, 256, 257, 512, 513, 1000, 1001, 1024, 1025, 2048, 3001, 4096, 4097, 8192, 8200, 20011]


@pytest.mark.gpu
@pytest.mark.parametrize('width', WIDTHS)
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
def test_forward(lib, width, kind):
    dt = DT[kind]
    for rows, residual, out, w_dt in ((1, False, dt, torch.float32), (37, True, dt, torch.float32),
                                      (5, True, torch.float32, dt), (301, False, torch.float32, dt)):
        x, r, w, b, _ = _inputs(rows, width, dt, width * 7 + rows, residual, w_dt)
        got = layer_norm(x.cuda(), w.cuda(), b.cuda(), EPS, residual=None if r is None else r.cuda(), out_dtype=out)
        y = got if r is None else got[0]
        assert y.shape == (rows, width) and y.dtype == out
        if r is not None:
            assert torch.equal(got[1].cpu(), _stream(x, r))
        _check_y(y, _stream(x, r), w, b, width)


def _grad_refs(s, w, gy, gsum):
    s, mu, sd, xh = _stats(s)
    gy, w = gy.double(), w.double()
    h = gy * w
    dx = (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True)) / sd
    if gsum is not None:
        dx = dx + gsum.double()
    return dx, (gy * xh).sum(0), gy.sum(0), mu, sd, xh, h


@pytest.mark.gpu
@pytest.mark.parametrize('width', [1, 7, 33, 256, 512, 1000, 1001, 1024, 2048, 4096, 4097, 8192, 9000])
@pytest.mark.parametrize('kind', ['fp32', 'bf16', 'fp16'])
def test_backward(lib, width, kind):
    dt = DT[kind]
    for rows, residual, out, w_dt in ((1, False, dt, torch.float32), (65, True, dt, torch.float32),
                                      (411, True, torch.float32, dt), (1203, False, dt, torch.float32)):
        x, r, w, b, g = _inputs(rows, width, dt, width * 3 + rows, residual, w_dt)
        gy = torch.randn(rows, width, generator=g).to(out)
        gs = torch.randn(rows, width, generator=g).to(dt) if residual else None
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b) + ((r,) if residual else ())]
        got = layer_norm(leaves[0], leaves[1], leaves[2], EPS, residual=leaves[3] if residual else None, out_dtype=out)
        grads = torch.autograd.grad(got, leaves, (gy.cuda(), gs.cuda()) if residual else gy.cuda())
        dx, dw, db, mu, sd, xh, h = _grad_refs(_stream(x, r), w, gy, gs)
        k = _k(width)
        lean = 1 + mu.abs() / sd
        size = h.abs() + h.abs().mean(1, keepdim=True) + (xh.abs() + lean) * (h * xh).abs().mean(1, keepdim=True)
        tol = UNIT[dt] * dx.abs() + 2 * k * lean * (1 + xh.abs()) * size / sd + 2.0 ** -24
        err = (grads[0].double().cpu() - dx).abs()
        assert not (err > tol).any(), f'dx: worst {float((err / tol).max()):.3g} of its tolerance'
        if residual:
            assert torch.equal(grads[3], grads[0])
        # column sums: each term to k of its size, the additions to (rows / 32 + 64) 2^-24 of the terms' sum
        wu = UNIT[w_dt]
        add = (rows / 32 + 64) * 2.0 ** -24
        for name, gt, ref, terms in (('dw', grads[1], dw, gy.double().abs() * (xh.abs() + lean)), ('db', grads[2], db, gy.double().abs())):
            tol = wu * ref.abs() + (k + add) * terms.sum(0) + 2.0 ** -24
            err = (gt.double().cpu() - ref).abs()
            assert gt.dtype == w_dt
            assert not (err > tol).any(), f'{name}: worst {float((err / tol).max()):.3g} of its tolerance'


@pytest.mark.gpu
def test_many_rows(lib):
    """More rows than any grid has places for, and few columns: 200,003 x 40."""
    x, _, w, b, g = _inputs(200003, 40, torch.bfloat16, 3, residual=False)
    gy = torch.randn(200003, 40, generator=g).bfloat16()
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    _check_y(y.detach(), x, w, b, 40)
    dx, dw, db = torch.autograd.grad(y, leaves, gy.cuda())
    rx, rw, rb, *_ = _grad_refs(x, w, gy, None)
    # sums of 200,003 terms of size 1 and random sign: fp32 rounding of the running sums, 2^-24 of their size each
    scale = (200003 / 32 + 64) * 2.0 ** -24 * 200003 ** 0.5
    assert (dw.cpu().double() - rw).abs().max() < scale and (db.cpu().double() - rb).abs().max() < scale


@pytest.mark.gpu
@pytest.mark.parametrize('width', [96, 512, 1001, 5000])
def test_gradient_against_differences(lib, width):
    """The directional derivative of sum(y gy) in fp32. The difference's own error: with h = 2^-7, each of the rows * width
    terms rounds to 4 * 2^-24 of its size 1, random in sign, over 2 h; and h^2 / 6 of a third derivative of at most 10 per
    row and unit of direction."""
    rows, h = 3, 2.0 ** -7
    x, _, w, b, g = _inputs(rows, width, torch.float32, width, residual=False)
    gy, v = torch.randn(rows, width, generator=g), torch.randn(rows, width, generator=g)
    vw, vb = torch.randn(width, generator=g), torch.randn(width, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, gy.cuda())

    def f(t):
        out = layer_norm((x + t * v).cuda(), (w + t * vw).cuda(), (b + t * vb).cuda())
        return float((out.cpu().double() * gy.double()).sum())

    want = (f(h) - f(-h)) / (2 * h)
    got = sum(float((a.cpu().double() * d.double()).sum()) for a, d in zip(grads, (v, vw, vb)))
    n = rows * width
    tol = n ** 0.5 * 4 * 2.0 ** -24 * 8 / h + h * h / 6 * 10 * n ** 0.5 * 3
    assert abs(got - want) < tol, (got, want, tol)


@pytest.mark.gpu
def test_large_mean_and_constant_rows(lib):
    x, _, w, b, _ = _inputs(16, 512, torch.float32, 1, residual=False, mean=1000.0)
    _check_y(layer_norm(x.cuda(), w.cuda(), b.cuda()), x, w, b, 512)
    c = torch.full((4, 512), 3.5).cuda()
    assert torch.equal(layer_norm(c, w.cuda(), b.cuda()), b.cuda().expand(4, 512))


@pytest.mark.gpu
@pytest.mark.parametrize('width', [512, 1001, 9000])
def test_bad_values_stay_in_their_rows(lib, width):
    x, r, w, b, _ = _inputs(9, width, torch.float32, 2)
    x[2, 5], x[4, 0], r[6, width - 1] = float('nan'), float('inf'), float('-inf')
    y, s = layer_norm(x.cuda(), w.cuda(), b.cuda(), residual=r.cuda())
    bad = torch.tensor([False, False, True, False, True, False, True, False, False])
    assert bool(y[bad.cuda()].isnan().any(1).all())
    good = ~bad
    _check_y(y[good.cuda()], _stream(x, r)[good], w, b, width)


@pytest.mark.gpu
def test_strides_shapes_and_missing_parameters(lib):
    x, r, w, b, _ = _inputs(24, 512, torch.bfloat16, 4)
    xc, rc, wc, bc = x.cuda(), r.cuda(), w.cuda(), b.cuda()
    want, total = layer_norm(xc, wc, bc, residual=rc)
    # leading axes
    y, t = layer_norm(xc.view(2, 3, 4, 512), wc, bc, residual=rc.view(2, 3, 4, 512))
    assert y.shape == (2, 3, 4, 512) and torch.equal(y.view(24, 512), want) and torch.equal(t.view(24, 512), total)
    assert torch.equal(layer_norm(xc[0], wc, bc), layer_norm(xc, wc, bc)[0])
    # rows apart, starts off any alignment, columns apart, a row repeated
    for pad, off in ((7, 1), (8, 0), (8, 8), (3, 2), (24, 5)):
        big = torch.full((24, 512 + pad), float('nan'), dtype=x.dtype, device='cuda')
        big[:, off:off + 512] = xc
        other = torch.full((24, 520), float('nan'), dtype=x.dtype, device='cuda')
        other[:, :512] = rc
        y, t = layer_norm(big[:, off:off + 512], wc, bc, residual=other[:, :512])
        assert torch.allclose(y.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -8) and torch.equal(t, total)
    turned = xc.t().contiguous().t()
    assert torch.equal(layer_norm(turned, wc, bc), layer_norm(xc, wc, bc))
    assert torch.equal(layer_norm(xc[:1].expand(24, 512), wc, bc), layer_norm(xc[:1], wc, bc).expand(24, 512))
    # weight and bias missing, or views
    for ww, bb in ((None, None), (w, None), (None, b)):
        y = layer_norm(xc, None if ww is None else ww.cuda(), None if bb is None else bb.cuda())
        _check_y(y, x, ww, bb, 512)
    wide = torch.zeros(512, 2, device='cuda')
    wide[:, 1] = wc
    assert torch.equal(layer_norm(xc, wide[:, 1], bc), layer_norm(xc, wc, bc))
    assert layer_norm(xc[:0], wc, bc).shape == (0, 512)


@pytest.mark.gpu
def test_gradients_of_parts_of_the_call(lib):
    x, r, w, b, g = _inputs(50, 512, torch.float32, 5)
    xc, rc, wc, bc = (t.cuda() for t in (x, r, w, b))
    gy = torch.randn(50, 512, generator=g).cuda()
    full = [t.clone().requires_grad_(True) for t in (xc, wc, bc)]
    want = torch.autograd.grad(layer_norm(*full), full, gy)
    for keep in range(3):   # one leaf at a time
        leaves = [xc, wc, bc]
        leaves[keep] = leaves[keep].clone().requires_grad_(True)
        got, = torch.autograd.grad(layer_norm(*leaves), [leaves[keep]], gy)
        assert torch.equal(got, want[keep])
    # only the stream is used; only y is used; a gradient that is one number repeated
    a, q = xc.clone().requires_grad_(True), rc.clone().requires_grad_(True)
    p = wc.clone().requires_grad_(True)
    y, s = layer_norm(a, p, bc, residual=q)
    da, dq, dp = torch.autograd.grad(s, [a, q, p], gy, retain_graph=True)
    assert torch.equal(da, gy) and torch.equal(dq, gy) and not dp.any()
    dy, = torch.autograd.grad(y, [a], gy)
    ref = _grad_refs(_stream(x, r), w, gy.cpu(), None)[0]
    assert torch.allclose(dy.cpu().double(), ref, rtol=0, atol=1e-5)
    y, s = layer_norm(a, p, bc, residual=q)
    (y.sum() + 0 * s.sum()).backward()
    assert torch.allclose(p.grad.cpu().double(), _stats(_stream(x, r))[3].sum(0), rtol=0, atol=1e-4)
    # nothing in the batch
    e = xc[:0].clone().requires_grad_(True)
    p = wc.clone().requires_grad_(True)
    layer_norm(e, p, bc).sum().backward()
    assert e.grad.shape == (0, 512) and not p.grad.any()
    # second derivatives are refused, not wrong
    a = xc.clone().requires_grad_(True)
    d, = torch.autograd.grad(layer_norm(a, wc, bc).square().sum(), [a], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.gpu
def test_same_bits_again_and_on_another_stream(lib):
    x, r, w, b, g = _inputs(5000, 512, torch.bfloat16, 6)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, r)]
    gy = torch.randn(5000, 512, generator=g).bfloat16().cuda()

    def once():
        y, s = layer_norm(*leaves[:3], residual=leaves[3])
        return [y, s, *torch.autograd.grad((y, s), leaves, (gy, gy))]

    first = once()
    q = torch.cuda.Stream()
    q.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(q):
        second = once()
    torch.cuda.current_stream().wait_stream(q)
    assert all(torch.equal(a, c) for a, c in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            y, s = layer_norm(*leaves[:3], residual=leaves[3])
    graph.replay()
    assert torch.equal(y, first[0]) and torch.equal(s, first[1])


@pytest.mark.gpu
def test_refusals(lib):
    x = torch.randn(4, 32, device='cuda')
    w = torch.ones(32, device='cuda')
    for args, kw in (((x.double(),), {}), ((x, w[:31]), {}), ((x, w, w.half()), {}), ((x, w, w), dict(residual=x[:3])),
                     ((x,), dict(residual=x.half())), ((x.half(),), dict(out_dtype=torch.bfloat16)), ((x, w.cpu()), {}),
                     ((torch.zeros(4, 0, device='cuda'),), {}), ((x.long(),), {}), ((x, w.double()), {}),
                     ((torch.tensor(1.0, device='cuda'),), {})):
        with pytest.raises(RuntimeError, match='layer_norm'):
            layer_norm(*args, **kw)


def test_refuses_the_cpu():
    with pytest.raises(RuntimeError, match='GPU only'):
        layer_norm(torch.randn(2, 8))


def test_c_entry_refusals():
    """Bad arguments come back as an error and a message before anything is launched (no GPU needed)."""
    import build
    lib = _lib(build.build())
    one = ctypes.c_void_p(16)

    def fwd(x=one, r=None, y=one, total=None, rows=1, width=8, xt=0, yt=0, wt=0):
        return lib.rl_norm_fwd(x, r, None, None, y, total, None, rows, width, 8, 8, xt, yt, wt, 1e-5, None)

    def bwd(gy=one, s=one, stats=one, dw=None, rows=1, width=8, xt=0, yt=0, work=None, nbytes=0):
        return lib.rl_norm_bwd(gy, None, s, stats, None, one, dw, None, rows, width, 8, 8, 8, xt, yt, 0, work, nbytes, None)

    for rc, word in ((fwd(rows=-1), b'rows'), (fwd(width=0), b'width'), (fwd(xt=3), b'type'), (fwd(xt=1, yt=2), b'type'),
                     (fwd(wt=-1), b'type'), (fwd(x=None), b'x, y'), (fwd(r=one), b'sum'), (bwd(rows=0), b'rows'),
                     (bwd(gy=None), b'gy'), (bwd(dw=one), b'work'), (bwd(dw=one, work=one, nbytes=4), b'work')):
        assert rc != 0
    fwd(width=0)
    assert b'width' in lib.rl_norm_error()
    assert fwd(rows=0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fp32', 'bf16'])
def test_gradients_through_views_that_are_not_aligned(lib, kind):
    """Rows that start one value off a 16-byte boundary, and a row's end inside a vector: the same gradients as from rows that
    lie end to end, to the tolerance of either."""
    dt = DT[kind]
    x, r, w, b, g = _inputs(300, 512, dt, 8)
    gy, gs = torch.randn(300, 512, generator=g).to(dt), torch.randn(300, 512, generator=g).to(dt)

    def wide(t):
        big = torch.full((300, 517), float('nan'), dtype=dt, device='cuda')
        big[:, 1:513] = t.cuda()
        return big

    bx, br = wide(x).requires_grad_(True), wide(r).requires_grad_(True)
    p = [t.cuda().requires_grad_(True) for t in (w, b)]
    out = layer_norm(bx[:, 1:513], *p, residual=br[:, 1:513])
    got = torch.autograd.grad(out, [bx, br, *p], (wide(gy)[:, 1:513], wide(gs)[:, 1:513]))
    dx, dw, db, mu, sd, xh, h = _grad_refs(_stream(x, r), w, gy, gs)
    k, lean = _k(512), 1 + mu.abs() / sd
    size = h.abs() + h.abs().mean(1, keepdim=True) + (xh.abs() + lean) * (h * xh).abs().mean(1, keepdim=True)
    tol = UNIT[dt] * dx.abs() + 2 * k * lean * (1 + xh.abs()) * size / sd + 2.0 ** -24
    for d in got[:2]:
        assert not ((d[:, 1:513].double().cpu() - dx).abs() > tol).any() and not d[:, 0].any() and not d[:, 513:].any()
    for d, ref, terms in ((got[2], dw, gy.double().abs() * (xh.abs() + lean)), (got[3], db, gy.double().abs())):
        assert ((d.double().cpu() - ref).abs() <= 2.0 ** -24 * ref.abs() + (k + (300 / 32 + 64) * 2.0 ** -24) * terms.sum(0)).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(lib):
    """4,200,000 x 512 values are more than 2^31: the last rows, forward and backward, are those of a batch of their own, bit for
    bit, and the column sums of gradients of 1 are the row count."""
    rows = 4_200_000
    g = torch.Generator(device='cuda').manual_seed(12)
    x = torch.randn(rows, 512, generator=g, device='cuda', dtype=torch.bfloat16).requires_grad_(True)
    w = (1 + 0.1 * torch.randn(512, generator=g, device='cuda')).requires_grad_(True)
    b = torch.randn(512, generator=g, device='cuda').requires_grad_(True)
    y = layer_norm(x, w, b)
    gy = torch.ones(512, device='cuda', dtype=torch.bfloat16).expand(rows, 512)
    dx, _, db = torch.autograd.grad(y, (x, w, b), gy)
    tail = x.detach()[-1000:].clone().requires_grad_(True)
    yt = layer_norm(tail, w, b)
    assert torch.equal(y[-1000:], yt)
    assert torch.equal(dx[-1000:], torch.autograd.grad(yt, tail, gy[-1000:])[0])
    assert torch.equal(db, torch.full((512,), float(rows), device='cuda'))   # whole numbers below 2^24
