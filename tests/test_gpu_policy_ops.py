"""The policy on the library's layer norm and head kernels (policy.Policy(fused=True)) against the same parameters on torch's
ops, and the small learner that runs them together (learn.py). The two paths share every linear layer; they differ in the
residual stream's rounding to bf16 after each sum (the same in both), and in the norms' outputs, fp32 rounded to bf16 in
either case: tolerance 8 bf16 roundings (2^-8) of the encoding's size 1, and of the gradients' largest."""
from __future__ import annotations

import pytest
import torch

from actions import PARTS, pack, unpack
from policy import Policy

pytestmark = pytest.mark.gpu


@pytest.fixture
def inputs(gpu_lib_path):
    import heads
    import norm
    import stem
    for m in (heads, norm, stem):
        m._lib(gpu_lib_path)
    B, dev = 96, torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(5)

    def bits(n, *shape):
        return torch.randint(0, n, shape, generator=g, device=dev, dtype=torch.int32).to(torch.uint8)

    masks = (torch.rand(B, 19, generator=g, device=dev) < 0.6).to(torch.uint8)
    for a, _ in PARTS:
        masks[:, a] = 1
    prev = [torch.randint(0, b - a, (B,), generator=g, device=dev) for a, b in PARTS]
    return dict(packed=bits(256, B, 4, 224, 180), emph=bits(8, B, 4, 224), timeline=bits(2, B, 8, 45), prev_parts=prev), masks, g


def _pair():
    torch.manual_seed(7)
    plain = Policy(torch.rand(512, 3)).cuda().to(memory_format=torch.channels_last)
    with torch.no_grad():   # tables and norms that are not where they start
        for k in range(5):
            for t in plain.cond[k]:
                t.weight.normal_(std=0.5)
        for m in (plain.ln, *[b.ln for b in plain.blocks]):
            m.weight.normal_(1.0, 0.1)
            m.bias.normal_(0.0, 0.1)
    fused = Policy(torch.rand(512, 3), fused=True).cuda().to(memory_format=torch.channels_last)
    fused.load_state_dict(plain.state_dict())
    fused.palette.copy_(plain.palette)
    return plain, fused


def test_encode_and_its_gradients(inputs):
    x, _, g = inputs
    plain, fused = _pair()
    outs, grads = [], []
    up = torch.randn(96, 512, generator=g, device='cuda')
    for pol in (plain, fused):
        with torch.autocast('cuda', dtype=torch.bfloat16):
            z = pol.encode(**x)
        assert z.dtype == torch.float32
        pol.zero_grad()
        (z * up).sum().backward()
        outs.append(z.detach())
        grads.append({n: p.grad.clone() for n, p in pol.named_parameters() if p.grad is not None})
    assert float((outs[0] - outs[1]).abs().max()) <= 8 * 2.0 ** -8 * float(outs[0].abs().max())
    assert grads[0].keys() == grads[1].keys() and 'blocks.1.ln.weight' in grads[0]
    for n, a in grads[0].items():
        b = grads[1][n]
        assert a.dtype == b.dtype
        assert float((a - b).norm()) <= 8 * 2.0 ** -8 * float(a.norm()), n


def test_draw_follows_act_and_evaluate(inputs):
    """The kernel's moves are legal, have the torch heads' log-probability, and come as often as the heads say."""
    _, masks, g = inputs
    _, pol = _pair()
    h = torch.randn(96, 512, generator=g, device='cuda')
    ids, logp = pol.draw(h, masks, g)
    chosen, want = unpack(ids), torch.zeros(96, device='cuda')
    for k, (a, b) in enumerate(PARTS):
        lg = pol.heads[k](h)
        for j in range(k):
            lg = lg + pol.cond[k][j](chosen[j])
        lp = lg.float().masked_fill(masks[:, a:b] == 0, -1e9).log_softmax(-1)
        assert bool((masks[torch.arange(96), a + chosen[k]] != 0).all())
        want = want + lp.gather(1, chosen[k][:, None]).squeeze(1)
    assert float((want - logp).detach().abs().max()) < 1e-4
    again, entropy = pol.evaluate(h, masks, ids)
    assert float((again - logp).detach().abs().max()) < 1e-4 and bool((entropy >= -1e-5).all())
    # 20,000 draws of one row: the first part's frequencies within 6 standard deviations (sqrt(p (1 - p) / n) <= 0.0036)
    hh, mm = h[:1].expand(20000, 512), masks[:1].expand(20000, 19)
    first = unpack(pol.draw(hh, mm, g)[0])[0]
    p = pol.heads[0](h[:1]).float().masked_fill(masks[:1, :9] == 0, -1e9).softmax(-1)[0]
    freq = torch.bincount(first, minlength=9) / 20000
    assert float((freq - p).detach().abs().max()) < 6 * 0.0036


def test_decide_is_the_same_surface(inputs):
    x, masks, g = inputs
    _, pol = _pair()
    h, starts = torch.zeros(96, 512, device='cuda'), torch.ones(96, dtype=torch.bool, device='cuda')
    mv, parts, logp, val, h2 = pol.decide(x['packed'], x['emph'], x['timeline'], x['prev_parts'], masks, h, starts, g, chunk=40)
    assert mv.dtype == torch.int16 and torch.equal(pack(parts), mv)
    assert val.shape == (96, 101) and h2.shape == (96, 512) and h2.dtype == torch.float32 and bool(torch.isfinite(logp).all())


def test_learner(inputs, gpu_lib_path):
    """Before the first update the policy that made the moves is the policy that is asked: their log-probabilities agree to
    the encoder's bf16 (batches of other sizes may round otherwise); every parameter that the losses reach gets a gradient."""
    from learn import Learner
    learner = Learner(envs=16, steps=4, lib_path=gpu_lib_path)
    batch, h0, last = learner.rollout()
    adv, returns = learner.advantages(batch, last)
    _, _, entropy, change = learner.losses(batch, h0, adv, returns)
    assert change.item() < 0.02 and 0 < entropy.item() < 6
    before = [p.detach().clone() for p in learner.policy.parameters()]
    said = learner.update(batch, h0, last)
    assert all(torch.isfinite(torch.tensor(v)) for v in said.values())
    moved = [n for (n, p), b in zip(learner.policy.named_parameters(), before) if not torch.equal(p, b)]
    assert {'blocks.0.ln.weight', 'ln.bias', 'cond.4.3.weight', 'heads.0.weight', 'stem.weight'} <= set(moved)
