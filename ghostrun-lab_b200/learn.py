"""A small learner on the library's kernels, end to end on one GPU: rollouts of the synthetic game with the policy choosing
the moves, then clipped policy-gradient updates through the policy's kernels in both directions.

    python ghostrun-lab_b200/learn.py [--envs 64] [--steps 16] [--iters 2] [--epochs 2]

Rollout: the env draws packed pictures (rlenv.RlEnv), Policy(fused=True).decide encodes them (stem, layer norms), steps the
GRU and samples the moves (heads.sample_moves). Update: the stored decisions are encoded again, the GRU runs along the
rollout with its memory cleared at episode starts, heads.moves_logp gives the moves' log-probabilities and entropies, and the
gradients come back through moves_logp, layer_norm and fused_stem. It shows how the pieces go together; it is not the
reference's trainer (rl/train.py)."""
from __future__ import annotations

import argparse

import torch

from policy import Policy
from rlenv import RlEnv

SPAN = 10.0   # the value bins' centres go from -SPAN to SPAN


def expected_value(logits):
    """The mean of the value head's distribution over its bins."""
    centres = torch.linspace(-SPAN, SPAN, logits.shape[-1], device=logits.device)
    return (logits.float().softmax(-1) * centres).sum(-1)


class Learner:
    def __init__(self, envs=64, steps=16, seed=1, lr=1e-4, device='cuda', lib_path=None):
        self.dev, self.N, self.T = torch.device(device), envs, steps
        self.env = RlEnv({'synth00': envs}, device=self.dev, seed=seed, lib_path=lib_path)
        self.packed = torch.empty(envs, 4, 224, 180, dtype=torch.uint8, device=self.dev)
        self.env.bind_obs_pack6(self.packed)
        self.env.start()
        torch.manual_seed(seed)
        palette = torch.rand(512, 3, generator=torch.Generator().manual_seed(seed))   # a seeded stand-in colour table
        self.policy = Policy(palette, fused=True).to(self.dev).to(memory_format=torch.channels_last)
        self.opt = torch.optim.AdamW(self.policy.parameters(), lr=lr, fused=True)
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        self.h = torch.zeros(envs, 512, device=self.dev)
        self.starts = torch.ones(envs, dtype=torch.bool, device=self.dev)
        self.prev = [torch.zeros(envs, dtype=torch.long, device=self.dev) for _ in range(5)]

    def rollout(self):
        """T decisions of every env: a dict of [T, N, ...] tensors, the GRU's memory before them, and the value after them."""
        env, keep = self.env, {k: [] for k in ('packed', 'emph', 'timeline', 'masks', 'prev', 'starts', 'ids', 'logp',
                                               'value', 'reward', 'done')}
        h0 = self.h
        for _ in range(self.T):
            for name, t in (('packed', self.packed), ('emph', env.emph), ('timeline', env.timeline), ('masks', env.masks),
                            ('prev', torch.stack(self.prev, 1)), ('starts', self.starts)):
                keep[name].append(t.clone())
            ids, parts, logp, value, self.h = self.policy.decide(self.packed, env.emph, env.timeline, self.prev, env.masks,
                                                                 self.h, self.starts, self.gen)
            env.actions.copy_(ids)
            env.step()
            done = env.done.bool()
            for name, t in (('ids', ids), ('logp', logp), ('value', expected_value(value)), ('reward', env.reward), ('done', done)):
                keep[name].append(t.clone())
            self.starts = done
            self.prev = [p * (~done).long() for p in parts]
        batch = {k: torch.stack(v) for k, v in keep.items()}
        _, _, _, value, _ = self.policy.decide(self.packed, env.emph, env.timeline, self.prev, env.masks, self.h, self.starts,
                                               self.gen)
        return batch, h0, expected_value(value)

    @staticmethod
    def advantages(batch, last, discount=0.99, trace=0.95):
        """Generalised advantage estimates [T, N], and the returns that the value head is fitted to."""
        adv, run, after = torch.zeros_like(batch['value']), torch.zeros_like(last), last
        for t in reversed(range(len(adv))):
            goes_on = (~batch['done'][t]).float()
            delta = batch['reward'][t] + discount * goes_on * after - batch['value'][t]
            run = delta + discount * trace * goes_on * run
            adv[t], after = run, batch['value'][t]
        return adv, (adv + batch['value']).clamp(-SPAN, SPAN)

    def losses(self, batch, h0, adv, returns, clip=0.2):
        """(policy loss, value loss, mean entropy, mean |change of log-probability|) of the rollout under the policy as it is."""
        pol, T, N = self.policy, *batch['ids'].shape
        with torch.autocast('cuda', dtype=torch.bfloat16):
            z = pol.encode(batch['packed'].flatten(0, 1), batch['emph'].flatten(0, 1), batch['timeline'].flatten(0, 1),
                           list(batch['prev'].flatten(0, 1).unbind(1)))
        z, h, hs = z.view(T, N, -1), h0, []
        for t in range(T):
            h = pol.gru(z[t], h * (~batch['starts'][t]).unsqueeze(1).float())
            hs.append(h)
        hs = torch.cat(hs)
        logp, entropy = pol.evaluate(hs, batch['masks'].flatten(0, 1), batch['ids'].flatten())
        a = ((adv - adv.mean()) / (adv.std() + 1e-6)).flatten()
        change = logp - batch['logp'].flatten()
        ratio = change.exp()
        policy = -torch.minimum(ratio * a, ratio.clamp(1 - clip, 1 + clip) * a).mean()
        value = (expected_value(pol.value(hs)) - returns.flatten()).square().mean()
        return policy, value, entropy.mean(), change.detach().abs().mean()

    def update(self, batch, h0, last, epochs=2, entropy_weight=0.01):
        adv, returns = self.advantages(batch, last)
        for _ in range(epochs):
            policy, value, entropy, change = self.losses(batch, h0, adv, returns)
            self.opt.zero_grad(set_to_none=True)
            (policy + 0.5 * value - entropy_weight * entropy).backward()
            norm = torch.nn.utils.clip_grad_norm_(self.policy.parameters(), 1.0)
            self.opt.step()
        return dict(policy=policy.item(), value=value.item(), entropy=entropy.item(), change=change.item(), grad_norm=norm.item())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--envs', type=int, default=64)
    ap.add_argument('--steps', type=int, default=16)
    ap.add_argument('--iters', type=int, default=2)
    ap.add_argument('--epochs', type=int, default=2)
    ap.add_argument('--seed', type=int, default=1)
    args = ap.parse_args()
    learner = Learner(args.envs, args.steps, args.seed)
    for it in range(args.iters):
        batch, h0, last = learner.rollout()
        said = learner.update(batch, h0, last, args.epochs)
        said['reward'] = float(batch['reward'].mean())
        print(f'iteration {it}: ' + ', '.join(f'{k} {v:.4g}' for k, v in said.items()), flush=True)


if __name__ == '__main__':
    main()
