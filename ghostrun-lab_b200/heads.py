"""The policy's action heads on the B200 library: moves sampled from given random numbers, and the log-probability and
entropy of given moves (rl/model.py:176-194, ordered heads masked by the legal parts).

    ids, logp = sample_moves(logits, cond, masks, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    logp, entropy = moves_logp(logits, cond, masks, ids)                    # differentiable (in reverse) in logits and cond
    choice, logp = sample(logits, u, legal=masks, top_p=0.95)               # rows of any width up to 4096

logits: [B, 19] fp32, bf16 or fp16, the five heads side by side in the mask bytes' order (actions.PARTS); cond: the ten
tables [choices of part j, choices of part k] for k = 1..4, j < k (policy.Policy.tables()), or None; masks: [B, 19] bytes, as
RlEnv.masks; u: fp32 random numbers in [0, 1), [B, 5] (sample: [B]); ids: int16 packed moves, as RlEnv.actions. sample's
legal is [B, V], or the 19 mask bytes for a flat head over the 324 packed moves, or None.

temperature (0: the best choice), top_k (0: all), top_p and min_p are numbers, or tensors [B] with one for each row. They
apply in this order: top-k of the logits / temperature, the shortest run of what is left that holds top_p of its probability,
those of it with at least min_p of the best one's. Numbers out of range are refused; a row's own count as the nearest that is
allowed (top_k, top_p and temperature below 0 as 0, min_p above 1 as 1), NaN as a temperature of 0 or as no cut. Equal logits
rank by index. The log-probability returned is that of the distribution drawn from. The same inputs give the same choice on
any launch shape (csrc/heads.cuh). The samplers' log-probabilities carry no gradient: moves_logp gives the moves' own. A part
(or row) with nothing legal answers 0, the neutral choice, with log-probability and entropy 0 and no gradient."""
from __future__ import annotations

import policy_ops

SIZES = (9, 3, 3, 2, 2)                                              # choices of each part
TABLES = [(SIZES[j], SIZES[k]) for k in range(5) for j in range(k)]   # shapes of the ten tables of cond

_lib = policy_ops.load
_ops = None


def _ready(lib_path):
    global _ops
    if _ops is None or lib_path is not None:
        _lib(lib_path)
        import policy_ops_b200
        _ops = policy_ops_b200
    return _ops


def sample_moves(logits, cond, masks, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lib_path=None):
    """One move for each row, part by part: (packed ids int16 [B], log-probabilities fp32 [B])."""
    return _ready(lib_path).sample_moves(logits, cond, masks, u, temperature, top_k, top_p, min_p)


def sample(logits, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lib_path=None):
    """One choice for each row of logits [B, V]: (choices int64 [B], log-probabilities fp32 [B])."""
    return _ready(lib_path).sample(logits, u, legal, temperature, top_k, top_p, min_p)


def moves_logp(logits, cond, masks, ids, lib_path=None):
    """(log-probability, entropy) fp32 [B] of the moves ids under the ordered heads, the entropy the sum of the parts'
    conditional entropies along the move. A move that the masks exclude has log-probability -inf, an id outside 0..323 NaN
    in both. The backward reads logits, cond, masks and ids again: give it copies of buffers that the env writes
    (RlEnv.masks, RlEnv.actions) where a step may come between."""
    return _ready(lib_path).moves_logp(logits, cond, masks, ids)
