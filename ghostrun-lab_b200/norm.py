"""Layer norm of the policy's blocks on the B200 library (rl_norm_fwd / rl_norm_bwd), with the residual sum before it:

    y = layer_norm(x, weight, bias, eps)                             # as torch.nn.functional.layer_norm over the last axis
    y, stream = layer_norm(x, weight, bias, eps, residual=branch)    # stream = x + branch, y = its norm

A SimBa block (rl/model.py:64-72) is x + mlp(norm(x)): the sum and the next block's norm read the stream once here. x and
residual: [..., D] fp32, bf16 or fp16, any leading shape and row strides; weight and bias: [D] of any of the three types,
each may be None; out_dtype: x's type (default) or fp32. The stream is kept in x's type, and what is kept is what is
normalised. Statistics and sums are fp32, every output is rounded once. Differentiable (once, in reverse; an input with a
forward-mode derivative is refused) in x, residual, weight and bias; the gradients of weight and bias are summed in a fixed
order, so the same inputs give the same bits."""
from __future__ import annotations

import policy_ops

_lib = policy_ops.load
_call = None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None, out_dtype=None, lib_path=None):
    """The norm of x's last axis; with a residual, (norm of x + residual, x + residual)."""
    global _call
    if _call is None or lib_path is not None:
        _lib(lib_path)
        from policy_ops_b200 import layer_norm as _call
    return _call(x, weight, bias, eps, residual, out_dtype)
