"""The binding of the policy operators and the library that it is given (policy_ops.py, csrc/policy_ops.cpp)."""
from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import PKG


def test_calls_before_a_library_is_bound():
    """An error, not a jump to no address."""
    import build
    build.build()
    code = ('import torch, policy_ops_b200 as p\n'
            'try:\n'
            '    p.sample(torch.zeros(1, 4), torch.zeros(1), None, 1.0, 0, 1.0, 0.0)\n'
            'except RuntimeError as e:\n'
            '    print(e)\n')
    said = subprocess.run([sys.executable, '-c', code], cwd=PKG, capture_output=True, text=True, timeout=300)
    assert said.returncode == 0 and 'policy_ops.load()' in said.stdout, (said.stdout, said.stderr)


@pytest.mark.gpu
def test_a_binding_that_fails_changes_nothing(gpu_lib_path):
    """The functions are taken over together: where one is missing, the earlier library stays whole."""
    import torch
    import policy_ops
    from norm import layer_norm
    policy_ops.load(gpu_lib_path)
    import policy_ops_b200
    x = torch.randn(3, 32, device='cuda')
    want = layer_norm(x)
    with pytest.raises(KeyError):
        policy_ops_b200.bind({'rl_norm_fwd': 1, 'rl_norm_error': 1})
    assert torch.equal(layer_norm(x), want)
