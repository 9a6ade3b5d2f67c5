"""The operators' workspace functions on the host: 0 for what the call refuses, whatever the numbers, and never a crash."""
import ctypes
import subprocess
import sys

import pytest

import conftest

# in a process of its own: a division by zero would end this one
PROGRAM = """
import ctypes, sys
sys.path.insert(0, %r)
import cdclq
from cdclq.abi import CPackedLayer
lib = cdclq.lib()
w = CPackedLayer()
big = 2 ** 64 - 1
got = []
for d_out, d_in in ((0, 0), (0, 64), (64, 0)):
    w.d_out, w.d_in = d_out, d_in
    for t in (1, 40, 4096, big):
        got.append(lib.cdclq_projection_forward_workspace(ctypes.byref(w), t, 2, 8))
        got.append(lib.cdclq_projection_backward_workspace(ctypes.byref(w), t, 2, 8, 1))
w.d_out = w.d_in = 64
for t in (2 ** 31, big):
    got.append(lib.cdclq_projection_forward_workspace(ctypes.byref(w), t, 2, 8))
    got.append(lib.cdclq_projection_backward_workspace(ctypes.byref(w), t, 2, 8, 1))
for n, r in ((big, 8), (2, big), (2 ** 15, 8), (2, 4097)):
    got.append(lib.cdclq_projection_forward_workspace(ctypes.byref(w), 40, n, r))
    got.append(lib.cdclq_projection_backward_workspace(ctypes.byref(w), 40, n, r, 1))
for a in ((big, 8, 8), (8, big, 8), (8, 8, big)):
    got.append(lib.cdclq_linear_cross_entropy_workspace(*a))
    got.append(lib.cdclq_linear_cross_entropy_backward_workspace(*a, 1, 1))
    got.append(lib.cdclq_checkpoint_weight_grad_workspace(*a))
assert not any(got), got
print("sound")
"""


def test_refused_sizes_have_no_workspace():
    import os

    out = subprocess.run([sys.executable, "-c", PROGRAM % os.path.join(conftest.ROOT, "cdcl-gptq_b200")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "sound", out.stderr[-500:]


@pytest.mark.parametrize("t", [1, 32, 33, 5000])
def test_sizes_of_calls_that_run(t):
    import cdclq
    from cdclq.abi import CPackedLayer

    lib = cdclq.lib()
    w = CPackedLayer()
    w.d_out, w.d_in, w.units, w.groups = 96, 128, 2, 1
    ref = ctypes.byref(w)
    assert lib.cdclq_projection_forward_workspace(ref, 0, 0, 0) == 0
    bare = lib.cdclq_projection_forward_workspace(ref, t, 0, 0)
    assert 0 < bare <= lib.cdclq_projection_forward_workspace(ref, t, 3, 16)
    assert lib.cdclq_projection_forward_workspace(ref, t, 0, 7) == bare  # a rank without adapters
    assert lib.cdclq_projection_backward_workspace(ref, t, 3, 16, 1) >= lib.cdclq_projection_backward_workspace(ref, t, 3, 16, 0) > 0
    assert lib.cdclq_linear_cross_entropy_workspace(t, 64, 100) > 0 and lib.cdclq_checkpoint_weight_grad_workspace(t, 64, 100) > 0
