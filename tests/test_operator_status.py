"""The status of the operators' pipeline waits: a word for each device, reported by the next call there, which does not run."""
import ctypes

import pytest

import conftest  # noqa: F401  (import paths)


def word(device):
    import cdclq

    p = cdclq.lib().cdclq_operator_word(device)
    return ctypes.cast(p, ctypes.POINTER(ctypes.c_int)) if p else None


def test_no_word_without_a_device():
    import cdclq
    import torch

    for device in (-1, 1000):
        assert not cdclq.lib().cdclq_operator_word(device)
    if not torch.cuda.is_available():
        assert not cdclq.lib().cdclq_operator_word(0)


@pytest.mark.gpu
def test_each_device_has_its_word(gpu):
    """Set by hand here, as a kernel would whose wait ran out.  A word of another device stops nothing on this one."""
    import torch

    from cdclq import CdclqError
    from cdclq import adapters as A
    from cdclq import checkpoint as C
    from cdclq import lib
    from cdclq import loss as L
    from test_gpu_adapters import bank, layer, tokens

    device = torch.cuda.current_device()
    mine, other = word(device), word(device + 1)
    assert mine and other and mine[0] == 0 and other[0] == 0
    packed, _ = layer(48, 72, [4], 32, 3)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 72, 48, "bf16", 1)
    x, index = tokens(40, 72, 2, "bf16", 2)
    dy, _ = tokens(40, 48, 2, "bf16", 3)
    head = torch.ones(9, 72, dtype=torch.bfloat16, device="cuda")
    target, ones = torch.zeros(40, dtype=torch.int64, device="cuda"), torch.ones(40, device="cuda")
    u = A.forward(x, p, a, b, scale, index, keep=True)[1]
    lse = L.linear_cross_entropy(x, head, target)[1]
    c = C.save(x)
    calls = [lambda: A.forward(x, p, a, b, scale, index), lambda: A.forward(x[:3], p), lambda: A.backward(dy, x, u, p, a, b, scale, index),
             lambda: C.save(x), lambda: C.restore(c), lambda: C.weight_grad(dy, c), lambda: L.linear_cross_entropy(x, head, target),
             lambda: L.linear_cross_entropy_backward(x, head, target, lse, ones), lambda: L.linear_cross_entropy(x[:, 1:8], head[:, 1:8], target)]
    try:
        for call in calls:
            other[0] = 1
            call()
            mine[0] = 1
            with pytest.raises(CdclqError, match="timed out"):
                call()
            assert mine[0] == 0 and other[0] == 1
            call()
        mine[0] = 1
        assert lib().cdclq_operator_status() != 0 and lib().cdclq_operator_status() == 0
        assert other[0] == 1
    finally:
        mine[0] = other[0] = 0
