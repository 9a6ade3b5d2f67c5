"""What is no tensor, no checkpoint and no projection is refused by name, not by an attribute that it lacks."""
import pytest

import conftest  # noqa: F401  (import paths)


def refused(calls):
    from cdclq import CdclqError

    for call, word in calls:
        with pytest.raises(CdclqError, match=word) as e:
            call()
        assert e.value.code == -3


def test_what_is_no_tensor_without_a_device():
    import numpy as np
    import torch

    from cdclq import adapters as A
    from cdclq import checkpoint as C
    from cdclq import loss as L

    n, x = np.zeros((4, 8), np.float32), torch.zeros(4, 8)
    refused([(lambda: A.PackedProjection(None, x, x, x, x, 8), "qweight: need a tensor"), (lambda: A.forward(x, None), "PackedProjection"),
             (lambda: C.save(None), "x: need a tensor"), (lambda: C.save(n), "x: need a tensor"), (lambda: C.save([x]), "x: need a tensor"),
             (lambda: C.Checkpoint(n, n, torch.float16), "codes: need a tensor"), (lambda: C.restore(None), "need a Checkpoint"),
             (lambda: C.restore(x), "need a Checkpoint"), (lambda: C.weight_grad(x, x), "need a Checkpoint"),
             (lambda: L.linear_cross_entropy(None, x, x), "h: need a tensor"), (lambda: L.linear_cross_entropy(n, n, n), "h: need a tensor"),
             (lambda: L.linear_cross_entropy_backward(n, n, n, n, n), "h: need a tensor")])


@pytest.mark.gpu
def test_what_is_no_tensor(gpu):
    import numpy as np
    import torch

    from cdclq import adapters as A
    from cdclq import checkpoint as C
    from cdclq import loss as L
    from test_gpu_adapters import bank, cdclq_status, layer, tokens

    packed, _ = layer(16, 64, [4], 32, 2)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 64, 16, "bf16", 1)
    x, index = tokens(5, 64, 2, "bf16", 2)
    dy, _ = tokens(5, 16, 2, "bf16", 3)
    u = A.forward(x, p, a, b, scale, index, keep=True)[1]
    n = np.zeros(2, np.float32)
    ones = torch.ones(5, device="cuda")
    target = torch.zeros(5, dtype=torch.int64, device="cuda")
    lse = L.linear_cross_entropy(x, a[0], target)[1]
    q, s, z, perm, gb, g = packed
    refused([(lambda: A.PackedProjection(q, s.cpu().numpy(), z, perm, gb, g), "scales: need a tensor"),
             (lambda: A.PackedProjection(q, s, z, perm, gb.cpu().numpy(), g), "gbits: need a tensor"),
             (lambda: A.forward(None, p), "x: need a tensor"), (lambda: A.forward(x.cpu().float().numpy(), p), "x: need a tensor"),
             (lambda: A.forward(x, p, [a], b, scale, index), "a: need a tensor"), (lambda: A.forward(x, p, a, [b], scale, index), "b: need a tensor"),
             (lambda: A.forward(x, p, a, b, n, index), "scale: need a tensor"), (lambda: A.forward(x, p, a, b, scale, [0] * 5), "index: need a tensor"),
             (lambda: A.backward(dy, None, u, p, a, b, scale, index), "x: need a tensor"),
             (lambda: A.backward(dy, x, None, p, a, b, scale, index), "u: need a tensor"),
             (lambda: A.backward(None, x, u, p, a, b, scale, index), "dy: need a tensor"),
             (lambda: C.weight_grad(None, C.save(x)), "dy: need a tensor"), (lambda: C.Checkpoint(C.save(x).codes, None, x.dtype), "scales: need a tensor"),
             (lambda: L.linear_cross_entropy(x, None, target), "w: need a tensor"), (lambda: L.linear_cross_entropy(x, a[0], [0] * 5), "target: need a tensor"),
             (lambda: L.linear_cross_entropy_backward(x, a[0], target, None, ones), "lse: need a tensor"),
             (lambda: L.linear_cross_entropy_backward(x, a[0], target, lse, 1.0), "dloss: need a tensor")])
    assert A.backward(dy, None, None, p, a, b, scale, index, need_da=False, need_db=False)[1:] == (None, None)
    assert cdclq_status() == 0
