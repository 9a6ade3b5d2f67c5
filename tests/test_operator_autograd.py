"""The operators' gradients come from their backward calls; what autograd would lose is refused."""
import pytest

import conftest  # noqa: F401  (import paths)


@pytest.mark.gpu
def test_inputs_that_want_gradients_are_refused(gpu):
    import torch

    from cdclq import CdclqError
    from cdclq import adapters as A
    from cdclq import checkpoint as C
    from cdclq import loss as L
    from cdclq import tune
    from test_gpu_adapters import bank, layer, tokens

    packed, _ = layer(48, 72, [4], 32, 3)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 72, 48, "bf16", 1)
    x, index = tokens(40, 72, 2, "bf16", 2)
    head = torch.ones(9, 48, dtype=torch.bfloat16, device="cuda")
    target = torch.zeros(40, dtype=torch.int64, device="cuda")
    y, u = A.forward(x, p, a, b, scale, index, keep=True)
    value, grads = tune.step(p, head, x, target, a, b, scale, index, need_head=True)
    for k in (x, a, b, scale, head):
        k.requires_grad_()
        if k is head:
            calls = [lambda: L.linear_cross_entropy(y, head, target)]
        else:
            calls = [lambda: A.forward(x, p, a, b, scale, index)]
        for call in calls:
            with pytest.raises(CdclqError, match="no_grad"):
                call()
            with torch.no_grad():
                call()
        # a step returns its gradients, serving has none, a checkpoint is data
        again, others = tune.step(p, head, x, target, a, b, scale, index, need_head=True)
        assert bool(again == value) and all(bool((others[n] == grads[n]).all()) for n in grads)
        assert tune.serve(p, head, x, a, b, scale, index).shape == (40, 9)
        C.restore(C.save(x))
        k.requires_grad_(False)
    lse = L.linear_cross_entropy(y, head, target)[1]
    y.requires_grad_()
    with pytest.raises(CdclqError, match="no_grad"):
        L.linear_cross_entropy(y, head, target)
    L.linear_cross_entropy_backward(y, head, target, lse, torch.ones(40, device="cuda"))
