"""Adapters, activation checkpoints and the vocabulary's loss in one training step, against autograd in 64 bits."""
import numpy as np
import pytest

import conftest  # noqa: F401  (import paths)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [7, 90])
def test_a_step_against_autograd(gpu, t):
    """float16 with a loss scale.  Against the same chain in 64 bits from the same (rounded) inputs: y, dy and v are rounded
    to 2^-11 each, x to half a step of its block, so a gradient is off by a few 2^-11 of the sum of its terms' sizes; these
    sums are random, so 2 % of the gradient's norm is five times what is expected of them."""
    import torch

    from cdclq import adapters as A
    from cdclq import tune
    from test_gpu_adapters import bank, layer, tokens

    packed, wd = layer(96, 136, [4], 64, 3)
    w = A.PackedProjection(*packed)
    a, b, scale = bank(3, 8, 136, 96, "f16", 1)
    x, index = tokens(t, 136, 3, "f16", 2)
    g = torch.Generator(device="cuda").manual_seed(5)
    head = (torch.randn(300, 96, generator=g, device="cuda") / 10).half()
    target = torch.randint(0, 300, (t,), generator=g, device="cuda")
    target[0] = -100
    value, got = tune.step(w, head, x, target, a, b, scale, index, need_head=True, loss_scale=64.0)
    xs, ad, bd, hd = (v.double().requires_grad_() for v in (x, a, b, head))
    y = xs @ wd.t()
    for i in range(3):
        y = y + (index == i)[:, None] * scale[i].double() * (xs @ ad[i].t() @ bd[i].t())
    want = torch.nn.functional.cross_entropy(y @ hd.t(), target, ignore_index=-100)
    want.backward()
    assert abs(float(value) - float(want.detach())) <= 2e-3 * abs(float(want.detach()))
    for name, ref in (("dx", xs), ("da", ad), ("db", bd), ("dhead", hd)):
        off = (got[name].double() / 64 - ref.grad).norm() / ref.grad.norm()
        assert float(off) <= 0.02, (name, float(off))


@pytest.mark.gpu
def test_training_teaches_what_serving_gives(gpu):
    from cdclq import tune

    losses, (before, after) = tune.demo(steps=40)
    assert np.isfinite(losses).all() and losses[-1] < 0.5 * losses[0]
    assert after > before


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 12, 90])
def test_a_captured_step_gives_the_same(gpu, t):
    """A decode step and a training step in a CUDA graph, replayed on new inputs: the same bits as calls."""
    import torch

    from cdclq import adapters as A
    from cdclq import tune
    from test_gpu_adapters import bank, layer, tokens

    packed, _ = layer(96, 136, [4], 64, 3)
    w = A.PackedProjection(*packed)
    a, b, scale = bank(3, 8, 136, 96, "bf16", 1)
    x, index = tokens(t, 136, 3, "bf16", 2)
    g = torch.Generator(device="cuda").manual_seed(5)
    head = (torch.randn(300, 96, generator=g, device="cuda") / 10).bfloat16()
    target = torch.randint(0, 300, (t,), generator=g, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tune.step(w, head, x, target, a, b, scale, index)
        A.forward(x, w, a, b, scale, index)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = A.forward(x, w, a, b, scale, index)
        value, grads = tune.step(w, head, x, target, a, b, scale, index)
    other, others = tokens(t, 136, 3, "bf16", 9)
    x.copy_(other)
    index.copy_(others)
    graph.replay()
    want = A.forward(x, w, a, b, scale, index)
    v, wg = tune.step(w, head, x, target, a, b, scale, index)
    assert bool((y == want).all()) and bool(value == v)
    assert all(bool((grads[k] == wg[k]).all()) for k in ("dx", "da", "db"))
