"""Adapters' gradients from inputs that start anywhere."""
import pytest

import conftest  # noqa: F401  (import paths)
from test_gpu_adapters import bank, layer, tokens


def gradients(t, d_in, d_out, n, r, name, sizes, seed=3):
    """Inputs with dy, b and x of the given standard deviations."""
    packed, w = layer(d_out, d_in, [4], 64, seed)
    a, b, scale = bank(n, r, d_in, d_out, name, seed)
    x, index = tokens(t, d_in, n, name, seed + 1)
    dy, _ = tokens(t, d_out, n, name, seed + 2)
    b = (b.double() * r ** 0.5 * sizes[1]).to(b.dtype)
    return packed, w, a, b, scale, (x.double() * sizes[2]).to(x.dtype), (dy.double() * sizes[0]).to(dy.dtype), index


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("first", [1, 3, 8])
@pytest.mark.parametrize("t,d_in,r", [(45, 64, 8), (300, 200, 16), (70, 133, 72)])
def test_x_that_starts_anywhere(gpu, t, d_in, r, first, name):
    """x in full whose rows start off 16 bytes beside factors that are read 16 bytes at a time: ranks below 64, tokens that do
    not fill a stage."""
    import torch

    from cdclq import adapters as A

    packed, w, a, b, scale, x, dy, index = gradients(t, d_in, 72, 3, r, name, (1, 1, 1))
    p = A.PackedProjection(*packed)
    u = A.forward(x, p, a, b, scale, index, keep=True)[1]
    want = A.backward(dy, x, u, p, a, b, scale, index)
    moved = torch.zeros(t * (d_in + 5) + 16, dtype=x.dtype, device="cuda")[first:first + t * (d_in + 5)].view(t, d_in + 5)[:, :d_in]
    moved.copy_(x)
    assert moved.stride(0) == d_in + 5
    assert all(bool((g == h).all()) for g, h in zip(A.backward(dy, moved, u, p, a, b, scale, index), want))
