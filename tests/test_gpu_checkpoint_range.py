"""Activation checkpoints at the ends of the types' ranges."""
import pytest

import conftest  # noqa: F401  (import paths)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 128, 131, 515])
@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
def test_the_largest_values_come_back_finite(gpu, d, name):
    """s = max / 127 rounded up makes 127 s pass the largest number of f32.  |off| <= s / 2 + 127 roundings of s (2^-24 s
    each, and one of x / s), and the result's own rounding: 2^-8 (bf16), 2^-11 (f16), 2^-24 (f32)."""
    import torch

    from cdclq import checkpoint as C
    from test_gpu_checkpoint import U, dtype_of

    dt = dtype_of(torch, name)
    top = torch.finfo(dt).max
    g = torch.Generator(device="cuda").manual_seed(d)
    x = (torch.rand(9, d, generator=g, device="cuda", dtype=torch.float64) * 2 - 1) * top
    x[:, 0], x[:, d - 1] = top, -top
    x[1] /= 3
    x = x.to(dt)
    c = C.save(x)
    back = C.restore(c)
    assert bool(back.isfinite().all())
    s = c.scales.double().repeat_interleave(128, 1)[:, :d]
    off = (back.double() - x.double()).abs()
    assert bool((off <= s * (0.5 + 128 * 2.0 ** -23) + U[name] * x.double().abs() * (1 + 2.0 ** -8)).all())
    x[2, 3] = float("nan")
    x[3, 0] = float("inf")
    back = C.restore(C.save(x))
    assert bool(back[2, :128].isnan().all()) and bool(back[3, :128].isnan().all()) and bool(back[4:].isfinite().all())
