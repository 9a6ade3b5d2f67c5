"""Adapters whose factors or gradients are small or large for their type, and inputs that start anywhere.

u = 2^-8 (bf16), 2^-11 (f16) is one rounding to nearest.  Of a gradient da whose elements are each rounded once, that is at most
u / sqrt(3) of its norm (and 2^-25 an element below f16's normal range); 20 % more stand for what is rounded before it.
"""
import pytest

import conftest  # noqa: F401  (import paths)
from test_gpu_adapters import U, acc, bank, layer, own, tokens, within


def gradients(t, d_in, d_out, n, r, name, sizes, seed=3):
    """Inputs with dy, b and x of the given standard deviations."""
    packed, w = layer(d_out, d_in, [4], 64, seed)
    a, b, scale = bank(n, r, d_in, d_out, name, seed)
    x, index = tokens(t, d_in, n, name, seed + 1)
    dy, _ = tokens(t, d_out, n, name, seed + 2)
    b = (b.double() * r ** 0.5 * sizes[1]).to(b.dtype)
    return packed, w, a, b, scale, (x.double() * sizes[2]).to(x.dtype), (dy.double() * sizes[0]).to(dy.dtype), index


def check_da(got, dy, x, b, scale, index, name):
    import torch

    want = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    for i in range(b.shape[0]):
        rows = own(index, i)
        want[i] = (scale[i].double() * (dy[rows].double() @ b[i].double())).t() @ x[rows].double()
    assert float(want.abs().max()) < 60000 and float(want.norm()) > 0
    off = float((got.double() - want).norm())
    assert off <= 1.2 * U[name] / 3 ** 0.5 * float(want.norm()) + 2.0 ** -25 * want.numel() ** 0.5, off / float(want.norm())


SIZES = [(1, 1, 1), (1e-3, 1e-2, 1), (1e-3, 1e-3, 1), (1e-3, 1e-4, 1), (1e-2, 1e-4, 0.05), (1e-2, 1e-2, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("t,r", [(2048, 16), (333, 24)])
def test_a_gradient_of_a_from_a_checkpoint(gpu, t, r, sizes, name):
    """Freshly started adapters have a small b, a mean's dy is small: neither costs da bits."""
    from cdclq import adapters as A
    from cdclq import checkpoint as C

    packed, w, a, b, scale, x, dy, index = gradients(t, 264, 1024, 2, r, name, sizes)
    c = C.save(x)
    da = A.backward(dy, c, None, A.PackedProjection(*packed), a, b, scale, index, need_dx=False, need_db=False)[1]
    check_da(da, dy, c.codes.double() * c.scales.double().repeat_interleave(128, 1)[:, :264], b, scale, index, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_a_gradient_of_a_from_a_checkpoint_of_large_v(gpu, name):
    """v past f16's range, x small: da is far inside it."""
    from cdclq import adapters as A
    from cdclq import checkpoint as C

    packed, w, a, b, scale, x, dy, index = gradients(700, 136, 1024, 2, 8, name, (100, 60, 1e-3))
    x[:, 1::2] = 0  # a zero code beside them
    c = C.save(x)
    da = A.backward(dy, c, None, A.PackedProjection(*packed), a, b, scale, index, need_dx=False, need_db=False)[1]
    check_da(da, dy, c.codes.double() * c.scales.double().repeat_interleave(128, 1)[:, :136], b, scale, index, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES + [(100, 60, 1e-3)])
@pytest.mark.parametrize("t,d_in,r", [(2048, 264, 16), (333, 264, 24), (150, 131, 70)])
def test_a_gradient_of_a_from_x_in_full(gpu, t, d_in, r, sizes, name):
    from cdclq import adapters as A

    packed, w, a, b, scale, x, dy, index = gradients(t, d_in, 1024, 2, r, name, sizes)
    da = A.backward(dy, x, None, A.PackedProjection(*packed), a, b, scale, index, need_dx=False, need_db=False)[1]
    check_da(da, dy, x, b, scale, index, name)


@pytest.mark.gpu
def test_gradients_of_unlike_tokens_and_adapters(gpu):
    """One adapter's v is 2^20 times another's, a third has none but infinities: each has its own bits."""
    import torch

    from cdclq import adapters as A

    packed, w, a, b, scale, x, dy, index = gradients(900, 136, 512, 4, 16, "f16", (1, 1, 1))
    b[0] /= 1024
    dy[index == 0] /= 1024
    dy[index == 3] = float("inf")
    p = A.PackedProjection(*packed)
    da = A.backward(dy, x, None, p, a, b, scale, index, need_dx=False, need_db=False)[1]
    for i in range(3):
        check_da(da[i:i + 1], dy, x, b[i:i + 1], scale[i:i + 1], torch.where(index == i, 0, -1), "f16")
    assert not bool(da[3].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("t,d_in,d_out,n,r", [(40, 512, 64, 3, 16), (300, 328, 515, 4, 100), (333, 2048, 256, 3, 8), (2100, 264, 1100, 3, 16),
                                              (129, 130, 77, 3, 5)])
def test_u_past_the_range_of_float16(gpu, t, d_in, d_out, n, r):
    """scale u is past 65504 for some tokens of some adapters, u and y are not.  Bounds as the forward pass has them elsewhere."""
    import torch

    from cdclq import adapters as A
    from test_gpu_adapters import check_forward, want_forward

    packed, w = layer(d_out, d_in, [4], 64, t)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(n, r, d_in, d_out, "f16", t)
    x, index = tokens(t, d_in, n, "f16", t + 1)
    scale[1] = 64.0
    b[1] = (b[1].double() / 4096).half()
    loud = torch.arange(t, device="cuda") % 3 == 0
    x[loud] = (x[loud].double() * 2000).half()
    wy, wu = want_forward(x, w, a, b, scale, index)[:2]
    assert float(wy.abs().max()) < 60000 and float(wu.abs().max()) < 60000
    assert float(wu[index == 1].abs().max()) * 64 > 70000
    y, u = A.forward(x, p, a, b, scale, index, keep=True)
    check_forward(y, u, x, w, a, b, scale, index, "f16")
    few = slice(0, 30)  # the same tokens, few at a time
    y2 = A.forward(x[few], p, a, b, scale, index[few])
    assert bool(y2.isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,d_in,d_out,n,r", [(40, 64, 512, 3, 16), (300, 515, 328, 4, 100), (333, 256, 2048, 3, 8), (2100, 1100, 264, 3, 16)])
def test_v_past_the_range_of_float16(gpu, t, d_in, d_out, n, r):
    """v under a loss scale is past 65504 for some tokens of one adapter, dx is not.  dx: the rounding of the weight and of v (u
    each, v's where it is inside the range), f32 sums, the output's own."""
    import torch

    from cdclq import adapters as A

    packed, w = layer(d_out, d_in, [4], 64, t)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(n, r, d_in, d_out, "f16", t)
    x, index = tokens(t, d_in, n, "f16", t + 1)
    dy, _ = tokens(t, d_out, n, "f16", t + 2)
    scale[1] = 40.0
    a[1] = (a[1].double() / 1024).half()
    b[1] = (b[1].double() * 4).half()
    loud = torch.arange(t, device="cuda") % 3 == 0
    dy[loud] = (dy[loud].double() * 500).half()
    uu, e, tiny = U["f16"], acc(d_out, r), 2.0 ** -25
    dd, ad = dy.double(), dy.double().abs()
    dx, bound = dd @ w, (uu + 2 * e) * (ad @ w.abs()) + 4 * tiny * ad.sum(1, keepdim=True) + tiny
    for i in range(n):
        rows = own(index, i)
        s, ai, bi = scale[i].double(), a[i].double(), b[i].double()
        v = s * (dd[rows] @ bi)
        assert (float(v.abs().max()) > 70000) == (i == 1)
        dx[rows] += v @ ai
        bound[rows] += (s * (ad[rows] @ bi.abs())) @ ai.abs() * (uu + 3 * e) + 4 * tiny * ai.abs().sum(0)
    assert float(dx.abs().max()) < 60000
    got = A.backward(dy, None, None, p, a, b, scale, index, need_da=False, need_db=False)[0]
    within(got, dx, bound + uu * dx.abs(), "dx")


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
