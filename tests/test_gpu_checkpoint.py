"""8-bit activation checkpoints against their definition in 64 bits.

A restored value is within s / 2 of x before its own rounding: s is off by one f32 rounding, x / s by another, so the
code differs from round(x / s) only within 2^-22 of a half, which adds 127 * 2^-22 s; the product's f32 rounding and the
type's add 2^-24 and u relative (u = 2^-8 bf16, 2^-11 f16, 2^-24 f32).
"""
import pytest

import conftest  # noqa: F401  (import paths)

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
SIZES = [(1, 1), (1, 128), (3, 127), (2, 129), (17, 200), (5, 1000), (300, 2048), (64, 136), (1, 4096), (1000, 8)]


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def activation(t, d, name, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    ranges = torch.exp(torch.randn(d, generator=g, device="cuda"))
    return (torch.randn(t, d, generator=g, device="cuda") * ranges).to(dtype_of(torch, name))


def scales_of(x):
    import torch

    return torch.stack([x[:, i:i + 128].double().abs().amax(1) for i in range(0, x.shape[1], 128)], 1) / 127


def wide(scales, d):
    return scales.repeat_interleave(128, 1)[:, :d]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,d", SIZES)
def test_save_and_restore(gpu, t, d, name):
    import torch
    from cdclq import checkpoint as C

    x = activation(t, d, name, t + d)
    c = C.save(x)
    s = scales_of(x)
    assert c.codes.shape == (t, d) and c.scales.shape == s.shape
    assert bool(((c.scales.double() - s).abs() <= 2.0 ** -24 * s).all())
    sw = wide(c.scales.double(), d)
    want = torch.where(sw > 0, x.double() / torch.where(sw > 0, sw, 1.0), 0.0)
    assert bool(((c.codes.double() - want).abs() <= 0.5 + 127 * 2.0 ** -22).all())
    back = C.restore(c)
    assert back.dtype == x.dtype
    exact = c.codes.double() * sw
    assert bool(((back.double() - exact).abs() <= (U[name] + 2.0 ** -24) * exact.abs() + 2.0 ** -25).all())
    assert bool(((back.double() - x.double()).abs() <= (0.5 + 127 * 2.0 ** -21) * sw + U[name] * x.double().abs() * 2).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,d", [(70, 4099), (33, 1004), (2000, 301), (40, 520)])
def test_rows_that_start_anywhere(gpu, t, d, name):
    """Codes and values do not depend on where the rows start: padded and shifted inputs, codes that begin on any byte."""
    import torch
    from cdclq import checkpoint as C

    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(t, d, generator=g, device="cuda").to(dtype_of(torch, name))
    pad = torch.zeros(t, -(-d // 128) * 128, dtype=torch.float64, device="cuda")
    pad[:, :d] = x.double()
    top = pad.reshape(t, -1, 128).abs().amax(2)
    want = C.save(x)
    s = want.scales.double()
    assert float((s - top / 127).abs().max()) <= 2.0 ** -24 * float(top.max())
    full = s.repeat_interleave(128, 1)[:, :d]
    assert bool(((want.codes.double() * full - x.double()).abs() <= full * (0.5 + 2.0 ** -15)).all())
    back = C.restore(want)
    exact = (want.codes.float() * want.scales.repeat_interleave(128, 1)[:, :d]).to(x.dtype)
    assert bool((back == exact).all())
    wide = torch.zeros(t, d + 5, dtype=x.dtype, device="cuda")
    for first in (0, 1, 5):
        part = wide[:, first:first + d]
        part.copy_(x)
        c = C.save(part)
        assert bool((c.codes == want.codes).all()) and bool((c.scales == want.scales).all())
    held = torch.empty(t * d + 3, dtype=torch.int8, device="cuda")
    moved = held[3:].view(t, d)
    moved.copy_(want.codes)
    assert bool((C.restore(C.Checkpoint(moved, want.scales, x.dtype)) == back).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_ties_zeros_and_non_finite_blocks(gpu, name):
    import torch
    from cdclq import checkpoint as C

    x = torch.zeros(4, 300, device="cuda")
    x[0, :128] = torch.arange(128, device="cuda") - 64 + 0.5  # scale 0.5: all exact
    x[0, 0] = 63.5
    x[1, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], device="cuda")  # ties go to even: 0, 2, -2
    x[2, 130] = float("nan")
    x[3, 5] = -float("inf")
    x[3, 299] = 2.0
    c = C.save(x.to(dtype_of(torch, name)))
    assert c.codes[1, :4].tolist() == [127, 0, 2, -2]
    assert not bool(c.codes[2].any()) and not bool(c.codes[1, 4:].any())
    assert c.scales[1].tolist() == [1.0, 0.0, 0.0]
    assert [bool(v.isnan()) for v in c.scales[2]] == [False, True, False]
    assert [bool(v.isnan()) for v in c.scales[3]] == [True, False, False] and c.codes[3, 299] == 127
    back = C.restore(c)
    assert bool(back[2, 128:256].isnan().all()) and not bool(back[2, :128].any()) and not bool(back[2, 256:].any())
    assert bool((back[0, :128].double() - x[0, :128].double()).abs().max() <= 0.25 + 0.25)
    tiny = torch.full((1, 128), 1e-44, device="cuda")  # below the smallest scale: nothing is left, nothing is NaN
    assert not bool(C.restore(C.save(tiny)).isnan().any())


@pytest.mark.gpu
def test_strides_streams_and_no_rows(gpu):
    import torch
    from cdclq import checkpoint as C

    x = activation(70, 515, "bf16", 1)
    ref = C.save(x)
    for view in (torch.cat([x, x], 1)[:, :515], torch.cat([x[:, :3], x], 1)[:, 3:], x.t().contiguous().t()):
        c = C.save(view)
        assert bool((c.codes == ref.codes).all()) and bool((c.scales == ref.scales).all())
    row = C.save(x[4:5].expand(6, 515))
    assert bool((row.codes == ref.codes[4]).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c = C.save(x, stream=s.cuda_stream)
    b = C.restore(c, stream=s.cuda_stream)
    s.synchronize()
    assert bool((c.codes == ref.codes).all()) and bool((b == C.restore(ref)).all())
    none = C.save(x[:0])
    assert none.codes.shape == (0, 515) and C.restore(none).shape == (0, 515)
    dw = C.weight_grad(torch.ones(0, 9, dtype=torch.bfloat16, device="cuda"), none)
    assert dw.shape == (9, 515) and not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d,n", [(1, 8, 8), (1, 1, 1), (3, 127, 5), (65, 200, 300), (127, 64, 129), (1025, 136, 72), (5000, 4096, 40)])
def test_weight_gradient(gpu, t, d, n, name):
    """|off| <= u of each restored value and of the result, and (t / 8 + 2) 2^-22 of the sum of |products| (f32 sums)."""
    import torch
    from cdclq import checkpoint as C

    c = C.save(activation(t, d, name, t))
    g = torch.Generator(device="cuda").manual_seed(n)
    dy = torch.randn(t, n, generator=g, device="cuda").to(dtype_of(torch, name))
    dw = C.weight_grad(dy, c)
    assert dw.dtype == dy.dtype and dw.shape == (n, d)
    x = c.codes.double() * wide(c.scales.double(), d)
    want, size = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
    u = U[name]
    bound = u * want.abs() + (u + 2.0 ** -23 + (t / 8 + 2) * 2.0 ** -22) * size * (1 + u) + 2.0 ** -25
    assert bool(((dw.double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_weight_gradient_against_differences(gpu):
    """d/dW of sum(dy * (x^ W^T)) by central differences in 64 bits: linear, so they are exact to rounding."""
    import torch
    from cdclq import checkpoint as C

    c = C.save(activation(37, 150, "f16", 3))
    x = c.codes.double() * wide(c.scales.double(), 150)
    g = torch.Generator(device="cuda").manual_seed(0)
    dy = torch.randn(37, 20, generator=g, device="cuda").half()
    dw = C.weight_grad(dy, c).double()
    w, v = torch.randn(20, 150, generator=g, device="cuda").double(), torch.randn(20, 150, generator=g, device="cuda").double()
    f = lambda m: (dy.double() * (x @ m.t())).sum()  # noqa: E731
    d = (f(w + 1e-3 * v) - f(w - 1e-3 * v)) / 2e-3
    size = (dy.double().abs().t() @ x.abs()) * v.abs()
    assert abs(float(d - (dw * v).sum())) <= float(3 * U["f16"] * size.sum() + 1e-6)


@pytest.mark.gpu
def test_refusals(gpu):
    import torch
    from cdclq import CdclqError
    from cdclq import checkpoint as C

    x = activation(8, 130, "bf16", 1)
    c = C.save(x)
    for call, word in [(lambda: C.save(x.double()), "unsupported"), (lambda: C.save(x[0]), "need shape"), (lambda: C.save(x.cpu()), "CUDA"),
                       (lambda: C.Checkpoint(c.codes, c.scales[:, :1], x.dtype), "need shape"),
                       (lambda: C.Checkpoint(c.codes.int(), c.scales, x.dtype), "need torch.int8"),
                       (lambda: C.Checkpoint(c.codes, c.scales, torch.float64), "unsupported"),
                       (lambda: C.weight_grad(x.float(), c), "float16 or bfloat16"), (lambda: C.weight_grad(x[:4], c), "need shape")]:
        with pytest.raises(CdclqError, match=word):
            call()


def test_refusals_without_a_device():
    import torch

    import cdclq
    from cdclq import checkpoint as C

    with pytest.raises(cdclq.CdclqError, match="CUDA tensor"):
        C.save(torch.zeros(2, 8))
    lib = cdclq.lib()
    assert lib.cdclq_checkpoint_save_device(None, 8, 7, 2, 8, None, None, None) == -3
    assert lib.cdclq_checkpoint_save_device(None, 8, 0, 2, 8, None, None, None) == -3
    assert lib.cdclq_checkpoint_save_device(None, 8, 0, 0, 8, None, None, None) == 0
    assert lib.cdclq_checkpoint_restore_device(None, None, 2, 8, None, 8, 1, None) == -3
    assert lib.cdclq_checkpoint_weight_grad_device(None, 8, 0, None, None, 2, 8, 8, None, 8, None, 0, None) == -3
    assert lib.cdclq_checkpoint_weight_grad_workspace(0, 8, 8) == 0
