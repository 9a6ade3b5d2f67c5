"""Cross entropy of a linear head without its logits, against its definition in 64 bits.

Tolerances.  u = 2^-8 (bf16) or 2^-11 (f16) bounds the relative error of one rounding to nearest: p significant bits
(8 and 11, the leading one included) are spaced 2^(1-p) at 1, and half of that is 2^-p.  A logit z = sum of d products, exact in f32, added by the tensor core
in groups of 16 or fewer: each of at most d / 8 + 2 additions is off by at most 2^-22 of the sum of |products|:
    dz = (d / 8 + 2) 2^-22 |h| |w|
loss and lse: a shift of all logits by dz moves lse and the label's logit by at most dz each; exp, log and the sums add
relative errors of a few 2^-23 to a sum of positive terms (2^-18 allowed), the last subtraction one of 2^-23 of lse.
g = (p - onehot) dloss: p is off by a factor exp(2 dz) (1 + 2^-18), then rounded once: u |g|.  The products' f32 sums
add (k / 8 + 2) 2^-22 of the sum of |products|, the output's rounding u |result| (f16: or half of 2^-24).
"""
import pytest

import conftest  # noqa: F401  (import paths)

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def head(t, d, v, name, seed, unlabelled=0.2, std=2.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(t, d, generator=g, device="cuda").to(dtype_of(torch, name))
    w = (torch.randn(v, d, generator=g, device="cuda") * std / d ** 0.5).to(dtype_of(torch, name))
    target = torch.randint(0, v, (t,), generator=g, device="cuda")
    target[torch.rand(t, generator=g, device="cuda") < unlabelled] = -100
    dloss = torch.rand(t, generator=g, device="cuda") + 0.5
    return h, w, target, dloss


def expected(h, w, target, dloss):
    """loss, lse, g, dh, dw and the bounds' ingredients, in f64; rows of h without a label count as zero in dw."""
    import torch

    v = w.shape[0]
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    lse = torch.logsumexp(z, 1)
    has = (target >= 0) & (target < v)
    label = target.clamp(0, v - 1)
    loss = torch.where(has, lse - z.gather(1, label[:, None])[:, 0], 0.0)
    g = torch.exp(z - lse[:, None])
    g[torch.arange(len(target), device="cuda"), label] -= 1
    g = torch.where(has[:, None], g * torch.where(has, dloss.double(), 0.0)[:, None], 0.0)
    hl = torch.where(has[:, None], hd, 0.0)
    return {"loss": loss, "lse": lse, "g": g, "dh": g @ wd, "dw": g.t() @ hl, "hl": hl, "has": has,
            "dz": (h.shape[1] / 8 + 2) * 2.0 ** -22 * (hd.abs() @ wd.abs().t()).amax(1)}


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g over a bound of %.3g" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound.expand_as(off)[bad].min()))


def check_loss(e, loss, lse):
    bound = 2 * e["dz"] + 2.0 ** -18 + 2.0 ** -22 * e["lse"].abs()
    within(lse, e["lse"], bound, "lse")
    within(loss, e["loss"], bound, "loss")


def check_gradient(e, h, w, dh, dw, name):
    import torch

    u, tiny = U[name], (2.0 ** -25 if name == "f16" else 1e-38)
    rel = u + 2.0 ** -18 + 2 * e["dz"]
    # p of the label is subtracted from 1: what is off in p counts against |g| + 2 |dloss| there
    ag = e["g"].abs()
    dg = rel[:, None] * ag
    one = (2 * e["dz"] + 2.0 ** -18) * e["g"].abs().amax(1).clamp(min=0) * 2
    peak = torch.zeros_like(ag).scatter_(1, ag.argmax(1, keepdim=True), one[:, None])
    dg = dg + peak
    if name == "f16":  # below 2^-28 of the largest |dloss| the gain leaves subnormal values
        dg = dg + 2.0 ** -38 * float(e["g"].abs().max())
    if dh is not None:
        acc = (w.shape[0] / 8 + 2) * 2.0 ** -22
        within(dh, e["dh"], dg @ w.double().abs() + acc * (ag @ w.double().abs()) + u * e["dh"].abs() + tiny, "dh")
    if dw is not None:
        acc = (h.shape[0] / 8 + 2) * 2.0 ** -22
        ha = e["hl"].abs()
        within(dw, e["dw"], dg.t() @ ha + acc * (ag.t() @ ha) + u * e["dw"].abs() + tiny, "dw")


SIZES = [(1, 8, 1), (1, 64, 2), (2, 72, 255), (127, 64, 257), (129, 200, 1000), (300, 2048, 97), (40, 128, 5003),
         (513, 8, 777)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d,v", SIZES)
def test_loss_and_gradient(gpu, t, d, v, name):
    from cdclq import loss as L

    h, w, target, dloss = head(t, d, v, name, t * 7 + v)
    e = expected(h, w, target, dloss)
    loss, lse = L.linear_cross_entropy(h, w, target)
    check_loss(e, loss, lse)
    dh, dw = L.linear_cross_entropy_backward(h, w, target, lse, dloss)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype and dw.shape == w.shape
    check_gradient(e, h, w, dh, dw, name)
    only, none = L.linear_cross_entropy_backward(h, w, target, lse, dloss, need_dw=False)
    assert none is None and bool((only == dh).all())
    none, only = L.linear_cross_entropy_backward(h, w, target, lse, dloss, need_dh=False)
    assert none is None and bool((only == dw).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_many_pieces_of_the_vocabulary(gpu, name):
    """More tokens x classes than one piece of the gradient holds; the last piece is shorter."""
    from cdclq import loss as L

    h, w, target, dloss = head(8200, 64, 33001, name, 5)
    dloss = dloss * (1.0 if name == "bf16" else 64.0)
    e = expected(h, w, target, dloss)
    loss, lse = L.linear_cross_entropy(h, w, target)
    check_loss(e, loss, lse)
    dh, dw = L.linear_cross_entropy_backward(h, w, target, lse, dloss)
    check_gradient(e, h, w, dh, dw, name)


@pytest.mark.gpu
def test_strides_and_rows_off_16_bytes(gpu):
    """Padded rows, a column window, odd widths, a transposed head and broadcast tokens."""
    import torch
    from cdclq import loss as L

    h, w, target, dloss = head(65, 203, 509, "bf16", 3)
    ref = L.linear_cross_entropy_backward(h, w, target, L.linear_cross_entropy(h, w, target)[1], dloss)
    check_gradient(expected(h, w, target, dloss), h, w, *ref, "bf16")
    wide_h, wide_w = torch.randn(65, 300, device="cuda").bfloat16(), torch.randn(203, 600, device="cuda").bfloat16()
    wide_h[:, 5:208] = h
    wide_w[:, 3:512] = w.t()
    target2 = torch.stack([target, target], 1)[:, 0]  # strided
    for hv, wv in [(wide_h[:, 5:208], w), (h, wide_w[:, 3:512].t()), (wide_h[:, 5:208], wide_w[:, 3:512].t())]:
        lse = L.linear_cross_entropy(hv, wv, target2)[1]
        got = L.linear_cross_entropy_backward(hv, wv, target2, lse, dloss)
        assert all(bool((a == b).all()) for a, b in zip(ref, got))
    one = h[:1].expand(65, 203)
    e = expected(one, w, target, dloss)
    loss, lse = L.linear_cross_entropy(one, w, target)
    check_loss(e, loss, lse)
    check_gradient(e, one, w, *L.linear_cross_entropy_backward(one, w, target, lse, dloss), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t", [13, 51, 205])
def test_a_mean_is_as_exact_as_its_output(gpu, t, name):
    """dloss = 1 / t, whose rounding would fall on every label's entry alike.  With labels of small probability these entries
    make up half of each row of g and are exact; the others' roundings are random among thousands.  What is left is the
    outputs' own rounding: u / sqrt(3) of the norm at most, and 10 % of it for the rest."""
    import torch
    from cdclq import loss as L

    h, w, target, _ = head(t, 264, 6000, name, t)
    dloss = torch.full((t,), 1.0 / t, device="cuda")
    target = torch.where(target < 0, torch.zeros_like(target), target % 6000)
    _, lse = L.linear_cross_entropy(h, w, target)
    dh, dw = L.linear_cross_entropy_backward(h, w, target, lse, dloss)
    g = torch.softmax(h.double() @ w.double().t(), 1)
    g[torch.arange(t, device="cuda"), target] -= 1
    g /= t
    for got, want in ((dh, g @ w.double()), (dw, g.t() @ h.double())):
        off = (got.double() - want).norm() / want.norm()
        assert float(off) <= 1.1 * U[name] / 3 ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_tokens_without_a_label_reach_nothing(gpu, name):
    """NaN and infinities in h, lse and dloss of unlabelled tokens; labels beyond the vocabulary count as none."""
    import torch
    from cdclq import loss as L

    h, w, target, dloss = head(200, 64, 300, name, 11, unlabelled=0.3)
    target[3], target[5] = 300, 2 ** 40
    bad = (target < 0) | (target >= 300)
    h[bad] = float("nan")
    h[3] = float("inf")
    e = expected(h, w, target, dloss)
    loss, lse = L.linear_cross_entropy(h, w, target)
    assert bool((loss[bad] == 0).all())
    check_loss({k: e[k][~bad] for k in ("loss", "lse", "dz")}, loss[~bad], lse[~bad])
    dloss[bad] = float("inf")
    dh, dw = L.linear_cross_entropy_backward(h, w, target, lse, dloss)
    assert bool((dh[bad] == 0).all())
    e["dz"][bad] = 0
    check_gradient(e, torch.where(bad[:, None], 0, h), w, dh, dw, name)
    nothing = torch.full_like(target, -1)
    dh, dw = L.linear_cross_entropy_backward(h, w, nothing, lse, dloss)
    assert not bool(dh.any()) and not bool(dw.any())


@pytest.mark.gpu
def test_large_logits_and_infinite_ones(gpu):
    """Logits of hundreds; a class at -inf has no probability; a NaN in h stays in its own row's loss."""
    import torch
    from cdclq import loss as L

    h, w, target, _ = head(64, 32, 700, "f16", 2, unlabelled=0.0, std=60.0)
    e = expected(h, w, target, torch.ones(64, device="cuda"))
    loss, lse = L.linear_cross_entropy(h, w, target)
    check_loss(e, loss, lse)
    h = h.abs()
    w[17] = 0
    w[17, 0] = -float("inf")
    target[target == 17] = 3
    z = h.double() @ w.double().t()
    loss, lse = L.linear_cross_entropy(h, w, target)
    e["dz"] = (32 / 8 + 2) * 2.0 ** -22 * (h.double() @ torch.nan_to_num(w.double(), 0, 0, 0).abs().t()).amax(1)
    e["lse"] = torch.logsumexp(z, 1)
    e["loss"] = e["lse"] - z.gather(1, target[:, None])[:, 0]
    check_loss(e, loss, lse)
    h[9] = float("nan")
    again, _ = L.linear_cross_entropy(h, w, target)
    assert bool(again[9].isnan()) and bool((again[:9] == loss[:9]).all()) and bool((again[10:] == loss[10:]).all())


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """Central differences of the 64-bit loss in random directions."""
    import torch
    from cdclq import loss as L

    h, w, target, dloss = head(33, 40, 61, "f16", 8)
    dh, dw = L.linear_cross_entropy_backward(h, w, target, L.linear_cross_entropy(h, w, target)[1], dloss)

    def total(hd, wd):
        z = hd @ wd.t()
        has = target >= 0
        at = z.gather(1, target.clamp(min=0)[:, None])[:, 0]
        return (torch.where(has, torch.logsumexp(z, 1) - at, 0.0) * dloss.double()).sum()

    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        a = torch.randn(h.shape, generator=gen, device="cuda").double()
        b = torch.randn(w.shape, generator=gen, device="cuda").double()
        eps = 1e-4
        d = (total(h.double() + eps * a, w.double() + eps * b) - total(h.double() - eps * a, w.double() - eps * b)) / (2 * eps)
        s = (dh.double() * a).sum() + (dw.double() * b).sum()
        # each entry within 2u relative of the formula's, times the direction's; the differences' own error is O(eps^2)
        bound = 4 * U["f16"] * ((dh.double() * a).abs().sum() + (dw.double() * b).abs().sum()) + 1e-5
        assert abs(float(d - s)) <= float(bound)


@pytest.mark.gpu
def test_no_tokens_streams_and_repeats(gpu):
    import torch
    from cdclq import loss as L

    h, w, target, dloss = head(130, 64, 1000, "bf16", 4)
    empty = L.linear_cross_entropy(h[:0], w, target[:0])
    assert all(x.numel() == 0 for x in empty)
    dh, dw = L.linear_cross_entropy_backward(h[:0], w, target[:0], empty[1], dloss[:0])
    assert dh.shape == (0, 64) and dw.shape == w.shape and not bool(dw.any())
    loss, lse = L.linear_cross_entropy(h, w, target)
    dh, dw = L.linear_cross_entropy_backward(h, w, target, lse, dloss)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a = L.linear_cross_entropy(h, w, target, stream=s.cuda_stream)
    b = L.linear_cross_entropy_backward(h, w, target, a[1], dloss, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        c = L.linear_cross_entropy(h, w, target)
    s.synchronize()
    assert all(bool((x == y).all()) for x, y in zip(a + b + c, (loss, lse, dh, dw, loss, lse)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = L.linear_cross_entropy(h, w, target)
    h2 = h.clone()
    h.copy_(h.flip(0))
    graph.replay()
    assert bool((captured[1] == L.linear_cross_entropy(h, w, target)[1]).all())
    h.copy_(h2)


@pytest.mark.gpu
def test_refusals(gpu):
    import torch
    from cdclq import CdclqError
    from cdclq import loss as L

    h, w, target, dloss = head(8, 64, 100, "bf16", 4)
    lse = torch.zeros(8, device="cuda")
    for args, word in [((h.float(), w, target), "float16 or bfloat16"), ((h, w.half(), target), "need torch.bfloat16"),
                       ((h, w[:, :32], target), "need shape"), ((h, w, target.int()), "need torch.int64"),
                       ((h, w, target[:4]), "need shape"), ((h.cpu(), w, target), "CUDA tensor"), ((h[0], w, target), "need shape"),
                       ((h, w[:0], target), "no rows")]:
        with pytest.raises(CdclqError, match=word):
            L.linear_cross_entropy(*args)
    for args in [(h, w, target, lse.double(), dloss), (h, w, target, lse, dloss[:3])]:
        with pytest.raises(CdclqError):
            L.linear_cross_entropy_backward(*args)


def test_refusals_without_a_device():
    import torch

    import cdclq
    from cdclq import loss as L

    h, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(9, 8, dtype=torch.bfloat16)
    with pytest.raises(cdclq.CdclqError, match="CUDA tensor") as e:
        L.linear_cross_entropy(h, w, torch.zeros(4, dtype=torch.int64))
    assert e.value.code == -3
    lib = cdclq.lib()
    assert lib.cdclq_linear_cross_entropy_workspace(0, 8, 9) == 0
    assert lib.cdclq_linear_cross_entropy_device(None, 8, None, 8, 0, 4, 8, 9, None, None, None, None, 0, None) == -3
    assert b"f16 or bf16" in lib.cdclq_last_error()
    assert lib.cdclq_linear_cross_entropy_device(None, 8, None, 8, 2, 4, 8, 9, None, None, None, None, 0, None) == -3
    assert lib.cdclq_linear_cross_entropy_backward_device(None, 4, None, 8, 2, 4, 8, 9, None, None, None, None, 8, None, 8,
                                                          None, 0, None) == -3
