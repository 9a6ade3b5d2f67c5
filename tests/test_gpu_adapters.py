"""The packed projection with low-rank adapters, forward and backward, against the definitions in 64 bits.

Tolerances: u = 2^-8 (bf16), 2^-11 (f16) for one rounding to nearest; acc = (k / 8 + 2) 2^-22 for an f32 sum of k products
(k the longest sum of the call) against the sum of |products|.  What is rounded: the expanded weight (or nothing, with few
tokens), u and scale u, v, every output; with a checkpoint v times the block's scale again.  f16: half of 2^-24 below
the normal range, for an operand times the sum of what it multiplies, and for the output.
"""
import numpy as np
import pytest

import conftest  # noqa: F401  (import paths)

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def layer(d_out, d_in, gbits, group, seed, act_order=True):
    """A random packed layer: the format's tensors and W in f64."""
    import torch

    rng = np.random.default_rng(seed)
    g = group if 0 < group < d_in else d_in
    ng = -(-d_in // g)
    gb = np.array([gbits[i % len(gbits)] for i in range(ng)], np.uint8)
    width = gb[np.arange(d_in) // g].astype(np.int64)
    codes = (rng.integers(0, 256, (d_out, d_in)) % (1 << width)).astype(np.uint8)
    stream = np.zeros((d_out, int(width.sum())), np.uint8)
    at = 0
    for j in range(d_in):
        for k in range(width[j]):
            stream[:, at] = (codes[:, j] >> k) & 1
            at += 1
    qweight = np.packbits(stream, axis=1, bitorder="little")
    zeros = (rng.integers(0, 256, (d_out, ng)) % (1 << gb.astype(np.int64))).astype(np.uint8)
    scales = (rng.uniform(0.5, 1.5, (d_out, ng)) / (1 << gb.astype(np.int64)) / d_in ** 0.5).astype(np.float16)
    perm = rng.permutation(d_in).astype(np.int32) if act_order else np.arange(d_in, dtype=np.int32)
    col = np.arange(d_in) // g
    w = np.zeros((d_out, d_in))
    w[:, perm] = scales[:, col].astype(np.float64) * (codes.astype(np.float64) - zeros[:, col])
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return (t(qweight), t(scales), t(zeros), t(perm), t(gb), g), t(w)


def bank(n, r, d_in, d_out, name, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = dtype_of(torch, name)
    a = (torch.randn(n, r, d_in, generator=g, device="cuda") / d_in ** 0.5).to(dt)
    b = (torch.randn(n, d_out, r, generator=g, device="cuda") / r ** 0.5).to(dt)
    return a, b, torch.rand(n, generator=g, device="cuda") + 0.5


def tokens(t, d, n, name, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, d, generator=g, device="cuda").to(dtype_of(torch, name))
    return x, torch.randint(-2, n + 1, (t,), generator=g, device="cuda").int()  # any order, some without an adapter


def own(index, i):
    return (index == i).nonzero()[:, 0]


def want_forward(x, w, a, b, scale, index):
    import torch

    xd, ax = x.double(), x.double().abs()
    r = a.shape[1]
    y, size = xd @ w.t(), ax @ w.abs().t()
    u = torch.zeros(len(x), r, dtype=torch.float64, device="cuda")
    usize = torch.zeros_like(u)
    add = torch.zeros_like(y)
    for i in range(a.shape[0]):
        rows = own(index, i)
        u[rows] = xd[rows] @ a[i].double().t()
        usize[rows] = ax[rows] @ a[i].double().abs().t()
        s = scale[i].double()
        y[rows] += s * (u[rows] @ b[i].double().t())
        add[rows] = s * (usize[rows] @ b[i].double().abs().t())
    return y, u, size, usize, add


def acc(*ks):
    return (max(ks) / 8 + 2) * 2.0 ** -22


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g over a bound of %.3g" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound[bad].min()))


def check_forward(y, kept, x, w, a, b, scale, index, name):
    u, tiny = U[name], 2.0 ** -25
    e = acc(w.shape[1], a.shape[1])
    wy, wu, size, usize, add = want_forward(x, w, a, b, scale, index)
    ax = x.double().abs().sum(1, keepdim=True) * (tiny if name == "f16" else 0)
    ab = b.double().abs().sum((1, 2)).max() * scale.max().double() * (2 * tiny if name == "f16" else 0)
    within(y, wy, u * wy.abs() + (u + e) * size + ax + (3 * u + 3 * e) * add + ab + tiny, "y")
    within(kept, wu, u * wu.abs() + e * usize + tiny, "u")
    bare = (index < 0) | (index >= a.shape[0])
    assert not bool(kept[bare].any())


CASES = [  # t, d_in, d_out, widths, group, adapters, rank
    (1, 64, 16, [4], 0, 1, 8), (1, 2056, 130, [3], 128, 3, 16), (7, 200, 1, [2], 64, 2, 1), (8, 40, 257, [8], 32, 3, 4),
    (9, 1000, 48, [4, 4, 8], 64, 40, 17), (17, 300, 31, [5, 6, 7], 32, 5, 3), (32, 512, 64, [3], 24, 3, 64),
    (33, 512, 64, [3], 128, 3, 16), (33, 16, 8, [2], 0, 1, 1), (64, 1000, 260, [4, 8], 128, 2, 24), (128, 72, 129, [7, 3], 40, 6, 8),
    (129, 328, 64, [6], 48, 4, 100), (300, 200, 515, [5], 100, 40, 16), (257, 2048, 1024, [3], 128, 3, 8), (130, 81, 77, [4], 16, 2, 5),
    (600, 64, 2048, [8, 2], 64, 3, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d_in,d_out,gbits,group,n,r", CASES)
def test_forward(gpu, t, d_in, d_out, gbits, group, n, r, name):
    from cdclq import adapters as A

    packed, w = layer(d_out, d_in, gbits, group, t + d_in)
    p = A.PackedProjection(*packed)
    assert (p.d_out, p.d_in) == (d_out, d_in)
    a, b, scale = bank(n, r, d_in, d_out, name, d_out)
    x, index = tokens(t, d_in, n, name, t)
    y, u = A.forward(x, p, a, b, scale, index, keep=True)
    assert y.dtype == x.dtype and y.shape == (t, d_out) and u.shape == (t, r)
    check_forward(y, u, x, w, a, b, scale, index, name)
    assert bool((A.forward(x, p, a, b, scale, index) == y).all())
    bare = A.forward(x, p)
    within(bare, x.double() @ w.t(), U[name] * (x.double() @ w.t()).abs() + (U[name] + acc(d_in)) * (x.double().abs() @ w.abs().t())
           + x.double().abs().sum(1, keepdim=True) * 2.0 ** -25 + 2.0 ** -25, "y alone")


def check_backward(got, dy, x, kept, w, a, b, scale, index, name, twice):
    import torch

    u, tiny = U[name], 2.0 ** -25
    e = acc(*dy.shape, w.shape[1], a.shape[1])
    dd, ad = dy.double(), dy.double().abs()
    dx, size = dd @ w, ad @ w.abs()
    add = torch.zeros_like(dx)
    small = 4 * tiny if name == "f16" else 0.0
    for i in range(a.shape[0]):
        rows = own(index, i)
        s, ai, bi = scale[i].double(), a[i].double(), b[i].double()
        v, vs = s * (dd[rows] @ bi), s * (ad[rows] @ bi.abs())
        dx[rows] += v @ ai
        add[rows] = vs @ ai.abs() * (u + 3 * e) + small * ai.abs().sum(0)
        da, das = v.t() @ x[rows], vs.t() @ x[rows].abs()
        within(got[1][i], da, u * da.abs() + ((2 if twice else 1) * u * (1 + u) + 3 * e) * das + small * x[rows].abs().sum(0) + tiny, "da")
        db, dbs = s * (dd[rows].t() @ kept[rows].double()), s * (ad[rows].t() @ kept[rows].double().abs())
        within(got[2][i], db, u * db.abs() + 2 * e * dbs + tiny, "db")
    within(got[0], dx, u * dx.abs() + (u + 2 * e) * size + small * ad.sum(1, keepdim=True) + add + tiny, "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d_in,d_out,gbits,group,n,r", CASES)
def test_backward(gpu, t, d_in, d_out, gbits, group, n, r, name):
    from cdclq import adapters as A
    from cdclq import checkpoint as C

    packed, w = layer(d_out, d_in, gbits, group, t + d_in)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(n, r, d_in, d_out, name, d_out)
    x, index = tokens(t, d_in, n, name, t)
    dy, _ = tokens(t, d_out, n, name, t + 1)
    kept = A.forward(x, p, a, b, scale, index, keep=True)[1]
    got = A.backward(dy, x, kept, p, a, b, scale, index)
    assert [g.shape for g in got] == [x.shape, a.shape, b.shape] and all(g.dtype == x.dtype for g in got)
    check_backward(got, dy, x.double(), kept, w, a, b, scale, index, name, False)
    c = C.save(x)
    xq = c.codes.double() * c.scales.double().repeat_interleave(128, 1)[:, :d_in]
    got8 = A.backward(dy, c, kept, p, a, b, scale, index)
    check_backward(got8, dy, xq, kept, w, a, b, scale, index, name, True)
    assert bool((got8[0] == got[0]).all()) and bool((got8[2] == got[2]).all())
    one = A.backward(dy, None, None, p, a, b, scale, index, need_da=False, need_db=False)
    assert bool((one[0] == got[0]).all()) and one[1] is None and one[2] is None
    two = A.backward(dy, x, kept, p, a, b, scale, index, need_dx=False)
    assert two[0] is None and bool((two[1] == got[1]).all()) and bool((two[2] == got[2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_many_tokens_of_one_adapter(gpu, name):
    """Adapters of thousands of tokens (their sums are split and joined), of a few, and of none."""
    import torch
    from cdclq import adapters as A

    packed, w = layer(96, 200, [4], 64, 5)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(5, 8, 200, 96, name, 1)
    x, _ = tokens(3000, 200, 5, name, 2)
    dy, _ = tokens(3000, 96, 5, name, 3)
    index = torch.full((3000,), 2, dtype=torch.int32, device="cuda")
    index[1000:1600] = 4
    index[2000:2003] = 0
    index[2500:2512] = -1
    y, kept = A.forward(x, p, a, b, scale, index, keep=True)
    check_forward(y, kept, x, w, a, b, scale, index, name)
    got = A.backward(dy, x, kept, p, a, b, scale, index)
    check_backward(got, dy, x.double(), kept, w, a, b, scale, index, name, False)
    assert not bool(got[1][1].any()) and not bool(got[2][3].any())
    again = A.backward(dy, x, kept, p, a, b, scale, index)
    assert all(bool((g == h).all()) for g, h in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [6, 200])
def test_requests_do_not_meet(gpu, t):
    """A NaN or an infinity in one request or one adapter stays there, forward and backward."""
    import torch
    from cdclq import adapters as A

    packed, w = layer(144, 136, [4], 64, 9)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(4, 16, 136, 144, "bf16", 1)
    x, _ = tokens(t, 136, 4, "bf16", 2)
    dy, _ = tokens(t, 144, 4, "bf16", 3)
    index = (torch.arange(t, device="cuda") % 4).int()
    y, kept = A.forward(x, p, a, b, scale, index, keep=True)
    got = A.backward(dy, x, kept, p, a, b, scale, index)
    bad_a, bad_b, bad_x, bad_dy, bad_scale = a.clone(), b.clone(), x.clone(), dy.clone(), scale.clone()
    bad_a[1], bad_b[1], bad_scale[1] = float("nan"), float("inf"), float("nan")
    bad_x[index == 2] = float("nan")
    bad_dy[index == 2] = -float("inf")
    y2, kept2 = A.forward(bad_x, p, bad_a, bad_b, bad_scale, index, keep=True)
    got2 = A.backward(bad_dy, bad_x, kept2, p, bad_a, bad_b, bad_scale, index)
    sound = (index == 0) | (index == 3)
    assert bool((y2[sound] == y[sound]).all()) and bool((kept2[sound] == kept[sound]).all())
    assert bool((got2[0][sound] == got[0][sound]).all())
    for i in (0, 3):
        assert bool((got2[1][i] == got[1][i]).all()) and bool((got2[2][i] == got[2][i]).all())
    assert bool(y2[index == 1].isnan().all()) and not bool(y2[sound].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [5, 70])
def test_strides_streams_and_no_tokens(gpu, t):
    import torch
    from cdclq import adapters as A

    packed, w = layer(100, 130, [3], 0, 2)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(3, 6, 130, 100, "f16", 1)
    x, index = tokens(t, 130, 3, "f16", 2)
    dy, _ = tokens(t, 100, 3, "f16", 3)
    y, kept = A.forward(x, p, a, b, scale, index, keep=True)
    got = A.backward(dy, x, kept, p, a, b, scale, index)
    wide = torch.cat([x[:, :3], x, x], 1)[:, 3:133]
    at, bt = a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 1).contiguous().transpose(0, 1)
    it = torch.stack([index, index], 1)[:, 0]
    assert bool((A.forward(wide, p, at, bt, scale, it) == y).all())
    dyt = dy.t().contiguous().t()
    assert all(bool((g == h).all()) for g, h in zip(got, A.backward(dyt, wide, kept, p, at, bt, scale, it)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y2, k2 = A.forward(x, p, a, b, scale, index, keep=True, stream=s.cuda_stream)
    got2 = A.backward(dy, x, k2, p, a, b, scale, index, stream=s.cuda_stream)
    s.synchronize()
    assert bool((y2 == y).all()) and all(bool((g == h).all()) for g, h in zip(got, got2))
    y0, u0 = A.forward(x[:0], p, a, b, scale, index[:0], keep=True)
    assert y0.shape == (0, 100) and u0.shape == (0, 6)
    none = A.backward(dy[:0], x[:0], u0, p, a, b, scale, index[:0])
    assert none[0].shape == (0, 130) and not bool(none[1].any()) and not bool(none[2].any())
    y1 = A.forward(x, p, a[:0], b[:0], scale[:0], index)
    assert bool((y1 == A.forward(x, p)).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = A.forward(x, p, a, b, scale, index)
    graph.replay()
    assert bool((captured == y).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [20, 60])
def test_gradient_against_differences(gpu, t):
    """Directional central differences of sum(dy * y) in 64 bits: y is bilinear, so they are exact to O(eps^2)."""
    import torch
    from cdclq import adapters as A

    packed, w = layer(40, 72, [4], 32, 2)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 72, 40, "f16", 1)
    x, index = tokens(t, 72, 2, "f16", 2)
    dy, _ = tokens(t, 40, 2, "f16", 3)
    kept = A.forward(x, p, a, b, scale, index, keep=True)[1]
    grads = A.backward(dy, x, kept, p, a, b, scale, index)
    f = lambda xx, aa, bb: (dy.double() * want_forward(xx, w, aa, bb, scale, index)[0]).sum()  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(7)
    for k, (value, grad) in enumerate(zip((x, a, b), grads)):
        v = torch.randn(value.shape, generator=g, device="cuda").double()
        args = lambda e: [q.double() + (e * v if j == k else 0) for j, q in enumerate((x, a, b))]  # noqa: E731
        d = (f(*args(1e-3)) - f(*args(-1e-3))) / 2e-3
        # each gradient is a sum of up to max(t, 72) terms, each within a few u of its size
        bound = 16 * U["f16"] * (grad.double().abs() * v.abs()).sum() + 1e-4
        assert abs(float(d - (grad.double() * v).sum())) <= float(bound)


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,kind", [(300, 300, "each its own"), (300, 200, "random"), (1290, 129, "random"), (1290, 700, "random"),
                                      (640, 3, "none"), (640, 1, "all"), (256, 4, "in turn")])
def test_adapters_among_a_tile_of_tokens(gpu, t, n, kind):
    """Tiles whose tokens have an adapter each, all the same, or none; more adapters than a CTA's threads."""
    import torch
    from cdclq import adapters as A

    packed, w = layer(72, 88, [4], 32, t + n)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(n, 4, 88, 72, "f16", 1)
    x, index = tokens(t, 88, n, "f16", 3)
    if kind == "none":
        index = torch.full_like(index, n)
    elif kind == "all":
        index = torch.zeros_like(index)
    elif kind != "random":
        index = (torch.arange(t, device="cuda") % n).int()
    y, u = A.forward(x, p, a, b, scale, index, keep=True)
    check_forward(y, u, x, w, a, b, scale, index, "f16")
    dy, _ = tokens(t, 72, n, "f16", 4)
    got = A.backward(dy, x, u, p, a, b, scale, index)
    check_backward(got, dy, x.double(), u, w, a, b, scale, index, "f16", False)
    again = A.backward(dy, x, u, p, a, b, scale, index)
    assert all(bool((g == h).all()) for g, h in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d_in,gbits,group", [(40, 14000, [4], 128), (40, 20000, [4], 128), (3, 20000, [3, 8], 96), (33, 40004, [3, 8], 100),
                                                (35, 60001, [2], 0)])
def test_long_rows(gpu, t, d_in, gbits, group, name):
    """Rows of which eight, four, two or one fit a CTA's shared memory."""
    from cdclq import adapters as A

    packed, w = layer(21, d_in, gbits, group, d_in)
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 8, d_in, 21, name, 1)
    x, index = tokens(t, d_in, 2, name, 3)
    y, u = A.forward(x, p, a, b, scale, index, keep=True)
    check_forward(y, u, x, w, a, b, scale, index, name)
    dy, _ = tokens(t, 21, 2, name, 4)
    check_backward(A.backward(dy, x, u, p, a, b, scale, index), dy, x.double(), u, w, a, b, scale, index, name, False)


@pytest.mark.gpu
def test_a_quantized_layer(gpu):
    """From quantize_layer through the packed tensors: the projection of unit vectors is the dequantized weight."""
    import torch

    import cdclq
    import oracle as orc
    from cdclq import adapters as A
    from cdclq.io import packed_tensors

    w, h = orc.problem(48, 256, 512, 3)
    for cfg in (cdclq.Config(bits=3, group=64, block=64, sub_block=32, passes=1),
                cdclq.Config(bits=4, group=64, block=64, sub_block=32, passes=1, skeleton_pct=25.0, skeleton_bits=8)):
        ql, _ = cdclq.quantize_layer(w, 48, 256, h, None, "l", cfg)
        p = A.PackedProjection.from_tensors(packed_tensors("l", ql), "l")
        dense = torch.from_numpy(ql.dequantize()).cuda()
        for rows in (torch.eye(256, device="cuda"), torch.eye(256, device="cuda")[100:120]):
            y = A.forward(rows.half(), p)
            assert bool((y.float() == (rows @ dense.t()).half().float()).all())


@pytest.mark.gpu
def test_refusals(gpu):
    import torch
    from cdclq import CdclqError
    from cdclq import adapters as A
    from cdclq import checkpoint as C

    packed, w = layer(16, 64, [4], 32, 2)
    q, s, z, perm, gb, g = packed
    p = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 64, 16, "bf16", 1)
    x, index = tokens(5, 64, 2, "bf16", 2)
    double = perm.clone()
    double[0] = double[1]
    high = z.clone()
    high[3, 1] = 16
    cases = [(lambda: A.PackedProjection(q[:, :-1], s, z, perm, gb, g), "bytes a row"), (lambda: A.PackedProjection(q, s.float(), z, perm, gb, g), "float16"),
             (lambda: A.PackedProjection(q, s, z, double, gb, g), "permutation"), (lambda: A.PackedProjection(q, s, high, perm, gb, g), "zero point"),
             (lambda: A.PackedProjection(q, s, z, perm + 1, gb, g), "permutation"), (lambda: A.PackedProjection(q, s, z, perm, gb[:1], g), "one width"),
             (lambda: A.PackedProjection(q[:, :8], s, z, perm, gb * 0 + 1, g), "2..=8"), (lambda: A.PackedProjection.from_tensors({}, "l"), "l.qweight: tensor not found"),
             (lambda: A.forward(x.float(), p), "float16 or bfloat16"), (lambda: A.forward(x[:, :32], p), "need shape"), (lambda: A.forward(x, w), "PackedProjection"),
             (lambda: A.forward(x, p, a), "go together"), (lambda: A.forward(x, p, a.half(), b, scale, index), "need torch.bfloat16"),
             (lambda: A.forward(x, p, a, b[:, :8], scale, index), "need shape"), (lambda: A.forward(x, p, a, b, scale, index.long()), "need torch.int32"),
             (lambda: A.forward(x, p, a, b, scale, index[:3]), "need shape"), (lambda: A.forward(x, p, a, b, scale.double(), index), "need torch.float32"),
             (lambda: A.forward(x, p, a[:, :0], b[:, :, :0], scale, index), "rank"), (lambda: A.forward(x.cpu(), p), "CUDA tensor")]
    dy = torch.zeros(5, 16, dtype=torch.bfloat16, device="cuda")
    u = torch.zeros(5, 4, dtype=torch.bfloat16, device="cuda")
    cases += [(lambda: A.backward(dy, x[:4], u, p, a, b, scale, index), "need shape"), (lambda: A.backward(dy, x, u[:, :2], p, a, b, scale, index), "need shape"),
              (lambda: A.backward(dy, C.save(x[:4]), u, p, a, b, scale, index), "need shape")]
    for call, word in cases:
        with pytest.raises(CdclqError, match=word):
            call()
    assert cdclq_status() == 0


def cdclq_status():
    import cdclq
    import torch

    torch.cuda.synchronize()
    return cdclq.lib().cdclq_operator_status()


def test_refusals_without_a_device():
    import ctypes

    import cdclq
    import torch
    from cdclq.abi import CAdapters, CPackedLayer
    from cdclq import adapters as A

    lib = cdclq.lib()
    with pytest.raises(cdclq.CdclqError, match="CUDA tensor"):
        A.PackedProjection(*[torch.zeros(2, 2, dtype=torch.uint8)] * 5, 2)
    gb = (ctypes.c_uint8 * 4)(3, 4, 8, 3)
    assert lib.cdclq_packed_layer_bytes(16, 200, 64, gb) > 0
    assert lib.cdclq_packed_layer_bytes(0, 200, 64, gb) == 0
    assert lib.cdclq_packed_layer_bytes(16, 200, 64, (ctypes.c_uint8 * 4)(3, 1, 8, 3)) == 0
    assert b"2..=8" in lib.cdclq_last_error()
    w = CPackedLayer()
    assert lib.cdclq_projection_forward_device(ctypes.byref(w), None, 8, 2, 1, None, None, 8, None, None, 0, None) == -3
    w.d_out, w.d_in, w.layout = 16, 64, 1
    assert lib.cdclq_projection_forward_device(ctypes.byref(w), None, 64, 0, 1, None, None, 16, None, None, 0, None) == -3
    ad = CAdapters(16, 16, 64, 8, 16, 16, 2, 0)
    assert lib.cdclq_projection_forward_device(ctypes.byref(w), 16, 64, 2, 1, ctypes.byref(ad), 16, 16, None, None, 0, None) == -3
    assert b"rank" in lib.cdclq_last_error()
    ad = CAdapters(16, 16, 60, 8, 16, 16, 2, 4)
    assert lib.cdclq_projection_backward_device(ctypes.byref(w), 16, 16, 2, 1, ctypes.byref(ad), None, 0, None, None, None, None, 0,
                                                None, None, None, 0, None) == -3
