"""Low-rank adapters of many requests beside a shared projection in the packed format.

    w = PackedProjection.from_tensors(tensors, layer)      # the packed tensors, laid out once
    y = forward(x, w, a, b, scale, index)                  # serving: one token a request, prompts, or both mixed
    y, u = forward(x, w, a, b, scale, index, keep=True)    # training
    dx, da, db = backward(dy, x, u, w, a, b, scale, index) # x in full, or its 8-bit cdclq.checkpoint.Checkpoint

    u_t = A_i x_t,  y_t = W x_t + scale_i B_i u_t,  i = index[t]

x: t x d_in, float16 or bfloat16; a: n x r x d_in and b: n x d_out x r of the same type; scale: n float32 (alpha / r);
index: t int32, the adapter of each token, in any order; outside [0, n) the token has none.  Without adapters (a = b =
scale = index = None) the projection is applied alone.  Outputs have x's type, sums are float32.  What one request or one
adapter holds (a NaN among it) does not reach another.  The calls are asynchronous on `stream` (torch's current one if
None).

Up to 32 tokens the codes and u enter as they are.  More tokens, and backward, round the weight and scale u (or v, for dx) to
x's type first, as the tensor cores take them: the same token's y differs by such roundings between 32 and 33 tokens (in
bfloat16 2.4e-3 of y's norm off in place of 1.7e-3, its own rounding).  In float16 entries of scale u and v past 65504 are kept
in float32; weights past it are infinite there.  Autograd does not see these calls: forward refuses inputs that require
gradients, unless gradients are off.
"""
import ctypes
import functools

import torch

from ._device import HALF, current_stream, half_code, operator, refuse, refuse_autograd, rows16, tensor, workspace
from ._lib import check, lib
from .abi import CAdapters, CPackedLayer
from .checkpoint import Checkpoint


class PackedProjection:
    """A packed layer on the GPU, laid out for products with activations: `.d_out` x `.d_in`.

    qweight u8 [d_out, row_bytes], scales f16 and qzeros u8 [d_out, groups], perm i32 [d_in] and gbits u8 [groups] as the
    packed format has them (src/io.rs:244-270), CUDA tensors; gsize: columns of a group, 0 for one group of all.  They are
    copied into the layout and not kept; building synchronises."""

    def __init__(self, qweight, scales, qzeros, perm, gbits, gsize):
        tensor(qweight, "qweight", 2, torch.uint8)
        with torch.cuda.device(qweight.device):
            self._build(qweight, scales, qzeros, perm, gbits, gsize)

    def _build(self, qweight, scales, qzeros, perm, gbits, gsize):
        dev = qweight.get_device()
        tensor(perm, "perm", 1, torch.int32, None, dev)
        if not isinstance(gbits, torch.Tensor):
            refuse("gbits: need a tensor, got %s" % type(gbits).__name__)
        gb = gbits.cpu().to(torch.uint8).contiguous()
        d_out, d_in, ng, gsize = qweight.shape[0], perm.shape[0], gb.numel(), int(gsize)
        gsize = gsize or max(d_in, 1)
        if gsize < 0 or gb.dim() != 1 or ng != -(-d_in // min(gsize, max(d_in, 1))):
            refuse("gbits: need one width for each group of %d of %d columns, got %d" % (gsize, d_in, ng))
        tensor(scales, "scales", 2, torch.float16, (d_out, ng), dev)
        tensor(qzeros, "qzeros", 2, torch.uint8, (d_out, ng), dev)
        row_bytes = int(lib().cdclq_row_bytes(d_in, gsize, gb.data_ptr())) if d_in else 0
        if qweight.shape[1] != row_bytes:
            refuse("qweight: need %d bytes a row, got %d" % (row_bytes, qweight.shape[1]))
        self._c = CPackedLayer()
        self._ref = ctypes.addressof(self._c)
        need = lib().cdclq_packed_layer_bytes(d_out, d_in, gsize, gb.data_ptr())
        self._layout = torch.empty(max(1, need), dtype=torch.uint8, device=qweight.device)
        qweight, scales, qzeros, perm = (x.contiguous() for x in (qweight, scales, qzeros, perm))
        check(lib().cdclq_packed_layer_build(qweight.data_ptr(), scales.data_ptr(), qzeros.data_ptr(), perm.data_ptr(), d_out,
                                             d_in, gsize, gb.data_ptr(), self._layout.data_ptr(), need, self._ref,
                                             current_stream(qweight)))
        self.d_out, self.d_in, self.device = d_out, d_in, qweight.device
        # workspace bytes by the sizes of a call
        self._forward_need = functools.lru_cache(256)(functools.partial(lib().cdclq_projection_forward_workspace, self._ref))
        self._backward_need = functools.lru_cache(256)(functools.partial(lib().cdclq_projection_backward_workspace, self._ref))

    @staticmethod
    def from_tensors(tensors, layer, device="cuda"):
        """From the six tensors of a packed layer (cdclq.io.packed_tensors, or a packed file's), numpy or torch."""

        def get(suffix):
            k = "%s.%s" % (layer, suffix)
            if k not in tensors:
                refuse("%s: tensor not found" % k)
            return torch.as_tensor(tensors[k])

        q, s, z, p = (get(x).to(device) for x in ("qweight", "scales", "qzeros", "perm"))
        return PackedProjection(q, s, z, p, get("gbits"), int(get("gsize").reshape(-1)[0]))

    @property
    def tensors(self):
        return (self._layout,)

    @property
    def nbytes(self):
        return self._layout.numel()


def _matrix(x, cols):
    """The rows of an n x rows x columns tensor, as rows16 gives them."""
    if cols % 8 == 0 and x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, cols
    return rows16(x.reshape(-1, cols))


def _refuse_adapters(w, like, a, b, scale, index, t):
    """The message for adapters that do not fit."""
    if a is None or b is None or scale is None or index is None:
        refuse("adapters: a, b, scale and index go together")
    dev = like.get_device()
    tensor(a, "a", 3, like.dtype, None, dev)
    n, r = a.shape[:2]
    tensor(a, "a", 3, shape=(n, r, w.d_in))
    tensor(b, "b", 3, like.dtype, (n, w.d_out, r), dev)
    tensor(scale, "scale", 1, torch.float32, (n,), dev)
    tensor(index, "index", 1, torch.int32, (t,), dev)
    refuse("a: the rank must be > 0")


class _Adapters:
    """The adapters of one call, checked and in the layout the kernels read."""

    __slots__ = ("n", "r", "c", "ref", "held")

    def __init__(self, w, like, a, b, scale, index, t):
        self.n = self.r = 0
        self.ref, self.held = None, ()
        if a is None and b is None and scale is None and index is None:
            return
        dev, dt = like.get_device(), like.dtype
        try:
            n, r, d_in = a.shape
            fit = (d_in == w.d_in and r and b.shape == (n, w.d_out, r) and scale.shape == (n,) and index.shape == (t,) and a.dtype is dt
                   and b.dtype is dt and scale.dtype is torch.float32 and index.dtype is torch.int32 and a.get_device() == dev
                   and b.get_device() == dev and scale.get_device() == dev and index.get_device() == dev)
        except (AttributeError, ValueError):  # no tensor, or one of other dimensions
            fit = False
        if not fit:
            _refuse_adapters(w, like, a, b, scale, index, t)
        self.n, self.r = n, r
        if n == 0:
            return
        ar, lda = _matrix(a, d_in)
        br, ldb = _matrix(b, r)
        scale, index = scale.contiguous(), index.contiguous()
        self.held = (a, b, ar, br, scale, index)
        self.c = CAdapters(ar.data_ptr(), br.data_ptr(), lda, ldb, scale.data_ptr(), index.data_ptr(), n, r)
        self.ref = ctypes.addressof(self.c)


def _projection(w, x, what, backward):
    if not isinstance(w, PackedProjection):
        refuse("w: need a PackedProjection")
    cols = w.d_out if backward else w.d_in
    if not isinstance(x, torch.Tensor):
        tensor(x, what, 2)
    code = HALF.get(x.dtype)
    if code is None or x.get_device() != w.device.index or x.dim() != 2 or x.shape[1] != cols:
        tensor(x, what, 2, device=w.device.index)
        half_code(x.dtype, what)
        tensor(x, what, 2, shape=(x.shape[0], cols))
    return code, x.shape[0]


@operator
def forward(x, w, a=None, b=None, scale=None, index=None, keep=False, *, stream=None):
    """y (t x d_out); with keep also u (t x r), which backward() takes.  Inputs that autograd would follow are refused."""
    code, t = _projection(w, x, "x", False)
    L = lib()
    ad = _Adapters(w, x, a, b, scale, index, t)
    refuse_autograd("forward", x, a, b, scale)
    y = x.new_empty(t, w.d_out)
    u = x.new_empty(t, ad.r) if keep else None
    if t:
        xr, ldx = rows16(x)
        need = w._forward_need(t, ad.n, ad.r)
        ws = workspace(need, x)
        check(L.cdclq_projection_forward_device(w._ref, xr.data_ptr(), ldx, code, t, ad.ref, y.data_ptr(), w.d_out,
                                                u.data_ptr() if keep and ad.n else None, ws.data_ptr(), need, current_stream(x)))
        if keep and not ad.n:
            u.zero_()
    return (y, u) if keep else y


@operator
def backward(dy, x, u, w, a, b, scale, index, need_dx=True, need_da=True, need_db=True, *, stream=None):
    """(dx, da, db) for the gradient dy of y; None in the place of one that is not needed.  x: the forward's input or its
    Checkpoint; u: what forward(keep=True) returned."""
    code, t = _projection(w, dy, "dy", True)
    L, dev = lib(), dy.get_device()
    ad = _Adapters(w, dy, a, b, scale, index, t)
    dx = dy.new_empty(t, w.d_in) if need_dx else None
    da = dy.new_empty(ad.n, ad.r, w.d_in) if need_da and a is not None else None
    db = dy.new_empty(ad.n, w.d_out, ad.r) if need_db and a is not None else None
    codes = scales = xr = None
    ldx = 0
    if da is not None:
        if isinstance(x, Checkpoint):
            codes, scales = tensor(x.codes, "x", 2, shape=(t, w.d_in), device=dev), x.scales
        else:
            tensor(x, "x", 2, dy.dtype, (t, w.d_in), dev)
            xr = x if x.stride(1) == 1 and (t <= 1 or x.stride(0) >= w.d_in) else x.contiguous()
            ldx = xr.stride(0) if t > 1 else w.d_in
    if db is not None:
        u = tensor(u, "u", 2, dy.dtype, (t, ad.r), dev).contiguous()
    if t == 0:
        return dx, da.zero_() if da is not None else None, db.zero_() if db is not None else None
    at = lambda v: None if v is None else v.data_ptr()  # noqa: E731
    src, ld = rows16(dy)
    need = w._backward_need(t, ad.n, ad.r, bool(need_dx))
    ws = workspace(need, dy)
    check(L.cdclq_projection_backward_device(w._ref, src.data_ptr(), ld, code, t, ad.ref, at(xr), ldx, at(codes), at(scales),
                                             u.data_ptr() if db is not None else None, at(dx), w.d_in, at(da), at(db),
                                             ws.data_ptr(), need, current_stream(dy)))
    return dx, da, db
