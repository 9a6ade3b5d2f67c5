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
"""
import ctypes

from ._device import half_code, on, ptr, refuse, rows16, tensor, workspace
from ._lib import check, lib
from .abi import CAdapters, CPackedLayer
from .checkpoint import Checkpoint


class PackedProjection:
    """A packed layer on the GPU, laid out for products with activations: `.d_out` x `.d_in`.

    qweight u8 [d_out, row_bytes], scales f16 and qzeros u8 [d_out, groups], perm i32 [d_in] and gbits u8 [groups] as the
    packed format has them (src/io.rs:244-270), CUDA tensors; gsize: columns of a group.  They are copied into the layout
    and not kept; building synchronises."""

    def __init__(self, qweight, scales, qzeros, perm, gbits, gsize, stream=None):
        import torch

        tensor(qweight, "qweight", torch.uint8, (None, None))
        dev = qweight.device
        tensor(perm, "perm", torch.int32, (None,), dev)
        gb = gbits.cpu().to(torch.uint8).contiguous()
        d_out, d_in, ng, gsize = qweight.shape[0], perm.shape[0], gb.numel(), int(gsize)
        if gsize <= 0 or gb.dim() != 1 or ng != -(-d_in // min(gsize, max(d_in, 1))):
            refuse("gbits: need one width for each group of %d of %d columns, got %d" % (gsize, d_in, ng))
        tensor(scales, "scales", torch.float16, (d_out, ng), dev)
        tensor(qzeros, "qzeros", torch.uint8, (d_out, ng), dev)
        row_bytes = int(lib().cdclq_row_bytes(d_in, gsize, ptr(gb))) if d_in else 0
        if qweight.shape[1] != row_bytes:
            refuse("qweight: need %d bytes a row, got %d" % (row_bytes, qweight.shape[1]))
        self._c = CPackedLayer()
        with on(torch, dev, stream) as call:
            need = lib().cdclq_packed_layer_bytes(d_out, d_in, gsize, ptr(gb))
            self._layout = torch.empty(max(1, need), dtype=torch.uint8, device=dev)
            qweight, scales, qzeros, perm = (x.contiguous() for x in (qweight, scales, qzeros, perm))
            check(lib().cdclq_packed_layer_build(ptr(qweight), ptr(scales), ptr(qzeros), ptr(perm), d_out, d_in, gsize, ptr(gb),
                                                 ptr(self._layout), need, ctypes.byref(self._c), call.handle))
            call.keep(self._layout, qweight, scales, qzeros, perm)
        self.d_out, self.d_in, self.device = d_out, d_in, dev

    @staticmethod
    def from_tensors(tensors, layer, device="cuda"):
        """From the six tensors of a packed layer (cdclq.io.packed_tensors, or a packed file's), numpy or torch."""
        import torch

        def get(suffix):
            k = "%s.%s" % (layer, suffix)
            if k not in tensors:
                refuse("%s: tensor not found" % k)
            return torch.as_tensor(tensors[k])

        q, s, z, p = (get(x).to(device) for x in ("qweight", "scales", "qzeros", "perm"))
        return PackedProjection(q, s, z, p, get("gbits"), int(get("gsize").reshape(-1)[0]))

    @property
    def nbytes(self):
        return self._layout.numel()


class _Call:
    """The adapters of one call, checked and in the layout the kernels read."""

    def __init__(self, torch, w, like, a, b, scale, index, t, call):
        given = [v is not None for v in (a, b, scale, index)]
        if any(given) and not all(given):
            refuse("adapters: a, b, scale and index go together")
        self.n = self.r = 0
        self.c, self.held = None, ()
        if not any(given):
            return
        tensor(a, "a", like.dtype, (None, None, w.d_in), like.device)
        self.n, self.r = a.shape[0], a.shape[1]
        tensor(b, "b", like.dtype, (self.n, w.d_out, self.r), like.device)
        tensor(scale, "scale", torch.float32, (self.n,), like.device)
        tensor(index, "index", torch.int32, (t,), like.device)
        if self.n == 0:
            return
        if self.r == 0:
            refuse("a: the rank must be > 0")
        ar, lda = rows16(torch, a.reshape(-1, w.d_in), call)
        br, ldb = rows16(torch, b.reshape(-1, self.r), call)
        scale, index = scale.contiguous(), index.contiguous()
        self.held = (a, b, ar, br, scale, index)
        self.c = ctypes.byref(CAdapters(ar.data_ptr(), br.data_ptr(), lda, ldb, scale.data_ptr(), index.data_ptr(), self.n, self.r))


def _projection(torch, w, x, what, cols):
    if not isinstance(w, PackedProjection):
        refuse("w: need a PackedProjection")
    tensor(x, what, shape=(None, cols), device=w.device)
    return half_code(torch, x.dtype, what)


def forward(x, w, a=None, b=None, scale=None, index=None, keep=False, stream=None):
    """y (t x d_out); with keep also u (t x r), which backward() takes."""
    import torch

    code = _projection(torch, w, x, "x", w.d_in if isinstance(w, PackedProjection) else None)
    t = x.shape[0]
    with on(torch, x.device, stream) as call:
        ad = _Call(torch, w, x, a, b, scale, index, t, call)
        y = torch.empty((t, w.d_out), dtype=x.dtype, device=x.device)
        u = torch.empty((t, ad.r), dtype=x.dtype, device=x.device) if keep else None
        if t:
            xr, ldx = rows16(torch, x, call)
            ws = workspace(torch, lib().cdclq_projection_forward_workspace(ctypes.byref(w._c), t, ad.n, ad.r), x.device, call)
            check(lib().cdclq_projection_forward_device(ctypes.byref(w._c), ptr(xr), ldx, code, t, ad.c, ptr(y), w.d_out,
                                                        ptr(u) if ad.n else None, ptr(ws), ws.numel(), call.handle))
            if keep and not ad.n:
                u.zero_()
            call.keep(x, xr, y, u, w._layout, *ad.held)
        return (y, u) if keep else y


def backward(dy, x, u, w, a, b, scale, index, need_dx=True, need_da=True, need_db=True, stream=None):
    """(dx, da, db) for the gradient dy of y; None in the place of one that is not needed.  x: the forward's input or its
    Checkpoint; u: what forward(keep=True) returned."""
    import torch

    code = _projection(torch, w, dy, "dy", w.d_out if isinstance(w, PackedProjection) else None)
    t = dy.shape[0]
    with on(torch, dy.device, stream) as call:
        ad = _Call(torch, w, dy, a, b, scale, index, t, call)
        new = lambda need, shape: torch.empty(shape, dtype=dy.dtype, device=dy.device) if need else None  # noqa: E731
        dx = new(need_dx, (t, w.d_in))
        da = new(need_da and a is not None, (ad.n, ad.r, w.d_in))
        db = new(need_db and a is not None, (ad.n, w.d_out, ad.r))
        codes = scales = xr = None
        ldx = 0
        if da is not None:
            if isinstance(x, Checkpoint):
                tensor(x.codes, "x", shape=(t, w.d_in), device=dy.device)
                codes, scales = x.codes, x.scales
            else:
                tensor(x, "x", dy.dtype, (t, w.d_in), dy.device)
                xr = x if x.stride(1) == 1 and (t <= 1 or x.stride(0) >= w.d_in) else x.contiguous()
                ldx = xr.stride(0) if t > 1 else w.d_in
        if db is not None:
            u = tensor(u, "u", dy.dtype, (t, ad.r), dy.device).contiguous()
        if t == 0:
            return dx, da.zero_() if da is not None else None, db.zero_() if db is not None else None
        src, ld = rows16(torch, dy, call)
        ws = workspace(torch, lib().cdclq_projection_backward_workspace(ctypes.byref(w._c), t, ad.n, ad.r, need_dx), dy.device, call)
        check(lib().cdclq_projection_backward_device(ctypes.byref(w._c), ptr(src), ld, code, t, ad.c, ptr(xr), ldx, ptr(codes),
                                                     ptr(scales), ptr(u if db is not None else None), ptr(dx), w.d_in, ptr(da),
                                                     ptr(db), ptr(ws), ws.numel(), call.handle))
        call.keep(dy, xr, codes, scales, u, dx, da, db, w._layout, *ad.held)
        return dx, da, db
