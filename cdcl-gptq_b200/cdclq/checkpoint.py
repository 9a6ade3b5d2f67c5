"""Activations kept in 8 bits between the forward and the backward pass, and the weight gradient computed from them.

    c = save(x)                    x: t x d, float16, bfloat16 or float32 on a CUDA device
    x^ = restore(c)                x's type
    dw = weight_grad(dy, c)        dy: t x n, float16 or bfloat16; dw = dy^T x^, n x d, dy's type

A block of 128 columns of a row shares the scale s = max |x| / 127 (float32); a value is kept as the nearest whole
multiple of it (ties to even), so it comes back within s / 2.  A block of zeros comes back as zeros; one that holds a
NaN or an infinity comes back as NaN.  A checkpoint takes d + 4 ceil(d / 128) bytes a row: 52 % of a 16-bit matrix.
The calls are asynchronous on `stream` (torch's current one if None).
"""
from ._device import half_code, on, ptr, refuse, rows16, tensor, workspace
from ._lib import check, lib
from .io import _dtype_code

BLOCK = 128


class Checkpoint:
    """`codes` int8 t x d, `scales` float32 t x ceil(d / 128), and the type that restore() gives back."""

    def __init__(self, codes, scales, dtype):
        import torch

        tensor(codes, "codes", torch.int8, (None, None))
        t, d = codes.shape
        tensor(scales, "scales", torch.float32, (t, -(-d // BLOCK)), codes.device)
        _dtype_code(torch, dtype)
        self.codes, self.scales, self.dtype = codes.contiguous(), scales.contiguous(), dtype

    @property
    def shape(self):
        return self.codes.shape


def save(x, stream=None):
    import torch

    tensor(x, "x", shape=(None, None))
    code = _dtype_code(torch, x.dtype)
    t, d = x.shape
    with on(torch, x.device, stream) as call:
        if d > 1 and x.stride(1) != 1 or t > 1 and x.stride(0) < d:
            x = x.contiguous()
        codes = torch.empty((t, d), dtype=torch.int8, device=x.device)
        scales = torch.empty((t, -(-d // BLOCK)), dtype=torch.float32, device=x.device)
        check(lib().cdclq_checkpoint_save_device(ptr(x), x.stride(0) if t > 1 else d, code, t, d, ptr(codes), ptr(scales),
                                                 call.handle))
        call.keep(x, codes, scales)
        return Checkpoint(codes, scales, x.dtype)


def restore(c, stream=None):
    import torch

    t, d = c.shape
    with on(torch, c.codes.device, stream) as call:
        out = torch.empty((t, d), dtype=c.dtype, device=c.codes.device)
        check(lib().cdclq_checkpoint_restore_device(ptr(c.codes), ptr(c.scales), t, d, ptr(out), d,
                                                    _dtype_code(torch, c.dtype), call.handle))
        call.keep(c.codes, c.scales, out)
        return out


def weight_grad(dy, c, stream=None):
    """dy^T x^ with the restored values rounded to dy's type, as the operand of the tensor cores."""
    import torch

    tensor(dy, "dy", shape=(c.shape[0], None), device=c.codes.device)
    code = half_code(torch, dy.dtype, "dy")
    (t, d), n = c.shape, dy.shape[1]
    if d == 0 or n == 0:
        refuse("weight_grad: no columns")
    with on(torch, dy.device, stream) as call:
        dw = torch.empty((n, d), dtype=dy.dtype, device=dy.device)
        src, ld = rows16(torch, dy, call) if t else (dy, n)
        ws = workspace(torch, lib().cdclq_checkpoint_weight_grad_workspace(t, d, n), dy.device, call)
        check(lib().cdclq_checkpoint_weight_grad_device(ptr(src), ld, code, ptr(c.codes), ptr(c.scales), t, d, n, ptr(dw), d,
                                                        ptr(ws), ws.numel(), call.handle))
        call.keep(dy, c.codes, c.scales, dw)
        return dw
