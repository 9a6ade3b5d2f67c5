"""Activations kept in 8 bits between the forward and the backward pass, and the weight gradient computed from them.

    c = save(x)                    x: t x d, float16, bfloat16 or float32 on a CUDA device
    x^ = restore(c)                x's type
    dw = weight_grad(dy, c)        dy: t x n, float16 or bfloat16; dw = dy^T x^, n x d, dy's type

A block of 128 columns of a row shares the scale s = max |x| / 127 (float32); a value is kept as the nearest whole
multiple of it (ties to even), so it comes back within s / 2, or within 1e-43 where that is more (blocks whose largest
value is below 3e-41; below 9e-44 they come back as zeros).  A block of finite values comes back finite, one of zeros as
zeros; one that holds a NaN or an infinity comes back as NaN.  A checkpoint takes d + 4 ceil(d / 128) bytes a row: 52 % of
a 16-bit matrix.
The calls are asynchronous on `stream` (torch's current one if None).
"""
import torch

from ._device import HALF, current_stream, half_code, operator, refuse, rows16, tensor, workspace
from ._lib import check, lib
from .io import _dtype_code

BLOCK = 128


class Checkpoint:
    """`codes` int8 t x d, `scales` float32 t x ceil(d / 128), and the type that restore() gives back."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes, scales, dtype):
        tensor(codes, "codes", 2, torch.int8)
        t, d = codes.shape
        tensor(scales, "scales", 2, torch.float32, (t, -(-d // BLOCK)), codes.get_device())
        _dtype_code(torch, dtype)
        self.codes, self.scales, self.dtype = codes.contiguous(), scales.contiguous(), dtype

    @classmethod
    def _made(cls, codes, scales, dtype):
        c = cls.__new__(cls)
        c.codes, c.scales, c.dtype = codes, scales, dtype
        return c

    @property
    def tensors(self):
        return self.codes, self.scales

    @property
    def shape(self):
        return self.codes.shape


def _held(c):
    if not isinstance(c, Checkpoint):
        refuse("c: need a Checkpoint, got %s" % type(c).__name__)


def _code(dt):
    code = HALF.get(dt)
    return _dtype_code(torch, dt) if code is None else code


@operator
def save(x, *, stream=None):
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not x.is_cuda:
        tensor(x, "x", 2)
    code = _code(x.dtype)
    t, d = x.shape
    ld, step = x.stride()
    if d > 1 and step != 1 or t > 1 and ld < d:
        x, ld = x.contiguous(), d
    codes = torch.empty(t, d, dtype=torch.int8, device=x.device)
    scales = torch.empty(t, -(-d // BLOCK), dtype=torch.float32, device=x.device)
    check(lib().cdclq_checkpoint_save_device(x.data_ptr(), ld if t > 1 else d, code, t, d, codes.data_ptr(), scales.data_ptr(),
                                             current_stream(x)))
    return Checkpoint._made(codes, scales, x.dtype)


@operator
def restore(c, *, stream=None):
    _held(c)
    codes, scales = c.codes, c.scales
    t, d = codes.shape
    out = torch.empty(t, d, dtype=c.dtype, device=codes.device)
    check(lib().cdclq_checkpoint_restore_device(codes.data_ptr(), scales.data_ptr(), t, d, out.data_ptr(), d, _code(c.dtype),
                                                current_stream(codes)))
    return out


@operator
def weight_grad(dy, c, *, stream=None):
    """dy^T x^ with the restored values rounded to dy's type, as the operand of the tensor cores."""
    _held(c)
    (t, d), codes = c.shape, c.codes
    tensor(dy, "dy", 2, device=codes.get_device())
    code = half_code(dy.dtype, "dy")
    n = dy.shape[1]
    tensor(dy, "dy", 2, shape=(t, n))
    if d == 0 or n == 0:
        refuse("weight_grad: no columns")
    L = lib()
    dw = dy.new_empty(n, d)
    src, ld = rows16(dy) if t else (dy, n)
    need = L.cdclq_checkpoint_weight_grad_workspace(t, d, n)
    ws = workspace(need, dy)
    check(L.cdclq_checkpoint_weight_grad_device(src.data_ptr(), ld, code, codes.data_ptr(), c.scales.data_ptr(), t, d, n,
                                                dw.data_ptr(), d, ws.data_ptr(), need, current_stream(dy)))
    return dw
