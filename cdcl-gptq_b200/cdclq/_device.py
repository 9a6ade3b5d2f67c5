"""What the operators on device tensors share: argument checks, row layout, streams and the errors they raise."""
import ctypes

from ._lib import CdclqError, check, lib
from .abi import CDCLQ_ERR_ARG
from .io import DTYPE_BF16, DTYPE_F16

_HALF = None


def refuse(msg):
    raise CdclqError(CDCLQ_ERR_ARG, msg)


def half_code(torch, dt, what):
    """CDCLQ_DTYPE_* of a 16-bit type."""
    global _HALF
    if _HALF is None:
        _HALF = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
    code = _HALF.get(dt)
    if code is None:
        refuse("%s: need float16 or bfloat16, got %s" % (what, dt))
    return code


def tensor(x, what, dtype=None, shape=None, device=None):
    """Checks one tensor argument; `shape` entries that are None are free."""
    if not x.is_cuda:
        refuse("%s: need a CUDA tensor, got one on %s" % (what, x.device))
    if device is not None and x.device != device:
        refuse("%s: is on %s, the other arguments on %s" % (what, x.device, device))
    if dtype is not None and x.dtype != dtype:
        refuse("%s: need %s, got %s" % (what, dtype, x.dtype))
    if shape is not None and (x.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, x.shape))):
        refuse("%s: need shape %s, got %s" % (what, "(" + ", ".join("any" if s is None else str(s) for s in shape) + ")",
                                             tuple(x.shape)))
    return x


def ptr(x):
    return ctypes.c_void_p(None if x is None else x.data_ptr())


class on:
    """The device of the tensors as the current one, and the stream of a call: `stream` as the library's other
    calls take it (a CUDA stream's handle, 0 for the legacy default stream), or None for torch's current stream.
    Tensors that the call allocates, and its arguments, stay alive for work on a stream that is not torch's current
    one: keep() marks them."""

    def __init__(self, torch, device, stream):
        self.torch, self.device, self.stream = torch, device, stream

    def __enter__(self):
        torch = self.torch
        self.other = torch.cuda.current_device() != self.device.index
        if self.other:
            self.before = torch.cuda.current_device()
            torch.cuda.set_device(self.device)
        current = torch.cuda.current_stream().cuda_stream
        self.apart = self.stream is not None and self.stream != current
        self.handle = ctypes.c_void_p(self.stream if self.apart else current)
        return self

    def keep(self, *tensors):
        if self.apart:
            s = self.torch.cuda.ExternalStream(self.stream) if self.stream else self.torch.cuda.default_stream()
            for t in tensors:
                if t is not None:
                    t.record_stream(s)

    def __exit__(self, *exc):
        if self.other:
            self.torch.cuda.set_device(self.before)
        return False


def rows16(torch, x, call):
    """(x, elements from row to row) of a 2-d 16-bit matrix in the layout the kernels read: columns contiguous, rows
    starting on 16 bytes.  x itself where it has that layout (any such row stride), else a copy."""
    t, d = x.shape
    ld = x.stride(0) if t > 1 else max(d, 1)
    if (d <= 1 or x.stride(1) == 1) and ld >= d:
        pad = -(-d // 8) * 8
        if t <= 1 and x.data_ptr() % 16 == 0:
            return x, pad
        if ld % 8 == 0 and x.data_ptr() % 16 == 0:
            return x, ld
    else:
        x = x.contiguous()
        ld = d
        if ld % 8 == 0:
            return x, ld
    pad = -(-d // 8) * 8
    out = torch.empty((t, pad), dtype=x.dtype, device=x.device)
    check(lib().cdclq_align_rows_device(ptr(x), t, d, ld, ptr(out), pad, call.handle))
    call.keep(x, out)
    return out, pad


def workspace(torch, nbytes, device, call):
    w = torch.empty(max(1, nbytes), dtype=torch.uint8, device=device)
    call.keep(w)
    return w
