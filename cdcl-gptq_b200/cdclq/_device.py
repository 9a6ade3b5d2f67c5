"""What the operators on device tensors share: argument checks, row layout, streams and the errors they raise."""
import functools

import torch

from ._lib import CdclqError, check, lib
from .abi import CDCLQ_ERR_ARG
from .io import DTYPE_BF16, DTYPE_F16

HALF = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
# absent from a torch built without CUDA
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def refuse(msg):
    raise CdclqError(CDCLQ_ERR_ARG, msg)


def half_code(dt, what):
    """CDCLQ_DTYPE_* of a 16-bit type."""
    code = HALF.get(dt)
    if code is None:
        refuse("%s: need float16 or bfloat16, got %s" % (what, dt))
    return code


def tensor(x, what, dims, dtype=None, shape=None, device=None):
    """Checks one tensor argument: on a CUDA device (the one with index `device` if given), `dims` dimensions, of type
    `dtype` and shape `shape` where given."""
    if not x.is_cuda:
        refuse("%s: need a CUDA tensor, got one on %s" % (what, x.device))
    if device is not None and x.get_device() != device:
        refuse("%s: is on %s, the other arguments on cuda:%d" % (what, x.device, device))
    if dtype is not None and x.dtype is not dtype:
        refuse("%s: need %s, got %s" % (what, dtype, x.dtype))
    if x.dim() != dims or (shape is not None and x.shape != shape):
        refuse("%s: need %s, got shape %s" % (what, "shape %s" % (tuple(shape),) if shape is not None else
                                             "shape of %d dimensions" % dims, tuple(x.shape)))
    return x


def on_device_of(position):
    """Runs an operator with the device of its argument at `position` as the current one."""

    def wrap(f):
        @functools.wraps(f)
        def g(*args, **kw):
            x = args[position] if len(args) > position else None
            if not isinstance(x, torch.Tensor):
                x = getattr(x, "codes", None)  # a Checkpoint
            if x is None or not x.is_cuda or x.get_device() == _current_device():
                return f(*args, **kw)
            with torch.cuda.device(x.device):
                return f(*args, **kw)

        return g

    return wrap


class Call:
    """The stream of one call: `stream` as the library's other calls take it (a CUDA stream's handle, 0 for the legacy
    default stream), or None for torch's current stream.  What a call allocates, and its arguments, stay alive for
    work on a stream that is not torch's current one: keep() marks them."""

    __slots__ = ("handle", "apart")

    def __init__(self, x, stream):
        current = _raw_stream(x.get_device())
        self.apart = stream is not None and stream != current
        self.handle = stream if self.apart else current

    def keep(self, *tensors):
        if self.apart:
            s = torch.cuda.ExternalStream(self.handle) if self.handle else torch.cuda.default_stream()
            for t in tensors:
                if t is not None:
                    t.record_stream(s)


def rows16(x, call):
    """(x, elements from row to row) of a 2-d 16-bit matrix in the layout the kernels read: columns contiguous, rows
    starting on 16 bytes.  x itself where it has that layout (any such row stride), else a copy."""
    t, d = x.shape
    ld, step = x.stride()
    if t <= 1:
        ld = -(-d // 8) * 8
    if (step == 1 or d <= 1) and ld >= d and ld % 8 == 0 and x.data_ptr() % 16 == 0:
        return x, ld
    if (step != 1 and d > 1) or (t > 1 and ld < d):
        x = x.contiguous()
        ld = d
    elif t <= 1:
        ld = max(d, 1)
    pad = -(-d // 8) * 8
    if ld == pad and x.data_ptr() % 16 == 0:
        return x, ld
    out = torch.empty((t, pad), dtype=x.dtype, device=x.device)
    check(lib().cdclq_align_rows_device(x.data_ptr(), t, d, ld, out.data_ptr(), pad, call.handle))
    call.keep(x, out)
    return out, pad


def workspace(nbytes, like, call):
    w = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    call.keep(w)
    return w
