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
    if not isinstance(x, torch.Tensor):
        refuse("%s: need a tensor, got %s" % (what, type(x).__name__))
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


def refuse_autograd(what, *inputs):
    """Refuses inputs that autograd would follow: it cannot see through the library's kernels, and their gradients would be
    lost without a word."""
    if torch.is_grad_enabled():
        for x in inputs:
            if x is not None and x.requires_grad:
                refuse("%s: an input requires a gradient, which comes from %s(), not from autograd: call it under torch.no_grad() "
                       "or with detached tensors" % (what, "linear_cross_entropy_backward" if what == "linear_cross_entropy" else "backward"))


def _tensors(args):
    for a in args:
        if isinstance(a, torch.Tensor):
            yield a
        elif a is not None:
            yield from getattr(a, "tensors", ())  # a Checkpoint, a PackedProjection


def operator(f):
    """An operator on the tensors of one CUDA device: runs with the device of its first tensor, by position or by name, as the
    current one and on `stream`, a CUDA stream's handle as the library's other calls take it (0: the legacy default stream),
    or on torch's current stream if None.  Results belong to that stream, as torch's own would."""

    @functools.wraps(f)
    def g(*args, stream=None, **kw):
        x = args[0] if args else None
        if not isinstance(x, torch.Tensor):
            x = next(_tensors((*args, *kw.values())), None)
        if x is None or not x.is_cuda or (stream is None and x.get_device() == _current_device()):
            return f(*args, **kw)
        with torch.cuda.device(x.device):
            if stream is None or stream == current_stream(x):
                return f(*args, **kw)
            s = torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
            with torch.cuda.stream(s):
                out = f(*args, **kw)
            for t in _tensors((*args, *kw.values())):
                t.record_stream(s)  # their memory is not reused while the stream reads it
            return out

    return g


def current_stream(x):
    """Handle of torch's current stream on x's device."""
    return _raw_stream(x.get_device())


def rows16(x):
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
    out = x.new_empty(t, pad)
    check(lib().cdclq_align_rows_device(x.data_ptr(), t, d, ld, out.data_ptr(), pad, current_stream(x)))
    return out, pad


def workspace(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
