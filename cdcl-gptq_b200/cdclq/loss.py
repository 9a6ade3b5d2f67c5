"""Softmax cross entropy of a linear head over a large vocabulary, without its logits, and its gradient.

    loss, lse = linear_cross_entropy(h, w, target)
    dh, dw = linear_cross_entropy_backward(h, w, target, lse, dloss)

h: t x d, the tokens' last hidden states; w: v x d, the head; both float16 or bfloat16 on one CUDA device.  target:
int64 labels; one outside [0, v) (such as -100) means that the token has none: its loss is 0 and it gets and gives no
gradient.  loss and lse are float32, one for each token; dloss is the gradient of each token's loss (for the mean over
labelled tokens: 1 / their number; in float16, times the loss scale).  The gradients have the inputs' type.

The logits exist a tile at a time in the tensor cores' accumulators; the backward pass computes them again, a piece of
the vocabulary at a time.  Matrices whose rows do not start on 16 bytes are copied first (a head of that kind is better
kept with padded rows: any row stride is taken as it is).  The calls are asynchronous on `stream` (torch's current one
if None).
"""
from ._device import half_code, on, ptr, refuse, rows16, tensor, workspace
from ._lib import check, lib


def _head(torch, h, w, target):
    tensor(h, "h", shape=(None, None))
    code = half_code(torch, h.dtype, "h")
    t, d = h.shape
    tensor(w, "w", h.dtype, (None, d), h.device)
    tensor(target, "target", torch.int64, (t,), h.device)
    if d == 0 or w.shape[0] == 0:
        refuse("w: the head has no rows or no columns")
    return code, t, d, w.shape[0]


def linear_cross_entropy(h, w, target, stream=None):
    """(loss, lse), float32, one for each row of h."""
    import torch

    code, t, d, v = _head(torch, h, w, target)
    with on(torch, h.device, stream) as call:
        loss = torch.empty(t, dtype=torch.float32, device=h.device)
        lse = torch.empty_like(loss)
        if t == 0:
            return loss, lse
        target = target.contiguous()
        hr, ldh = rows16(torch, h, call)
        wr, ldw = rows16(torch, w, call)
        ws = workspace(torch, lib().cdclq_linear_cross_entropy_workspace(t, d, v), h.device, call)
        check(lib().cdclq_linear_cross_entropy_device(ptr(hr), ldh, ptr(wr), ldw, code, t, d, v, ptr(target), ptr(loss),
                                                      ptr(lse), ptr(ws), ws.numel(), call.handle))
        call.keep(h, w, target, loss, lse)
        return loss, lse


def linear_cross_entropy_backward(h, w, target, lse, dloss, need_dh=True, need_dw=True, stream=None):
    """(dh, dw) for the gradient dloss of each token's loss; None in the place of one that is not needed."""
    import torch

    code, t, d, v = _head(torch, h, w, target)
    tensor(lse, "lse", torch.float32, (t,), h.device)
    tensor(dloss, "dloss", torch.float32, (t,), h.device)
    with on(torch, h.device, stream) as call:
        dh = torch.empty((t, d), dtype=h.dtype, device=h.device) if need_dh else None
        dw = torch.empty((v, d), dtype=h.dtype, device=h.device) if need_dw else None
        if t == 0 or not (need_dh or need_dw):
            return dh, dw.zero_() if dw is not None else None
        target, lse, dloss = target.contiguous(), lse.contiguous(), dloss.contiguous()
        hr, ldh = rows16(torch, h, call)
        wr, ldw = rows16(torch, w, call)
        need = lib().cdclq_linear_cross_entropy_backward_workspace(t, d, v, need_dh, need_dw)
        ws = workspace(torch, need, h.device, call)
        check(lib().cdclq_linear_cross_entropy_backward_device(ptr(hr), ldh, ptr(wr), ldw, code, t, d, v, ptr(target),
                                                               ptr(lse), ptr(dloss), ptr(dh), d, ptr(dw), d, ptr(ws),
                                                               ws.numel(), call.handle))
        call.keep(h, w, target, lse, dloss, dh, dw)
        return dh, dw
