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
import torch

from ._device import current_stream, half_code, operator, refuse, refuse_autograd, rows16, tensor, workspace
from ._lib import check, lib


def _head(h, w, target):
    tensor(h, "h", 2)
    code = half_code(h.dtype, "h")
    (t, d), dev = h.shape, h.get_device()
    tensor(w, "w", 2, h.dtype, None, dev)
    v = w.shape[0]
    tensor(w, "w", 2, shape=(v, d))
    tensor(target, "target", 1, torch.int64, (t,), dev)
    if d == 0 or v == 0:
        refuse("w: the head has no rows or no columns")
    return code, t, d, v


@operator
def linear_cross_entropy(h, w, target, *, stream=None):
    """(loss, lse), float32, one for each row of h.  Inputs that autograd would follow are refused."""
    code, t, d, v = _head(h, w, target)
    refuse_autograd("linear_cross_entropy", h, w)
    loss = torch.empty(t, dtype=torch.float32, device=h.device)
    lse = torch.empty_like(loss)
    if t == 0:
        return loss, lse
    L = lib()
    target = target.contiguous()
    hr, ldh = rows16(h)
    wr, ldw = rows16(w)
    need = L.cdclq_linear_cross_entropy_workspace(t, d, v)
    ws = workspace(need, h)
    check(L.cdclq_linear_cross_entropy_device(hr.data_ptr(), ldh, wr.data_ptr(), ldw, code, t, d, v, target.data_ptr(),
                                              loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), need, current_stream(h)))
    return loss, lse


@operator
def linear_cross_entropy_backward(h, w, target, lse, dloss, need_dh=True, need_dw=True, *, stream=None):
    """(dh, dw) for the gradient dloss of each token's loss; None in the place of one that is not needed."""
    code, t, d, v = _head(h, w, target)
    dev = h.get_device()
    tensor(lse, "lse", 1, torch.float32, (t,), dev)
    tensor(dloss, "dloss", 1, torch.float32, (t,), dev)
    dh = h.new_empty(t, d) if need_dh else None
    dw = h.new_empty(v, d) if need_dw else None
    if t == 0 or not (need_dh or need_dw):
        return dh, dw.zero_() if dw is not None else None
    L = lib()
    target, lse, dloss = target.contiguous(), lse.contiguous(), dloss.contiguous()
    hr, ldh = rows16(h)
    wr, ldw = rows16(w)
    need = L.cdclq_linear_cross_entropy_backward_workspace(t, d, v, need_dh, need_dw)
    ws = workspace(need, h)
    check(L.cdclq_linear_cross_entropy_backward_device(
        hr.data_ptr(), ldh, wr.data_ptr(), ldw, code, t, d, v, target.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
        dh.data_ptr() if need_dh else None, d, dw.data_ptr() if need_dw else None, d, ws.data_ptr(), need, current_stream(h)))
    return dh, dw
