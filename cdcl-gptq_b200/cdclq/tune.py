"""Low-rank adapters trained on a quantized layer and then served from it: adapters, checkpoint and loss together.

    python -m cdclq.tune [--tokens T] [--adapters N] [--rank R] [--steps K]

quantizes a random layer (quantize_layer, with the Hessian of its inputs), lays it out once, and teaches each of N adapters
to give, through the packed layer and a head, the labels that a layer of its own gives.  A training step keeps the layer's
input in 8 bits, never holds the logits, and never expands the layer beyond one call; afterwards the same calls serve one
token of every adapter at a time.  step() is the part to take along:

    loss, grads = step(w, head, x, target, a, b, scale, index)     # grads: da, db, dx and, if wanted, dhead
    logits = serve(w, head, x, a, b, scale, index)
"""
import argparse

import numpy as np
import torch

from . import adapters, checkpoint, loss


@torch.no_grad()
def step(w, head, x, target, a, b, scale, index, need_head=False, loss_scale=1.0):
    """The mean loss over the labelled tokens of head(w(x)), a 0-d tensor, and loss_scale times its gradients by name."""
    y, u = adapters.forward(x, w, a, b, scale, index, keep=True)
    kept = checkpoint.save(x)  # a deeper model lets go of x here
    each, lse = loss.linear_cross_entropy(y, head, target)
    labelled = (target >= 0) & (target < head.shape[0])
    share = labelled.float() / labelled.sum().clamp(min=1)
    dy, dhead = loss.linear_cross_entropy_backward(y, head, target, lse, share * loss_scale, need_dw=need_head)
    dx, da, db = adapters.backward(dy, kept, u, w, a, b, scale, index)
    return (each * share).sum(), {"da": da, "db": db, "dx": dx, "dhead": dhead}


@torch.no_grad()
def serve(w, head, x, a, b, scale, index):
    """The logits (t x v) of a few tokens, each with its own adapter."""
    return adapters.forward(x, w, a, b, scale, index) @ head.t()


def demo(tokens=512, d_in=256, d_out=192, vocab=500, n=4, rank=8, steps=40, seed=0, dtype=torch.bfloat16):
    """(losses of the steps, share of served tokens whose label comes first): before and after training."""
    from . import Config, quantize_layer
    from .io import packed_tensors

    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(d_out, d_in, generator=g) / d_in ** 0.5
    x = torch.randn(tokens, d_in, generator=g)
    ql, _ = quantize_layer(weight.numpy(), d_out, d_in, (x.t() @ x).numpy(), None, "demo", Config(bits=4, group=64, passes=1))
    w = adapters.PackedProjection.from_tensors(packed_tensors("demo", ql), "demo")
    head = torch.randn(vocab, d_out, generator=g)
    index = torch.randint(0, n, (tokens,), generator=g).int()
    # each adapter's own layer: the weight and a change of low rank
    change = torch.randn(n, d_out, rank, generator=g) @ torch.randn(n, rank, d_in, generator=g) / (rank * d_in) ** 0.5
    target = torch.empty(tokens, dtype=torch.int64)
    for i in range(n):
        mine = index == i
        target[mine] = (x[mine] @ (weight + change[i]).t() @ head.t()).argmax(1)
    scale = torch.ones(n, device="cuda")
    x, index, target, head = x.to("cuda", dtype), index.cuda(), target.cuda(), head.to("cuda", dtype)
    # 32-bit masters of the adapters; b starts at 0, so that training starts from the quantized layer
    a = (torch.randn(n, rank, d_in, generator=g) / d_in ** 0.5).cuda().requires_grad_()
    b = torch.zeros(n, d_out, rank, device="cuda").requires_grad_()
    opt = torch.optim.Adam([a, b], lr=2e-2)

    def right():
        """Served a token of every adapter at a time."""
        with torch.no_grad():
            first = [torch.nonzero(index == i)[:, 0][:16] for i in range(n)]
            rounds = [torch.stack([f[k] for f in first if k < len(f)]) for k in range(max(len(f) for f in first))]
            hits = [serve(w, head, x[r], a.to(dtype), b.to(dtype), scale, index[r]).argmax(1) == target[r] for r in rounds]
        return float(torch.cat(hits).float().mean())

    before, losses = right(), []
    for _ in range(steps):
        value, grads = step(w, head, x, target, a.detach().to(dtype), b.detach().to(dtype), scale, index)
        a.grad, b.grad = grads["da"].float(), grads["db"].float()
        opt.step()
        losses.append(value)
    return torch.stack(losses).cpu().numpy().astype(np.float64), (before, right())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--adapters", type=int, default=4)
    ap.add_argument("--rank", type=int, default=8)
    ap.add_argument("--steps", type=int, default=40)
    args = ap.parse_args(argv)
    losses, (before, after) = demo(tokens=args.tokens, n=args.adapters, rank=args.rank, steps=args.steps)
    print("loss %.3f -> %.3f over %d steps; labels served first: %.0f %% -> %.0f %%"
          % (losses[0], losses[-1], len(losses), 100 * before, 100 * after))


if __name__ == "__main__":
    main()
