"""Infinite logits in the vocabulary's loss: lse = log sum exp z is +inf for a row with a logit at +inf, and so is the loss
of every other label (of the infinite label it is inf - inf); a row with a NaN stays NaN; -inf adds nothing."""
import pytest

import conftest  # noqa: F401  (import paths)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("t,d,v", [(5, 64, 700), (400, 1100, 300), (4800, 32, 130), (3, 16, 1)])
def test_a_logit_at_infinity(gpu, t, d, v, name):
    import torch

    from cdclq import loss as L
    from test_gpu_loss import check_loss, head

    h, w, target, _ = head(t, d, v, name, t + v, unlabelled=0.1)
    h[:, 0] = torch.where(torch.arange(t, device="cuda") % 2 == 0, 1.5, -1.5)  # the sign decides the infinite logit's
    odd = v // 2
    w[odd] = 0
    w[odd, 0] = float("inf")
    nan = torch.zeros(t, dtype=torch.bool, device="cuda")
    if t > 4:
        h[4] = float("nan")
        nan[4] = True
    loss, lse = L.linear_cross_entropy(h, w, target)
    z = h.double() @ w.double().t()
    has = target >= 0
    up = (h[:, 0] > 0) & ~nan
    assert bool((lse[up] == float("inf")).all())
    assert bool((loss[up & has & (target != odd)] == float("inf")).all())
    assert bool(loss[up & (target == odd)].isnan().all())
    assert bool(lse[nan].isnan().all()) and not bool(loss[~has].any())
    rest = ~up & ~nan & (target != odd)
    if v == 1:  # the only logit is -inf: log of an empty sum
        assert bool((lse[~up & ~nan] == -float("inf")).all())
        return
    e = {"lse": torch.logsumexp(z, 1), "dz": (d / 8 + 2) * 2.0 ** -22 * (h.double().abs() @ torch.nan_to_num(w.double(), 0, 0, 0).abs().t()).amax(1)}
    e["loss"] = torch.where(has, e["lse"] - z.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0)
    check_loss({k: x[rest] for k, x in e.items()}, loss[rest], lse[rest])
