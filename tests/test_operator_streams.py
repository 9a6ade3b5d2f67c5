"""Operators called with every argument by name run on the stream and the device that they are given."""
import contextlib

import pytest

import conftest  # noqa: F401  (import paths)


@pytest.mark.parametrize("by_name", [False, True])
@pytest.mark.parametrize("held", [False, True])
def test_a_call_reaches_its_stream_and_device(monkeypatch, by_name, held):
    """A tensor (or what holds some) that says it is on another device; the switches are recorded instead of made."""
    import torch

    from cdclq import _device as D

    class Far(torch.Tensor):
        is_cuda = property(lambda self: True)
        device = property(lambda self: torch.device("cuda", 3))

        def get_device(self):
            return 3

        def record_stream(self, s):
            seen.append(("kept for", s))

    class Holder:
        def __init__(self, *tensors):
            self.tensors = tensors

    @contextlib.contextmanager
    def note(kind, what):
        seen.append((kind, what))
        yield

    seen = []
    monkeypatch.setattr(D, "_current_device", lambda: 0)
    monkeypatch.setattr(D, "current_stream", lambda x: 7)
    monkeypatch.setattr(torch.cuda, "device", lambda d: note("device", d.index))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s: s)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: note("stream", s))
    x = torch.zeros(2).as_subclass(Far)
    f = D.operator(lambda x, keep=False: seen.append(("runs", None)))
    first = Holder(x) if held else x
    if by_name:
        f(keep=True, x=first, stream=99)
    else:
        f(first, keep=True, stream=99)
    assert seen == [("device", 3), ("stream", 99), ("runs", None), ("kept for", 99)]
    seen.clear()
    f(x=first) if by_name else f(first)
    assert seen == [("device", 3), ("runs", None)]


@pytest.mark.gpu
def test_every_argument_by_name(gpu, monkeypatch):
    """The streams' handles that reach the library, and the same results as calls by position."""
    import torch

    from cdclq import adapters as A
    from cdclq import checkpoint as C
    from cdclq import loss as L
    from test_gpu_adapters import bank, layer, tokens

    packed, _ = layer(48, 72, [4], 32, 3)
    w = A.PackedProjection(*packed)
    a, b, scale = bank(2, 4, 72, 48, "bf16", 1)
    x, index = tokens(40, 72, 2, "bf16", 2)
    dy, _ = tokens(40, 48, 2, "bf16", 3)
    g = torch.Generator(device="cuda").manual_seed(1)
    head = torch.randn(90, 72, generator=g, device="cuda").bfloat16()
    target = torch.randint(0, 90, (40,), generator=g, device="cuda")
    ones = torch.ones(40, device="cuda")
    y, u = A.forward(x, w, a, b, scale, index, True)
    each, lse = L.linear_cross_entropy(x, head, target)
    kept = C.save(x)
    want = [y, u, *A.backward(dy, x, u, w, a, b, scale, index), each, lse, *L.linear_cross_entropy_backward(x, head, target, lse, ones),
            kept.codes, kept.scales, C.restore(kept), C.weight_grad(dy, kept)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    seen = []
    for m in (A, C, L):
        real = m.current_stream
        monkeypatch.setattr(m, "current_stream", lambda t, real=real: seen.append(real(t)) or seen[-1])
    h = s.cuda_stream
    ad = dict(a=a, b=b, scale=scale, index=index)
    got = [*A.forward(x=x, w=w, keep=True, stream=h, **ad), *A.backward(dy=dy, x=x, u=u, w=w, stream=h, **ad),
           *L.linear_cross_entropy(h=x, w=head, target=target, stream=h),
           *L.linear_cross_entropy_backward(h=x, w=head, target=target, lse=lse, dloss=ones, stream=h)]
    c = C.save(x=x, stream=h)
    got += [c.codes, c.scales, C.restore(c=c, stream=h), C.weight_grad(dy=dy, c=c, stream=h)]
    s.synchronize()
    assert len(seen) == 7 and set(seen) == {h}
    assert all(bool((p == q).all()) for p, q in zip(got, want))
