"""What the gated block's nodes save for their backward passes, in other hands: saved-tensor hooks that bring tensors back
from the host, in another layout or wrongly, checkpointing, and several threads at once."""
import threading

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from flashmlp_amd import GatedFlashMLP, block_join, block_norm

pytestmark = pytest.mark.gpu
BF, FL = torch.bfloat16, torch.float32


def normal(*shape, dt=BF, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


class Case:
    """a call, its differentiable inputs and its outputs' gradients"""

    def __init__(self, what, dt=BF, rdt=None, seed=0):
        H, B, D, E = 3, 20, 32, 48
        n = lambda *s, k=0, t=dt: normal(*s, dt=t, seed=10 * seed + k)  # noqa: E731
        if what in ("module", "shared"):
            torch.manual_seed(seed)
            m = GatedFlashMLP(H, D, E, dtype=dt)
            x = n(B, D) if what == "shared" else n(H, B, D)
            self.inputs, self.call = [x, *m.parameters()], lambda x, *_: (m(x),)
        elif what == "join":
            self.inputs = [n(B, H * D, t=rdt or dt), n(H, B, D, k=1), n(H * D, k=2), n(2, H * D, k=3), n(H * D, k=4)]
            self.call = lambda r, o, w, g, p: block_join(r, o, w, g, 0.5, pre_weight=p)
        else:
            self.inputs, self.call = [n(B, H * D, t=rdt or dt), n(H * D, k=1)], lambda x, w: (block_norm(x, w, heads=H),)
        self.inputs = [t if t.is_leaf and t.requires_grad else t.requires_grad_(True) for t in self.inputs]

    def grads(self, outs):
        return torch.autograd.grad(outs, self.inputs, [torch.ones_like(o) * 0.5 + o.detach() for o in outs])

    def step(self):
        return self.grads(self.call(*self.inputs))


CASES = [("module", BF, None), ("module", FL, None), ("shared", BF, None), ("join", BF, None), ("join", BF, FL), ("norm", BF, FL)]


def same(a, b):
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


def other_layout(t):
    """t's values and sizes over other strides"""
    if t.dim() < 2:
        return torch.stack([t, t], -1)[..., 0]
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


def odd_base(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("what,dt,rdt", CASES)
def test_hooks_that_keep_values(what, dt, rdt):
    c = Case(what, dt, rdt)
    want = c.step()
    with save_on_cpu():
        same(c.step(), want)
    for unpack in (other_layout, odd_base, lambda t: torch._neg_view(-t)):
        with saved_tensors_hooks(lambda t: t, unpack):
            outs = c.call(*c.inputs)
            got = c.grads(outs)
        if unpack is odd_base and what in ("join", "norm"):  # (read element by element: another order of a row's sum)
            for a, b in zip(got, want):
                assert (a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm()
        else:
            same(got, want)


@pytest.mark.parametrize("what,dt,rdt", CASES)
@pytest.mark.parametrize("unpack", [lambda t: t.double(), lambda t: t[..., :1], lambda t: t.cpu(), lambda t: t[:1]])
def test_hooks_that_do_not(what, dt, rdt, unpack):
    c = Case(what, dt, rdt)
    with saved_tensors_hooks(lambda t: t, unpack):
        outs = c.call(*c.inputs)
        with pytest.raises(RuntimeError, match="came back"):
            c.grads(outs)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("what,dt,rdt", CASES)
def test_checkpointing(what, dt, rdt, reentrant):
    c = Case(what, dt, rdt)
    want = c.step()
    outs = checkpoint(c.call, *c.inputs, use_reentrant=reentrant)
    if not reentrant:
        same(c.grads(outs), want)
        return
    for t in c.inputs:
        t.grad = None
    torch.autograd.backward(outs, [torch.ones_like(o) * 0.5 + o.detach() for o in outs])
    same([t.grad for t in c.inputs], want)


def test_threads_on_streams_of_their_own():
    cases = [Case(w, dt, rdt, seed=i) for i, (w, dt, rdt) in enumerate(CASES)]
    want = [c.step() for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = cases[i].step()
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        same(a, b)
