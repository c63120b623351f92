"""The gated block's operators under torch.jit.trace: the graph holds each as one operation, which computes on new
inputs, and not the allocations of one call. What has no operation to stand there refuses."""
import pytest
import torch

from flashmlp_amd import (GatedFlashMLP, block_join, block_join_bwd, block_join_fwd, block_norm, clip_grads,
                          flashmlp_gated_bwd, flashmlp_gated_fwd, grad_norm)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def normal(*shape, dt=BF, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


def module(H=3, D=32, E=48, dt=BF):
    torch.manual_seed(0)
    return GatedFlashMLP(H, D, E, dtype=dt)


def poison():
    """what an uninitialised tensor of the next calls would hold"""
    for n in (1 << 10, 1 << 14, 1 << 16, 1 << 20):
        torch.full((n,), float("nan"), device="cuda")


@pytest.mark.parametrize("shape", [(3, 20, 32), (20, 32)])
@pytest.mark.parametrize("grad", [False, True])
def test_trace_of_the_module(shape, grad):
    m = module().requires_grad_(grad)
    f = torch.jit.trace(m, (normal(*shape),))
    for seed in (1, 2):
        x = normal(*shape, seed=seed)
        poison()
        y = f(x)
        assert torch.equal(y, m(x))
        if grad:
            g = normal(*shape, seed=seed + 5)
            for a, b in zip(torch.autograd.grad(y, list(f.parameters()), g), torch.autograd.grad(m(x), list(m.parameters()), g)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("grad", [False, True])
def test_trace_of_join_and_norm(grad):
    r, o, w = normal(20, 96), normal(3, 20, 32, seed=1), normal(96, seed=2).requires_grad_(grad)

    def step(r, o, w):
        r2, y = block_join(r, o, w, None, 0.5, pre_weight=w)
        return r2 * 2, y * 2, block_norm(r, w, heads=3) * 2, block_join(r, o, w, pre=False)[0]

    f = torch.jit.trace(step, (r, o, w))
    for seed in (3, 4):
        a, b = normal(20, 96, seed=seed), normal(3, 20, 32, seed=seed + 9)
        poison()
        for u, v in zip(f(a, b, w), step(a, b, w)):
            assert torch.equal(u, v)


def test_trace_of_the_plain_calls():
    """the registered operators stand in the graph; what has none refuses"""
    x, wg, wu, w2 = normal(2, 10, 32), normal(2, 32, 48, seed=1), normal(2, 32, 48, seed=2), normal(2, 48, 32, seed=3)
    f = torch.jit.trace(lambda t: flashmlp_gated_fwd(t, wg, wu, w2, "silu") * 2, (x,))
    g = torch.jit.trace(lambda t: tuple(v * 2 for v in flashmlp_gated_bwd(t, wg, wu, w2, t, "silu")), (x,))
    y = normal(2, 10, 32, seed=4)
    poison()
    assert torch.equal(f(y), flashmlp_gated_fwd(y, wg, wu, w2, "silu") * 2)
    poison()
    for a, b in zip(g(y), flashmlp_gated_bwd(y, wg, wu, w2, y, "silu")):
        assert torch.equal(a, b * 2)
    part = torch.jit.trace(lambda t: flashmlp_gated_bwd(t, wg, wu, w2, t, "silu", _needs=(True, False))[0] * 2, (x,))
    poison()
    assert torch.equal(part(y), flashmlp_gated_bwd(y, wg, wu, w2, y, "silu")[0] * 2)
    r, o = normal(10, 64), normal(2, 10, 32)
    rs = torch.ones(10, device="cuda")
    for call in (lambda t: grad_norm([t]), lambda t: clip_grads([t.clone()], 1.0)[1],
                 lambda t: block_join_fwd(t, o)[0], lambda t: block_join_bwd(t, o, rs, rs, t, o)[0]):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (r,))
