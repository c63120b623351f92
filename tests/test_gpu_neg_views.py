"""Lazily negated tensors (a view with the negative bit set: its memory holds the opposite sign) as inputs, incoming
gradients and outputs, dense and aligned ones among them, which no layout copy would resolve."""
import pytest
import torch

from flashmlp_amd import (GatedFlashMLP, block_join, block_join_bwd, block_join_fwd, block_norm, clip_grads,
                          flashmlp_bwd, flashmlp_fwd, flashmlp_gated_bwd, flashmlp_gated_fwd, grad_norm)

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def neg(t):
    """a view with t's values over memory that holds -t"""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def normal(*shape, dt=BF, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


def same(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("dt", [BF, FL])
@pytest.mark.parametrize("D,E", [(64, 96), (64, 45), (256, 20)])
def test_plain(dt, D, E):
    t = [normal(*s, dt=dt, seed=i) for i, s in enumerate([(2, 40, D), (2, D, E), (2, E, D), (2, 40, D)])]
    want = (flashmlp_fwd(*t[:3], "silu"), *flashmlp_bwd(*t, "silu"))
    for i in range(4):
        u = [neg(v) if j == i else v for j, v in enumerate(t)]
        same((flashmlp_fwd(*u[:3], "silu"), *flashmlp_bwd(*u, "silu")), want)


@pytest.mark.parametrize("dt", [BF, FL])
def test_gated(dt):
    t = [normal(*s, dt=dt, seed=i) for i, s in enumerate([(2, 40, 64), (2, 64, 96), (2, 64, 96), (2, 96, 64), (2, 40, 64)])]
    want = (flashmlp_gated_fwd(*t[:4], "silu"), *flashmlp_gated_bwd(*t, "silu"))
    for i in range(5):
        u = [neg(v) if j == i else v for j, v in enumerate(t)]
        same((flashmlp_gated_fwd(*u[:4], "silu"), *flashmlp_gated_bwd(*u, "silu")), want)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_gated_module(shared, both):
    """incoming gradients of the autograd nodes, and (both) inputs"""
    torch.manual_seed(0)
    m = GatedFlashMLP(2, 64, 96, dtype=BF)
    shape = (40, 64) if shared else (2, 40, 64)
    x, g = normal(*shape), normal(*shape, seed=1)

    def step(x, g):
        x = x.detach().requires_grad_(True)
        o = m(x)
        return (o, *torch.autograd.grad(o, (x, m.wg, m.wu, m.w2), g))

    same(step(neg(x) if both else x, neg(g)), step(x, g))


@pytest.mark.parametrize("D", [64, 50])
def test_join(D):
    B, H, C = 30, 3, 3 * D
    t = dict(r=normal(B, C), o=normal(H, B, D, seed=1), w_post=normal(C, seed=2), gate=normal(2, C, seed=3),
             w_pre=normal(C, seed=4), dr2=normal(B, C, seed=5), dy=normal(H, B, D, seed=6))

    def step(t):
        ins = [t[k].detach().requires_grad_(True) for k in ("r", "o", "w_post", "gate", "w_pre")]
        r2, y = block_join(*ins[:4], 0.5, pre_weight=ins[4])
        return (r2, y, *torch.autograd.grad((r2, y), ins, (t["dr2"], t["dy"])), block_norm(t["r"], t["w_pre"], heads=H))

    def direct(t):
        a, w = (t["o"], t["w_post"], t["gate"], 0.5), t["w_pre"]
        r2, y, rs_o, rs_r = block_join_fwd(t["r"], *a, pre_weight=w, _save=True)
        return (r2, y, *block_join_bwd(r2, t["o"], rs_o, rs_r, t["dr2"], t["dy"], *a[1:], pre_weight=w))

    for f in (step, direct):
        want = f(t)
        for k in t:
            same(f(dict(t, **{k: neg(t[k])})), want)


def test_clip():
    g = [normal(1000, dt=FL), normal(30, 40, seed=1)]
    want = [torch.empty(v.shape, dtype=FL, device="cuda") for v in g]
    _, norm = clip_grads(g, 0.5, out=want)
    assert torch.equal(grad_norm([neg(v) for v in g]), norm)
    outs = [torch.empty_like(v) for v in want]
    clip_grads([neg(v) for v in g], 0.5, out=outs)
    same(outs, want)
    outs = [torch._neg_view(torch.empty_like(v)) for v in want]
    clip_grads(g, 0.5, out=outs)
    same(outs, want)
    inplace = [neg(v.float()) for v in g]
    clip_grads(inplace, 0.5)
    same(inplace, want)
