"""The gated block's operators where torch asks for derivatives that they do not have: forward mode and second
derivatives are refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from flashmlp_amd import GatedFlashMLP, block_join, block_norm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def normal(*shape, dt=BF, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


def module(H=3, D=32, E=48, dt=BF):
    torch.manual_seed(0)
    return GatedFlashMLP(H, D, E, dtype=dt)


def test_forward_mode_is_refused():
    m = module()
    r, o, w, gate = normal(20, 96), normal(3, 20, 32, seed=1), normal(96, seed=2), normal(2, 96, seed=3)
    strided = torch.stack([r, r], -1).flatten(1)[:, ::2]
    calls = [lambda d: block_norm(d(r), heads=3), lambda d: block_norm(r, d(w)), lambda d: block_norm(d(strided)),
             lambda d: block_join(d(r), o), lambda d: block_join(r, d(o)), lambda d: block_join(r, o, d(w)),
             lambda d: block_join(r, o, None, d(gate)), lambda d: block_join(r, o, pre_weight=d(w)),
             lambda d: block_join(d(r), o, pre=False), lambda d: m(d(o)), lambda d: m(d(o[0]))]
    with fwd_ad.dual_level():
        for i, call in enumerate(calls):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="jvp"):
                    call(lambda t: fwd_ad.make_dual(t, torch.ones_like(t)))
        with torch.no_grad():  # (nothing dual: as ever)
            y = block_norm(r, w, heads=3)
    assert torch.equal(y, block_norm(r, w, heads=3))


@pytest.mark.parametrize("path", ["dense", "strided"])
@pytest.mark.parametrize("what", ["module", "shared", "join", "norm"])
@pytest.mark.parametrize("wrt", ["output", "linear"])
def test_first_derivatives_under_create_graph_and_no_second(path, what, wrt):
    """create_graph=True gives the ordinary first derivatives, on the kernels' own layouts (nodes in C++) and on others
    (in Python); differentiating those raises, also where the incoming gradient itself is a constant"""
    m = module()
    shape = dict(module=(3, 20, 32), shared=(20, 32), join=(20, 96), norm=(20, 96))[what]
    x = normal(*shape)
    if path == "strided":
        x = torch.stack([x, x], -1).flatten(-2)[..., ::2]
    x.requires_grad_(True)
    o, w = normal(3, 20, 32, seed=1), normal(96, seed=2).requires_grad_(True)
    run = dict(module=lambda: m(x), shared=lambda: m(x), join=lambda: block_join(x, o, w, pre_weight=w)[1],
               norm=lambda: block_norm(x, w))[what]
    y = run()
    loss = y.float().square().sum() if wrt == "output" else y.float().sum()
    inputs = [x, *(m.parameters() if what in ("module", "shared") else [w])]
    want = torch.autograd.grad(loss, inputs, retain_graph=True)
    got = torch.autograd.grad(loss, inputs, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(sum(g.float().square().sum() for g in got), inputs, allow_unused=True)
