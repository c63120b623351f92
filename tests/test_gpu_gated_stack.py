"""The gated block's operators together: the example's stack of blocks, its gradients against the same stack of
plain operations in 64 bits, a training run that learns, single rows, CUDA-graph replay of a forward, and the
registered operator under torch.compile."""
import importlib.util
from pathlib import Path

import pytest
import torch

from flashmlp_amd import GatedFlashMLP, block_join, block_norm, flashmlp_gated_bwd, flashmlp_gated_fwd

pytestmark = pytest.mark.gpu
spec = importlib.util.spec_from_file_location("gated_stack", Path(__file__).parents[1] / "examples" / "gated_stack.py")
gated_stack = importlib.util.module_from_spec(spec)
spec.loader.exec_module(gated_stack)


def plain(model, params, x):
    """the stack in plain operations on 64-bit copies of the parameters"""
    p = iter(params)
    L, H = len(model.mlps), model.heads
    w = [[next(p) for _ in range(3)] for _ in range(L)]
    pre, post, gate = [next(p) for _ in range(L + 1)], [next(p) for _ in range(L)], [next(p) for _ in range(L)]
    rms = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    for i in range(L):
        y = (rms(x) * pre[i]).view(x.shape[0], H, -1).transpose(0, 1)
        wg, wu, w2 = w[i]
        z = y @ wg
        o = (z * torch.sigmoid(z) * (y @ wu)) @ w2
        x = x + model.scale * gate[i] * rms(o.transpose(0, 1).reshape(x.shape)) * post[i]
    return rms(x) * pre[L]


@pytest.mark.parametrize("dtype,rows,tol", [(torch.float32, 70, 2e-5), (torch.bfloat16, 70, 5e-2), (torch.float32, 1, 2e-5)])
def test_stack_and_gradients(dtype, rows, tol):
    """normwise: fp32 sums of up to 200 terms through three blocks; bf16 rounds some 8 times a block (2^-9 each on
    average) on a path of 3 blocks, and as often on the way back."""
    torch.manual_seed(3)
    model = gated_stack.GatedStack(3, 4, 32, 96, dtype=dtype)
    x = torch.randn(rows, 128, device="cuda")
    gy = torch.randn(rows, 128, device="cuda")
    params = list(model.parameters())
    y = model(x)
    g = torch.autograd.grad((y.float() * gy).sum(), params)
    ref = [p.detach().double().cpu().requires_grad_(True) for p in params]
    want = plain(model, ref, x.double().cpu())
    wg = torch.autograd.grad((want * gy.double().cpu()).sum(), ref)
    for a, b in zip((y, *g), (want, *wg)):
        a, b = a.double().cpu(), b.detach()
        assert (a - b).norm() <= tol * b.norm(), ((a - b).norm() / b.norm()).item()


def test_training_learns_and_generates():
    torch.manual_seed(0)
    model = gated_stack.GatedStack(2, 4, 64, 128)
    losses, norms = gated_stack.train(model, 512, 40)
    assert losses[-1] < 0.8 * losses[0] and all(n == n and n > 0 for n in norms)
    out = gated_stack.generate(model, torch.randn(3, 256, device="cuda"), 4)
    assert out.shape == (4, 3, 256) and out.isfinite().all()


def test_rows_do_not_depend_on_their_company():
    """a row alone and among others: the same up to the order of the sums over E"""
    torch.manual_seed(1)
    model = gated_stack.GatedStack(2, 4, 64, 256)
    x = torch.randn(300, 256, device="cuda")
    with torch.no_grad():
        many, one = model(x), torch.cat([model(x[i:i + 1]) for i in (0, 150, 299)])
    assert torch.allclose(many[[0, 150, 299]].float(), one.float(), rtol=0.05, atol=0.05)


def test_forward_in_a_graph():
    torch.manual_seed(2)
    model = gated_stack.GatedStack(2, 4, 64, 128)
    x = torch.randn(4, 256, device="cuda")
    with torch.no_grad():
        model(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x)
        for i in range(4):
            x.copy_(torch.randn(4, 256, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, model(x))


def test_registered_operator_and_compile():
    torch.manual_seed(0)
    m = GatedFlashMLP(2, 32, 64, dtype=torch.bfloat16)
    x = torch.randn(2, 40, 32, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = [p.detach() for p in (m.wg, m.wu, m.w2)]
    o = torch.ops.flashmlp_amd.gated_fwd(x.detach(), *w, "silu")
    assert torch.equal(o, flashmlp_gated_fwd(x.detach(), *w, "silu"))
    do = torch.randn_like(o)
    g = torch.ops.flashmlp_amd.gated_bwd(x.detach(), *w, do, "silu")
    assert all(torch.equal(a, b) for a, b in zip(g, flashmlp_gated_bwd(x.detach(), *w, do, "silu")))
    f = torch.compile(lambda t: m(t), backend="aot_eager", fullgraph=True)
    (dx,) = torch.autograd.grad(f(x), (x,), do)
    assert torch.equal(f(x), o) and torch.equal(dx, g[0])
    shared = torch.randn(40, 32, dtype=torch.bfloat16, device="cuda")
    # (compiled, the mean is torch's over the heads' rounded results)
    assert torch.allclose(f(shared).float(), m(shared).float(), rtol=2.0 ** -6, atol=2.0 ** -6)


def test_join_and_norm_under_compile():
    """they break the graph, and give the same results"""
    r = torch.randn(20, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    o = torch.randn(2, 20, 32, device="cuda", dtype=torch.bfloat16)
    f = torch.compile(lambda a, b: block_join(a * 2, block_norm(a, heads=2) + b)[1] * 3, backend="aot_eager")
    e = block_join(r * 2, block_norm(r, heads=2) + o)[1] * 3
    assert torch.equal(f(r, o), e)
