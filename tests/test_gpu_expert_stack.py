"""The experts' operators and the orthogonalised updates together: the example's stack of mixtures, its gradients against the
same stack of plain operations in 64 bits, a few training steps, single rows, and replays of a captured forward."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

import flashmlp_amd.experts as experts_module

pytestmark = pytest.mark.gpu
spec = importlib.util.spec_from_file_location("expert_stack", Path(__file__).parents[1] / "examples" / "expert_stack.py")
expert_stack = importlib.util.module_from_spec(spec)
spec.loader.exec_module(expert_stack)


def kept(choice, N, capacity):
    load, keep = [0] * N, torch.zeros_like(choice, dtype=torch.bool)
    for t, row in enumerate(choice.tolist()):
        for j, e in enumerate(row):
            keep[t, j] = load[e] < capacity
            load[e] += 1
    return keep


def plain(model, params, x, choices):
    """the stack in plain operations on 64-bit copies of the parameters, with the choices that the model made"""
    p = iter(params)
    L, H = len(model.mixtures), model.heads
    w = [[next(p) for _ in range(4)] for _ in range(L)]
    pre, post, gate = [next(p) for _ in range(L + 1)], [next(p) for _ in range(L)], [next(p) for _ in range(L)]
    rms = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    for i, m in enumerate(model.mixtures):
        router, wg, wu, w2 = w[i]
        y = (rms(x) * pre[i]).view(x.shape[0], H, -1).transpose(0, 1).reshape(-1, wg.shape[1])
        N, k, T = m.num_experts, m.experts_per_token, y.shape[0]
        choice = choices[i]
        s = torch.softmax(y @ router, 1).gather(1, choice)
        s = s / s.sum(1, keepdim=True)
        keep = kept(choice, N, math.ceil(T * k / N * m.capacity_factor))
        o = torch.zeros_like(y)
        for e in range(N):
            t, j = torch.nonzero((choice == e) & keep, as_tuple=True)
            z = y[t] @ wg[e]
            o = o.index_add(0, t, ((z * torch.sigmoid(z) * (y[t] @ wu[e])) @ w2[e]) * s[t, j][:, None])
        o = o.view(H, x.shape[0], -1)
        x = x + model.scale * gate[i] * rms(o.transpose(0, 1).reshape(x.shape)) * post[i]
    return rms(x) * pre[L]


@pytest.mark.parametrize("rows,factor", [(60, 1.0), (60, 2.0), (1, 1.5)])
def test_stack_and_gradients(rows, factor, monkeypatch):
    """normwise, fp32: sums of up to 128 terms (7.6e-6 at worst) in four products a block and way, two blocks, and the norms
    between them: 1e-4"""
    torch.manual_seed(4)
    model = expert_stack.ExpertStack(2, 4, 32, 48, 6, dtype=torch.float32, capacity_factor=factor)
    choices, route = [], experts_module.expert_route

    def recorded(*args, **kw):
        w, e = route(*args, **kw)
        choices.append(e.cpu().long())
        return w, e

    monkeypatch.setattr(experts_module, "expert_route", recorded)
    x, gy = torch.randn(rows, 128, device="cuda"), torch.randn(rows, 128, device="cuda")
    params = list(model.parameters())
    y = model(x)
    g = torch.autograd.grad((y * gy).sum(), params)
    ref = [p.detach().double().cpu().requires_grad_(True) for p in params]
    want = plain(model, ref, x.double().cpu(), choices)
    wg = torch.autograd.grad((want * gy.double().cpu()).sum(), ref)
    for i, (a, b) in enumerate(zip((y, *g), (want, *wg))):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).norm() <= 1e-4 * b.norm() + 1e-6, (i, ((a - b).norm() / b.norm()).item())


def test_steps_of_training_change_every_matrix():
    torch.manual_seed(0)
    model = expert_stack.ExpertStack(2, 4, 64, 96, 8)
    before = [p.detach().clone() for p in model.parameters()]
    losses, norms = expert_stack.train(model, 200, 4)
    assert all(math.isfinite(v) for v in losses + norms) and all(n > 0 for n in norms)
    for p, b in zip(model.parameters(), before):
        assert torch.isfinite(p).all()
        if p.dim() > 1:  # (small changes of vectors around one are below bf16's rounding)
            assert not torch.equal(p, b)


def test_captured_forward():
    """replays on new rows between eager work, against the eager forward"""
    torch.manual_seed(1)
    model = expert_stack.ExpertStack(2, 4, 64, 96, 8)
    x = torch.randn(50, 256, device="cuda")
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            model(x)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x)
        for i in range(4):
            x.copy_(torch.randn(50, 256, generator=torch.Generator().manual_seed(i)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, model(x.clone())), i
