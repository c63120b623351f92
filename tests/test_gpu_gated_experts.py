"""GatedExperts against its parts and against a plain mixture in 64 bits: every token through its own experts, gradients of
the router, the experts and the input.

Against 64 bits a result's error is that of the gated MLP's 16-bit operands (h rounded, relative 2^-8 in bf16), its own
rounding and the combination's: 4 roundings of the values' size; the gradients have twice as many. The choice of experts is
made from the module's own logits, so that both sides agree on it."""
import math

import pytest
import torch

from flashmlp_amd import GatedExperts, expert_route
from oracle.gated import UNIT

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def plain(m, tokens, do, capacity):
    """(o, gradients of tokens, router, wg, wu, w2) in 64 bits, with the module's choices"""
    with torch.no_grad():
        _, choice = expert_route(tokens @ m.router, m.experts_per_token, normalize=m.normalize)
    x, r, wg, wu, w2 = (t.detach().double().cpu().requires_grad_(True)
                        for t in (tokens, m.router, m.experts.wg, m.experts.wu, m.experts.w2))
    choice = choice.cpu().long()
    p = torch.softmax(x @ r, 1).gather(1, choice)
    w = p / p.sum(1, keepdim=True) if m.normalize else p
    o, load = torch.zeros_like(x), [0] * m.num_experts
    kept = torch.zeros_like(choice, dtype=torch.bool)
    for t, row in enumerate(choice.tolist()):
        for j, e in enumerate(row):
            kept[t, j] = load[e] < capacity
            load[e] += 1
    for e in range(m.num_experts):
        t, j = torch.nonzero((choice == e) & kept, as_tuple=True)
        h = torch.nn.functional.silu(x[t] @ wg[e]) * (x[t] @ wu[e])
        o = o.index_add(0, t, (h @ w2[e]) * w[t, j][:, None])
    return o.detach(), torch.autograd.grad(o, (x, r, wg, wu, w2), do.double().cpu())


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("N,D,E,k,factor,normalize,shape", [(4, 32, 40, 2, None, True, (50,)), (8, 64, 96, 2, 1.0, True, (3, 67)),
                                                           (3, 16, 33, 1, 2.0, False, (1,)), (6, 128, 64, 3, 0.5, False, (2, 5, 20)),
                                                           (2, 256, 48, 2, None, True, (37,))])
def test_module(N, D, E, k, factor, normalize, shape, dtype):
    torch.manual_seed(N + D)
    m = GatedExperts(N, D, E, k, factor, normalize=normalize, dtype=dtype)
    x = torch.randn(*shape, D, device="cuda").to(dtype).requires_grad_(True)
    do = torch.randn(*shape, D, device="cuda").to(dtype)
    o = m(x)
    assert o.shape == x.shape and o.dtype == dtype
    grads = torch.autograd.grad(o, (x, m.router, m.experts.wg, m.experts.wu, m.experts.w2), do)
    T = math.prod(shape)
    want, wants = plain(m, x.reshape(T, D), do.reshape(T, D), T if factor is None else math.ceil(T * k / N * factor))
    u = max(UNIT[dtype], 2.0 ** -20)

    def off(a, b):
        return ((a.detach().double().cpu().reshape(b.shape) - b).norm() / b.norm().clamp(min=1e-30)).item()

    assert off(o, want) <= 4 * u
    for a, b in zip(grads, wants):
        assert a.dtype == dtype and off(a, b) <= 8 * u


def test_heads_of_the_mlp_layout_are_tokens():
    torch.manual_seed(0)
    m = GatedExperts(4, 64, 128, dtype=BF)
    x = torch.randn(3, 50, 64, device="cuda", dtype=BF)
    assert torch.equal(m(x).reshape(-1, 64), m(x.reshape(-1, 64)))
    assert m(x[:, :0]).shape == (3, 0, 64)


def test_tokens_do_not_depend_on_others_without_capacity():
    """a token alone, as in generation, and among others"""
    torch.manual_seed(1)
    m = GatedExperts(8, 64, 96, dtype=FL)
    x = torch.randn(9, 64, device="cuda")
    assert (m(x)[4:5] - m(x[4:5])).abs().max() <= 1e-5
