"""More tokens than one launch has threads for: four tokens a workgroup of 256 threads (columns or experts past 256) are 2^32 at 2^26
tokens. Tokens and logits are overlapping rows of one small buffer; chosen tokens are compared with calls for them alone."""
import pytest
import torch

from flashmlp_amd import ExpertPlan, expert_combine, expert_dispatch, expert_plan, expert_route

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
T = (1 << 26) + 5
AT = (0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, T - 1)


def rows_of(columns, seed):
    """(T, columns), each row an element further on"""
    base = torch.randn(T + columns, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF)
    return base.as_strided((T, columns), (1, 1))


@pytest.mark.parametrize("normalize", [True, False])
def test_route(normalize):
    N, k = 260, 2
    at = torch.tensor(AT, device="cuda")
    logits = rows_of(N, 1).requires_grad_(True)
    few = logits.detach()[at].contiguous().requires_grad_(True)
    w, e = expert_route(logits, k, normalize=normalize)
    w1, e1 = expert_route(few, k, normalize=normalize)
    assert torch.equal(w[at], w1) and torch.equal(e[at], e1)
    dw = torch.randn(T, k, device="cuda")
    (dl,) = torch.autograd.grad(w, logits, dw)
    (dl1,) = torch.autograd.grad(w1, few, dw[at])
    assert torch.equal(dl[at], dl1)


def test_dispatch_and_combine():
    N, capacity, D, k = 3, 3, 264, 2
    at = torch.tensor(AT, device="cuda")
    experts = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    experts[at, 0] = torch.arange(len(AT), dtype=torch.int32, device="cuda") % N
    experts[at[::3], 1] = 2
    plan, few = expert_plan(experts, N, capacity), expert_plan(experts[at], N, capacity)
    assert torch.equal(plan.slots[at], few.slots) and torch.equal(plan.counts, few.counts) and (plan.slots >= 0).sum() == (few.slots >= 0).sum()
    x = rows_of(D, 2)
    rows = expert_dispatch(x, plan)
    assert torch.equal(rows, expert_dispatch(x[at].contiguous(), few))
    weights = torch.randn(T, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    r, r1 = (rows.clone().requires_grad_(True) for _ in range(2))
    w, w1 = weights.requires_grad_(True), weights.detach()[at].requires_grad_(True)
    o, o1 = expert_combine(r, plan, w), expert_combine(r1, few, w1)
    assert torch.equal(o[at], o1) and (o[:4096].float().abs().sum(1) > 0).sum() == 2
    del o1
    do = rows_of(D, 4)
    dr, dw = torch.autograd.grad(o, (r, w), do)
    dr1, dw1 = torch.autograd.grad(expert_combine(r1, few, w1), (r1, w1), do[at].contiguous())
    assert torch.equal(dr, dr1) and torch.equal(dw[at], dw1) and (dw != 0).sum() == (dw1 != 0).sum()
