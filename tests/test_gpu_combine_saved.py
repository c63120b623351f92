"""What expert_combine holds until its backward: the experts' rows where the weights' gradient is asked for, and no rows otherwise."""
import pytest
import torch

from flashmlp_amd import expert_combine, expert_plan, experts
from oracle import experts as ox

pytestmark = pytest.mark.gpu
T, k, N, capacity, D = 50, 2, 5, 18, 24


@pytest.fixture(params=[True, False], ids=["C++", "Python"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(experts, "_fast", None)


@pytest.mark.parametrize("weighted,learns", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved(path, weighted, learns, dtype):
    g = torch.Generator().manual_seed(0)
    choice = torch.stack([torch.randperm(N, generator=g)[:k] for _ in range(T)]).int()
    plan = expert_plan(choice.cuda(), N, capacity)
    slots = plan.slots.cpu()
    rows0 = torch.randn(N, capacity, D, generator=g).to(dtype)
    w0 = torch.randn(T, k, generator=g) if weighted else None
    do = torch.randn(T, D, generator=g).to(dtype)
    leaf = rows0.cuda().requires_grad_(True)
    rows = leaf * 1
    w = None if w0 is None else w0.cuda().requires_grad_(learns)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(tuple(t.shape)) or t, lambda t: t):
        o = expert_combine(rows, plan, w)
    assert ((N, capacity, D) in saved) == learns
    ref, bound = ox.gather64(rows0, slots, w0)
    assert ox.over(o, ref, bound) <= 1
    if learns:
        dr, dw = torch.autograd.grad(o, (leaf, w), do.cuda())
        assert ox.over(dw, *ox.dot64(rows0, do, slots)) <= 1
    else:
        with torch.no_grad():
            rows.fill_(float("nan"))  # no gradient depends on the values
        (dr,) = torch.autograd.grad(o, leaf, do.cuda())
    assert ox.over(dr, *ox.scatter64(do, slots, N, capacity, w0)) <= 1


def test_weights_alone(path):
    """rows that need no gradient"""
    g = torch.Generator().manual_seed(1)
    plan = expert_plan(torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2) % 4, 4, 2)
    rows, do = torch.randn(4, 2, 8, generator=g), torch.randn(3, 8, generator=g)
    w = torch.randn(3, 2, generator=g).cuda().requires_grad_(True)
    (dw,) = torch.autograd.grad(expert_combine(rows.cuda(), plan, w), w, do.cuda())
    assert ox.over(dw, *ox.dot64(rows, do, plan.slots.cpu())) <= 1
