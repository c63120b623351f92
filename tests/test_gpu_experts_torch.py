"""The experts' operators and the orthogonalised updates in torch's hands: the nodes in C++ and those in Python alike, saved
tensors that hooks bring back, checkpointing, threads, derivatives that they do not have, tracing and compiling, views that
negate, tensors without memory, and sizes past 2^32 bytes."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

import flashmlp_amd.experts as experts_module
import flashmlp_amd.muon as muon_module
from flashmlp_amd import ExpertPlan, GatedExperts, expert_combine, expert_dispatch, expert_plan, expert_route, muon_step, orthogonalize
from oracle import experts as ox
from test_gpu_join_wrappers import Wrapper

pytestmark = pytest.mark.gpu
BF, FL = torch.bfloat16, torch.float32


def normal(*shape, dt=FL, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


class Case:
    """a call of one operator, its differentiable inputs and the gradients of its outputs"""

    def __init__(self, what, dt=BF, seed=0):
        T, N, k, D, cap = 40, 6, 2, 24, 15
        with torch.no_grad():
            plan = expert_plan(expert_route(normal(T, N, seed=9), k)[1], N, cap)
        if what.startswith("route"):
            self.inputs = [normal(T, N, dt=dt, seed=seed)]
            self.call = lambda l: expert_route(l, k, normalize=what == "route")[0]
        elif what == "dispatch":
            self.inputs, self.call = [normal(T, D, dt=dt, seed=seed)], lambda x: expert_dispatch(x, plan)
        elif what == "combine":
            self.inputs = [normal(N, cap, D, dt=dt, seed=seed), normal(T, k, seed=seed + 1).abs()]
            self.call = lambda rows, w: expert_combine(rows, plan, w)
        else:
            self.inputs, self.call = [normal(N, cap, D, dt=dt, seed=seed)], lambda rows: expert_combine(rows, plan)
        self.inputs = [t.requires_grad_(True) for t in self.inputs]

    def step(self):
        o = self.call(*self.inputs)
        return (o.detach(), *torch.autograd.grad(o, self.inputs, torch.ones_like(o) + o.detach()))


WHATS = ["route", "route_plain", "dispatch", "combine", "combine_sum"]


def same(a, b):
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.fixture(params=["fast", "general"])
def path(request, monkeypatch):
    if request.param == "general":
        monkeypatch.setattr(experts_module, "_fast", None)
        monkeypatch.setattr(muon_module, "_fast", None)
    elif experts_module._fast is None:
        pytest.skip("the fast path is not built")
    return request.param


@pytest.mark.parametrize("dt", [BF, FL])
@pytest.mark.parametrize("what", WHATS)
def test_both_paths_are_the_same(what, dt, monkeypatch):
    case = Case(what, dt)
    want = case.step()
    monkeypatch.setattr(experts_module, "_fast", None)
    same(Case(what, dt).step(), want)


def test_both_paths_of_the_updates_are_the_same(monkeypatch):
    w, g, m = normal(3, 40, 72), normal(3, 40, 72, dt=BF, seed=1), normal(3, 40, 72, seed=2)
    a = w.clone(), m.clone()
    muon_step([a[0]], [g], [a[1]], 0.1, weight_decay=0.1)
    o = orthogonalize(g)
    monkeypatch.setattr(muon_module, "_fast", None)
    b = w.clone(), m.clone()
    muon_step([b[0]], [g], [b[1]], 0.1, weight_decay=0.1)
    same(a, b)
    assert torch.equal(o, orthogonalize(g))


def other_layout(t):
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else torch.stack([t, t], -1)[..., 0]


@pytest.mark.parametrize("what", WHATS)
def test_saved_tensors_that_come_back(what, path):
    case = Case(what)
    want = case.step()
    with save_on_cpu():
        same(case.step(), want)
    with saved_tensors_hooks(lambda t: t, other_layout):
        same(case.step(), want)


@pytest.mark.parametrize("what", WHATS)
@pytest.mark.parametrize("wrong", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.double() if t.is_floating_point() else t.long()])
def test_wrong_saved_tensors_are_refused(what, wrong, path):
    case = Case(what)
    with saved_tensors_hooks(lambda t: t, wrong), pytest.raises(RuntimeError, match="came back with another"):
        case.step()


def test_checkpoint_and_threads(path):
    torch.manual_seed(0)
    m = GatedExperts(5, 32, 40, capacity_factor=1.25, dtype=BF)
    x = normal(70, 32, dt=BF).requires_grad_(True)
    inputs = [x, *m.parameters()]
    want = torch.autograd.grad(m(x), inputs, torch.ones_like(x))
    same(torch.autograd.grad(checkpoint(m, x, use_reentrant=False), inputs, torch.ones_like(x)), want)
    got = {}

    def run(i):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = torch.autograd.grad(m(x), inputs, torch.ones_like(x))
        s.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4
    for g in got.values():
        same(g, want)


@pytest.mark.parametrize("what", WHATS)
def test_first_derivatives_only(what, path):
    case = Case(what, FL)
    o = case.call(*case.inputs)
    loss = o.square().sum()
    want = torch.autograd.grad(loss, case.inputs, retain_graph=True)
    got = torch.autograd.grad(loss, case.inputs, create_graph=True)
    same([g.detach() for g in got], want)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(sum(g.square().sum() for g in got), case.inputs, allow_unused=True)
    with fwd_ad.dual_level():
        for mode in (torch.enable_grad, torch.no_grad):
            for i in range(len(case.inputs)):
                args = [fwd_ad.make_dual(t.detach(), torch.ones_like(t)) if j == i else t.detach() for j, t in enumerate(case.inputs)]
                with mode(), pytest.raises(RuntimeError, match="jvp"):
                    case.call(*args)


def test_tracing_is_refused_and_compiling_breaks_the_graph():
    case = Case("combine")
    x, logits = normal(40, 24, dt=BF), normal(40, 6)
    _, e = expert_route(logits, 2)
    plan = expert_plan(e, 6)
    calls = [lambda: expert_route(logits, 2)[0], lambda: expert_plan(e, 6).slots, lambda: expert_dispatch(x, plan),
             lambda: expert_combine(expert_dispatch(x, plan), plan), lambda: orthogonalize(x)]
    for call in calls:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda t: call() + t.sum().to(torch.int32), (x,), check_trace=False)
    step = torch.compile(lambda rows, w: case.call(rows * 2, w) + 1, backend="eager")
    same([step(*case.inputs)], [case.call(case.inputs[0] * 2, case.inputs[1]) + 1])


def test_lazily_negated_views(path):
    z = torch.complex(normal(40, 24), normal(40, 24, seed=1))
    neg = torch._neg_view(z.real.contiguous())
    logits = torch._neg_view(normal(40, 6, seed=2))
    w, e = expert_route(logits, 2)
    a, b = expert_route(logits.resolve_neg(), 2)
    assert torch.equal(w, a) and torch.equal(e, b)
    plan = expert_plan(e, 6)
    rows = expert_dispatch(neg, plan)
    assert torch.equal(rows, expert_dispatch(neg.resolve_neg(), plan))
    assert torch.equal(expert_combine(torch._neg_view(rows), plan, w), -expert_combine(rows, plan, w))
    assert torch.equal(orthogonalize(neg), orthogonalize(neg.resolve_neg()))
    g, m, p, q = normal(40, 24, seed=3), torch.zeros(40, 24, device="cuda"), normal(40, 24, seed=4), normal(40, 24, seed=4)
    muon_step([p], [torch._neg_view(g)], [m], 0.1)
    muon_step([q], [-g], [torch.zeros_like(m)], 0.1)
    assert torch.equal(p, q)


def test_tensors_without_memory_are_refused(path):
    x, logits = normal(40, 24), normal(40, 6)
    w, e = expert_route(logits, 2)
    plan = expert_plan(e, 6)
    rows = expert_dispatch(x, plan)
    bad = ExpertPlan(Wrapper(plan.slots), plan.counts, 6, 40), ExpertPlan(plan.slots, Wrapper(plan.counts), 6, 40)
    calls = [lambda: expert_route(Wrapper(logits), 2), lambda: expert_plan(Wrapper(e), 6), lambda: expert_dispatch(Wrapper(x), plan),
             lambda: expert_dispatch(x, bad[0]), lambda: expert_dispatch(x, bad[1]), lambda: expert_combine(Wrapper(rows), plan, w),
             lambda: expert_combine(rows, plan, Wrapper(w)), lambda: expert_combine(rows, bad[0]), lambda: orthogonalize(Wrapper(x)),
             lambda: muon_step([x], [Wrapper(x)], [x.clone()], 0.1)]
    for call in calls:
        with pytest.raises(TypeError, match="memory of its own"):
            call()


def test_refusals_on_the_device(path):
    x, logits = normal(40, 24), normal(40, 6)
    w, e = expert_route(logits, 2)
    plan = expert_plan(e, 6)
    rows = expert_dispatch(x, plan)
    for call, error in ((lambda: expert_route(logits.double(), 2), TypeError), (lambda: expert_route(logits.int(), 2), TypeError),
                        (lambda: expert_plan(e.short(), 6), TypeError), (lambda: expert_plan(e.float(), 6), TypeError),
                        (lambda: expert_dispatch(x.double(), plan), TypeError), (lambda: expert_dispatch(x[:9], plan), AssertionError),
                        (lambda: expert_dispatch(x.cpu(), plan), RuntimeError),
                        (lambda: expert_dispatch(x, plan._replace(slots=plan.slots.cpu())), RuntimeError),
                        (lambda: expert_dispatch(x, plan._replace(slots=plan.slots.long())), TypeError),
                        (lambda: expert_dispatch(x, plan._replace(counts=plan.counts[:2])), AssertionError),
                        (lambda: expert_combine(rows.double(), plan), TypeError), (lambda: expert_combine(rows, plan, w.half()), TypeError),
                        (lambda: expert_combine(rows, plan, w[:, :1]), AssertionError), (lambda: expert_combine(rows, plan, w.cpu()), RuntimeError),
                        (lambda: expert_combine(rows[:, :9], plan), AssertionError), (lambda: expert_plan(e, 1025), RuntimeError),
                        (lambda: expert_route(normal(2, 1025), 2), RuntimeError), (lambda: expert_route(normal(2, 64), 33), RuntimeError),
                        (lambda: expert_plan(e, 6, 2 ** 31), RuntimeError),
                        (lambda: orthogonalize(normal(2, 300, 300)), RuntimeError), (lambda: orthogonalize(x.double()), TypeError),
                        (lambda: orthogonalize(x, out=x.half()), ValueError),
                        (lambda: muon_step([x], [x.double()], [x.clone()], 0.1), TypeError),
                        (lambda: muon_step([x], [x.cpu()], [x.clone()], 0.1), RuntimeError)):
        with pytest.raises(error):
            call()


def test_tokens_and_rows_past_32_bits():
    """more than 2^32 bytes of tokens and of rows: every offset of the copies is 64 bits wide"""
    T, N, D = (1 << 24) + 3, 3, 160
    e = torch.arange(T, device="cuda", dtype=torch.int32).view(T, 1) % N
    x = torch.empty(T, D, device="cuda", dtype=BF)
    x.copy_((torch.arange(T, device="cuda") % 251).to(BF).view(T, 1))
    plan = expert_plan(e, N, T // N + 1)
    t = torch.arange(T, device="cuda")
    assert torch.equal(plan.slots[:, 0].long(), (t % N) * (T // N + 1) + t // N)
    rows = expert_dispatch(x, plan)
    assert rows.numel() * 2 > 1 << 32
    flat = rows.view(-1, D)
    for i in (0, 1, 2, T // 2, T - 2, T - 1):
        assert (flat[plan.slots[i, 0].long()] == x[i]).all()
    assert (flat.sum(0, dtype=torch.float64) == x.sum(0, dtype=torch.float64)).all()
    w = torch.full((T, 1), 2.0, device="cuda")
    o = expert_combine(rows, plan, w)
    assert torch.equal(o, x * 2)


def test_a_stack_past_32_bits():
    """more than 2^32 bytes of matrices, the last ones as the first"""
    H = (1 << 32) // (64 * 512 * 4) + 5
    one = normal(7, 64, 512)
    x = one.repeat((H + 6) // 7, 1, 1)[:H]
    o = orthogonalize(x, out=x)
    want = orthogonalize(one)
    for i in (0, 1, 6, H // 2, H - 2, H - 1):
        assert (o[i] - want[i % 7]).abs().max() <= 1e-4
    assert torch.equal(o[:7], o[7 * (H // 14):7 * (H // 14) + 7])


def test_slots_that_a_user_makes_are_bounded():
    plan = ExpertPlan(torch.full((9, 2), 10 ** 9, dtype=torch.int32, device="cuda"), torch.full((3,), -5, dtype=torch.int32, device="cuda"), 3, 4)
    x = normal(9, 16)
    rows = expert_dispatch(x, plan)
    assert (rows == 0).all()
    assert (expert_combine(rows + 1, plan) == 0).all()
    assert ox.over(expert_combine(rows, plan), torch.zeros(9, 16, dtype=torch.float64), torch.zeros(9, 16, dtype=torch.float64)) == 0
