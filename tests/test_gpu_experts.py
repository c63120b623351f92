"""expert_route, expert_plan, expert_dispatch and expert_combine against 64-bit definitions: every type, one token to many,
experts and columns of any number, ties, masked experts, rows that drop, gradients, views, other streams, graphs.

Bounds are those that oracle/experts.py derives from the kernels' roundings; slots, counts and experts are exact."""
import pytest
import torch

from flashmlp_amd import ExpertPlan, expert_combine, expert_dispatch, expert_plan, expert_route
from oracle import experts as ox

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
TYPES = (BF, HF, FL)


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- route ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,N,k", [(1, 1, 1), (1, 2, 2), (3, 7, 1), (130, 8, 8), (129, 9, 3), (65, 16, 2), (257, 64, 8),
                                   (33, 100, 5), (20, 256, 6), (9, 512, 4), (8, 513, 4), (5, 1000, 32), (3, 1024, 7)])
def test_route(T, N, k, normalize, dtype):
    g = gen(T * N + k)
    logits = (2 * torch.randn(T, N, generator=g)).to(dtype)
    dw = torch.randn(T, k, generator=g)
    x = logits.cuda().requires_grad_(True)
    w, e = expert_route(x, k, normalize=normalize)
    (dx,) = torch.autograd.grad(w, x, dw.cuda())
    rw, bw, re, rdl, bdl = ox.route64(logits, k, normalize, dw)
    assert w.dtype == FL and e.dtype == torch.int32 and dx.dtype == dtype
    assert torch.equal(e.cpu().long(), re)
    assert ox.over(w, rw, bw) <= 1
    assert ox.over(dx, rdl, bdl) <= 1


@pytest.mark.parametrize("normalize", [True, False])
def test_route_ties_go_to_the_lowest_index(normalize):
    logits = torch.randint(-2, 3, (200, 40), generator=gen(1)).float()
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    for dtype in TYPES:
        w, e = expert_route(logits.to(dtype).cuda(), 9, normalize=normalize)
        rw, bw, re, _, _ = ox.route64(logits.to(dtype), 9, normalize)
        assert torch.equal(e.cpu().long(), re) and ox.over(w, rw, bw) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_masked_experts(normalize, dtype):
    """-infinity and the type's lowest value; rows with fewer experts than choices, and with none"""
    g = gen(2)
    logits = torch.randn(60, 24, generator=g).to(dtype)
    logits[torch.rand(60, 24, generator=g) < 0.7] = float("-inf")
    logits[5], logits[6] = float("-inf"), torch.finfo(dtype).min
    logits[7, 3:] = float("-inf")
    logits[8, 4] = torch.finfo(dtype).max
    dw = torch.randn(60, 6, generator=g)
    x = logits.cuda().requires_grad_(True)
    w, e = expert_route(x, 6, normalize=normalize)
    (dx,) = torch.autograd.grad(w, x, dw.cuda())
    rw, bw, re, rdl, bdl = ox.route64(logits, 6, normalize, dw)
    assert torch.equal(e.cpu().long(), re)
    assert (e[5] == -1).all() and (w[5] == 0).all() and (dx[5] == 0).all()
    assert e[6].tolist() == list(range(6))
    assert ox.over(w, rw, bw) <= 1 and ox.over(dx, rdl, bdl) <= 1


@pytest.mark.parametrize("normalize", [True, False])
def test_route_rows_that_are_not_finite(normalize):
    """NaN and +infinity spoil their own row only"""
    for bad in (float("nan"), float("inf")):
        logits = torch.randn(20, 12, generator=gen(3))
        clean = expert_route(logits.cuda(), 3, normalize=normalize)
        logits[7, 5] = bad
        x = logits.cuda().requires_grad_(True)
        w, e = expert_route(x, 3, normalize=normalize)
        assert e[7, 0].item() == 5 and torch.isnan(w[7]).all()
        rest = [i for i in range(20) if i != 7]
        assert torch.equal(w[rest], clean[0][rest]) and torch.equal(e[rest], clean[1][rest])
        (dx,) = torch.autograd.grad(w, x, torch.ones_like(w))
        assert torch.isfinite(dx[rest]).all()


def test_route_views():
    base = torch.randn(50, 40, generator=gen(4)).to(BF).cuda()
    for v in (base[:, 3:20], base.t()[2:30], base[::3, ::2], base[:1].expand(9, 40), base.T[:, 5:6]):
        k = min(2, v.shape[1])
        a, b = expert_route(v, k), expert_route(v.contiguous(), k)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- plan ----
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("T,k,N", [(0, 2, 3), (1, 1, 1), (1, 32, 5), (63, 1, 2), (64, 1, 64), (65, 3, 7), (2047, 2, 32),
                                   (2048, 2, 32), (2049, 2, 1000), (8191, 2, 1024), (8192, 2, 16), (8193, 2, 16), (40000, 3, 12), (30000, 3, 1000),
                                   (300000, 4, 5), (60000, 4, 700)])
def test_plan(T, k, N, wide):
    g = gen(T + k + N)
    experts = (N * torch.rand(T, k, generator=g) ** 2).long().clamp(max=N - 1)
    experts[torch.rand(T, k, generator=g) < 0.05] = -1
    if T > 10:
        experts[3], experts[5, 0], experts[9, -1] = 0, N, -7
    if wide and T > 10:
        experts[4, 0] = 2 ** 40
    dev = experts.cuda() if wide else experts.int().cuda()
    for capacity in (None, 0, 1, max(1, T * k // N), 3 * T * k):
        p = expert_plan(dev, N, capacity)
        slots, counts = ox.plan(experts if wide else experts.int(), N, T if capacity is None else capacity)
        assert p.num_experts == N and p.capacity == (T if capacity is None else capacity)
        assert torch.equal(p.slots.cpu(), slots) and torch.equal(p.counts.cpu(), counts)


def test_plan_one_expert_takes_all():
    for T in (100, 5000, 70000):
        p = expert_plan(torch.full((T, 1), 3, dtype=torch.int32, device="cuda"), 8, T)
        assert torch.equal(p.slots[:, 0].cpu().long(), 3 * T + torch.arange(T)) and p.counts.tolist() == [0, 0, 0, T] + [0] * 4


# ---- copies ----
def choice(T, k, N, g):
    return torch.stack([torch.randperm(N, generator=g)[:k] for _ in range(T)]).int() if T else torch.zeros(0, k, dtype=torch.int32)


COPIES = [(1, 1, 1, 16, None), (7, 2, 3, 64, None), (130, 2, 8, 128, 20), (65, 3, 5, 100, 40), (33, 5, 9, 201, 7), (50, 1, 4, 1, 9),
          (20, 4, 4, 256, 20), (9, 2, 3, 1030, 4), (12, 2, 6, 3000, None), (3, 2, 2, 8, 0), (40, 7, 11, 33, 25), (0, 2, 3, 32, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N,D,capacity", COPIES)
def test_dispatch(T, k, N, D, capacity, dtype):
    g = gen(T + D)
    experts = choice(T, k, N, g)
    x = torch.randn(T, D, generator=g).to(dtype)
    p = expert_plan(experts.cuda(), N, capacity)
    xd = x.cuda().requires_grad_(True)
    rows = expert_dispatch(xd, p)
    slots, _ = ox.plan(experts, N, p.capacity)
    want, _ = ox.scatter64(x, slots, N, p.capacity)
    assert rows.shape == (N, p.capacity, D) and rows.dtype == dtype
    assert torch.equal(rows.detach().cpu().double(), want)
    drows = torch.randn(N, p.capacity, D, generator=g).to(dtype)
    (dx,) = torch.autograd.grad(rows, xd, drows.cuda())
    want, bound = ox.gather64(drows, slots)
    assert dx.dtype == dtype and ox.over(dx, want, bound) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N,D,capacity", COPIES)
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(T, k, N, D, capacity, weighted, dtype):
    g = gen(T + D + 1)
    experts = choice(T, k, N, g)
    p = expert_plan(experts.cuda(), N, capacity)
    slots, _ = ox.plan(experts, N, p.capacity)
    rows = torch.randn(N, p.capacity, D, generator=g).to(dtype)
    do = torch.randn(T, D, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g) if weighted else None
    rd = rows.cuda().requires_grad_(True)
    wd = w.cuda().requires_grad_(True) if weighted else None
    o = expert_combine(rd, p, wd)
    want, bound = ox.gather64(rows, slots, w)
    assert o.shape == (T, D) and o.dtype == dtype and ox.over(o, want, bound) <= 1
    grads = torch.autograd.grad(o, (rd, wd) if weighted else (rd,), do.cuda())
    want, bound = ox.scatter64(do, slots, N, p.capacity, w)
    assert grads[0].dtype == dtype and ox.over(grads[0], want, bound) <= 1
    if weighted:
        want, bound = ox.dot64(rows, do, slots)
        assert grads[1].dtype == FL and ox.over(grads[1], want, bound) <= 1


def test_gradients_of_one_side_alone():
    g = gen(5)
    experts = choice(40, 2, 6, g)
    p = expert_plan(experts.cuda(), 6, 9)
    rows, w, do = torch.randn(6, 9, 64, generator=g).cuda(), torch.rand(40, 2, generator=g).cuda(), torch.randn(40, 64, generator=g).cuda()
    both = torch.autograd.grad(expert_combine(rows.requires_grad_(), p, w.requires_grad_()), (rows, w), do)
    one = torch.autograd.grad(expert_combine(rows, p, w.detach()), rows, do)
    two = torch.autograd.grad(expert_combine(rows.detach(), p, w), w, do)
    assert torch.equal(both[0], one[0]) and torch.equal(both[1], two[0])


def test_dropped_choices_bring_nothing_of_what_is_not_finite():
    """infinities and NaN of dropped tokens, of rows without a token and of weights of dropped choices stay where they are"""
    experts = torch.zeros(4, 2, dtype=torch.int32)
    experts[:, 1] = 1
    p = expert_plan(experts.cuda(), 2, 2)  # tokens 2 and 3 are dropped
    x = torch.ones(4, 32)
    x[2], x[3] = float("inf"), float("nan")
    rows = expert_dispatch(x.cuda(), p)
    assert torch.equal(rows, torch.ones_like(rows))
    w = torch.ones(4, 2)
    w[2:] = float("nan")
    rd, wd = rows.requires_grad_(True), w.cuda().requires_grad_(True)
    o = expert_combine(rd, p, wd)
    assert torch.equal(o[:2], torch.full_like(o[:2], 2.0)) and (o[2:] == 0).all()
    drows, dw = torch.autograd.grad(o, (rd, wd), x.cuda())
    assert torch.equal(drows, torch.ones_like(drows)) and (dw[:2] == 32).all() and (dw[2:] == 0).all()
    p = expert_plan(experts[:1].cuda(), 2, 3)  # rows 1 and 2 of each expert have no token
    rows = torch.full((2, 3, 32), float("nan"), device="cuda")
    rows[:, 0] = 1
    assert (expert_combine(rows, p, w[:1].cuda()) == 2).all()


def test_views_and_guards():
    """tokens in any layout; what lies beside the rows is not written"""
    g = gen(6)
    experts = choice(60, 2, 5, g).cuda()
    p = expert_plan(experts, 5, 30)
    base = torch.randn(70, 90, generator=g).to(BF).cuda()
    for x in (base[:60, 1:70], base[3:63, :64], base.t()[:60, 5:69], base[:1, :33].expand(60, 33), base[:60, ::2]):
        assert torch.equal(expert_dispatch(x, p), expert_dispatch(x.contiguous(), p))
    rows = torch.randn(5, 33, 70, generator=g).to(BF).cuda()
    w = torch.rand(60, 4, generator=g).cuda()
    v = rows[:, :30, 3:69]
    assert torch.equal(expert_combine(v, p, w[:, ::2]), expert_combine(v.contiguous(), p, w[:, ::2].contiguous()))
    assert torch.equal(expert_plan(experts.t().contiguous().t(), 5, 30).slots, p.slots)
    q = ExpertPlan(p.slots.t().contiguous().t(), p.counts, 5, 30)
    assert torch.equal(expert_dispatch(base[:60, :64], q), expert_dispatch(base[:60, :64], p))


def test_slots_out_of_range_count_as_dropped():
    p = ExpertPlan(torch.tensor([[0, 6], [-5, 1], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device="cuda"),
                   torch.tensor([2, 0], dtype=torch.int32, device="cuda"), 2, 3)
    x = torch.arange(96.0, device="cuda").view(3, 32) + 1
    rows = expert_dispatch(x, p)
    assert torch.equal(rows[0, :2], x[:2]) and (rows[0, 2:] == 0).all() and (rows[1] == 0).all()
    o = expert_combine(rows, p)
    assert torch.equal(o[:2], x[:2]) and (o[2] == 0).all()


def test_repeatable_on_another_stream():
    g = gen(7)
    experts = choice(3000, 4, 16, g).cuda()
    x = torch.randn(3000, 128, generator=g).to(BF).cuda()
    w = torch.rand(3000, 4, generator=g).cuda()
    torch.cuda.synchronize()

    def once():
        p = expert_plan(experts, 16, 700)
        rows = expert_dispatch(x, p)
        return (*p[:2], rows, expert_combine(rows, p, w))

    first = once()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_graph_of_a_step():
    """route, plan, dispatch, combine and their gradients, captured once and replayed on new inputs"""
    g = gen(8)
    T, N, k, D = 5000, 12, 2, 64
    logits, x, do = torch.zeros(T, N, device="cuda"), torch.zeros(T, D, device="cuda", dtype=HF), torch.zeros(T, D, device="cuda", dtype=HF)
    logits.requires_grad_(True)
    x.requires_grad_(True)

    def step(logits, x):
        w, e = expert_route(logits, k)
        p = expert_plan(e, N, 900)
        rows = expert_dispatch(x, p)
        o = expert_combine(rows, p, w)
        return (o, p.slots, p.counts, *torch.autograd.grad(o, (logits, x), do))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(logits, x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(logits, x)
    for i in range(4):
        with torch.no_grad():
            logits.copy_(torch.randn(T, N, generator=g))
            x.copy_(torch.randn(T, D, generator=g))
            do.copy_(torch.randn(T, D, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(logits.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_differences():
    """gradients along a direction against differences, in full precision"""
    g = gen(9)
    T, N, k, D = 30, 6, 2, 32
    # logits half a unit apart, so that no choice changes on the way
    logits = torch.stack([torch.randperm(N, generator=g) for _ in range(T)]).cuda() / 2
    x = torch.randn(T, D, generator=g).cuda()
    do = torch.randn(T, D, generator=g).cuda()
    scale = torch.arange(1, N + 1, device="cuda").view(N, 1, 1).float()  # the experts: a factor of each

    def loss(logits, x):
        w, e = expert_route(logits, k, normalize=False)
        p = expert_plan(e, N, 9)
        return (expert_combine(expert_dispatch(x, p) * scale, p, w).double() * do).sum()

    a, b = logits.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ga, gb = torch.autograd.grad(loss(a, b), (a, b))
    da, db = torch.rand(T, N, generator=g).cuda() * 2 - 1, torch.randn(T, D, generator=g).cuda()
    h = 2.0 ** -8
    diff = ((loss(logits + h * da, x + h * db) - loss(logits - h * da, x - h * db)) / (2 * h)).item()
    want = ((ga.double() * da).sum() + (gb.double() * db).sum()).item()
    # third derivatives times h^2 / 6, and fp32 sums over h
    size = (ga.double() * da).abs().sum().item() + (gb.double() * db).abs().sum().item() + 1
    assert abs(diff - want) <= size * (h * h + 64 * 2.0 ** -24 / h)
