"""grad_norm, clip_grads and clip_grad_norm_ against 64-bit sums: types in any mix, sizes from none to past a
workgroup's chunk, hundreds of tensors, odd bases, layouts, non-finite values and refusals.

The norm is a 64-bit sum rounded once to fp32 (2^-24, its root and the coefficient's division a few more); a
clipped value has the coefficient's error, 2^-22 at most, and its own rounding."""
import pytest
import torch

from flashmlp_amd import GatedFlashMLP, clip_grad_norm_, clip_grads, grad_norm
from oracle.gated import UNIT

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def tensors(shapes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * 10.0 ** (i % 3 - 1) * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]).cuda()
            for i, s in enumerate(shapes)]


def norm64(ts):
    return sum(t.double().pow(2).sum().item() for t in ts) ** 0.5


def check(grads, outs, norm, before, max_norm):
    want = norm64(before)
    assert norm.dtype == FL and norm.dim() == 0 and abs(norm.item() - want) <= 2.0 ** -22 * want
    coef = min(1.0, max_norm / (want + 1e-6)) if want > 0 else 1.0
    for b, o in zip(before, outs):
        w = b.double() * coef
        u = UNIT[o.dtype]
        tiny = 2.0 ** -25 if o.dtype == HF else 0.0
        assert o.shape == b.shape
        if coef == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b)
        assert ((o.double() - w).abs() <= 1.01 * (u + 2.0 ** -21) * w.abs() + tiny).all()


SHAPES = {
    "one": [(1,)],
    "small": [(3,), (0,), (17, 5), (2, 3, 4), (1,), (4096,)],
    "chunks": [(8191,), (8192,), (8193,), (100003,), (7,)],
    "large": [(3000, 1001), (70001,), (2048, 2048)],
    "many": [(i % 37 * 13,) for i in range(400)],
}


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("dtypes", [(BF,), (HF,), (FL,), (BF, FL, HF)])
def test_norm_and_clipping(name, dtypes):
    grads = tensors(SHAPES[name], dtypes)
    before = [g.clone() for g in grads]
    want = norm64(before)
    n = grad_norm(grads)
    assert abs(n.item() - want) <= 2.0 ** -22 * want
    for max_norm in (0.5, 1e9):
        for odt in (FL, BF, HF):
            outs = [torch.full(g.shape, 7.0, dtype=odt, device="cuda") for g in grads]
            r, norm = clip_grads(grads, max_norm, out=outs)
            assert all(a is b for a, b in zip(r, outs))
            check(grads, outs, norm, before, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    r, norm = clip_grads(grads, 0.5)
    check(grads, grads, norm, before, 0.5)


def test_in_place_within_the_limit_changes_nothing():
    grads = tensors([(1000,), (33, 7)], (BF,))
    before = [g.clone() for g in grads]
    clip_grads(grads, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_guards_and_odd_bases():
    """views one after the other in one buffer, each at an element's alignment; nothing beside them is written"""
    sizes = [1, 8191, 5, 20000, 3]
    for dt in (BF, FL):
        flat = torch.randn(1 + sum(sizes) + 1, device="cuda").to(dt)
        buf = torch.full((1 + sum(sizes) + len(sizes) + 1,), 7.0, dtype=FL, device="cuda")
        grads, outs, i, j = [], [], 1, 1
        for n in sizes:
            grads.append(flat[i:i + n])
            outs.append(buf[j:j + n])
            i, j = i + n, j + n + 1
        before = flat.clone()
        _, norm = clip_grads(grads, 1.0, out=outs)
        check(grads, outs, norm, [g.clone() for g in grads], 1.0)
        assert torch.equal(flat, before)
        at, ends = 1, []
        for n in sizes:
            at += n
            ends.append(at)
            at += 1
        assert buf[0] == 7 and all(buf[e] == 7 for e in ends) and buf[-1] == 7
        clip_grads(grads, 1.0)
        assert flat[0] == before[0] and flat[-1] == before[-1]


def test_layouts():
    """transposed and strided gradients and outputs"""
    a, b = tensors([(40, 70), (30, 50)], (BF,))
    for grads in ([a.t(), b], [a[:, ::2], b[::3]], [a.t()[5:], b[:, 3:9].t()]):
        want = [g.clone() for g in grads]
        outs = [torch.zeros(g.shape[::-1], dtype=FL, device="cuda").t() for g in grads]
        _, norm = clip_grads(grads, 0.1, out=outs)
        check(grads, outs, norm, want, 0.1)
        outs = [torch.zeros(*g.shape, 2, dtype=FL, device="cuda")[..., 0] for g in grads]
        _, norm = clip_grads(grads, 0.1, out=outs)
        check(grads, outs, norm, want, 0.1)
        assert abs(grad_norm(grads).item() - norm64(want)) <= 2.0 ** -22 * norm64(want)
        _, norm = clip_grads(grads, 0.1)
        check(grads, grads, norm, want, 0.1)


def test_extreme_values():
    big = torch.full((1000,), 1e30, device="cuda").to(BF)  # squares beyond fp32
    want = norm64([big])
    assert abs(grad_norm([big]).item() - want) <= 2.0 ** -22 * want
    small = torch.full((1000,), 1e-30, device="cuda")  # squares below fp32
    want = norm64([small])
    assert abs(grad_norm([small]).item() - want) <= 2.0 ** -22 * want
    zero = torch.zeros(100, device="cuda")
    out, norm = clip_grads([zero], 1.0)
    assert norm == 0 and not zero.any()
    for bad in (float("inf"), float("nan")):
        g = torch.ones(100, device="cuda")
        g[7] = bad
        ref = [torch.nn.Parameter(torch.zeros(100, device="cuda"))]
        ref[0].grad = g.clone()
        torch.nn.utils.clip_grad_norm_(ref, 1.0)
        _, norm = clip_grads([g], 1.0)
        assert not norm.isfinite() and torch.equal(g.isnan(), ref[0].grad.isnan())
        assert torch.equal(g.nan_to_num(), ref[0].grad.nan_to_num())


def test_max_norm_zero_and_infinite():
    (g,) = tensors([(500,)], (FL,))
    before = g.clone()
    clip_grads([g], float("inf"))
    assert torch.equal(g, before)
    clip_grads([g], 0.0)
    assert not g.any()


def test_module_parameters_and_torch():
    torch.manual_seed(0)
    m = GatedFlashMLP(2, 64, 96, dtype=FL)
    x = torch.randn(2, 50, 64, device="cuda")
    m(x).square().sum().backward()
    m.extra = torch.nn.Parameter(torch.zeros(3, device="cuda"))  # without a gradient
    before = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    n = clip_grad_norm_(m.parameters(), 0.7)
    check(None, [p.grad for p in m.parameters() if p.grad is not None], n, before, 0.7)
    assert m.extra.grad is None
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.full((4,), float("inf"), device="cuda")
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert p.grad.isinf().all()
    assert clip_grad_norm_([], 1.0) == 0 and grad_norm([]) == 0
    assert grad_norm([torch.zeros(0, device="cuda")]) == 0


def test_repeatable_on_streams_and_in_graphs():
    grads = tensors([(70001,), (300, 41), (5,)] * 60, (BF, FL))
    ref = [g.clone() for g in grads]
    outs, norm = clip_grads(grads, 1.0, out=ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, n2 = clip_grads(grads, 1.0, out=[g.clone() for g in grads])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(outs, o2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    o3 = [torch.zeros_like(g) for g in grads]
    with torch.cuda.graph(graph):
        _, n3 = clip_grads(grads, 1.0, out=o3)
    for i in range(4):
        grads[0].mul_(1.5)
        n3.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        o4, n4 = clip_grads(grads, 1.0, out=[g.clone() for g in grads])
        assert torch.equal(n3, n4) and all(torch.equal(a, b) for a, b in zip(o3, o4))


def test_autograd_notices_a_saved_tensor_that_was_clipped():
    for g in (torch.full((64,), 3.0, device="cuda"), torch.full((8, 16), 3.0, device="cuda").t(),
              torch.full((8, 16), 3.0, device="cuda")[:, ::2]):
        w = torch.ones_like(g).requires_grad_(True)
        y = (w * g).sum()  # saves g
        clip_grads([g], 0.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():
            h = torch.full((64,), 3.0, device="cuda")
            clip_grads([h, torch.full((8, 16), 3.0, device="cuda").t()], 0.5)
        clip_grads([h], 0.25)
        assert abs(h.norm().item() - 0.25) <= 1e-5


def test_a_parameter_listed_twice_counts_once():
    p, q = (torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (100001, 7))
    p.grad, q.grad = torch.full_like(p, 2.0), torch.full_like(q, 3.0)
    before = [p.grad.clone(), q.grad.clone()]
    norm = clip_grad_norm_([p, q, p], 1.0)
    check(None, [p.grad, q.grad], norm, before, 1.0)


def test_refusals():
    g = tensors([(4,), (5,)], (FL,))
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads(g, -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads(g, float("nan"))
    with pytest.raises(ValueError, match="outputs"):
        clip_grads(g, 1.0, out=g[:1])
    with pytest.raises(ValueError, match="shape"):
        clip_grads(g, 1.0, out=[g[1], g[0]])
    with pytest.raises(TypeError):
        grad_norm([g[0].double()])
    with pytest.raises(TypeError):
        clip_grads(g, 1.0, out=[t.double() for t in g])
    with pytest.raises(RuntimeError, match="GPU"):
        grad_norm([g[0].cpu()])
    with pytest.raises(RuntimeError, match="one device"):
        grad_norm([g[0], g[1].cpu()])
