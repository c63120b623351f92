"""orthogonalize and muon_step against 64 bits: both orientations, small sides at and around every padded size, long sides from
one on, spectra of several decades, types in any mix, many stacks in a call, steps and coefficients, refusals.

Bounds are those that oracle/muon.py derives."""
import pytest
import torch

from flashmlp_amd import GatedFlashMLP, clip_grads, muon_step, orthogonalize
from oracle import muon as om
from oracle.gated import UNIT

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
TYPES = (BF, HF, FL)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check(x, o, steps=5, coefficients=om.COEFFICIENTS, eps=1e-7):
    want = om.orthogonal64(x, steps, coefficients, eps)
    got = o.double().cpu()
    assert o.shape == x.shape and o.dtype == x.dtype and torch.isfinite(got).all()
    tol = UNIT[x.dtype] * want.abs() + 1.01 * om.bound(x, steps, coefficients, x.dtype == FL)
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


SHAPES = [(3, 16, 40), (2, 32, 32), (2, 33, 70), (1, 64, 683), (3, 64, 1), (2, 100, 300), (2, 128, 129), (2, 129, 300), (1, 201, 640),
          (2, 256, 256), (3, 256, 1031), (1, 1, 1), (2, 1, 1000), (1, 7, 2049), (5, 128, 64), (4, 300, 20), (1, 5000, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("H,R,C", SHAPES)
def test_orthogonalize(H, R, C, tall, dtype):
    x = torch.randn(H, R, C, generator=gen(R + C)).mul(1e-3)
    x = (x.mT.contiguous() if tall else x).to(dtype)
    check(x, orthogonalize(x.cuda()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,e", [(24, 100), (64, 500), (128, 128), (128, 700), (200, 256)])
@pytest.mark.parametrize("decades", [1, 4])
def test_spectra_of_several_decades(n, e, decades, dtype):
    """singular values that fall evenly in their logarithm, in stacks of both orientations"""
    g = gen(n + e)
    q, r = torch.linalg.qr(torch.randn(2, n, n, generator=g, dtype=torch.float64))[0], torch.linalg.qr(
        torch.randn(2, e, n, generator=g, dtype=torch.float64))[0]
    s = 10.0 ** (-decades * torch.arange(n, dtype=torch.float64) / n)
    x = ((q * s) @ r.mT).to(dtype)
    check(x, orthogonalize(x.cuda()))
    t = x.mT.contiguous()
    check(t, orthogonalize(t.cuda()))


@pytest.mark.parametrize("dtype,steps", [(FL, 1), (FL, 2), (FL, 3), (FL, 4), (BF, 1), (BF, 6), (HF, 10), (FL, 10)])
@pytest.mark.parametrize("n", [50, 128, 256])
def test_steps(n, steps, dtype):
    x = torch.randn(2, n, 300, generator=gen(n)).to(dtype)
    check(x, orthogonalize(x.cuda(), steps=steps), steps)


@pytest.mark.parametrize("R,C", [(32, 33), (64, 64), (64, 128), (96, 128), (100, 400), (140, 128), (201, 220), (256, 256), (300, 256), (256, 400)])
def test_full_precision_is_that_of_the_products(R, C):
    """fp32 results of noise around a low rank, whose singular values reach over two to three decades: at most twice as far off, in norm,
    as fp32 products of the matrices themselves, which have the same number of roundings of the same size"""
    g = gen(R + C)
    x = torch.randn(3, R, 8, generator=g) @ torch.randn(3, 8, C, generator=g) / 8 ** 0.5 + 0.5 * torch.randn(3, R, C, generator=g)
    want = om.orthogonal64(x)
    y = x.mT if R > C else x
    y = y / (torch.linalg.matrix_norm(y, keepdim=True) + 1e-7)
    for a, b, c in om.triples(om.COEFFICIENTS, 5):
        t = y @ y.mT
        y = a * y + (b * t + c * (t @ t)) @ y
    y = y.mT if R > C else y
    off = (orthogonalize(x.cuda()).double().cpu() - want).norm()
    assert off <= 2 * (y.double() - want).norm()


def test_coefficients_of_every_step():
    x = torch.randn(3, 60, 200, generator=gen(1))
    c = [(3.4445, -4.775, 2.0315), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)]
    check(x, orthogonalize(x.cuda(), steps=4, coefficients=c), 4, c)
    o = orthogonalize(x.cuda(), steps=10, coefficients=(1.875, -1.25, 0.375)).double()
    assert (o @ o.mT - torch.eye(60, device="cuda")).abs().max() < 1e-4  # (this one ends at orthogonal matrices)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-7, 1.0, 1e12])
def test_sizes_of_the_values(scale):
    """the norm, not the values' size, decides; values far below eps stay small"""
    for n in (40, 128, 256):
        x = torch.randn(2, n, 300, generator=gen(2)) * scale
        want = om.orthogonal64(x)
        got = orthogonalize(x.cuda()).double().cpu()
        tol = 1.01 * om.bound(x, full=True) * min(1.0, want.abs().max().item() * 8)
        assert ((got - want).abs() <= 2.0 ** -22 * want.abs() + tol).all()
    tiny = (torch.randn(1, 64, 300, generator=gen(3)) * 3e-7).half()  # most of them below fp16's normal numbers
    check(tiny, orthogonalize(tiny.cuda()))


def test_zero_and_non_finite_matrices_keep_to_themselves():
    for dtype in TYPES:
        for n in (64, 256):
            x = torch.randn(4, n, 260, generator=gen(4)).to(dtype)
            clean = orthogonalize(x.cuda())
            x[1] = 0
            x[2, 3, 5] = float("nan")
            x[3, 1, 1] = float("inf")
            o = orthogonalize(x.cuda())
            assert torch.equal(o[0], clean[0]) and (o[1] == 0).all() and torch.isnan(o[2]).any() and torch.isnan(o[3]).any()


def test_in_place_out_and_views():
    x = torch.randn(3, 48, 90, generator=gen(5)).cuda()
    want = orthogonalize(x)
    out = torch.empty_like(x)
    assert orthogonalize(x, out=out) is out and torch.equal(out, want)
    y = x.clone()
    v = y._version
    assert orthogonalize(y, out=y) is y and torch.equal(y, want) and y._version > v
    flat = torch.full((1 + x.numel() + 1,), 7.0, device="cuda")
    z = flat[1:-1].view(x.shape)
    z.copy_(x)
    orthogonalize(z, out=z)
    assert torch.equal(z, want) and flat[0] == 7 and flat[-1] == 7
    base = torch.randn(3, 90, 48, generator=gen(6)).cuda()
    assert torch.equal(orthogonalize(base.mT), orthogonalize(base.mT.contiguous()))
    wide = torch.zeros(3, 48, 99, device="cuda")
    orthogonalize(x, out=wide[..., 3:93])
    assert torch.equal(wide[..., 3:93], want) and (wide[..., :3] == 0).all() and (wide[..., 93:] == 0).all()
    assert torch.equal(orthogonalize(x[1]), want[1]) and torch.equal(orthogonalize(x.view(3, 1, 48, 90)).view(3, 48, 90), want)
    assert orthogonalize(x[:0]).shape == (0, 48, 90) and orthogonalize(x[..., :0]).shape == (3, 48, 0)


def stacks(shapes, types, seed):
    g = gen(seed)
    w = [torch.randn(s, generator=g).div(s[-2] ** 0.5).to(types[0]) for s in shapes]
    gr = [(10.0 ** -(i % 3) * torch.randn(s, generator=g)).to(types[1]) for i, s in enumerate(shapes)]
    m = [(10.0 ** -(i % 3) * 0.5 * torch.randn(s, generator=g)).to(types[2]) for i, s in enumerate(shapes)]
    return w, gr, m


LISTS = {
    "one": [(64, 100)],
    "layer": [(6, 64, 200), (6, 64, 200), (6, 200, 64)],
    "mixed": [(2, 32, 50), (3, 128, 130), (1, 256, 300), (2, 300, 256), (0, 16, 16), (5, 16, 7), (2, 70, 64), (100, 3)],
    "many": [(1 + i % 3, 16 + i % 40, 20 + 7 * (i % 11)) for i in range(150)],
}


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("types", [(FL, BF, FL), (BF, BF, BF), (HF, FL, HF), (FL, FL, FL), (BF, HF, FL)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(name, types, nesterov):
    w, g, m = stacks(LISTS[name], types, 7)
    dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
    muon_step(dw, dg, dm, 0.02, nesterov=nesterov, weight_decay=0.1)
    for i in range(len(w)):
        want = om.step64(w[i], g[i], m[i], 0.02, nesterov=nesterov, weight_decay=0.1)
        assert torch.equal(dg[i].cpu(), g[i])
        for t, got in (("w", dw[i]), ("m", dm[i])):
            ref, tol = want[t]
            tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -130
            assert ((got.double().cpu() - ref).abs() <= 1.01 * tol + tiny).all(), (i, t)


def test_options():
    w, g, m = stacks([(2, 40, 90), (2, 90, 40)], (FL, FL, FL), 8)
    for kw in (dict(scale=0.2), dict(momentum=0.0), dict(momentum=1.0), dict(steps=7), dict(eps=1e-3, steps=2), dict(weight_decay=0.5)):
        dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
        muon_step(dw, dg, dm, 0.1, **kw)
        for i in range(2):
            want = om.step64(w[i], g[i], m[i], 0.1, **kw)
            for t, got in (("w", dw[i]), ("m", dm[i])):
                assert ((got.double().cpu() - want[t][0]).abs() <= 1.01 * want[t][1] + 2.0 ** -130).all(), (kw, i, t)


def test_layouts_single_tensors_and_versions():
    w, g, m = (v[0].cuda() for v in stacks([(3, 40, 70)], (FL, BF, FL), 9))
    w2, m2 = w.clone(), m.clone()
    p = torch.nn.Parameter(w2)
    v = p._version
    muon_step(p, g, m2, 0.1)
    assert p._version > v and m2._version > 0
    wt, mt, gt = (t.mT.contiguous().mT for t in (w, m, g))
    muon_step([wt], [gt], [mt], 0.1)
    assert torch.equal(wt, p.detach()) and torch.equal(mt, m2)


def test_flat_buffers_guards_and_streams():
    """parameters and momenta as views of one buffer at odd places, gradients clipped into another one"""
    shapes = [(2, 33, 45), (1, 16, 7), (3, 64, 65)]
    w, g, m = stacks(shapes, (FL, BF, FL), 10)
    n = sum(t.numel() for t in w)
    flat = [torch.full((n + len(w) + 1,), 7.0, device="cuda") for _ in range(3)]
    views, at = [[], [], []], 1
    for t in w:
        for v, f in zip(views, flat):
            v.append(f[at:at + t.numel()].view(t.shape))
        at += t.numel() + 1
    for v, t in zip(views[0] + views[1], w + m):
        v.copy_(t)
    dg = [t.cuda() for t in g]
    clip_grads(dg, 1.0, out=views[2])
    alone = [t.cuda() for t in w], [t.clone() for t in views[2]], [t.cuda() for t in m]
    muon_step(*alone, 0.05)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        muon_step(views[0], views[2], views[1], 0.05)
    s.synchronize()
    for k, v in ((0, views[0]), (2, views[1])):
        assert all(torch.equal(a, b) for a, b in zip(alone[k], v))
    at = 0
    for t in [*w, None]:
        assert all(f[at] == 7 for f in flat[:2])
        at += 1 + (t.numel() if t is not None else 0)


def test_graph():
    """captured once, replayed with new gradients between eager work, against eager steps"""
    shapes = [(4, 64, 96), (4, 96, 64), (2, 200, 256)]
    w, g, m = ([t.cuda() for t in v] for v in stacks(shapes, (FL, BF, FL), 11))
    we, me = [t.clone() for t in w], [t.clone() for t in m]
    muon_step([t.clone() for t in w], g, [t.clone() for t in m], 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(w, g, m, 0.1)
    for i in range(4):
        for t in g:
            t.copy_(torch.randn(t.shape, generator=gen(20 + i)))
        graph.replay()
        muon_step(we, g, me, 0.1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(w + m, we + me)), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H", [1, 12, 13, 31, 32])
@pytest.mark.parametrize("n,e", [(130, 137), (192, 64 * 5), (256, 2000)])
def test_few_wide_matrices(H, n, e, dtype):
    """and a matrix alone in the middle of its memory: what lies around it stays"""
    x = torch.randn(H, n, e, generator=gen(n + H)).to(dtype)
    buf = torch.full((H * n * e + 128,), 7.0, dtype=dtype, device="cuda")
    out = buf[64:-64].view(H, n, e)
    check(x, orthogonalize(x.cuda(), out=out))
    assert (buf[:64] == 7).all() and (buf[-64:] == 7).all()
    t = x.mT.contiguous()
    check(t, orthogonalize(t.cuda()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("n,e", [(7, 300), (32, 20), (50, 129), (64, 128), (100, 65), (128, 200)])
def test_many_matrices(n, e, tall, dtype):
    """as many as take a workgroup each from end to end"""
    x = torch.randn(700, n, e, generator=gen(n * e)).mul(1e-2)
    x = (x.mT.contiguous() if tall else x).to(dtype)
    check(x, orthogonalize(x.cuda()))


@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("H,n,e", [(70, 200, 210), (64, 256, 300), (65, 129, 136), (400, 140, 150)])
def test_many_wide_matrices(H, n, e, dtype):
    x = torch.randn(H, n, e, generator=gen(n * e)).to(dtype)
    check(x, orthogonalize(x.cuda()))
    check(x[:3].mT.contiguous(), orthogonalize(x.mT.contiguous().cuda())[:3])


@pytest.mark.parametrize("types", [(FL, BF, FL), (BF, HF, BF)])
def test_muon_step_of_many_matrices(types):
    """the same with weights and momenta, in stacks of both orientations and several sizes"""
    shapes = [(300, 40, 70), (400, 70, 40), (350, 64, 33), (350, 128, 140), (513, 20, 30), (1, 20, 31), (3, 140, 128)]
    w, g, m = stacks(shapes, types, 13)
    dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
    muon_step(dw, dg, dm, 0.02, weight_decay=0.1)
    for i in range(len(w)):
        want = om.step64(w[i], g[i], m[i], 0.02, weight_decay=0.1)
        for t, got in (("w", dw[i]), ("m", dm[i])):
            ref, tol = want[t]
            tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -130
            assert ((got.double().cpu() - ref).abs() <= 1.01 * tol + tiny).all(), (i, t)


@pytest.mark.parametrize("types", [(FL, BF, FL), (HF, FL, BF)])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(3, 256, 264), (2, 1000, 133)], [(9, 150, 300)], [(7, 200, 131), (8, 256, 512), (1, 256, 1)], [(30, 129, 200)],
                                    [(40, 256, 260), (30, 201, 150)]])
def test_muon_step_of_wide_matrices(shapes, types, nesterov):
    """small sides above 128: Gram matrices by tiles and by parts, products of few and of many, a small side shorter than a tile's"""
    w, g, m = stacks(shapes, types, 15)
    dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
    muon_step(dw, dg, dm, 0.02, nesterov=nesterov)
    for i in range(len(w)):
        want = om.step64(w[i], g[i], m[i], 0.02, nesterov=nesterov)
        for t, got in (("w", dw[i]), ("m", dm[i])):
            ref, tol = want[t]
            tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -130
            assert ((got.double().cpu() - ref).abs() <= 1.01 * tol + tiny).all(), (i, t)


def test_a_matrix_does_not_depend_on_what_is_beside_it():
    x = torch.randn(9, 64, 500, generator=gen(12)).to(BF).cuda()
    assert (orthogonalize(x)[4].float() - orthogonalize(x[4]).float()).abs().max() <= 2.0 ** -8 * 0.3


def test_refusals_of_overlap():
    t = torch.zeros(2, 8, 9, device="cuda")
    a, b, c = t.clone(), t.clone(), t.clone()
    for args in (([a, a], [b, b], [c, t]), ([a], [b], [a]), ([a], [a], [c])):
        with pytest.raises(RuntimeError, match="overlap"):
            muon_step(*args, 0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        orthogonalize(t[0:1], out=t.view(-1)[9:81].view(1, 8, 9))
    muon_step([a, c], [b, b], [t, t.clone()], 0.1)  # (gradients are only read)


def test_refusals_of_overlap_in_other_layouts():
    """nothing is written before the refusal; the parts of a fused weight are taken"""
    t = torch.ones(2, 8, 9, device="cuda")
    g, other = torch.ones(2, 9, 8, device="cuda"), torch.ones(2, 9, 8, device="cuda")
    for w, m in ((t.mT, t.view(2, 9, 8)), (other, other.new_ones(2, 9, 1).expand(2, 9, 8))):
        with pytest.raises(RuntimeError, match="overlap"):
            muon_step([w], [g], [m], 0.1)
        assert (w == 1).all() and (m == 1).all()
    fused, g, m = (v[0].cuda() for v in stacks([(2, 24, 40)], (FL, FL, FL), 13))
    parts = [[v[..., :17], v[..., 17:]] for v in (fused, g, m)]
    alone = [[v.contiguous() for v in p] for p in parts]
    muon_step(*alone, 0.1)
    muon_step(*parts, 0.1)
    for p, a in zip(parts, alone):
        assert all(torch.equal(u, v) for u, v in zip(p, a))


def test_learns_with_the_gated_mlp_stacks():
    """the shapes a module's parameters have, gradients from its backward, clipped into full precision"""
    torch.manual_seed(0)
    mlp = GatedFlashMLP(4, 64, 96, dtype=BF)
    x = torch.randn(4, 100, 64, device="cuda", dtype=BF)
    mlp(x).float().square().mean().backward()
    params = list(mlp.parameters())
    out = [torch.empty(p.shape, device="cuda") for p in params]
    clip_grads([p.grad for p in params], 1.0, out=out)
    momenta = [torch.zeros(p.shape, device="cuda") for p in params]
    before = [p.detach().cpu() for p in params]
    muon_step(params, out, momenta, 0.02)
    for b, p, g in zip(before, params, out):
        ref, tol = om.step64(b, g.cpu(), torch.zeros(b.shape), 0.02)["w"]
        assert ((p.detach().double().cpu() - ref).abs() <= 1.01 * tol).all()
