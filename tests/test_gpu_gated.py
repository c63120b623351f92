"""The gated MLP against its definition in 64 bits, elementwise within the bounds of oracle/gated.py.

Sizes at the edges of the kernels' tiles (32 columns of E, 32 to 256 rows), one row, one column, no row;
every io type, activation and D; views, streams, graphs and repeatability.
"""
import pytest
import torch

from flashmlp_amd import GatedFlashMLP, GatedFlashMLPFunction, flashmlp_gated_bwd, flashmlp_gated_fwd
from oracle.gated import excess, gated64

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
NAMES = ("o", "dx", "dwg", "dwu", "dw2")


def make(H, B, D, E, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = (n(H, B, D), n(H, D, E) / D ** 0.5, n(H, D, E) / D ** 0.5, n(H, E, D) / E ** 0.5, n(H, B, D))
    return tuple(v.to(dt).cuda() for v in t)


def both(x, wg, wu, w2, do, act):
    return (flashmlp_gated_fwd(x, wg, wu, w2, act), *flashmlp_gated_bwd(x, wg, wu, w2, do, act))


def check(got, t, act):
    want, bounds = gated64(*t, act)
    for name, a, w, b in zip(NAMES, got, want, bounds):
        assert a.shape == w.shape and a.dtype == t[0].dtype and a.is_contiguous(), name
        e = excess(a, w, b, t[0].dtype)
        assert e <= 1.0, (name, e)


CASES = [
    # H, B, D, E, dtype, act
    (2, 1, 16, 1, BF, "silu"), (1, 1, 64, 64, HF, "silu"), (3, 2, 128, 32, BF, "sigmoid"),
    (2, 33, 16, 8, HF, "leaky_relu"), (2, 31, 32, 45, BF, "silu"), (3, 64, 32, 96, HF, ""),
    (2, 127, 64, 96, BF, "silu"), (2, 129, 64, 264, HF, "sigmoid"), (1, 300, 64, 683, BF, "leaky_relu"),
    (2, 65, 128, 31, HF, "silu"), (2, 257, 128, 129, BF, "silu"), (1, 512, 128, 256, BF, ""),
    (3, 100, 128, 683, HF, "leaky_relu"), (1, 5, 128, 2048, BF, "silu"), (40, 4, 64, 160, BF, "silu"),
    (1, 33, 256, 64, BF, "silu"), (2, 160, 256, 200, HF, "sigmoid"), (1, 290, 256, 37, BF, "leaky_relu"),
    (1, 1000, 64, 64, BF, "silu"), (1, 2100, 128, 40, HF, "silu"), (9, 70, 32, 72, BF, "sigmoid"),
    (2, 1, 16, 3, FL, "silu"), (2, 70, 32, 45, FL, "leaky_relu"), (2, 129, 64, 132, FL, "silu"),
    (1, 260, 128, 96, FL, "sigmoid"), (2, 33, 128, 77, FL, ""), (1, 65, 256, 40, FL, "silu"),
    (1, 700, 64, 64, FL, "silu"),
]


@pytest.mark.parametrize("H,B,D,E,dt,act", CASES)
def test_forward_and_gradients(H, B, D, E, dt, act):
    print(f"[gated] H={H} B={B} D={D} E={E} {dt} act='{act}'", flush=True)
    t = make(H, B, D, E, dt, seed=B + E)
    check(both(*t, act), t, act)


LARGE_CASES = [
    # many heads of one to a few tiles: more workgroups than run at once, the larger row tiles of every D
    (200, 70, 32, 64, BF, "silu"), (1200, 40, 32, 100, HF, "sigmoid"), (300, 100, 64, 64, HF, "silu"),
    (800, 130, 64, 32, BF, "leaky_relu"), (300, 200, 128, 64, BF, "silu"), (260, 250, 128, 93, HF, ""),
    (520, 120, 128, 64, BF, "silu"), (600, 40, 256, 64, BF, "silu"), (300, 130, 256, 40, HF, "leaky_relu"),
    # few heads of many rows: the weight gradients' rows are split, down to one subtile of 32 rows in the last range
    (2, 9000, 32, 64, BF, "silu"), (1, 20000, 64, 72, HF, "silu"), (1, 9000, 128, 100, BF, "sigmoid"),
    (1, 6000, 256, 72, BF, "silu"), (1, 6049, 256, 33, HF, ""), (1, 700, 256, 130, BF, "silu"),
    (2, 9000, 32, 64, FL, "silu"), (1, 9000, 128, 100, FL, "silu"), (1, 6000, 256, 72, FL, "sigmoid"),
    (400, 40, 64, 36, FL, "silu"),
]


@pytest.mark.parametrize("H,B,D,E,dt,act", LARGE_CASES)
def test_many_workgroups(H, B, D, E, dt, act):
    print(f"[gated] H={H} B={B} D={D} E={E} {dt} act='{act}'", flush=True)
    t = make(H, B, D, E, dt, seed=B + E)
    check(both(*t, act), t, act)


@pytest.mark.parametrize("B", [1, 32, 33, 64, 65, 96, 97, 128, 129, 160, 224])
def test_weight_gradients_over_few_subtiles(B):
    """Every fill of the ring of row subtiles at D = 256, where two waves share a subtile's sums."""
    t = make(2, B, 256, 70, BF, seed=B)
    check(both(*t, "silu"), t, "silu")


@pytest.mark.parametrize("D", [16, 64, 128, 256])
def test_no_rows(D):
    t = make(2, 0, D, 40, BF)
    o, dx, *dw = both(*t, "silu")
    assert o.shape == (2, 0, D) and dx.shape == (2, 0, D)
    assert all(not g.any() for g in dw)


def test_partial_backward_is_the_full_one():
    for D, E in ((64, 96), (128, 264), (256, 64)):
        x, wg, wu, w2, do = make(2, 150, D, E, BF)
        full = flashmlp_gated_bwd(x, wg, wu, w2, do, "silu")
        dx, *none = flashmlp_gated_bwd(x, wg, wu, w2, do, "silu", _needs=(True, False))
        assert none == [None] * 3 and torch.equal(dx, full[0])
        none, *dw = flashmlp_gated_bwd(x, wg, wu, w2, do, "silu", _needs=(False, True))
        assert none is None and all(torch.equal(a, b) for a, b in zip(dw, full[1:]))


@pytest.mark.parametrize("dt", [BF, FL])
def test_views(dt):
    """x and do with any head distance (one matrix for every head too), rows, weights and gradients in
    other orders than the dense one, and bases that are not 16-byte aligned."""
    H, B, D, E = 3, 70, 64, 100
    x, wg, wu, w2, do = make(H, B, D, E, dt)
    want = both(x, wg, wu, w2, do, "silu")

    def heads(v):  # heads in reverse distance: a slice of a larger tensor
        big = torch.empty(H, 2, *v.shape[1:], dtype=v.dtype, device="cuda")
        big[:, 1] = v
        return big[:, 1]

    def token_major(v):
        return v.transpose(0, 1).contiguous().transpose(0, 1)

    def odd_base(v):
        return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)

    def transposed(v):
        return v.transpose(1, 2).contiguous().transpose(1, 2)

    for make_view in (heads, token_major, odd_base, transposed):
        got = both(*(make_view(v) for v in (x, wg, wu, w2, do)), "silu")
        for name, a, b in zip(NAMES, got, want):
            assert torch.equal(a, b), (make_view.__name__, name)
    xe = x[:1].expand(H, B, D)
    got, ref = both(xe, wg, wu, w2, do, "silu"), both(xe.contiguous(), wg, wu, w2, do, "silu")
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("dt,H,B,D,E", [(BF, 4, 50, 64, 96), (HF, 12, 33, 128, 100), (FL, 3, 40, 64, 45), (FL, 2, 9, 256, 20),
                                        (BF, 1, 1, 16, 8)])
@pytest.mark.parametrize("view", [False, True])
def test_module_and_shared_input(dt, H, B, D, E, view):
    """2-D input: through every head, mean over heads. Each output is a sum over heads of the heads' own results, whose
    operands are rounded as ever and which is rounded once itself: the bounds of the heads add up."""
    torch.manual_seed(1)
    m = GatedFlashMLP(H, D, E, dtype=dt)
    x = torch.randn(B, D, device="cuda").to(dt)
    gy = torch.randn(B, D, device="cuda").to(dt)
    if view:  # columns that are not dense: the general path
        x, gy = (torch.stack([v, v], -1).flatten(-2)[:, ::2] for v in (x, gy))
    x.requires_grad_(True)
    o = m(x)
    got = (o, *torch.autograd.grad(o, (x, m.wg, m.wu, m.w2), gy))
    t = (x.detach().expand(H, B, D), m.wg.detach(), m.wu.detach(), m.w2.detach(), gy.expand(H, B, D))
    want, bounds = gated64(*t, "silu")
    for name, a, w, (rounded, summed) in zip(NAMES, got, want, bounds):
        if name in ("o", "dx"):
            w, rounded, summed = (v.sum(0) for v in (w, rounded, summed))
        e = excess(a, w / H, (rounded / H, summed * 1.01 / H), dt)  # (1.01: the sum over heads in fp32)
        assert e <= 1.0, (name, e)


def test_gradients_against_differences():
    """fp32: the derivative along a direction v is (L(t + e v) - L(t - e v)) / 2e up to e^2 times the third
    derivative; e = 2^-7 leaves 6e-5 of it, and the loss' fp32 rounding (2^-24 |O| |dO| sqrt(n) / e) about 1e-4
    of a derivative of the size of |O| |dO|."""
    t = make(2, 40, 64, 72, FL, seed=5)
    do = t[4].double()
    g = torch.Generator().manual_seed(7)
    grads = flashmlp_gated_bwd(*t, "silu")
    for i in range(4):
        v = torch.randn(t[i].shape, generator=g).cuda() * t[i].std()
        e = 2.0 ** -7
        loss = []
        for s in (e, -e):
            u = list(t[:4])
            u[i] = u[i] + s * v
            loss.append((flashmlp_gated_fwd(*u, "silu").double() * do).sum())
        diff = ((loss[0] - loss[1]) / (2 * e)).item()
        along = (grads[i].double() * v.double()).sum().item()
        scale = (grads[i].double().norm() * v.double().norm()).item()
        assert abs(diff - along) <= 1e-3 * scale, (i, diff, along)


def test_repeatable_and_on_another_stream():
    t = make(3, 200, 128, 264, BF)
    ref = both(*t, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = both(*t, "silu")
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_graph_replays():
    t = make(2, 100, 64, 200, BF)
    both(*t, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*t, "silu")
    for i in range(4):
        t[0].copy_(make(2, 100, 64, 200, BF, seed=10 + i)[0])
        for o in out:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both(*t, "silu")))


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_a_row_of_infinities_stays_in_its_row(D):
    """A non-finite input row makes its own output row non-finite and no other, cut tiles included."""
    for B, E in ((33, 45), (70, 64)):
        x, wg, wu, w2, do = make(2, B, D, E, BF)
        ref = flashmlp_gated_fwd(x, wg, wu, w2, "silu")
        x[1, 5] = float("inf")
        o = flashmlp_gated_fwd(x, wg, wu, w2, "silu")
        keep = torch.ones(2, B, dtype=torch.bool, device="cuda")
        keep[1, 5] = False
        assert torch.equal(o[keep], ref[keep]) and not o[1, 5].isfinite().any()
        do[0, 3, 1] = float("nan")
        dx, *_ = flashmlp_gated_bwd(x, wg, wu, w2, do, "silu")
        keep[0, 3] = False
        assert dx[keep].isfinite().all() and dx[0, 3].isnan().all()


def test_autograd_skips_what_is_not_needed():
    x, wg, wu, w2, do = make(2, 40, 64, 64, BF)
    wu.requires_grad_(True)
    o = GatedFlashMLPFunction.apply(x, wg, wu, w2, "silu")
    (g,) = torch.autograd.grad(o, (wu,), do)
    assert torch.equal(g, flashmlp_gated_bwd(x, wg, wu.detach(), w2, do, "silu")[2])


def test_refusals():
    x, wg, wu, w2, do = make(2, 8, 64, 32, BF)
    with pytest.raises(AssertionError, match="Gate and up"):
        flashmlp_gated_fwd(x, wg, wu[:, :, :16], w2)
    with pytest.raises(AssertionError, match="Number of heads"):
        flashmlp_gated_fwd(x[:1], wg, wu, w2)
    with pytest.raises(AssertionError, match="Hidden dimension"):
        flashmlp_gated_fwd(x[:, :, :32], wg, wu, w2)
    with pytest.raises(AssertionError, match="Intermediate dimension"):
        flashmlp_gated_fwd(x, wg, wu, w2[:, :16])
    with pytest.raises(AssertionError, match="Gradient shape"):
        flashmlp_gated_bwd(x, wg, wu, w2, do[:, :4])
    with pytest.raises(TypeError):
        flashmlp_gated_fwd(x, wg, wu, w2.float())
    with pytest.raises(TypeError):
        flashmlp_gated_fwd(*(t.double() for t in (x, wg, wu, w2)))
    with pytest.raises(RuntimeError, match="cuda|GPU"):
        flashmlp_gated_fwd(*(t.cpu() for t in (x, wg, wu, w2)))
    y = torch.randn(2, 8, 48, dtype=BF, device="cuda")
    w = torch.randn(2, 48, 32, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="supported D"):
        flashmlp_gated_fwd(y, w, w, w.transpose(1, 2).contiguous())
