"""block_join and block_norm against their definition in 64 bits, elementwise within the bounds of
oracle/join.py: every io type and stream type, row widths from one column to the largest, gates shared, per
group and per row, the parts that can be left out, views, streams and refusals."""
import pytest
import torch

from flashmlp_amd import block_join, block_join_bwd, block_join_fwd, block_norm
from oracle.join import excess, join64

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def rows(t, H):
    """(H, B, D) as (B, C)"""
    return t.transpose(0, 1).reshape(t.shape[1], -1)


def make(B, H, D, groups, dt, rdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    C = H * D
    return dict(r=n(B, C).to(rdt).cuda(), o=(0.7 * n(H, B, D)).to(dt).cuda(), w_post=(1 + 0.1 * n(C)).to(dt).cuda(),
                gate=(0.5 + 0.3 * n(groups, C)).to(dt).cuda(), w_pre=(1 + 0.1 * n(C)).to(dt).cuda(),
                dr2=n(B, C).to(rdt).cuda(), dy=n(H, B, D).to(dt).cuda())


def check(t, post=True, scale=0.5, grads=True):
    """run forward and backward under autograd on the entries of t that are there, and compare"""
    r, o, w_post, gate, w_pre = (t.get(k) for k in ("r", "o", "w_post", "gate", "w_pre"))
    H, B, D = o.shape
    ins = [v.detach().clone().requires_grad_(True) if v is not None else None for v in (r, o, w_post, gate, w_pre)]
    with_y, with_r2 = t.get("dy") is not None, t.get("dr2") is not None
    r2, y = block_join(*ins[:4], scale, pre_weight=ins[4], post=post, pre=with_y or ins[4] is not None, eps=EPS)
    outs = [(v, t[k]) for v, k, there in ((r2, "dr2", with_r2), (y, "dy", with_y)) if there]
    have = [v for v in ins if v is not None]
    g = iter(torch.autograd.grad([a for a, _ in outs], have, [b for _, b in outs], allow_unused=True))
    g = [next(g) if v is not None else None for v in ins]
    if gate is not None and gate.dim() == 1:
        gate = gate[None]
    want, bound = join64(r, rows(o, H), w_post, gate, w_pre, scale, EPS, post, t.get("dr2"),
                         rows(t["dy"], H) if with_y else None)
    got = dict(r2=r2, dr=g[0], do=rows(g[1], H))
    if y is not None:
        assert y.shape == (H, B, D) and y.is_contiguous()
        got["y"] = rows(y, H)
    for k, v in (("dw_post", g[2]), ("dgate", g[3]), ("dw_pre", g[4])):
        if v is not None:
            got[k] = v
    for k, v in got.items():
        assert v.dtype == (r.dtype if k in ("r2", "dr") else o.dtype), k
        if k == "dw_pre" and not with_y:
            assert not v.any()
            continue
        e = excess(v, want[k], bound[k], v.dtype)
        assert e <= 1.0, (k, e)


CASES = [
    # B, H, D, groups, dtype, stream's dtype
    (1, 1, 1, 1, BF, BF), (2, 1, 7, 2, HF, FL), (3, 2, 8, 1, FL, FL), (5, 3, 16, 5, BF, FL), (33, 4, 100, 1, BF, BF),
    (64, 8, 64, 1, BF, BF), (65, 9, 64, 1, HF, HF), (63, 8, 128, 3, BF, FL), (7, 1, 1025, 7, FL, FL),
    (130, 12, 64, 2, BF, FL), (300, 16, 64, 300, HF, HF), (40, 32, 128, 4, BF, BF), (17, 32, 256, 1, BF, FL),
    (9, 64, 128, 1, FL, FL), (4, 64, 256, 2, BF, BF), (3, 5, 3001, 1, HF, FL), (2000, 2, 32, 1, BF, BF),
    (2100, 1, 64, 3, FL, FL), (1500, 5, 201, 5, BF, BF), (4099, 1, 256, 1, HF, HF),
]


@pytest.mark.parametrize("B,H,D,groups,dt,rdt", CASES)
def test_forward_and_gradients(B, H, D, groups, dt, rdt):
    print(f"[join] B={B} H={H} D={D} groups={groups} {dt} {rdt}", flush=True)
    check(make(B, H, D, groups, dt, rdt, seed=B + D))


@pytest.mark.parametrize("drop", [("w_post",), ("gate",), ("w_pre",), ("w_post", "gate", "w_pre"), ("dy",), ("dr2",),
                                  ("dy", "w_pre"), ("gate", "dr2")])
@pytest.mark.parametrize("D", [64, 50])
def test_parts_left_out(drop, D):
    t = make(60, 4, D, 2, BF, BF)
    check({k: v for k, v in t.items() if k not in drop})


def test_without_the_post_norm():
    t = make(50, 4, 64, 1, BF, FL)
    del t["w_post"]
    check(t, post=False, scale=-2.0)
    t["gate"] = t["gate"][0]  # one row, as a vector
    check(t, post=False)


@pytest.mark.parametrize("heads,dt,rdt", [(None, BF, BF), (4, BF, FL), (4, FL, FL), (8, HF, HF)])
def test_norm_alone(heads, dt, rdt):
    t = make(70, heads or 1, 512 // (heads or 1), 1, dt, rdt)
    x, w = t["r"].clone().requires_grad_(True), t["w_pre"].clone().requires_grad_(True)
    y = block_norm(x, w, heads=heads, eps=EPS)
    dy = t["dy"] if heads else t["dy"][0]
    assert y.shape == dy.shape and y.dtype == dt
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    dyr = rows(dy, heads) if heads else dy
    want, bound = join64(t["r"], None, None, None, t["w_pre"], 1.0, EPS, True, None, dyr)
    for k, v in (("y", rows(y, heads) if heads else y), ("dr", dx), ("dw_pre", dw)):
        assert excess(v, want[k], bound[k], v.dtype) <= 1.0, k
    plain = block_norm(t["r"], heads=heads, dtype=dt)
    want, bound = join64(t["r"], None, None, None, None, 1.0, EPS, True, None, dyr)
    assert excess(rows(plain, heads) if heads else plain, want["y"], bound["y"], dt) <= 1.0


def test_rows_of_zeros_and_of_extremes():
    """A row of zeros has 1 / rms = 1 / sqrt(eps), rows near the type's largest values stay finite through the
    norm in 32 bits, a non-finite row stays in its row."""
    t = make(8, 2, 64, 1, BF, BF)
    t["o"][:, 1], t["r"][1] = 0, 0
    t["o"][:, 2] = 1e15
    check(t)
    o = t["o"].clone()
    ref = block_join(t["r"], o, t["w_post"], t["gate"], pre_weight=t["w_pre"])
    o[0, 4, 3], o[1, 5, 0] = float("inf"), float("nan")
    got = block_join(t["r"], o, t["w_post"], t["gate"], pre_weight=t["w_pre"])
    keep = [0, 1, 2, 3, 6, 7]
    assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[1][:, keep], ref[1][:, keep])
    assert not got[1][:, [4, 5]].isfinite().all(2).any()


@pytest.mark.parametrize("groups", [1, 3])
def test_no_rows(groups):
    t = make(0, 2, 64, groups, BF, BF)
    t = {k: v.requires_grad_(True) if k in ("r", "o", "w_post", "gate", "w_pre") else v for k, v in t.items()}
    r2, y = block_join(t["r"], t["o"], t["w_post"], t["gate"], pre_weight=t["w_pre"])
    assert r2.shape == (0, 128) and y.shape == (2, 0, 64)
    g = torch.autograd.grad((r2, y), [t[k] for k in ("r", "o", "w_post", "gate", "w_pre")], (t["dr2"], t["dy"]))
    assert all(not v.any() for v in g) and g[3].shape == (groups, 128)


@pytest.mark.parametrize("D", [64, 50])
@pytest.mark.parametrize("dt", [BF, FL])
def test_views(D, dt):
    """the same bits from streams and blocks in other orders, with padded rows and odd bases"""
    B, H = 40, 4
    t = make(B, H, D, 2, dt, dt)

    def step(t):
        ins = [t[k].detach().requires_grad_(True) for k in ("r", "o", "w_post", "gate", "w_pre")]
        r2, y = block_join(*ins[:4], 0.5, pre_weight=ins[4])
        return (r2, y, *torch.autograd.grad((r2, y), ins, (t["dr2"], t["dy"])))

    def padded(v):
        big = torch.full((*v.shape[:-1], v.shape[-1] + 8), 9.0, dtype=v.dtype, device="cuda")
        big[..., :-8] = v
        return big[..., :-8]

    def odd_base(v):
        return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)

    def token_major(v):
        return v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() == 3 else v

    def column_major(v):
        return v.transpose(-1, -2).contiguous().transpose(-1, -2) if v.dim() > 1 else v

    def spread(v):  # column stride 2
        return torch.stack([v, v + 1], -1).flatten(-2)[..., ::2]

    # the element-wise kernels sum a row in another order than the vector ones
    want = step(t)
    for view in (padded, odd_base, token_major, column_major, spread):
        got = step({k: view(v) for k, v in t.items()})
        for a, b in zip(got, want):
            assert a.shape == b.shape
            if view in (token_major, column_major, spread):
                assert torch.equal(a, b), view.__name__
            else:
                tol = 2 ** -7 if dt == BF else 2e-5
                assert torch.allclose(a.double(), b.double(), rtol=tol, atol=tol), view.__name__
    # one gradient for every row
    e = dict(t, dr2=t["dr2"][:1].expand(B, -1), dy=t["dy"][:, :1].expand(-1, B, -1))
    for a, b in zip(step(e), step(dict(e, dr2=e["dr2"].contiguous(), dy=e["dy"].contiguous()))):
        assert torch.equal(a, b)


def test_rows_layout_is_the_head_layout_of_one_head():
    t = make(30, 1, 96, 1, BF, BF)
    a = block_join(t["r"], t["o"], t["w_post"], t["gate"], pre_weight=t["w_pre"])
    b = block_join(t["r"], t["o"][0], t["w_post"], t["gate"], pre_weight=t["w_pre"])
    assert b[1].shape == (30, 96) and torch.equal(a[0], b[0]) and torch.equal(a[1][0], b[1])


def test_gradients_against_differences():
    """fp32, along a direction: see the gated MLP's test; here the results are of the size of one."""
    t = make(24, 2, 40, 3, FL, FL, seed=4)
    names = ("r", "o", "w_post", "gate", "w_pre")
    ins = [t[k].detach().requires_grad_(True) for k in names]
    r2, y = block_join(*ins[:4], 0.5, pre_weight=ins[4])
    grads = torch.autograd.grad((r2, y), ins, (t["dr2"], t["dy"]))
    gen = torch.Generator().manual_seed(9)
    for i, k in enumerate(names):
        v = torch.randn(t[k].shape, generator=gen).cuda()
        e, loss = 2.0 ** -7, []
        for s in (e, -e):
            u = [x.detach() for x in ins]
            u[i] = u[i] + s * v
            a, b = block_join(*u[:4], 0.5, pre_weight=u[4])
            loss.append((a.double() * t["dr2"].double()).sum() + (b.double() * t["dy"].double()).sum())
        diff = ((loss[0] - loss[1]) / (2 * e)).item()
        along = (grads[i].double() * v.double()).sum().item()
        scale = (grads[i].double().norm() * v.double().norm()).item()
        assert abs(diff - along) <= 1e-3 * scale, (k, diff, along)


def test_repeatable_on_streams_and_in_graphs():
    t = make(500, 8, 64, 1, BF, BF)
    args = [t[k] for k in ("r", "o", "w_post", "gate")]

    def step():
        r2, y, rs_o, rs_r = block_join_fwd(*args, 0.5, pre_weight=t["w_pre"], _save=True)
        return (r2, y, *block_join_bwd(r2, t["o"], rs_o, rs_r, t["dr2"], t["dy"], t["w_post"], t["gate"], 0.5,
                                       pre_weight=t["w_pre"]))

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        t["o"].copy_(make(500, 8, 64, 1, BF, BF, seed=20 + i)["o"])
        for v in out:
            v.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_only_the_wanted_gradients():
    t = make(40, 4, 64, 2, BF, BF)
    args = [t[k] for k in ("r", "o", "w_post", "gate")]
    r2, y, rs_o, rs_r = block_join_fwd(*args, 0.5, pre_weight=t["w_pre"], _save=True)

    def bwd(needs):
        return block_join_bwd(r2, t["o"], rs_o, rs_r, t["dr2"], t["dy"], t["w_post"], t["gate"], 0.5,
                              pre_weight=t["w_pre"], _needs=needs)

    full = bwd((True,) * 5)
    for i in range(5):
        g = bwd([j == i for j in range(5)])
        assert all((v is None) == (j != i) for j, v in enumerate(g)) and torch.equal(g[i], full[i])


def test_refusals():
    t = make(12, 4, 64, 1, BF, BF)
    r, o, w, gate = t["r"], t["o"], t["w_post"], t["gate"]
    for bad, match in (((r, o[:2], w), "Columns"), ((r[:5], o, w), "rows"), ((r, o, w[:9]), "Post norm"),
                       ((r, o, w, torch.ones(5, 256, dtype=BF, device="cuda")), "divide"),
                       ((r, o, w, gate[:, :8]), "gate")):
        with pytest.raises(AssertionError, match=match):
            block_join(*bad)
    with pytest.raises(AssertionError, match="post norm"):
        block_join(r, o, w, post=False)
    with pytest.raises(AssertionError, match="pre norm"):
        block_join(r, o, w, pre_weight=w, pre=False)
    with pytest.raises(AssertionError, match="heads"):
        block_norm(r, heads=3)
    with pytest.raises(TypeError):
        block_join(r.half(), o, w)
    with pytest.raises(TypeError):
        block_join(r, o, w.float())
    with pytest.raises(TypeError):
        block_norm(r, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        block_norm(r.cpu())
    with pytest.raises(RuntimeError, match="at most"):
        block_norm(torch.zeros(1, 16392, dtype=BF, device="cuda"))
    with pytest.raises(RuntimeError, match="eps"):
        block_norm(r, eps=-1.0)


@pytest.mark.parametrize("B,H,D,groups,dt", [(1, 3, 64, 1, BF), (95, 2, 128, 95, BF), (300, 3, 50, 2, HF), (64, 12, 128, 1, HF),
                                             (40, 32, 128, 4, BF), (70, 64, 130, 1, BF), (12, 64, 200, 1, HF)])
@pytest.mark.parametrize("drop", [(), ("w_post", "gate"), ("w_pre",), ("dr2",)])
def test_gradients_of_a_16_bit_stream_lose_nothing_to_its_rounding(B, H, D, groups, dt, drop):
    """made from r again, the backward's stream is the unrounded one: bounds without its rounding"""
    t = {k: v for k, v in make(B, H, D, groups, dt, dt, seed=B).items() if k not in drop}
    names = [k for k in ("r", "o", "w_post", "gate", "w_pre") if k in t]
    ins = {k: t[k].detach().requires_grad_(True) for k in names}
    r2, y = block_join(ins["r"], ins["o"], ins.get("w_post"), ins.get("gate"), 0.5, pre_weight=ins.get("w_pre"), eps=EPS)
    outs, dout = ((r2, y), (t["dr2"], t["dy"])) if "dr2" in t else ((y,), (t["dy"],))
    auto = dict(zip(names, torch.autograd.grad(outs, list(ins.values()), dout)))
    a = (t["o"], t.get("w_post"), t.get("gate"), 0.5)
    r2, y, rs_o, rs_r = block_join_fwd(t["r"], *a, pre_weight=t.get("w_pre"), eps=EPS, _save=True)
    direct = block_join_bwd(None, t["o"], rs_o, rs_r, t.get("dr2"), t["dy"], *a[1:], pre_weight=t.get("w_pre"), eps=EPS,
                            residual=t["r"])
    want, bound = join64(t["r"], rows(t["o"], H), *a[1:3], t.get("w_pre"), 0.5, EPS, True, t.get("dr2"),
                         rows(t["dy"], H), stream_rounded=False)
    for (k, name), d in zip((("r", "dr"), ("o", "do"), ("w_post", "dw_post"), ("gate", "dgate"), ("w_pre", "dw_pre")), direct):
        if k not in t:
            assert d is None
            continue
        assert torch.equal(d, auto[k]), name
        v = rows(d, H) if k == "o" else d
        assert excess(v, want[name], bound[name], dt) <= 1.0, name
