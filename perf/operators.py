"""The gated feed-forward block's operators, as cases that can be timed and checked.

Three operators of one training or serving step:

* ``gated``: the gated multi-head MLP  O = (act(X Wg) * (X Wu)) W2  per head (``flashmlp_gated_fwd``),
  and with its backward (``flashmlp_gated_bwd``, or the ``GatedFlashMLP`` module under autograd);
* ``join``: a block's output brought back to the residual stream and the next block's input taken from
  it in one pass,  R' = R + scale * gate * (RMSnorm(O) * w_post),  Y = RMSnorm(R') * w_pre
  (``block_join``), forward alone or with its gradients under autograd;
* ``clip``: the global norm of many gradients and their clipping into the optimizer's buffers
  (``clip_grads``).

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits.
Inputs: X ~ N(0, 1), Wg, Wu ~ N(0, 1/D), W2 ~ N(0, 1/E), dO ~ N(0, 1); a residual stream R ~ N(0, 1),
norm weights around 1, gates of size 0.5; gradients whose scale differs from tensor to tensor.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_EPS = 1e-6  # under the root of the norms
_CLIP_EPS = 1e-6  # beside the norm in the clipping coefficient


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _gated(kind, dtype, act, H, B, D, E, name=None):
    c = {"op": "gated", "kind": kind, "dtype": dtype, "act": act, "H": H, "B": B, "D": D, "E": E}
    if name is not None:
        c["name"] = name
    return c


def _join(kind, dtype, res, B, H, D, groups, name=None):
    # groups: rows of the gate, each for B / groups consecutive rows of the stream
    c = {"op": "join", "kind": kind, "dtype": dtype, "res": res, "B": B, "H": H, "D": D, "groups": groups}
    if name is not None:
        c["name"] = name
    return c


def _clip(dtype, out, layers, H, D, E, flat, max_norm, name=None):
    # layers x (two norm weights, a gate, Wg, Wu, W2); flat: the gradients too are views of one buffer, and both
    # buffers' views follow one another without padding
    c = {"op": "clip", "dtype": dtype, "out": out, "layers": layers, "H": H, "D": D, "E": E, "flat": flat,
         "max_norm": max_norm}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one new token of each of four requests through the block's matrices: all of the weights for a few rows
        _gated("fwd", "bf16", "silu", 32, 4, 128, 1024, name="gated_token"),
        # a prompt of some hundred tokens, piecewise linear gate
        _gated("fwd", "fp16", "leaky_relu", 12, 300, 64, 768, name="gated_prompt"),
        # a middle-sized training step through the module, one activation matrix shared by every head
        _gated("shared", "bf16", "silu", 16, 4096, 128, 512, name="gated_module"),
        # a large training step
        _gated("step", "bf16", "silu", 32, 16384, 128, 1024, name="gated_step_large"),
        # an intermediate size that is no multiple of anything (2/3 of 1024), ragged rows
        _gated("step", "fp16", "sigmoid", 16, 4095, 64, 683, name="gated_step_odd"),
        # wide heads
        _gated("step", "bf16", "silu", 8, 2048, 256, 1024, name="gated_step_wide"),
        # full precision training
        _gated("step", "fp32", "silu", 12, 1024, 64, 768, name="gated_step_fp32"),
        # the stream of a few requests between two blocks while they generate
        _join("fwd", "bf16", "bf16", 4, 32, 128, 1, name="join_token"),
        # the same between the blocks of a large training step
        _join("step", "bf16", "bf16", 16384, 32, 128, 1, name="join_step_large"),
        # a full precision stream beside 16-bit blocks, a gate for each of three sequences of odd length
        _join("step", "bf16", "fp32", 4101, 12, 64, 3, name="join_step_groups"),
        # clipping a small model's gradients, views of one flat buffer, into the optimizer's full precision buffer
        _clip("bf16", "fp32", 4, 12, 64, 683, True, 1.0, name="clip_small"),
        # clipping a large model's gradients, tensors of their own
        _clip("bf16", "fp32", 24, 32, 128, 1024, False, 1.0, name="clip_large"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# The most work a drawn case may have: the largest listed case's of its type, in u = H B D E.
_U_MAX = {"fp16": 32 * 16384 * 128 * 1024, "bf16": 32 * 16384 * 128 * 1024, "fp32": 12 * 1024 * 64 * 768}


def draw(rng):
    """One more case: sizes over the whole range of the listed ones, odd ones among them."""
    op = rng.choice(["gated", "gated", "gated", "join", "join", "clip"])
    if op == "gated":
        while True:
            kind = rng.choice(["fwd", "step", "step", "shared"])
            dtype = rng.choice(["fp16", "bf16", "bf16", "bf16", "fp32"])
            act = rng.choice(["silu", "silu", "leaky_relu", "sigmoid", ""])
            H = _log_int(rng, 1, 32)
            B = _log_int(rng, 1, 16384)
            D = rng.choice([16, 32, 64, 64, 128, 128, 256])
            E = _log_int(rng, 64, 2048)
            if rng.random() < 0.6:
                E = max(64, E // 64 * 64)
            if B > 64 and rng.random() < 0.5:
                B = B // 64 * 64
            if 1 << 16 <= H * B * D * E <= _U_MAX[dtype] * (1 if D >= 64 else 0.25):
                return _gated(kind, dtype, act, H, B, D, E)
    if op == "join":
        while True:
            kind = rng.choice(["fwd", "step", "step"])
            dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
            res = rng.choice([dtype, dtype, "fp32"])
            B = _log_int(rng, 1, 16384)
            H = _log_int(rng, 1, 32)
            D = rng.choice([16, 32, 64, 64, 100, 128, 128, 201, 256])
            groups = rng.choice([1, 1, 2, 3, B])
            if H * D <= 8192 and B * H * D <= 16384 * 4096 and B % groups == 0:
                return _join(kind, dtype, res, B, H, D, groups)
    while True:
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        out = rng.choice(["fp32", dtype])
        layers = _log_int(rng, 1, 40)
        H, D, E = _log_int(rng, 1, 32), rng.choice([16, 32, 64, 128, 256]), _log_int(rng, 64, 2048)
        if layers * H * D * E <= 24 * 32 * 128 * 1024:
            return _clip(dtype, out, layers, H, D, E, rng.random() < 0.5, rng.choice([0.1, 1.0, 10.0, 1e6]))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
class _Normal:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def __call__(self, shape, std, dtype, mean=0.0):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return t.mul_(std).add_(mean).to(dtype)


def _gated_inputs(case, seed):
    """x, wg, wu, w2 and the gradient of the output."""
    H, B, D, E = case["H"], case["B"], case["D"], case["E"]
    dt, normal = _DTYPES[case["dtype"]], _Normal(seed)
    rows = (B, D) if case["kind"] == "shared" else (H, B, D)
    x = normal(rows, 1.0, dt)
    wg = normal((H, D, E), 1.0 / math.sqrt(D), dt)
    wu = normal((H, D, E), 1.0 / math.sqrt(D), dt)
    w2 = normal((H, E, D), 1.0 / math.sqrt(E), dt)
    dout = normal(rows, 1.0, dt) if case["kind"] != "fwd" else None
    return x, wg, wu, w2, dout


def _join_inputs(case, seed):
    """the stream, the block's output, w_post, gate, w_pre and the gradients of both outputs."""
    B, H, D, C = case["B"], case["H"], case["D"], case["H"] * case["D"]
    dt, rdt, normal = _DTYPES[case["dtype"]], _DTYPES[case["res"]], _Normal(seed)
    r = normal((B, C), 1.0, rdt)
    o = normal((H, B, D), 0.7, dt)
    w_post = normal((C,), 0.1, dt, 1.0)
    gate = normal((case["groups"], C), 0.3, dt, 0.5)
    w_pre = normal((C,), 0.1, dt, 1.0)
    if case["kind"] == "fwd":
        return r, o, w_post, gate, w_pre, None, None
    return r, o, w_post, gate, w_pre, normal((B, C), 1.0, rdt), normal((H, B, D), 1.0, dt)


def _clip_shapes(case):
    H, D, E = case["H"], case["D"], case["E"]
    layer = [(H * D,), (H * D,), (H * D,), (H, D, E), (H, D, E), (H, E, D)]
    return layer * case["layers"]


def _views(buffer, shapes, align):
    """one view of the buffer for each shape, its start a multiple of `align` elements"""
    views, at = [], 0
    for s in shapes:
        n = math.prod(s)
        views.append(buffer[at:at + n].view(s))
        at += -(-n // align) * align
    return views


def _clip_inputs(case, seed):
    """the gradients, and the optimizer's buffer with the views they are clipped into."""
    dt, odt, normal = _DTYPES[case["dtype"]], _DTYPES[case["out"]], _Normal(seed)
    shapes = _clip_shapes(case)
    align = 1 if case["flat"] else 128
    total = sum(-(-math.prod(s) // align) * align for s in shapes)
    buffer = torch.zeros(total, dtype=odt, device="cuda")
    grads = [normal(s, 10.0 ** (-(i % 5) / 2.0 - 2.0), dt) for i, s in enumerate(shapes)]
    if case["flat"]:
        flat = _views(torch.empty(total, dtype=dt, device="cuda"), shapes, 1)
        grads = [v.copy_(g) for v, g in zip(flat, grads)]
    return grads, buffer, _views(buffer, shapes, align)


_SCALE = 0.5  # the residual branch's scale in every join case


def prepare(case, seed):
    op, kind = case["op"], case.get("kind")
    state = {"op": op, "kind": kind}
    if op == "gated":
        x, wg, wu, w2, dout = _gated_inputs(case, seed)
        state.update(act=case["act"], x=x, wg=wg, wu=wu, w2=w2, dout=dout)
        if kind == "shared" and own:
            from flashmlp_amd import GatedFlashMLP

            m = GatedFlashMLP(case["H"], case["D"], case["E"], activation=case["act"], dtype=_DTYPES[case["dtype"]],
                              device="cuda")
            with torch.no_grad():
                for p, w in ((m.wg, wg), (m.wu, wu), (m.w2, w2)):
                    p.copy_(w)
            state.update(module=m, x=x.requires_grad_(True))
    elif op == "join":
        names = ("r", "o", "w_post", "gate", "w_pre", "dr", "dy")
        state.update(zip(names, _join_inputs(case, seed)))
        if kind == "step" and own:
            for n in names[:5]:
                state[n].requires_grad_(True)
    else:
        state["grads"], state["buffer"], state["outs"] = _clip_inputs(case, seed)
        state["max_norm"] = case["max_norm"]
    return state


# ---------------------------------------------------------------------------------------------
# the operators' plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------
def _act_plain(name, z, grad):
    """act(z), and act'(z) where the gradient is wanted."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s)) if grad else None
    if name == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s, s * (1.0 - s) if grad else None
    if name == "leaky_relu":
        p = z > 0
        return torch.where(p, z, 0.01 * z), torch.where(p, 1.0, 0.01) if grad else None
    return z, torch.ones_like(z) if grad else None


def _gated_plain(st):
    dt = st["x"].dtype
    shared, step = st["kind"] == "shared", st["dout"] is not None
    x, wg, wu, w2 = (st[k].float() for k in ("x", "wg", "wu", "w2"))
    H = wg.shape[0]
    if shared:
        x = x.expand(H, *x.shape)
    a, da = _act_plain(st["act"], x @ wg, step)
    u = x @ wu
    h = a * u
    o = h @ w2
    if shared:
        o = o.mean(0)
    if not step:
        return (o.to(dt),)
    g = st["dout"].float()
    if shared:
        g = (g / H).expand(H, *g.shape)
    dh = g @ w2.transpose(1, 2)
    dg, du = dh * u * da, dh * a
    dx = dg @ wg.transpose(1, 2) + du @ wu.transpose(1, 2)
    if shared:
        dx = dx.sum(0)
    xt = x.transpose(1, 2)
    dw2 = h.transpose(1, 2) @ g
    return tuple(t.to(dt) for t in (o, dx, xt @ dg, xt @ du, dw2))


def _heads_to_rows(t):
    return t.transpose(0, 1).reshape(t.shape[1], -1)


def _rows_to_heads(t, H):
    return t.reshape(t.shape[0], H, -1).transpose(0, 1).contiguous()


def _join_plain(st):
    H, B, D = st["o"].shape
    rdt, dt = st["r"].dtype, st["o"].dtype
    r, w_post, w_pre = st["r"].float(), st["w_post"].float(), st["w_pre"].float()
    gate = st["gate"].float()
    G = gate.shape[0]
    rows = gate.repeat_interleave(B // G, 0) if G > 1 else gate
    o = _heads_to_rows(st["o"].float())
    rs_o = 1.0 / torch.sqrt((o * o).mean(1, keepdim=True) + _EPS)
    n = o * rs_o
    p = n * w_post
    r2 = r + _SCALE * rows * p
    rs_r = 1.0 / torch.sqrt((r2 * r2).mean(1, keepdim=True) + _EPS)
    m = r2 * rs_r
    y = _rows_to_heads(m * w_pre, H)
    if st["kind"] == "fwd":
        return r2.to(rdt), y.to(dt)
    dy = _heads_to_rows(st["dy"].float())
    dm = dy * w_pre
    dr = st["dr"].float() + rs_r * (dm - m * (dm * m).mean(1, keepdim=True))
    dgate = (_SCALE * dr * p).reshape(G, B // G, -1).sum(1)
    dp = _SCALE * rows * dr
    dn = dp * w_post
    do = rs_o * (dn - n * (dn * n).mean(1, keepdim=True))
    return (r2.to(rdt), y.to(dt), dr.to(rdt), _rows_to_heads(do, H).to(dt), (dp * n).sum(0).to(dt), dgate.to(dt),
            (dy * m).sum(0).to(dt))


def _clip_plain(st):
    sq = [(g.float() * g.float()).sum() for g in st["grads"]]
    norm = torch.sqrt(torch.stack(sq).sum())
    coef = torch.clamp(st["max_norm"] / (norm + _CLIP_EPS), max=1.0)
    for g, b in zip(st["grads"], st["outs"]):
        b.copy_(g.float() * coef)
    return norm, st["buffer"]


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if not own:
        return {"gated": _gated_plain, "join": _join_plain, "clip": _clip_plain}[op](state)
    import flashmlp_amd as fm

    if op == "gated":
        x, dout, act = state["x"], state["dout"], state["act"]
        if state["kind"] == "shared":
            m = state["module"]
            o = m(x)
            return (o.detach(), *torch.autograd.grad(o, (x, m.wg, m.wu, m.w2), dout))
        w = state["wg"], state["wu"], state["w2"]
        o = fm.flashmlp_gated_fwd(x, *w, act)
        return (o,) if dout is None else (o, *fm.flashmlp_gated_bwd(x, *w, dout, act))
    if op == "join":
        r, o, w_post, gate, w_pre = (state[k] for k in ("r", "o", "w_post", "gate", "w_pre"))
        r2, y = fm.block_join(r, o, w_post, gate, _SCALE, pre_weight=w_pre, eps=_EPS)
        if state["kind"] == "fwd":
            return r2, y
        g = torch.autograd.grad((r2, y), (r, o, w_post, gate, w_pre), (state["dr"], state["dy"]))
        return (r2.detach(), y.detach(), *g)
    _, norm = fm.clip_grads(state["grads"], state["max_norm"], out=state["outs"])
    return norm, state["buffer"]


def work(case):
    """What a pass cannot do without. The gated forward has three products of 2u FLOPs, u = H B D E; its
    backward, which is given no projections, computes both again, dO W2^T, two products into dX and three
    weight gradients (16u). The other two operators move data: each input and output once."""
    if case["op"] == "gated":
        H, B, D, E = case["H"], case["B"], case["D"], case["E"]
        s, u = _BYTES[case["dtype"]], H * B * D * E
        rows = (1 if case["kind"] == "shared" else H) * B * D * s
        weights = 3 * H * D * E * s
        if case["kind"] == "fwd":
            return {"bytes": 2 * rows + weights, "flops": 6 * u}
        return {"bytes": 5 * rows + 3 * weights, "flops": 22 * u}
    if case["op"] == "join":
        n, s, sr = case["B"] * case["H"] * case["D"], _BYTES[case["dtype"]], _BYTES[case["res"]]
        vectors = (2 + case["groups"]) * case["H"] * case["D"] * s
        if case["kind"] == "fwd":  # r, o -> r', y
            return {"bytes": 2 * n * (s + sr) + vectors, "flops": 12 * n}
        # and r', o, dr', dy -> dr, do and the vectors' gradients
        return {"bytes": 2 * n * (s + sr) + vectors + n * (3 * sr + 3 * s) + 2 * vectors, "flops": 45 * n}
    n = sum(math.prod(s) for s in _clip_shapes(case))
    return {"bytes": n * (_BYTES[case["dtype"]] + _BYTES[case["out"]]), "flops": 3 * n}


# ---------------------------------------------------------------------------------------------
# the same outputs in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_gated(case, seed):
    x, wg, wu, w2, dout = _gated_inputs(case, seed)
    H, shared, act = case["H"], case["kind"] == "shared", case["act"]
    cols = [[] for _ in range(5)]
    for h in range(H):
        xh = (x if shared else x[h]).double()
        a, b, c = wg[h].double(), wu[h].double(), w2[h].double()
        z, up = xh.matmul(a), xh.matmul(b)
        sig = torch.sigmoid(z)
        if act == "silu":
            f, df = z * sig, sig + z * sig * (1 - sig)
        elif act == "sigmoid":
            f, df = sig, sig * (1 - sig)
        elif act == "leaky_relu":
            f, df = torch.nn.functional.leaky_relu(z, 0.01), torch.where(z > 0, 1.0, 0.01).double()
        else:
            f, df = z, torch.ones_like(z)
        if act == "leaky_relu":
            # the literal 0.01 in 64 bits on both sides
            f = torch.where(z > 0, z, z * 0.01)
        cols[0].append((f * up).matmul(c))
        if dout is None:
            continue
        g = dout.double() / H if shared else dout[h].double()
        dh = g.matmul(c.t().contiguous())
        dz, dup = dh * up * df, dh * f
        xt = xh.t().contiguous()
        cols[1].append(dz.matmul(a.t().contiguous()) + dup.matmul(b.t().contiguous()))
        cols[2].append(xt.matmul(dz))
        cols[3].append(xt.matmul(dup))
        cols[4].append((f * up).t().contiguous().matmul(g))
    out = [torch.stack(c) for c in cols if c]
    if shared:
        out[0], out[1] = out[0].mean(0), out[1].sum(0)
    return tuple(out)


def _exact_join(case, seed):
    # gradients by autograd over the definition in 64 bits
    t = _join_inputs(case, seed)
    r, o, w_post, gate, w_pre = (v.double().requires_grad_(True) for v in t[:5])
    H, B, D = o.shape

    def norm(v):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + _EPS)

    flat = o.permute(1, 0, 2).reshape(B, H * D)
    branch = (norm(flat) * w_post).view(case["groups"], -1, H * D) * gate[:, None, :]
    r2 = r + _SCALE * branch.reshape(B, H * D)
    y = (norm(r2) * w_pre).view(B, H, D).permute(1, 0, 2)
    if case["kind"] == "fwd":
        return r2.detach(), y.detach()
    g = torch.autograd.grad((r2, y), (r, o, w_post, gate, w_pre), (t[5].double(), t[6].double()))
    return (r2.detach(), y.detach(), *g)


def _exact_clip(case, seed):
    grads, buffer, _ = _clip_inputs(case, seed)
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in grads))
    coef = min(1.0, case["max_norm"] / (norm + _CLIP_EPS))
    clipped = torch.zeros_like(buffer, dtype=torch.float64)
    for v, g in zip(_views(clipped, [g.shape for g in grads], 1 if case["flat"] else 128), grads):
        v.copy_(g.double() * coef)
    return torch.tensor(norm, dtype=torch.float64, device="cuda"), clipped


def exact(case, seed):
    return {"gated": _exact_gated, "join": _exact_join, "clip": _exact_clip}[case["op"]](case, seed)
