"""The operators around a mixture of gated experts and its training, as cases that can be timed and checked.

* ``route``: each token's experts from its logits, the k largest of a softmax and their weights
  (``expert_route``), forward alone or with the logits' gradient;
* ``dispatch``: tokens sorted by expert (``expert_plan``) and copied to the experts' rows, the (H, B, D) layout
  of the multi-head MLPs (``expert_dispatch``), forward alone or with the tokens' gradient;
* ``combine``: the experts' rows back at their tokens, summed with the tokens' weights (``expert_combine``),
  forward alone or with the gradients of rows and weights;
* ``ortho``: stacks of matrices orthogonalised by Newton-Schulz products (``orthogonalize``);
* ``muon``: the same as an optimizer's step: momentum, orthogonalised update, weights (``muon_step``).

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits.
Inputs: logits ~ N(0, 1) with a popularity of size 0.5 for each expert, so that loads differ and a capacity drops
some tokens; tokens, rows and gradients ~ N(0, 1); weights ~ N(0, 1 / rows of the matrix), their gradients and
momenta a product of rank 8 under noise, as gradients of a layer are.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_STEPS, _EPS = 5, 1e-7
# lr of a large run whose updates have an element's rms of 0.2 at 4e-4: 0.2 sqrt(1024) 4e-4
_LR, _MOMENTUM, _DECAY = 2.5e-3, 0.95, 0.1


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _case(op, name, **c):
    c = {"op": op, **c}
    if name is not None:
        c["name"] = name
    return c


def _route(kind, dtype, T, N, k, normalize, name=None):
    return _case("route", name, kind=kind, dtype=dtype, T=T, N=N, k=k, normalize=normalize)


def _tokens(op, kind, dtype, T, D, N, k, capacity, name=None):
    # capacity: rows of an expert; 0: as many as there are tokens, none is dropped
    return _case(op, name, kind=kind, dtype=dtype, T=T, D=D, N=N, k=k, capacity=capacity)


def _ortho(dtype, H, R, C, name=None):
    return _case("ortho", name, dtype=dtype, H=H, R=R, C=C)


def _muon(dtype, grad, moment, layers, H, D, E, nesterov, name=None):
    # layers of a gated MLP's three stacks: weights of `dtype`, their gradients, their momenta
    return _case("muon", name, dtype=dtype, grad=grad, moment=moment, layers=layers, H=H, D=D, E=E, nesterov=nesterov)


def _capacity(T, N, k, factor):
    return max(1, math.ceil(T * k / N * factor))


def listed():
    big = 32 * 16384  # a large training step's rows of 32 heads
    return [
        # a few requests of 32 heads each choosing while they generate
        _route("fwd", "bf16", 4 * 32, 16, 2, True, name="route_token"),
        # a training step's choice among many experts, as many as a token takes
        _route("step", "bf16", 4 * 16384, 64, 8, True, name="route_step"),
        # the tokens of a few requests to their experts, none dropped
        _tokens("dispatch", "fwd", "bf16", 4 * 32, 128, 32, 2, 0, name="dispatch_token"),
        # a large training step
        _tokens("dispatch", "step", "bf16", big, 128, 32, 2, _capacity(big, 32, 2, 1.25), name="dispatch_step"),
        # ragged tokens of narrow heads, no spare rows: the popular experts drop many
        _tokens("dispatch", "step", "fp16", 16 * 4095, 64, 12, 3, _capacity(16 * 4095, 12, 3, 1.0), name="dispatch_odd"),
        # back again, for a few requests
        _tokens("combine", "fwd", "bf16", 4 * 32, 128, 32, 2, 0, name="combine_token"),
        # the large training step
        _tokens("combine", "step", "bf16", big, 128, 32, 2, _capacity(big, 32, 2, 1.25), name="combine_step"),
        # full precision training, one expert a token, ample rows
        _tokens("combine", "step", "fp32", 12 * 1024, 64, 8, 1, _capacity(12 * 1024, 8, 1, 2.0), name="combine_fp32"),
        # one stack, an intermediate size that is no multiple of anything
        _ortho("bf16", 16, 64, 683, name="ortho_odd"),
        # wide heads in full precision
        _ortho("fp32", 8, 256, 1024, name="ortho_wide"),
        # a small model's layer: 16-bit gradients, full precision momenta and weights
        _muon("fp32", "bf16", "fp32", 1, 12, 64, 768, True, name="muon_small"),
        # a large model
        _muon("fp32", "bf16", "fp32", 24, 32, 128, 1024, True, name="muon_large"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes over the whole range of the listed ones, odd ones among them."""
    op = rng.choice(["route", "dispatch", "dispatch", "combine", "combine", "ortho", "muon", "muon"])
    if op == "route":
        N = _log_int(rng, 2, 256)
        T = _log_int(rng, 1, min(4 * 16384, 4 * 16384 * 64 // N))
        k = min(N, rng.choice([1, 2, 2, 4, 6, 8]))
        # (one expert a token with its weight brought to one would learn nothing)
        return _route(rng.choice(["fwd", "step"]), rng.choice(["bf16", "fp16", "fp32"]), T, N, k, k > 1 and rng.random() < 0.6)
    if op in ("dispatch", "combine"):
        while True:
            T, N, k = _log_int(rng, 1, 32 * 16384), _log_int(rng, 2, 64), rng.choice([1, 2, 2, 3, 4])
            D = rng.choice([16, 32, 64, 64, 100, 128, 128, 201, 256])
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            factor = rng.choice([0.0, 1.0, 1.25, 1.25, 2.0])
            k = min(k, N)
            cap = _capacity(T, N, k, factor) if factor else 0
            if N * (cap or T) * D * _BYTES[dtype] <= 32 * 40960 * 256 and T * k * N <= 1 << 25 and T * D * _BYTES[dtype] <= 32 * 16384 * 256:
                return _tokens(op, rng.choice(["fwd", "step", "step"]), dtype, T, D, N, k, cap)
    if op == "ortho":
        D, E = rng.choice([16, 32, 64, 64, 100, 128, 128, 201, 256]), _log_int(rng, 64, 2048)
        R, C = (D, E) if rng.random() < 0.5 else (E, D)
        return _ortho(rng.choice(["bf16", "fp16", "fp32"]), _log_int(rng, 1, 32), R, C)
    while True:
        layers, H = _log_int(rng, 1, 32), _log_int(rng, 1, 32)
        D, E = rng.choice([16, 32, 64, 64, 128, 128, 256]), _log_int(rng, 64, 2048)
        dtype = rng.choice(["fp32", "fp32", "bf16"])
        if layers * H * D * E * max(1, D / 128) <= 24 * 32 * 128 * 1024:
            return _muon(dtype, rng.choice(["bf16", "fp32", "fp16"]), rng.choice(["fp32", "fp32", dtype]), layers, H, D, E,
                         rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
class _Normal:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def __call__(self, shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    def low_rank(self, shape, std, dtype):
        """a product of rank 8 and half as much noise, elements of size std"""
        *h, r, c = shape
        t = torch.matmul(self((*h, r, 8)), self((*h, 8, c)))
        return t.mul_(std / math.sqrt(8)).add_(self(shape, 0.5 * std)).to(dtype)


def _logits(normal, T, N):
    return normal((T, N)) + normal((N,), 0.5)


def _choice(normal, T, N, k):
    """experts (T, k) int32, different ones for each token, and their weights in fp32: their shares of the softmax,
    which sum to one where there are several"""
    p, e = torch.topk(torch.softmax(_logits(normal, T, N), 1), k, dim=1)
    return e.int(), p / p.sum(1, keepdim=True) if k > 1 else p


def _rows_of(case):
    return case["capacity"] or case["T"]


def _slots(experts, N, cap):
    """a plan's two tensors: the row of each assignment (-1: dropped) and the experts' loads"""
    flat = experts.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    load = torch.bincount(flat, minlength=N)
    at = torch.empty_like(flat)
    at[order] = torch.arange(flat.numel(), device=flat.device) - (load.cumsum(0) - load)[flat[order]]
    return torch.where(at < cap, flat * cap + at, -1).int().view(experts.shape), load.int()


def _stack_shapes(case):
    H, D, E = case["H"], case["D"], case["E"]
    return [(H, D, E), (H, D, E), (H, E, D)] * case["layers"]


def _views(buffer, shapes):
    """one view of the buffer for each shape, one after the other"""
    sizes = [math.prod(s) for s in shapes]
    return [v.view(s) for v, s in zip(buffer.split(sizes), shapes)]


def _muon_inputs(case, seed):
    """the weights' and the momenta's buffers, their views, and the gradients."""
    normal, shapes = _Normal(seed), _stack_shapes(case)
    n = sum(math.prod(s) for s in shapes)
    w = torch.empty(n, dtype=_DTYPES[case["dtype"]], device="cuda")
    m = torch.empty(n, dtype=_DTYPES[case["moment"]], device="cuda")
    ws, ms, gs = _views(w, shapes), _views(m, shapes), []
    for i, (s, wv, mv) in enumerate(zip(shapes, ws, ms)):
        std = 10.0 ** (-(i % 5) / 2.0 - 2.0)
        wv.copy_(normal(s, 1.0 / math.sqrt(s[1])))
        mv.copy_(normal.low_rank(s, 0.5 * std, torch.float32))
        gs.append(normal.low_rank(s, std, _DTYPES[case["grad"]]))
    return w, m, ws, ms, gs


def prepare(case, seed):
    op, kind = case["op"], case.get("kind")
    state = {"op": op, "kind": kind}
    normal = _Normal(seed)
    if op == "route":
        T, N, k = case["T"], case["N"], case["k"]
        x = _logits(normal, T, N).to(_DTYPES[case["dtype"]])
        state.update(logits=x.requires_grad_(kind == "step"), k=k, normalize=case["normalize"], dw=normal((T, k)))
    elif op in ("dispatch", "combine"):
        T, D, N, k, cap, dt = case["T"], case["D"], case["N"], case["k"], _rows_of(case), _DTYPES[case["dtype"]]
        experts, weights = _choice(normal, T, N, k)
        state.update(experts=experts, N=N, capacity=case["capacity"] or None, cap=cap)
        if op == "dispatch":
            state["x"] = normal((T, D), 1.0, dt).requires_grad_(kind == "step")
            state["drows"] = normal((N, cap, D), 1.0, dt) if kind == "step" else None
        else:
            state["slots"], state["counts"] = _slots(experts, N, cap)
            state["rows"] = normal((N, cap, D), 1.0, dt).requires_grad_(kind == "step")
            state["weights"] = weights.requires_grad_(kind == "step")
            state["do"] = normal((T, D), 1.0, dt) if kind == "step" else None
    elif op == "ortho":
        state["x"] = normal.low_rank((case["H"], case["R"], case["C"]), 1e-3, _DTYPES[case["dtype"]])
    else:
        w, m, ws, ms, gs = _muon_inputs(case, seed)
        state.update(w=w, m=m, ws=ws, ms=ms, gs=gs, nesterov=case["nesterov"])
    return state


# ---------------------------------------------------------------------------------------------
# the operators' plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------
def _route_plain(st):
    x, k = st["logits"].detach().float(), st["k"]
    e = torch.exp(x - x.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    experts = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    sel = p.gather(1, experts)
    total = sel.sum(1, keepdim=True)
    w = sel / total if st["normalize"] else sel
    if st["kind"] == "fwd":
        return w, experts.int()
    dw = st["dw"]
    inner = (w * dw).sum(1, keepdim=True)
    if st["normalize"]:
        dx = torch.zeros_like(x).scatter_(1, experts, w * (dw - inner))
    else:
        dx = (p * -inner).scatter_add_(1, experts, w * dw)
    return w, experts.int(), dx.to(st["logits"].dtype)


def _plan_plain(experts, N, cap):
    flat = experts.reshape(-1).long()
    one = (torch.arange(N, device=flat.device)[:, None] == flat).int()
    at = one.cumsum(1, dtype=torch.int32).gather(0, flat[None])[0] - 1
    slots = torch.where(at < cap, flat.int() * cap + at, -1)
    return slots.view(experts.shape), one.sum(1, dtype=torch.int32)


def _gathered(rows, slots):
    """rows (N cap, D) at slots (T, k), zeros where a slot is -1, in fp32"""
    t = rows[slots.long().clamp(min=0)].float()
    return t * (slots >= 0)[..., None]


def _scattered(values, slots, n):
    """(n, D) with values (T, k, D) at their slots, zeros elsewhere"""
    out = values.new_zeros(n + 1, values.shape[-1])
    at = torch.where(slots < 0, n, slots).long()
    out[at.reshape(-1)] = values.reshape(-1, values.shape[-1])
    return out[:n]


def _dispatch_plain(st):
    x, N, cap = st["x"].detach(), st["N"], st["cap"]
    slots, counts = _plan_plain(st["experts"], N, cap)
    D = x.shape[1]
    rows = _scattered(x[:, None].expand(-1, slots.shape[1], -1), slots, N * cap).view(N, cap, D)
    if st["kind"] == "fwd":
        return rows, slots, counts
    return rows, slots, counts, _gathered(st["drows"].view(-1, D), slots).sum(1).to(x.dtype)


def _combine_plain(st):
    rows, w, slots = st["rows"].detach(), st["weights"].detach(), st["slots"]
    N, cap, D = rows.shape
    t = _gathered(rows.view(-1, D), slots)
    o = (t * w[..., None]).sum(1).to(rows.dtype)
    if st["kind"] == "fwd":
        return (o,)
    do = st["do"].float()
    drows = _scattered((do[:, None] * w[..., None]).to(rows.dtype), slots, N * cap).view(N, cap, D)
    return o, drows, (t * do[:, None]).sum(2)


def _orthogonal_plain(u):
    a, b, c = _COEFFICIENTS
    x = u / ((u * u).sum((-2, -1), keepdim=True).sqrt() + _EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    for _ in range(_STEPS):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def _muon_plain(st):
    for w, m, g in zip(st["ws"], st["ms"], st["gs"]):
        gf = g.float()
        m.copy_(_MOMENTUM * m.float() + (1 - _MOMENTUM) * gf)
        u = (1 - _MOMENTUM) * gf + _MOMENTUM * m.float() if st["nesterov"] else m.float()
        R, C = w.shape[-2:]
        lr = _LR * math.sqrt(max(1.0, R / C))
        w.copy_(w.float() * (1 - _LR * _DECAY) - lr * _orthogonal_plain(u))
    return st["w"], st["m"]


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if not own:
        if op == "ortho":
            return _orthogonal_plain(state["x"].float()).to(state["x"].dtype)
        return {"route": _route_plain, "dispatch": _dispatch_plain, "combine": _combine_plain, "muon": _muon_plain}[op](state)
    import flashmlp_amd as fm

    step = state["kind"] == "step"
    if op == "route":
        x = state["logits"]
        w, experts = fm.expert_route(x, state["k"], normalize=state["normalize"])
        if not step:
            return w, experts
        return w.detach(), experts, torch.autograd.grad(w, x, state["dw"])[0]
    if op == "dispatch":
        x = state["x"]
        plan = fm.expert_plan(state["experts"], state["N"], state["capacity"])
        rows = fm.expert_dispatch(x, plan)
        if not step:
            return rows, plan.slots, plan.counts
        return rows.detach(), plan.slots, plan.counts, torch.autograd.grad(rows, x, state["drows"])[0]
    if op == "combine":
        rows, w = state["rows"], state["weights"]
        plan = fm.ExpertPlan(state["slots"], state["counts"], state["N"], state["cap"])
        o = fm.expert_combine(rows, plan, w)
        if not step:
            return (o,)
        return (o.detach(), *torch.autograd.grad(o, (rows, w), state["do"]))
    if op == "ortho":
        return fm.orthogonalize(state["x"], steps=_STEPS, coefficients=_COEFFICIENTS, eps=_EPS)
    fm.muon_step(state["ws"], state["gs"], state["ms"], _LR, momentum=_MOMENTUM, nesterov=state["nesterov"],
                 weight_decay=_DECAY, steps=_STEPS, coefficients=_COEFFICIENTS, eps=_EPS)
    return state["w"], state["m"]


def work(case):
    """What a pass cannot do without: each input read once, each output written once. Newton-Schulz products on the
    small side n of a matrix n x e: its symmetric Gram matrix (n n e), 17 symmetric products of n x n for five steps (n n n
    each) and the result (2 n n e)."""
    op, s = case["op"], _BYTES[case["dtype"]]
    if op == "route":
        T, N, k = case["T"], case["N"], case["k"]
        step = case["kind"] == "step"
        return {"bytes": T * N * s * (2 if step else 1) + T * k * (12 if step else 8), "flops": T * (N * (k + 4) + (6 * k if step else 0))}
    if op in ("dispatch", "combine"):
        T, D, N, k, cap = case["T"], case["D"], case["N"], case["k"], _rows_of(case)
        x, rows, kept = T * D * s, N * cap * D * s, min(T * k, N * cap) * D * s
        step = case["kind"] == "step"
        if op == "dispatch":
            return {"bytes": x + rows + 8 * T * k + 4 * N + (kept + x if step else 0), "flops": T * k * D if step else T * k}
        return {"bytes": kept + x + 8 * T * k + (x + rows + 4 * T * k if step else 0), "flops": T * k * D * (5 if step else 2)}

    def products(h, r, c):
        n, e = min(r, c), max(r, c)
        return h * (3 * n * n * e + 17 * n ** 3)

    if op == "ortho":
        H, R, C = case["H"], case["R"], case["C"]
        return {"bytes": 2 * H * R * C * s, "flops": products(H, R, C)}
    shapes = _stack_shapes(case)
    n = sum(math.prod(v) for v in shapes)
    return {"bytes": n * (_BYTES[case["grad"]] + 2 * _BYTES[case["moment"]] + 2 * s),
            "flops": sum(products(*v) for v in shapes) + 8 * n}


# ---------------------------------------------------------------------------------------------
# the same outputs in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_route(case, seed):
    st = prepare(case, seed)
    x = st["logits"].detach().double().requires_grad_(True)
    p = torch.softmax(x, 1)
    # the order of (logit, lowest index): distinct keys, the index a step below any difference of two logits
    N = case["N"]
    rank = x.detach().unique(return_inverse=True)[1] * N + (N - 1 - torch.arange(N, device=x.device))
    experts = rank.topk(case["k"], dim=1).indices
    w = p.gather(1, experts)
    if case["normalize"]:
        w = w / w.sum(1, keepdim=True)
    if case["kind"] == "fwd":
        return w.detach(), None
    return w.detach(), None, torch.autograd.grad(w, x, st["dw"].double())[0]


def _exact_dispatch(case, seed):
    st = prepare(case, seed)
    N, cap = case["N"], _rows_of(case)
    slots, _ = _slots(st["experts"], N, cap)
    x = st["x"].detach().double()
    D = x.shape[1]
    token, j = torch.nonzero(slots >= 0, as_tuple=True)
    rows = torch.zeros(N * cap, D, dtype=torch.float64, device="cuda")
    rows.index_copy_(0, slots[token, j].long(), x[token])
    rows = rows.view(N, cap, D)
    if case["kind"] == "fwd":
        return rows, None, None
    dx = torch.zeros_like(x).index_add_(0, token, st["drows"].view(-1, D)[slots[token, j].long()].double())
    return rows, None, None, dx


def _exact_combine(case, seed):
    st = prepare(case, seed)
    slots = st["slots"]
    token, j = torch.nonzero(slots >= 0, as_tuple=True)
    at = slots[token, j].long()
    N, cap, D = st["rows"].shape
    flat = st["rows"].detach().view(-1, D)
    w = st["weights"].detach().double()
    o = torch.zeros(case["T"], D, dtype=torch.float64, device="cuda")
    o.index_add_(0, token, flat[at].double() * w[token, j][:, None])
    if case["kind"] == "fwd":
        return (o,)
    do = st["do"].double()
    drows = torch.zeros(N * cap, D, dtype=torch.float64, device="cuda").index_copy_(0, at, do[token] * w[token, j][:, None])
    dw = torch.zeros_like(w)
    dw[token, j] = (flat[at].double() * do[token]).sum(1)
    return o, drows.view(N, cap, D), dw


def _exact_orthogonal(u):
    # on the side of the smaller Gram matrix: O = P X with P and G polynomials of it
    a, b, c = _COEFFICIENTS
    tall = u.shape[-2] > u.shape[-1]
    x = (u.mT if tall else u).contiguous()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + _EPS)
    g = torch.matmul(x, x.mT.contiguous())
    eye = torch.eye(g.shape[-1], dtype=g.dtype, device=g.device)
    p = eye.expand_as(g)
    for i in range(_STEPS):
        q = a * eye + b * g + c * torch.matmul(g, g)
        p = torch.matmul(q, p)
        if i + 1 < _STEPS:
            g = torch.matmul(torch.matmul(q, g), q)
    o = torch.matmul(p, x)
    return o.mT if tall else o


def _exact_muon(case, seed):
    w, m, ws, ms, gs = _muon_inputs(case, seed)
    w2, m2 = torch.empty_like(w, dtype=torch.float64), torch.empty_like(m, dtype=torch.float64)
    shapes = [g.shape for g in gs]
    for wv, mv, gv, wo, mo in zip(ws, ms, gs, _views(w2, shapes), _views(m2, shapes)):
        g = gv.double()
        mo.copy_(torch.lerp(g, mv.double(), _MOMENTUM))
        kept = mo.to(mv.dtype).double()  # the momentum as it is stored is what the update reads
        u = torch.lerp(g, kept, _MOMENTUM) if case["nesterov"] else kept
        R, C = g.shape[-2:]
        wo.copy_(wv.double() * (1 - _LR * _DECAY)).sub_(_exact_orthogonal(u), alpha=_LR * max(1.0, R / C) ** 0.5)
    return w2, m2


def exact(case, seed):
    if case["op"] == "ortho":
        return _exact_orthogonal(prepare(case, seed)["x"].double())
    return {"route": _exact_route, "dispatch": _exact_dispatch, "combine": _exact_combine, "muon": _exact_muon}[case["op"]](case, seed)
