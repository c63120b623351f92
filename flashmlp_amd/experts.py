"""Experts: tokens that choose among the heads of a multi-head MLP, and the way to their rows and back.

    expert_route(logits, k, *, normalize=True) -> (weights, experts)            (T, k), (T, k)
    expert_plan(experts, num_experts, capacity=None) -> ExpertPlan
    expert_dispatch(x, plan) -> rows                                            (N, capacity, D)
    expert_combine(rows, plan, weights=None) -> o                               (T, D)
    GatedExperts(num_experts, hidden_dim, intermediate_dim, experts_per_token=2, capacity_factor=None, ...)

    p = softmax(logits), the k largest of each token (ties: the lowest index), weights = p / sum of the k
    rows[slot(t, j)] = x[t],  o[t] = sum over j of weights[t, j] * rows[slot(t, j)]

`rows` is the (H, B, D) layout that flashmlp_fwd and flashmlp_gated_fwd read, a head for each expert. An expert takes its
tokens in their order up to `capacity`, further ones are dropped, their weights not given to others (capacity=None: a row
for every token, none is); rows without a token are zeros. Nothing waits for the loads: sizes do not depend on them. All
but the plan are differentiable; sums are fp32, in a fixed order. Tokens and rows are fp16, bf16 or fp32, weights fp32.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from .block import _dense_cols, _input
from .flashmlp import _DTYPES, _alloc_ws, _fast, _ptr
from .gated import GatedFlashMLP, _not_traced, _On, first_derivatives_only

_MAX_ROWS = 2 ** 31 - 1


class ExpertPlan(NamedTuple):
    """Where tokens go (expert_plan): slots (T, k) int32, the row e * capacity + position of each choice, -1 for one that
    is dropped; counts (num_experts,) int32, the choices of each expert, dropped ones too. To leave a choice out (a padded
    token's), give expert_plan -1 for its expert: the counts say which rows are zeros, and have to go with the slots (rows
    below an expert's count that no slot names are not written)."""
    slots: torch.Tensor
    counts: torch.Tensor
    num_experts: int
    capacity: int


def _gpu(t: torch.Tensor):
    if t.device.type != "cuda":
        raise RuntimeError(f"FlashMLP runs on an AMD GPU through HIP; got a tensor on {t.device} (move inputs to 'cuda')")
    return t.device


def _io(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError(f"FlashMLP supports float16, bfloat16 and float32 {what}, got {t.dtype}")
    return _DTYPES[t.dtype]


def _beside(t: torch.Tensor, dev, dtype, what: str):
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise RuntimeError(f"all tensors must be on one device ({dev} vs {t.device})")


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t.resolve_neg().contiguous()


def _needs_function(*ts) -> bool:
    # for its gradients, or to refuse forward mode
    ts = [t for t in ts if t is not None]
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts) or any(unpack_dual(t).tangent is not None for t in ts)


def _save(ctx, *ts):
    ctx.save_for_backward(*ts)
    ctx.saved_as = [None if t is None else (t.shape, t.dtype, t.device) for t in ts]


def _saved(ctx):
    # hooks may bring a tensor back in any layout: the kernels are given dense ones of the size, type and device that were saved
    ts = ctx.saved_tensors  # (each is unpacked once)
    for t, was in zip(ts, ctx.saved_as):
        if t is not None and (t.shape, t.dtype, t.device) != was:
            raise RuntimeError("a saved tensor of the experts' operators came back with another size, type or device")
    return ts


# ---------------------------------------------------------------------------------------------
# route
# ---------------------------------------------------------------------------------------------
def _route_fwd(logits, k, normalize):
    T, N = logits.shape
    logits = _dense_cols(logits)
    weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    experts = torch.empty((T, k), dtype=torch.int32, device=logits.device)
    with _On(logits.get_device()) as stream:
        st = _lib.lib().fmlp_route_fwd(_input(logits), weights.data_ptr(), experts.data_ptr(), T, N, logits.stride(0), k,
                                       int(normalize), _DTYPES[logits.dtype], stream)
    _lib.check(st, "route forward")
    return weights, experts


class _RouteFunction(torch.autograd.Function):
    """Saves the weights and experts, and the logits where the weights are not brought to a sum of one."""

    @staticmethod
    def forward(ctx, logits, k, normalize):
        weights, experts = _route_fwd(logits, k, normalize)
        _save(ctx, None if normalize else logits, weights, experts)
        ctx.args = (logits.shape, logits.dtype, normalize)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @first_derivatives_only
    def backward(ctx, dw, _):
        logits, weights, experts = _saved(ctx)
        (T, N), dtype, normalize = ctx.args
        weights, experts, dw = _dense(weights), _dense(experts), _dense(dw)
        logits = None if logits is None else _dense_cols(logits)
        dlogits = torch.empty((T, N), dtype=dtype, device=weights.device)
        with _On(weights.get_device()) as stream:
            st = _lib.lib().fmlp_route_bwd(None if logits is None else _input(logits), _input(weights), _input(experts),
                                           _input(dw), dlogits.data_ptr(), T, N, 0 if logits is None else logits.stride(0),
                                           weights.shape[1], int(normalize), _DTYPES[dtype], stream)
        _lib.check(st, "route backward")
        return dlogits, None, None


@torch.compiler.disable  # (torch.compile breaks its graph here)
def expert_route(logits: torch.Tensor, k: int, *, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each token's k experts and their weights.

    Args:
        logits: (T, N), fp16, bf16 or fp32; -infinity masks an expert; N <= 1024, k <= 32;
        normalize: the weights are softmax probabilities over their sum over the k; else as they are. (With k = 1 the
        weight is 1 whatever the logits, which get no gradient then.)
    Returns:
        (weights, experts): (T, k) fp32, and (T, k) int32 in falling order of the logits. A token with fewer
        than k experts that are not masked has -1 with the weight 0 in place of the rest.
    """
    if _fast is not None:  # tensors that need no copies and no error: else None
        r = _fast.expert_route(logits, k, normalize)
        if r is not None:
            return r
    _not_traced("expert_route")
    assert logits.dim() == 2, "Logits must be (tokens, experts)"
    T, N = logits.shape
    assert 1 <= k <= N, "A token takes at least one expert and at most all"
    _gpu(logits)
    _io(logits, "logits")
    if _needs_function(logits):
        return _RouteFunction.apply(logits, int(k), bool(normalize))
    return _route_fwd(logits, int(k), normalize)


# ---------------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------------
@torch.compiler.disable
def expert_plan(experts: torch.Tensor, num_experts: int, capacity: Optional[int] = None) -> ExpertPlan:
    """The row of each token's choices: a stable sort by expert.

    Args:
        experts: (T, k) int32 or int64; values outside [0, num_experts) are no choice (expert_route's -1);
        num_experts: at most 1024; capacity: rows of each expert, None for T, so that none is dropped (as long as a
        token's choices differ).
    """
    if _fast is not None:  # as in expert_route
        rows = capacity if capacity is not None else experts.shape[0] if experts.dim() else -1
        r = _fast.expert_plan(experts, num_experts, rows)
        if r is not None:
            return ExpertPlan(*r, num_experts, rows)
    _not_traced("expert_plan")
    assert experts.dim() == 2, "Experts must be (tokens, choices)"
    T, k = experts.shape
    capacity = T if capacity is None else capacity
    assert num_experts >= 1 and capacity >= 0 and k >= 1, "Experts, choices and rows must be counted"
    _gpu(experts)
    if experts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"experts must be int32 or int64, got {experts.dtype}")
    experts, dev = experts.contiguous(), experts.device
    slots = torch.empty((T, k), dtype=torch.int32, device=dev)
    counts = torch.empty((num_experts,), dtype=torch.int32, device=dev)
    L = _lib.lib()
    with _On(dev.index) as stream:
        n = L.fmlp_expert_plan_workspace_bytes(T, k, num_experts)
        ws = _alloc_ws(n, dev)
        st = L.fmlp_expert_plan(_input(experts), experts.element_size(), slots.data_ptr(), counts.data_ptr(), T, k,
                                num_experts, capacity, _ptr(ws), n, stream)
    _lib.check(st, "expert plan")
    return ExpertPlan(slots, counts, int(num_experts), int(capacity))


def _check_plan(plan, dev):
    slots, counts, N, capacity = plan
    assert slots.dim() == 2 and counts.shape == (N,), "The plan's slots must be (tokens, choices), its counts one per expert"
    _beside(slots, dev, torch.int32, "the plan's slots")
    _beside(counts, dev, torch.int32, "the plan's counts")
    return slots.shape


# ---------------------------------------------------------------------------------------------
# dispatch and combine
# ---------------------------------------------------------------------------------------------
def _scatter(x, weights, slots, counts, N, capacity, rows_in, want_rows, want_dw):
    """(rows, dweights); those that are not wanted None"""
    x, slots, counts = _dense_cols(x), _dense(slots), _dense(counts)
    (T, k), D, dev = slots.shape, x.shape[1], x.device
    weights = None if weights is None else _dense(weights)
    rows_in = _dense(rows_in) if want_dw else None
    rows = torch.empty((N, capacity, D), dtype=x.dtype, device=dev) if want_rows else None
    dw = torch.empty((T, k), dtype=torch.float32, device=dev) if want_dw else None
    if rows is None and dw is None:
        return rows, dw
    with _On(dev.index) as stream:
        st = _lib.lib().fmlp_expert_scatter(_input(x), x.stride(0), None if weights is None else _input(weights), _input(slots),
                                            _input(counts), None if rows_in is None else _input(rows_in), _ptr(rows), _ptr(dw),
                                            T, k, N, capacity, D, _DTYPES[x.dtype], stream)
    _lib.check(st, "expert scatter")
    return rows, dw


def _gather(rows, weights, slots):
    rows, slots = _dense(rows), _dense(slots)
    weights = None if weights is None else _dense(weights)
    (N, capacity, D), (T, k) = rows.shape, slots.shape
    o = torch.empty((T, D), dtype=rows.dtype, device=rows.device)
    with _On(rows.get_device()) as stream:
        st = _lib.lib().fmlp_expert_gather(_input(rows), None if weights is None else _input(weights), _input(slots), o.data_ptr(),
                                           T, k, N, capacity, D, _DTYPES[rows.dtype], stream)
    _lib.check(st, "expert gather")
    return o


class _DispatchFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, counts, N, capacity):
        _save(ctx, slots)
        return _scatter(x, None, slots, counts, N, capacity, None, True, False)[0]

    @staticmethod
    @first_derivatives_only
    def backward(ctx, drows):
        return (_gather(drows, None, *_saved(ctx)),) + (None,) * 4


class _CombineFunction(torch.autograd.Function):
    """Saves the rows for the weights' gradient alone."""

    @staticmethod
    def forward(ctx, rows, weights, slots, counts):
        _save(ctx, rows if weights is not None and ctx.needs_input_grad[1] else None, weights, slots, counts)
        ctx.args = rows.shape[:2]
        return _gather(rows, weights, slots)

    @staticmethod
    @first_derivatives_only
    def backward(ctx, do):
        rows, weights, slots, counts = _saved(ctx)
        drows, dw = _scatter(do, weights, slots, counts, *ctx.args, rows, ctx.needs_input_grad[0],
                             weights is not None and ctx.needs_input_grad[1])
        return drows, dw, None, None


@torch.compiler.disable
def expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Tokens x (T, D) at their experts' rows: (num_experts, capacity, D), zeros where no token is."""
    if _fast is not None:  # as in expert_route
        rows = _fast.expert_dispatch(x, *plan)
        if rows is not None:
            return rows
    _not_traced("expert_dispatch")
    assert x.dim() == 2 and x.shape[1] >= 1, "Tokens must be (tokens, columns)"
    dev = _gpu(x)
    _io(x, "tokens")
    assert _check_plan(plan, dev)[0] == x.shape[0], "Number of tokens must match"
    if _needs_function(x):
        return _DispatchFunction.apply(x, *plan)
    return _scatter(x, None, *plan, None, True, False)[0]


@torch.compiler.disable
def expert_combine(rows: torch.Tensor, plan: ExpertPlan, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The tokens' sums of their experts' rows (num_experts, capacity, D), with weights (T, k) fp32 or plainly: (T, D) in
    the rows' dtype. A choice that was dropped adds nothing."""
    if _fast is not None:  # as in expert_route
        o = _fast.expert_combine(rows, weights, *plan)
        if o is not None:
            return o
    _not_traced("expert_combine")
    assert rows.dim() == 3 and rows.shape[2] >= 1, "Rows must be (experts, capacity, columns)"
    assert rows.shape[:2] == (plan.num_experts, plan.capacity), "Rows must be the plan's"
    dev = _gpu(rows)
    _io(rows, "rows")
    shape = _check_plan(plan, dev)
    if weights is not None:
        assert weights.shape == shape, "Weights must be one per choice"
        _beside(weights, dev, torch.float32, "weights")
    if _needs_function(rows, weights):
        return _CombineFunction.apply(rows, weights, plan.slots, plan.counts)
    return _gather(rows, weights, plan.slots)


class GatedExperts(torch.nn.Module):
    """A mixture of gated experts: the heads of a GatedFlashMLP, of which each token takes experts_per_token.

    Args:
        num_experts: number of experts N; hidden_dim: D; intermediate_dim: E; activation, dtype, device: as GatedFlashMLP's
        experts_per_token: k
        capacity_factor: an expert has ceil(T k / N * capacity_factor) rows for T tokens, what comes beyond is
            dropped; None: T rows, none is dropped, and the experts' MLP runs on N T rows for the T k that hold tokens,
            N / k times their work
        normalize: as expert_route's; None: where experts_per_token is above one, so that the router always learns

    The input is (..., D): rows of tokens, or the MLP's (H, B, D) layout, whose heads' rows are tokens of their own.
    Parameters: router (D, N) ~ randn / sqrt(D), and the experts' (experts.wg, experts.wu, experts.w2).
    """

    def __init__(self, num_experts: int, hidden_dim: int, intermediate_dim: int, experts_per_token: int = 2,
                 capacity_factor: Optional[float] = None, activation: str = "silu",
                 normalize: Optional[bool] = None, dtype=torch.float16, device="cuda"):
        super().__init__()
        self.num_experts, self.experts_per_token = num_experts, experts_per_token
        self.capacity_factor, self.normalize = capacity_factor, experts_per_token > 1 if normalize is None else normalize
        self.router = torch.nn.Parameter(torch.randn(hidden_dim, num_experts, dtype=dtype, device=device) / hidden_dim ** 0.5)
        self.experts = GatedFlashMLP(num_experts, hidden_dim, intermediate_dim, activation, dtype=dtype, device=device)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        tokens = x.reshape(-1, x.shape[-1])
        T, N, k = tokens.shape[0], self.num_experts, self.experts_per_token
        weights, experts = expert_route(tokens @ self.router, k, normalize=self.normalize)
        capacity = None if self.capacity_factor is None else math.ceil(T * k / N * self.capacity_factor)
        plan = expert_plan(experts, N, capacity)
        rows = self.experts(expert_dispatch(tokens, plan))
        return expert_combine(rows, plan, weights).view(x.shape)
