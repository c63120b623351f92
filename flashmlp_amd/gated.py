"""Gated multi-head MLP:  O = (act(X Wg) * (X Wu)) W2  per head, with a recomputing backward.

    flashmlp_gated_fwd(x, wg, wu, w2, activation="") -> o                            (H,B,D)
    flashmlp_gated_bwd(x, wg, wu, w2, do, activation="") -> (dx, dwg, dwu, dw2)
    GatedFlashMLPFunction.apply(x, wg, wu, w2, activation)
    GatedFlashMLP(num_heads, hidden_dim, intermediate_dim, activation="silu", dtype, device)

The gated form of flashmlp_fwd / flashmlp_bwd / FlashMLPFunction / FlashMLP, in their manner: x
(H, B, D), wg and wu (H, D, E), w2 (H, E, D); act in {"", "silu", "leaky_relu", "sigmoid"}; fp16, bf16
and fp32 tensors on one GPU, D in {16, 32, 64, 128, 256}, any E >= 1. An x or do of dense rows is read in
place whatever the distance of its heads, other views are copied. Every call launches the HIP kernels
of libflashmlp.so asynchronously on torch's current stream of the tensors' device.
"""
from __future__ import annotations

import functools
from typing import Tuple

import numpy as np
import torch

from . import _lib
from .flashmlp import (_DTYPES, _act_code, _alloc_ws, _current_device, _dense_all, _empty_as, _fast, _io_code, _ptr,
                       _rows, _stream_of)


def _check(x, wg, wu, w2) -> Tuple[int, int, int, int]:
    H, B, D = x.shape
    Hg, Dg, E = wg.shape
    H2, E2, D2 = w2.shape
    assert H == Hg and H == H2, "Number of heads must match"
    assert wu.shape == wg.shape, "Gate and up projections must match"
    assert D == Dg, "Hidden dimension mismatch"
    assert E == E2, "Intermediate dimension mismatch"
    assert D == D2, "Output dimension mismatch"
    return H, B, D, E


def _not_traced(what: str):
    # (the graph would hold the outputs' allocation and not the launch that fills them)
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced by torch.jit.trace: it is no operation that a graph can hold")


class _On:
    """The library launches on the current device: make it the tensors'."""

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.prev = _current_device()
        if self.prev != self.index:
            torch.cuda.set_device(self.index)
        return _stream_of(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)


def _workspace(L, n: int, H: int, D: int, E: int, dtype: int, device):
    """(tensor or None, its size): the call's workspace; where it does not fit, the least the call runs with"""
    try:
        return _alloc_ws(n, device), n
    except torch.OutOfMemoryError:
        least = L.fmlp_gated_min_workspace_bytes(H, D, E, dtype)
        if least >= n:
            raise
        return _alloc_ws(least, device), least


def _fwd(x, wg, wu, w2, activation, out_f32=False):
    """the general path: views and bases that the kernels do not read are copied first"""
    H, B, D, E = _check(x, wg, wu, w2)
    dtype = _io_code(x, wg, wu, w2)
    o = torch.empty((H, B, D), dtype=torch.float32, device=x.device) if out_f32 else _empty_as(x, (H, B, D))
    dtype |= _lib.FMLP_OUT_F32 if out_f32 else 0
    L = _lib.lib()
    with _On(x.get_device()) as stream:
        x = _rows(x)
        wg, wu, w2 = _dense_all(wg, wu, w2)
        ws, n = _workspace(L, L.fmlp_gated_fwd_workspace_bytes(H, B, D, E, dtype), H, D, E, dtype, x.device)
        st = L.fmlp_gated_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), w2.data_ptr(), o.data_ptr(), H, B, D, E,
                              x.stride(0), dtype, _act_code(activation), _ptr(ws), n, stream)
    _lib.check(st, "gated forward")
    return o


def _bwd(x, wg, wu, w2, do, activation, need_dx, need_dw, out_f32=False, dw_scale=1.0):
    H, B, D, E = _check(x, wg, wu, w2)
    assert x.shape == do.shape, "Gradient shape mismatch"
    dtype = _io_code(x, wg, wu, w2, do)
    dx = None
    if need_dx:
        dx = torch.empty((H, B, D), dtype=torch.float32, device=x.device) if out_f32 else _empty_as(x, (H, B, D))
    dwg, dwu, dw2 = ((_empty_as(t, t.shape) for t in (wg, wu, w2)) if need_dw else (None, None, None))
    if not (need_dx or need_dw):
        return dx, dwg, dwu, dw2
    dtype |= (0 if need_dx else _lib.FMLP_BWD_NO_DX) | (0 if need_dw else _lib.FMLP_BWD_NO_DW)
    dtype |= _lib.FMLP_OUT_F32 if out_f32 else 0
    L = _lib.lib()
    with _On(x.get_device()) as stream:
        x, do = _rows(x), _rows(do)
        wg, wu, w2 = _dense_all(wg, wu, w2)
        ws, n = _workspace(L, L.fmlp_gated_bwd_workspace_bytes(H, B, D, E, dtype), H, D, E, dtype, x.device)
        st = L.fmlp_gated_bwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), w2.data_ptr(), do.data_ptr(), _ptr(dx),
                              _ptr(dwg), _ptr(dwu), _ptr(dw2), H, B, D, E, x.stride(0), do.stride(0), dtype,
                              _act_code(activation), dw_scale, _ptr(ws), n, stream)
    _lib.check(st, "gated backward")
    return dx, dwg, dwu, dw2


def _head_sum(t: torch.Tensor, scale: float, dtype: torch.dtype) -> torch.Tensor:
    """scale * the sum over heads of fp32 (H, B, D), rounded once"""
    out = torch.empty(t.shape[1:], dtype=dtype, device=t.device)
    with _On(t.get_device()) as stream:
        st = _lib.lib().fmlp_head_sum(t.data_ptr(), out.data_ptr(), t.shape[0], out.numel(), scale, _DTYPES[dtype], stream)
    _lib.check(st, "head sum")
    return out


def flashmlp_gated_fwd(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, w2: torch.Tensor,
                       activation: str = "") -> torch.Tensor:
    """O = (act(x @ wg) * (x @ wu)) @ w2 per head.

    Args:
        x: (H, B, D); wg, wu: (H, D, E); w2: (H, E, D); activation: "silu", "leaky_relu",
        "sigmoid" or "" (linear: a bilinear product).
    Returns:
        o (H, B, D), dtype of x. The products are summed in fp32 and h = act(.) * (.) is rounded to
        the io dtype before the last one.
    """
    if _fast is not None:  # one GPU, tensors that the kernels read in place: else None
        o = _fast.gated_fwd(x, wg, wu, w2, _act_code(activation))
        if o is not None:
            return o
    if torch.jit.is_tracing():  # the operation that the graph holds
        return torch.ops.flashmlp_amd.gated_fwd(x, wg, wu, w2, activation)
    return _fwd(x, wg, wu, w2, activation)


def flashmlp_gated_bwd(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, w2: torch.Tensor, do: torch.Tensor,
                       activation: str = "", *, _needs: Tuple[bool, bool] = (True, True)):
    """Gradients of flashmlp_gated_fwd: (dx, dwg, dwu, dw2), shaped like (x, wg, wu, w2).

    Recomputes both projections from x instead of reading stored activations. `_needs` (need dx,
    need the weights' gradients; GatedFlashMLPFunction passes autograd's needs_input_grad) skips the
    programs of gradients that nobody asked for and returns None in their place.
    """
    need_dx, need_dw = bool(_needs[0]), bool(_needs[1])
    if _fast is not None:  # as in flashmlp_gated_fwd
        g = _fast.gated_bwd(x, wg, wu, w2, do, _act_code(activation), need_dx, need_dw)
        if g is not None:
            return g
    if torch.jit.is_tracing():  # as in flashmlp_gated_fwd; it computes them all
        g = torch.ops.flashmlp_amd.gated_bwd(x, wg, wu, w2, do, activation)
        return tuple(v if n else None for v, n in zip(g, (need_dx, need_dw, need_dw, need_dw)))
    return _bwd(x, wg, wu, w2, do, activation, need_dx, need_dw)


class _NoSecond(torch.autograd.Function):
    @staticmethod
    def forward(ctx, n, *ts):
        return ts[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("FlashMLP's gradients cannot be differentiated again")


def first_derivatives_only(backward):
    """A Function's backward that cannot be differentiated: under create_graph=True its gradients come with a node
    between them and what they are made of that raises once it is. (torch's once_differentiable adds one where the
    incoming gradients are differentiable, with no connection to the inputs: torch.autograd.grad goes past it, and
    where the saved tensors alone are differentiable a second derivative is silently left out.)"""

    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        of = [t for t in (*grads, *ctx.saved_tensors) if t is not None and t.requires_grad]
        if not of:
            return out
        there = [t for t in out if t is not None]
        marked = iter(_NoSecond.apply(len(there), *there, *of))
        return tuple(t if t is None else next(marked) for t in out)

    return run


class GatedFlashMLPFunction(torch.autograd.Function):
    """Autograd binding of the gated MLP. Saves only (x, wg, wu, w2)."""

    @staticmethod
    def forward(ctx, x, wg, wu, w2, activation=""):
        o = flashmlp_gated_fwd(x, wg, wu, w2, activation)
        ctx.save_for_backward(x, wg, wu, w2)
        ctx.activation = activation
        return o

    @staticmethod
    @first_derivatives_only
    def backward(ctx, do):
        x, wg, wu, w2 = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, *dw = flashmlp_gated_bwd(x, wg, wu, w2, do, ctx.activation, _needs=(need[0], any(need[1:4])))
        return (dx, *(g if n else None for g, n in zip(dw, need[1:4])), None)


class _SharedGatedFunction(torch.autograd.Function):
    """One input (B, D) through every head, the mean over heads: per head in fp32, rounded once behind the sum. The
    gradient of the mean is the same for every head; its 1 / H goes into the sums' and gradients' rounding."""

    @staticmethod
    def forward(ctx, x, wg, wu, w2, activation):
        H = wg.shape[0]
        o = _fwd(x.unsqueeze(0).expand(H, *x.shape), wg, wu, w2, activation, out_f32=True)
        ctx.save_for_backward(x, wg, wu, w2)
        ctx.activation = activation
        return _head_sum(o, 1.0 / H, x.dtype)

    @staticmethod
    @first_derivatives_only
    def backward(ctx, do):
        x, wg, wu, w2 = ctx.saved_tensors
        H, need = wg.shape[0], ctx.needs_input_grad
        dx, *dw = _bwd(x.unsqueeze(0).expand(H, *x.shape), wg, wu, w2, do.unsqueeze(0).expand(H, *do.shape),
                       ctx.activation, need[0], any(need[1:4]), out_f32=True, dw_scale=1.0 / H)
        dx = _head_sum(dx, 1.0 / H, x.dtype) if need[0] else None
        return (dx, *(g if n else None for g, n in zip(dw, need[1:4])), None)


class GatedFlashMLP(torch.nn.Module):
    """Gated multi-head MLP module (the gated form of FlashMLP).

    Args:
        num_heads: number of heads H
        hidden_dim: hidden dimension D
        intermediate_dim: intermediate dimension E
        activation: "silu", "leaky_relu", "sigmoid" or ""
        dtype: weight dtype (float16, bfloat16 or float32)
        device: device of the weights

    Parameters wg, wu (H, D, E) ~ randn / sqrt(D) and w2 (H, E, D) ~ randn / sqrt(E). A 2-D input
    (B, D) goes through every head and the output is the mean over heads, as in FlashMLP; the heads'
    results, and the gradient of x, are summed in fp32 and rounded once (under torch.compile, which traces the
    registered per-head operator, each head's are rounded first).
    """

    def __init__(self, num_heads: int, hidden_dim: int, intermediate_dim: int, activation: str = "silu",
                 dtype=torch.float16, device="cuda"):
        super().__init__()
        self.num_heads = num_heads
        self.hidden_dim = hidden_dim
        self.intermediate_dim = intermediate_dim
        self.activation = activation

        def weight(rows, cols):
            return torch.nn.Parameter(torch.randn(num_heads, rows, cols, dtype=dtype, device=device) / np.sqrt(rows))

        self.wg = weight(hidden_dim, intermediate_dim)
        self.wu = weight(hidden_dim, intermediate_dim)
        self.w2 = weight(intermediate_dim, hidden_dim)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w, act = (self.wg, self.wu, self.w2), self.activation
        shared = x.dim() == 2
        if torch.compiler.is_compiling():  # the registered operator is what torch.compile traces through
            xh = x.unsqueeze(0).expand(self.num_heads, -1, -1) if shared else x
            o = torch.ops.flashmlp_amd.gated_fwd(xh, *w, act)
            return o.mean(dim=0) if shared else o
        if _fast is not None:  # the same autograd nodes in C++ where the kernels read the tensors in place
            o = (_fast.gated_shared if shared else _fast.gated)(x, *w, _act_code(act))
            if o is not None:
                return o
        # (under torch.jit.trace too, whose graph holds these Functions)
        return (_SharedGatedFunction if shared else GatedFlashMLPFunction).apply(x, *w, act)
