"""The norms, gate and residual around a block, one launch each way.

    block_norm(x, weight=None, *, heads=None, dtype=None, eps=1e-6) -> y
    block_join(residual, o, post_weight=None, gate=None, scale=1.0, *, pre_weight=None, post=True, pre=True,
               eps=1e-6) -> (residual', y)

    n = o / rms(o), p = n * post_weight                (RMS norm after the block; post=False: p = o)
    residual' = residual + scale * gate * p
    y = residual' / rms(residual') * pre_weight        (RMS norm before the next block)

The stream `residual` is (B, C). The block's output `o` and its next input `y` are (H, B, D) with
H D = C, the layout of flashmlp_gated_fwd and flashmlp_fwd (head h has the columns h D .. of the stream), or
(B, C). block_norm is the first block's input: y alone, from the stream as it is. `gate` is (C,) for every
row or (G, C), row g for the rows g B/G .. (one per sequence, or per token with G = B); `scale` is a number.
The stream may be fp32 beside 16-bit blocks; weights and gate have the blocks' dtype. Sums are fp32, and y is
taken from the unrounded residual'. Both functions are differentiable; strides and alignments are any
as long as the columns are dense (other views are copied).
"""
from __future__ import annotations

import numbers
from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from .flashmlp import _DTYPES, _alloc_ws, _fast, _ptr
from .gated import _not_traced, _On, first_derivatives_only


def _dense_cols(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    # unit column stride and no lazily negated data
    if t is None or (t.stride(-1) == 1 or t.shape[-1] <= 1) and not t.is_neg():
        return t
    return t.resolve_neg().contiguous()


def _heads3(t: torch.Tensor) -> Tuple[int, int]:
    """head and row stride of a (H, B, D) or (B, C) tensor"""
    return (t.stride(0), t.stride(1)) if t.dim() == 3 else (0, t.stride(0))


def _check_join(r, o, w_post, gate, w_pre, heads, dtype, post, pre):
    """shapes, dtypes and devices; the sizes (B, H, D, groups)"""
    assert r.dim() == 2, "The stream must be (rows, columns)"
    B, C = r.shape
    if o is not None:
        assert o.dim() in (2, 3), "The block's output must be (heads, rows, columns) or (rows, columns)"
        H, Bo, D = o.shape if o.dim() == 3 else (1, *o.shape)
        assert Bo == B, "Number of rows must match"
        assert H * D == C, "Columns of the stream and the block must match"
    else:
        H = 1 if heads is None else heads
        assert H >= 1 and C % H == 0, "Columns must divide into the heads"
        D = C // H
        assert w_post is None and gate is None, "A post norm or gate needs the block's output"
    assert C >= 1, "The stream needs columns"
    for w, name in ((w_post, "Post norm weight"), (w_pre, "Pre norm weight")):
        assert w is None or w.shape == (C,), f"{name} must have one value per column"
    assert w_post is None or post, "A post norm weight needs the post norm"
    assert w_pre is None or pre, "A pre norm weight needs the pre norm"
    groups = 1
    if gate is not None:
        assert gate.dim() in (1, 2) and gate.shape[-1] == C, "The gate must have one value per column"
        groups = gate.shape[0] if gate.dim() == 2 else 1
        assert groups >= 1 and B % groups == 0, "Rows must divide into the gate's rows"
    dev = r.device
    if dev.type != "cuda":
        raise RuntimeError(f"FlashMLP runs on an AMD GPU through HIP; got a tensor on {dev} (move inputs to 'cuda')")
    if dtype not in _DTYPES or r.dtype not in (dtype, torch.float32):
        raise TypeError(f"the stream must be {dtype} or float32 beside float16, bfloat16 or float32 blocks, got {r.dtype}")
    for t in (o, w_post, gate, w_pre):
        if t is not None and t.device != dev:
            raise RuntimeError(f"all tensors must be on one device ({dev} vs {t.device})")
        if t is not None and t.dtype != dtype:
            raise TypeError(f"block output, weights and gate must share one dtype ({dtype} vs {t.dtype})")
    return B, H, D, groups


def _check_number(v, name):
    # (a tensor would be read on the host, and get no gradient)
    if not isinstance(v, numbers.Real):
        raise TypeError(f"{name} must be a number, got {type(v).__name__}")


def _input(t):
    # an input's address, None for one that is not there: what has no memory of its own (a wrapper around other tensors, a
    # fake one) would pass for that
    p = _ptr(t)
    if p == 0 and t.numel() > 0:
        raise TypeError(f"a tensor without memory of its own ({type(t).__name__}) cannot be read by the kernels")
    return p


def _row_values(t, B, dev, name):
    # the rows' 1 / rms as the kernels read them: one fp32 number a row, dense (None where no kernel does)
    if t is None:
        return None
    assert t.shape == (B,), f"{name} must have one value per row"
    if t.dtype != torch.float32 or t.device != dev:
        raise TypeError(f"{name} must be float32 on {dev}, got {t.dtype} on {t.device}")
    return t.resolve_neg().contiguous()


def _call(B, H, D, groups, scale, eps, dtype, r_dtype, post) -> _lib.Join:
    j = _lib.Join()
    j.B, j.H, j.D, j.groups = B, H, D, groups
    j.scale, j.eps, j.post = scale, eps, int(post)
    j.dtype, j.r_dtype = _DTYPES[dtype], _DTYPES[r_dtype]
    return j


def _flat(w):
    # weights and gate as dense rows
    return None if w is None else w.resolve_neg().contiguous()


def block_join_fwd(residual, o, post_weight=None, gate=None, scale=1.0, *, pre_weight=None, post=True, pre=True,
                   eps=1e-6, heads=None, dtype=None, _save=False):
    """(residual', y, rs_o, rs_r): block_join without autograd. residual' is None without o; y is None with
    pre=False; rs_o, rs_r (the rows' 1 / rms, what the backward reads) are None unless `_save`."""
    _not_traced("block_join_fwd")
    return _join_fwd(residual, o, post_weight, gate, scale, pre_weight, post, pre, eps, heads, dtype, _save)


def _join_fwd(residual, o, post_weight, gate, scale, pre_weight, post, pre, eps, heads, dtype, _save):
    _check_number(scale, "scale")
    _check_number(eps, "eps")
    dtype = (o.dtype if o is not None else dtype or residual.dtype)
    B, H, D, groups = _check_join(residual, o, post_weight, gate, pre_weight, heads, dtype, post, pre)
    dev = residual.device
    as_rows = o.dim() == 2 if o is not None else heads is None
    r2 = torch.empty(residual.shape, dtype=residual.dtype, device=dev) if o is not None else None
    y = torch.empty((B, D) if as_rows else (H, B, D), dtype=dtype, device=dev) if pre else None
    rs = torch.empty((2, B), dtype=torch.float32, device=dev) if _save else None
    if r2 is None and y is None:
        return None, None, None, None
    r, oo = _dense_cols(residual), _dense_cols(o)
    ws = [_flat(w) for w in (post_weight, gate, pre_weight)]
    j = _call(B, H, D, groups, scale, eps, dtype, residual.dtype, post)
    j.r, j.o, j.w_post, j.gate, j.w_pre = (_input(t) for t in (r, oo, *ws))
    j.r_out, j.y = _ptr(r2), _ptr(y)
    if rs is not None:
        j.rs_o, j.rs_r = rs[0].data_ptr(), rs[1].data_ptr()
    j.r_stride = r.stride(0)
    if oo is not None:
        j.o_head_stride, j.o_row_stride = _heads3(oo)
    if y is not None:
        j.y_head_stride, j.y_row_stride = _heads3(y)
    L = _lib.lib()
    with _On(dev.index) as stream:
        st = L.fmlp_join_fwd(j, stream)
    _lib.check(st, "join forward")
    return r2, y, rs[0] if _save else None, rs[1] if _save else None


def block_join_bwd(residual_out, o, rs_o, rs_r, dresidual, dy, post_weight=None, gate=None, scale=1.0, *,
                   pre_weight=None, post=True, eps=1e-6, heads=None, dtype=None, residual=None, _needs=(True,) * 5):
    """Gradients (dresidual_in, do, dpost_weight, dgate, dpre_weight) of block_join_fwd's outputs, which gave
    residual_out (the stream itself without o), rs_o and rs_r. With `residual`, a 16-bit stream
    before the join, the unrounded residual' is made again from it and residual_out is not read: the gradients lose
    nothing to the stream's rounding, as under autograd. dresidual or dy may be None (zero). `_needs`
    says which are wanted; the others, and those of inputs that are None, come back as None."""
    _not_traced("block_join_bwd")
    return _join_bwd(residual_out, o, rs_o, rs_r, dresidual, dy, post_weight, gate, scale, pre_weight, post, eps, heads,
                     dtype, residual, _needs)


def _join_bwd(residual_out, o, rs_o, rs_r, dresidual, dy, post_weight, gate, scale, pre_weight, post, eps, heads, dtype,
              residual, _needs):
    _check_number(scale, "scale")
    _check_number(eps, "eps")
    from_r = residual is not None and o is not None and residual.dtype != torch.float32
    if from_r:
        residual_out = residual
    assert residual_out is not None, "The stream behind the join is needed (or a 16-bit one before it as residual=)"
    dtype = (o.dtype if o is not None else dtype or residual_out.dtype)
    pre = dy is not None
    B, H, D, groups = _check_join(residual_out, o, post_weight, gate, pre_weight if pre else None, heads, dtype, post, pre)
    dev, C = residual_out.device, H * D
    for t, dt, what in ((dresidual, residual_out.dtype, "stream"), (dy, dtype, "block")):
        if t is not None and (t.dtype != dt or t.device != dev):
            raise TypeError(f"the {what}'s gradient must be {dt} on {dev}, got {t.dtype} on {t.device}")
    assert dresidual is None or dresidual.shape == residual_out.shape, "Gradient shape mismatch"
    assert dy is None or tuple(dy.shape) in ((H, B, D), (B, C)) and (dy.dim() == 3 or H == 1), "Gradient shape mismatch"
    rs_o = _row_values(rs_o if o is not None and post else None, B, dev, "rs_o")
    rs_r = _row_values(rs_r if pre else None, B, dev, "rs_r")
    nr, no, npost, ngate, npre = _needs

    def new(shape, dt, want):
        return torch.empty(shape, dtype=dt, device=dev) if want else None

    dr = new((B, C), residual_out.dtype, nr)
    d_o = new(o.shape if o is not None else (), dtype, no and o is not None)
    dpost = new((C,), dtype, npost and post_weight is not None)
    dgate = new(gate.shape if gate is not None else (), dtype, ngate and gate is not None)
    dpre = new((C,), dtype, npre and pre_weight is not None)
    if dpre is not None and dy is None:
        dpre.zero_()
    r2, oo = _dense_cols(residual_out), _dense_cols(o)
    dres, dyy = _dense_cols(dresidual), _dense_cols(dy)
    ws_ = [_flat(w) for w in (post_weight, gate, pre_weight if pre else None)]
    j = _call(B, H, D, groups, scale, eps, dtype, residual_out.dtype, post)
    j.r, j.r_out = (_input(r2), None) if from_r else (None, _input(r2))
    j.o, j.w_post, j.gate, j.w_pre = (_input(t) for t in (oo, *ws_))
    j.rs_o, j.rs_r, j.dr_out, j.dy = (_input(t) for t in (rs_o, rs_r, dres, dyy))
    j.dr, j.d_o, j.dw_post, j.dgate, j.dw_pre = (_ptr(t) for t in (dr, d_o, dpost, dgate, dpre if pre else None))
    j.r_stride = r2.stride(0)
    if oo is not None:
        j.o_head_stride, j.o_row_stride = _heads3(oo)
    if dyy is not None:
        j.y_head_stride, j.y_row_stride = _heads3(dyy)
    if dres is not None:
        j.dr_out_stride = dres.stride(0)
    if d_o is not None:
        j.d_o_head_stride, j.d_o_row_stride = _heads3(d_o)
    L = _lib.lib()
    with _On(dev.index) as stream:
        n = L.fmlp_join_bwd_workspace_bytes(j)
        ws = _alloc_ws(n, dev)
        st = L.fmlp_join_bwd(j, _ptr(ws), n, stream)
    _lib.check(st, "join backward")
    return dr, d_o, dpost, dgate, dpre


class BlockJoinFunction(torch.autograd.Function):
    """Autograd binding of the join. Saves the stream (a 16-bit one before it, else after it), o, the weights and two
    floats a row."""

    @staticmethod
    def forward(ctx, residual, o, post_weight, gate, pre_weight, scale, post, pre, eps, heads, dtype):
        r2, y, rs_o, rs_r = _join_fwd(residual, o, post_weight, gate, scale, pre_weight, post, pre, eps, heads, dtype, True)
        before = r2 is None or residual.dtype != torch.float32
        ctx.save_for_backward(residual if before else r2, o, rs_o, rs_r, post_weight, gate, pre_weight)
        ctx.args = (scale, post, eps, heads, dtype)
        ctx.set_materialize_grads(False)
        return r2, y

    @staticmethod
    @first_derivatives_only
    def backward(ctx, dr2, dy):
        r2, o, rs_o, rs_r, post_weight, gate, pre_weight = ctx.saved_tensors
        scale, post, eps, heads, dtype = ctx.args
        if dr2 is None and dy is None:
            return (None,) * 11
        g = _join_bwd(r2, o, rs_o, rs_r, dr2, dy, post_weight, gate, scale, pre_weight, post, eps, heads, dtype, r2,
                      ctx.needs_input_grad[:5])
        return (*g, *(None,) * 6)


def _through_function(*ts) -> bool:
    # whether a call is to be a Function: for its gradients, as the operation that a traced graph holds, or to refuse
    # forward mode
    if torch.jit.is_tracing():
        return True
    ts = [t for t in ts if t is not None]
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts) or any(unpack_dual(t).tangent is not None for t in ts)


@torch.compiler.disable  # (torch.compile breaks its graph here)
def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, heads: Optional[int] = None,
               dtype: Optional[torch.dtype] = None, eps: float = 1e-6) -> torch.Tensor:
    """RMS norm of a stream x (B, C) into the first block's input.

    Args:
        weight: (C,) or None; heads: the result is (heads, B, C / heads), or (B, C) where None;
        dtype: of the result (the weight's, or x's without a weight); x may be fp32 beside a 16-bit one.
    """
    dtype = dtype or (weight.dtype if weight is not None else x.dtype)
    if _fast is not None and dtype in _DTYPES and heads != 0:  # tensors that need no copies and no error: else None
        r = _fast.join(x, None, None, None, weight, 1.0, True, eps, heads or 0, _DTYPES[dtype])
        if r is not None:
            return r[1]
    if _through_function(x, weight):
        return BlockJoinFunction.apply(x, None, None, None, weight, 1.0, True, True, eps, heads, dtype)[1]
    return _join_fwd(x, None, None, None, 1.0, weight, True, True, eps, heads, dtype, False)[1]


@torch.compiler.disable
def block_join(residual: torch.Tensor, o: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: float = 1.0, *, pre_weight: Optional[torch.Tensor] = None,
               post: bool = True, pre: bool = True, eps: float = 1e-6):
    """(residual', y) of a block's output and its residual stream; y is None with pre=False.

    Args:
        residual: (B, C); o: (H, B, D) with H D = C, or (B, C); post_weight, pre_weight: (C,) or None;
        gate: (C,) or (G, C) with B % G == 0, or None; scale: a number; post=False joins o without its
        norm; pre=False leaves y out.
    """
    if _fast is not None and pre and o is not None:  # as in block_norm
        r = _fast.join(residual, o, post_weight, gate, pre_weight, scale, post, eps, 0, 0)
        if r is not None:
            return r
    if _through_function(residual, o, post_weight, gate, pre_weight):
        return BlockJoinFunction.apply(residual, o, post_weight, gate, pre_weight, scale, post, pre, eps, None, None)
    return _join_fwd(residual, o, post_weight, gate, scale, pre_weight, post, pre, eps, None, None, False)[:2]
