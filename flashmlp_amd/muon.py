"""Stacks of matrices orthogonalised by Newton-Schulz products, and the Muon optimizer's step around it.

    orthogonalize(x, *, steps=5, coefficients=(3.4445, -4.775, 2.0315), eps=1e-7, out=None) -> like x
    muon_step(params, grads, momenta, lr, *, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, ...)

    X = u / (|u| + eps),  `steps` times  X <- a X + b (X X^T) X + c (X X^T)^2 X        |u| the Frobenius norm
    m = momentum m + (1 - momentum) g,  u = (1 - momentum) g + momentum m (nesterov) or m
    w = (1 - lr weight_decay) w - lr scale X

Every matrix of a stack (..., R, C) stands by itself, as the heads of the MLPs' weights (H, D, E) and (H, E, D) do; min(R, C) <=
256, the other side is any. torch.optim.Muon, whose momentum, decoupled decay and scale these are, takes single matrices
only, decays by 0.1 by default where this does not, and divides by the norm or eps, whichever is more, where this divides by their
sum, which differs for gradients near eps alone. fp16, bf16 or fp32; weights, gradients and momenta each of its own type, so that
gradients clipped into full precision buffers (clip_grads) or 16-bit ones go with full precision weights. Calls are asynchronous on
torch's current stream.

The steps are taken on the smaller side's Gram matrix in 32 bits. 16-bit results, and the update that weights take, are off by up
to 4e-4 in norm and 1.4e-3 in directions whose singular values are far below the largest (measured with the usual coefficients; a
bf16 result's rounding is 1.7e-3 and 3e-3, an fp16 one's an eighth of that); an fp32 `orthogonalize` is as exact as the formula's products in fp32. |u|^2 has to be
within fp32's range; coefficients under which singular values up to one may grow beyond 2^8 in between are refused.
"""
from __future__ import annotations

import ctypes
import math
import numbers
from typing import Iterable, Optional, Sequence, Tuple, Union

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from .block import _input
from .flashmlp import _DTYPES, _alloc_ws, _fast, _ptr
from .gated import _not_traced, _On

_COEFFICIENTS = (3.4445, -4.775, 2.0315)
_MAX_STEPS = 10


def _coefficients(coefficients, steps):
    """a, b, c of every step as the library takes them"""
    if not 1 <= steps <= _MAX_STEPS:
        raise ValueError(f"steps must be 1 to {_MAX_STEPS}, got {steps}")
    c = list(coefficients)
    if len(c) == 3 and all(isinstance(v, numbers.Real) for v in c):
        c = [c] * steps
    if len(c) != steps or any(len(v) != 3 for v in c):
        raise ValueError(f"coefficients must be three numbers, or three for each of {steps} steps")
    return (ctypes.c_float * (3 * steps))(*(float(v) for s in c for v in s))


def _stack(t: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(H, R, C)"""
    if t.dim() < 2:
        raise ValueError(f"{what} must be matrices or stacks of them, got {t.dim()} dimensions")
    R, C = t.shape[-2:]
    return math.prod(t.shape[:-2]), R, C


def _check(t: torch.Tensor, what: str, dev=None):
    if t.device.type != "cuda":
        raise RuntimeError(f"FlashMLP runs on an AMD GPU through HIP; got a tensor on {t.device} (move inputs to 'cuda')")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"all tensors must be on one device ({dev} vs {t.device})")
    if t.dtype not in _DTYPES:
        raise TypeError(f"FlashMLP supports float16, bfloat16 and float32 {what}, got {t.dtype}")
    if t.layout != torch.strided:
        raise TypeError(f"{what} must be dense tensors, got {t.layout}")
    _input(t)  # (memory of its own)
    if unpack_dual(t).tangent is not None:
        raise RuntimeError(f"orthogonalised updates have no forward mode (jvp): {what} with a tangent")


def _number(v, name):
    # (a tensor would be read on the host)
    if not isinstance(v, numbers.Real):
        raise TypeError(f"{name} must be a number, got {type(v).__name__}")
    return float(v)


def _plain(t: torch.Tensor) -> bool:
    return t.is_contiguous() and not t.is_neg()


def _box(t: torch.Tensor):
    """({stride: size} in bytes, largest first), None where two elements may be in one place"""
    dims = [(s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if n > 1] + [(1, t.element_size())]
    dims.sort(reverse=True)
    if any(s * n > outer for (outer, _), (s, n) in zip(dims, dims[1:])) or dims[-1][0] == 0:
        return None
    return dict(dims)


def _refuse_overlap(written):
    """Raises where two of the tensors may share memory, or two elements of one. A tensor's bytes are numbers whose digits
    have its strides as bases; two tensors are apart where a digit is, as long as all digits stay within the bases."""
    ts = sorted((t for t in written if t.numel()), key=lambda t: t.data_ptr())
    boxes = [_box(t) for t in ts]
    for i, (t, a) in enumerate(zip(ts, boxes)):
        end = 0 if a is None else t.data_ptr() + 1 + sum(s * (n - 1) for s, n in a.items())
        for u, b in zip(ts[i + 1:], boxes[i + 1:]):
            if a is None or b is None or u.data_ptr() >= end:
                break
            rest, outer, apart = u.data_ptr() - t.data_ptr(), math.inf, False
            for s in sorted({*a, *b}, reverse=True):
                digit, rest = divmod(rest, s)
                if max(a.get(s, 1), digit + b.get(s, 1)) * s > outer:
                    apart = False
                    break
                outer, apart = s, apart or digit >= a.get(s, 1)
            if not apart:
                a = None
        if a is None:
            raise RuntimeError("parameters and momenta must not overlap, nor may one's elements share a place")


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients: Sequence = _COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The matrices of x (..., R, C) orthogonalised: singular values brought towards one, singular vectors kept.

    Args:
        steps: 1 to 10; coefficients: (a, b, c), or one such triple for each step;
        out: of x's shape and type, or x itself.
    No gradient is kept; forward mode is refused.
    """
    if _fast is not None:  # dense tensors on one GPU and no error: else None
        r = _fast.orthogonalize(x, out, steps, coefficients, eps)
        if r is not None:
            return out if out is not None else r
    _not_traced("orthogonalize")
    H, R, C = _stack(x, "x")
    abc = _coefficients(coefficients, steps)
    eps = _number(eps, "eps")
    _check(x, "matrices")
    if out is not None:
        _check(out, "outputs", x.device)
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError(f"out must be {x.dtype} of shape {tuple(x.shape)}, got {out.dtype} of {tuple(out.shape)}")
    same = out is x
    x = x.detach()
    xd = x if _plain(x) else x.resolve_neg().contiguous()
    o = out if out is not None and _plain(out) else xd if same else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    L = _lib.lib()
    with _On(x.get_device()) as stream:
        n = L.fmlp_orthogonalize_workspace_bytes_for(H, R, C, _DTYPES[x.dtype], steps, abc)
        ws = _alloc_ws(n, x.device)
        st = L.fmlp_orthogonalize(xd.data_ptr(), o.data_ptr(), H, R, C, _DTYPES[x.dtype], steps, abc, eps, _ptr(ws), n, stream)
    _lib.check(st, "orthogonalisation")
    if out is None:
        return o
    if o is out:
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)
    else:
        with torch.no_grad():
            out.copy_(o)
    return out


def muon_step(params: Union[torch.Tensor, Iterable[torch.Tensor]], grads: Union[torch.Tensor, Iterable[torch.Tensor]],
              momenta: Union[torch.Tensor, Iterable[torch.Tensor]], lr: float, *, momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, scale: Optional[float] = None, steps: int = 5,
              coefficients: Sequence = _COEFFICIENTS, eps: float = 1e-7) -> None:
    """One step of Muon for many stacks of matrices, in place.

    Args:
        params, grads, momenta: tensors, or as many of each, of equal shapes (..., R, C); momenta start as zeros;
        weight_decay: decoupled: w (1 - lr weight_decay);
        scale: of the update; None: sqrt(max(1, R / C)) (0.2 * sqrt(max(R, C)) has the rms of AdamW's updates);
        steps, coefficients, eps: as orthogonalize's.
    A tensor that is in the call twice, or overlaps another one that is written, is refused.
    """
    params, grads, momenta = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (params, grads, momenta))
    if _fast is not None and _fast.muon_step(params, grads, momenta, lr, momentum, nesterov, weight_decay, scale, steps, coefficients,
                                             eps):  # as in orthogonalize
        return
    _not_traced("muon_step")
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients, {len(momenta)} momenta")
    lr, momentum, weight_decay, eps = (_number(v, n) for v, n in ((lr, "lr"), (momentum, "momentum"),
                                                                  (weight_decay, "weight_decay"), (eps, "eps")))
    scale = None if scale is None else _number(scale, "scale")
    abc = _coefficients(coefficients, steps)
    if not (lr >= 0 and weight_decay >= 0 and 0 <= momentum <= 1):
        raise ValueError(f"lr and weight_decay must not be negative, momentum within [0, 1]: {lr}, {weight_decay}, {momentum}")
    if not params:
        return
    dev = params[0].device
    calls, held, back = (_lib.MuonTensor * len(params))(), [], []
    for c, w, g, m in zip(calls, params, grads, momenta):
        c.H, c.R, c.C = _stack(w, "parameters")
        if g.shape != w.shape or m.shape != w.shape:
            raise ValueError(f"a parameter of shape {tuple(w.shape)} with a gradient of {tuple(g.shape)}, a momentum of {tuple(m.shape)}")
        for t, what in ((w, "parameters"), (g, "gradients"), (m, "momenta")):
            _check(t, what, dev)
        g = g if _plain(g) else g.detach().resolve_neg().contiguous()
        held.append(g)
        dense = []
        for t in (w, m):  # other layouts through dense tensors
            d = t
            if not _plain(t):
                d = t.detach().resolve_neg().contiguous()
                back.append((t, d))
            dense.append(d)
        held.extend(dense)
        c.w, c.g, c.m = dense[0].data_ptr(), g.data_ptr(), dense[1].data_ptr()
        c.w_dtype, c.g_dtype, c.m_dtype = _DTYPES[w.dtype], _DTYPES[g.dtype], _DTYPES[m.dtype]
        c.scale = math.sqrt(max(1.0, c.R / c.C if c.C else 1.0)) if scale is None else scale
    if back:  # (dense ones alone: the library's own check)
        _refuse_overlap([*params, *momenta])
    L = _lib.lib()
    with _On(dev.index) as stream:
        n = L.fmlp_muon_workspace_bytes_for(len(params), calls, steps, abc)
        ws = _alloc_ws(n, dev)
        st = L.fmlp_muon_step(len(params), calls, lr, momentum, int(nesterov), weight_decay, steps, abc, eps, _ptr(ws), n, stream)
    _lib.check(st, "muon step")
    seen = {id(t) for t, _ in back}
    torch.autograd.graph.increment_version([t for t in (*params, *momenta) if id(t) not in seen and not t.is_inference()])
    with torch.no_grad():
        for t, d in back:
            t.copy_(d)
