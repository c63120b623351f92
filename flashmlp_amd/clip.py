"""Global gradient norm over many tensors, and clipping.

    grad_norm(grads) -> norm
    clip_grads(grads, max_norm, *, out=None) -> (out, norm)
    clip_grad_norm_(parameters, max_norm, *, error_if_nonfinite=False) -> norm

    norm = sqrt(sum of all squares),  out = grad * min(1, max_norm / (norm + 1e-6))

The norm is an fp32 number on the tensors' device; nothing waits for it (error_if_nonfinite does).
Gradients are fp16, bf16 or fp32 in any mix, on one GPU. The squares are summed in 64 bits in a fixed order:
results repeat bitwise, and finite gradients whose norm is beyond fp32, which comes back as infinity, are clipped by
their true norm. A norm that is infinite or NaN because a gradient is scales by 0 or NaN, as
torch.nn.utils.clip_grad_norm_ does.
"""
from __future__ import annotations

import ctypes
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .flashmlp import _DTYPES, _fast
from .gated import _not_traced, _On


def _one_run(t: torch.Tensor) -> bool:
    # the tensor's elements are one run of memory, each once, in whatever order
    if t.is_contiguous():
        return not t.is_neg()
    return torch.ops.aten.is_non_overlapping_and_dense.default(t) and not t.is_neg()


def _check(ts: Sequence[torch.Tensor], what: str):
    dev = ts[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"FlashMLP runs on an AMD GPU through HIP; got a tensor on {dev} (move inputs to 'cuda')")
    for t in ts:
        if t.device != dev:
            raise RuntimeError(f"all {what} must be on one device ({dev} vs {t.device})")
        if t.dtype not in _DTYPES:
            raise TypeError(f"FlashMLP supports float16, bfloat16 and float32 {what}, got {t.dtype}")
        if t.layout != torch.strided:
            raise TypeError(f"{what} must be dense tensors, got {t.layout}")
    return dev


def _pointers(ts):
    return (ctypes.c_void_p * len(ts))(*(t.data_ptr() for t in ts))


def _codes(ts):
    return (ctypes.c_int * len(ts))(*(_DTYPES[t.dtype] for t in ts))


def _run(grads, outs, max_norm, dev):
    L, n = _lib.lib(), len(grads)
    numels = (ctypes.c_int64 * n)(*(g.numel() for g in grads))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with _On(dev.index) as stream:
        size = L.fmlp_clip_workspace_bytes(n, numels)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        if outs is None:
            st = L.fmlp_grad_norm(n, _pointers(grads), numels, _codes(grads), norm.data_ptr(), ws.data_ptr(), size, stream)
        else:
            st = L.fmlp_clip_grads(n, _pointers(grads), _pointers(outs), numels, _codes(grads), _codes(outs), max_norm,
                                   norm.data_ptr(), ws.data_ptr(), size, stream)
    _lib.check(st, "gradient norm" if outs is None else "gradient clipping")
    return norm


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """The L2 norm over all elements of all tensors, a 0-dim fp32 tensor."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    norm = _fast.clip(grads, None, 0.0) if _fast is not None else None  # dense tensors on one GPU: else None
    if norm is not None:
        return norm
    _not_traced("grad_norm")
    dev = _check(grads, "gradients")
    return _run([g if _one_run(g) else g.contiguous() for g in grads], None, 0.0, dev)


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, *,
               out: Optional[Iterable[torch.Tensor]] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """Gradients scaled so that their global norm is at most max_norm.

    Args:
        out: tensors of the gradients' shapes, each of any of the dtypes (an optimizer's full precision
            buffers, say); None clips in place. Outputs that overlap each other, or a gradient that is
            not clipped in place, are refused.
    Returns:
        (out, norm): the clipped tensors and the norm before the clipping.
    """
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(outs)} outputs")
    if not grads:
        return outs, torch.zeros(())
    norm = _fast.clip(grads, outs, max_norm) if _fast is not None else None  # as in grad_norm
    if norm is not None:
        return outs, norm
    _not_traced("clip_grads")
    dev = _check(grads, "gradients")
    if out is not None:
        if _check(outs, "outputs") != dev:
            raise RuntimeError(f"gradients and outputs must be on one device ({dev} vs {outs[0].device})")
        for g, o in zip(grads, outs):
            if g.shape != o.shape:
                raise ValueError(f"output of shape {tuple(o.shape)} for a gradient of {tuple(g.shape)}")
    src, dst, back = [], [], []
    for g, o in zip(grads, outs):
        if _one_run(o) and (g is o or g.stride() == o.stride()):
            src.append(g if g is o or _one_run(g) else g.resolve_neg().contiguous())
            dst.append(o)
            continue
        # other layouts through dense tensors
        s = g.resolve_neg().contiguous()
        d = o if o.is_contiguous() and not o.is_neg() else torch.empty(o.shape, dtype=o.dtype, device=dev)
        src.append(s)
        dst.append(d)
        if d is not o:
            back.append((o, d))
    if len({(o.data_ptr(), o.shape, o.stride()) for o, _ in back}) < len(back):  # (dense ones: the library's own check)
        raise RuntimeError("an output is listed twice: outputs must not overlap")
    norm = _run(src, dst, max_norm, dev)
    # autograd notices a saved tensor that has changed (copy_ below says so itself)
    torch.autograd.graph.increment_version([o for o, d in zip(outs, dst) if d is o and not o.is_inference()])
    with torch.no_grad():
        for o, d in back:
            o.copy_(d)
    return outs, norm


def _memory(t: torch.Tensor):
    # equal for tensors that are one and the same memory
    if t.layout != torch.strided or t.numel() == 0:
        return id(t)
    return t.data_ptr(), t.dtype, t.shape, t.stride()


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, *,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ (L2) on these kernels: clips the parameters' .grad in place and
    returns their norm. A gradient that is there twice (a parameter listed twice, or parameters that share one
    gradient) counts and is scaled once. error_if_nonfinite waits for the norm, and raises before any gradient is
    changed."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = list({_memory(p.grad): p.grad for p in params if p.grad is not None}.values())
    if error_if_nonfinite and grads and not torch.isfinite(grad_norm(grads)):
        raise RuntimeError("the total norm of the gradients is not finite, so it cannot be clipped")
    return clip_grads(grads, max_norm)[1]
