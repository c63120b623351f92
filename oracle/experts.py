"""Routing, the sort by expert and the copies between tokens and experts' rows in 64 bits, with elementwise error bounds
(test infrastructure only; CPU tensors).

    p = softmax(l), the k largest (ties: lowest index; -infinity is never chosen); w = p, or p / sum of the k
    dl = w (dw - sum w dw) at the chosen, or p ([chosen] dw - sum over the chosen of p dw)
    slot(t, j) = e capacity + number of earlier choices of e, or -1

The kernels work in fp32: e^(l - top) as 2^((l - top) log2 e) has the difference's rounding (2^-24 |d|), the product's and its
constant's (1.5 2^-24 |d|) and the exponential's own (2^-23); sums of n terms n 2^-24 relative.
"""
from __future__ import annotations

import torch

from .gated import UNIT

E = 2.0 ** -24


def route64(logits, k, normalize, dw=None):
    """(weights, their bound, experts, dlogits, its bound); the last two None without dw"""
    l = logits.double()
    T, N = l.shape
    experts = torch.empty(T, k, dtype=torch.int64)
    for t in range(T):
        row = l[t].tolist()
        order = sorted((i for i in range(N) if row[i] != float("-inf")), key=lambda i: (-row[i], i))[:k]
        experts[t] = torch.tensor(order + [-1] * (k - len(order)))
    chosen = experts >= 0
    top = l.amax(1, keepdim=True) if T else l[:, :1]
    d = torch.where(torch.isinf(l), torch.zeros_like(l), l - top)
    e = torch.where(torch.isinf(l), torch.zeros_like(l), torch.exp(d))
    at = experts.clamp(min=0)
    es = torch.where(chosen, e.gather(1, at), torch.zeros(T, k, dtype=torch.float64))
    total = (es if normalize else e).sum(1, keepdim=True)
    w = torch.where(chosen, es / total, torch.zeros_like(es))
    rel_e = E * (2.5 * d.abs() + 3)  # of an exponential
    rel_sum = ((es * torch.where(chosen, rel_e.gather(1, at), 0.0)).sum(1, keepdim=True) if normalize
               else (e * rel_e).sum(1, keepdim=True)) / total.clamp(min=1e-300) + (N + 3) * E
    rel = torch.where(chosen, rel_e.gather(1, at), 0.0) + rel_sum
    bw = 1.01 * rel * w + 2.0 ** -120
    if dw is None:
        return w, bw, experts, None, None
    dw = torch.where(chosen, dw.double(), torch.zeros(T, k, dtype=torch.float64))
    terms = w * dw
    inner = terms.sum(1, keepdim=True)
    b_inner = (bw * dw.abs()).sum(1, keepdim=True) + (k + 2) * E * terms.abs().sum(1, keepdim=True)
    dl, b = torch.zeros_like(l), torch.zeros_like(l)
    if normalize:
        v = w * (dw - inner)
        bv = bw * (dw - inner).abs() + w * (b_inner + 3 * E * (dw.abs() + inner.abs()))
        for j in range(k):
            rows = chosen[:, j]
            dl[rows, experts[rows, j]] += v[rows, j]
            b[rows, experts[rows, j]] += bv[rows, j]
    else:
        p = e / total.clamp(min=1e-300)
        dl = -p * inner
        b = p * (rel_e + rel_sum) * inner.abs() + p * (b_inner + 4 * E * inner.abs())
        for j in range(k):
            rows = chosen[:, j]
            dl[rows, experts[rows, j]] += terms[rows, j]
            b[rows, experts[rows, j]] += (bw * dw.abs() + 3 * E * terms.abs())[rows, j]
    return w, bw, experts, dl, UNIT[logits.dtype] * dl.abs() + 1.01 * b + (2.0 ** -25 if logits.dtype == torch.float16 else 2.0 ** -120)


def plan(experts, N, capacity):
    """(slots, counts) by counting in the choices' order"""
    T, k = experts.shape
    slots, counts = torch.full((T, k), -1, dtype=torch.int32), [0] * N
    for t, row in enumerate(experts.tolist()):
        for j, e in enumerate(row):
            if 0 <= e < N:
                if counts[e] < capacity:
                    slots[t, j] = e * capacity + counts[e]
                counts[e] += 1
    return slots, torch.tensor(counts, dtype=torch.int32)


def gather64(rows, slots, weights=None):
    """(o, its bound)"""
    N, capacity, D = rows.shape
    flat = rows.double().reshape(-1, D)
    there = (slots >= 0)[..., None]
    t = torch.zeros(*slots.shape, D, dtype=torch.float64)
    if flat.numel():
        t = torch.where(there, flat[slots.long().clamp(min=0)], t)
    w = torch.ones(slots.shape, dtype=torch.float64) if weights is None else weights.double()
    t = torch.where(there, t * w[..., None], torch.zeros_like(t))
    o = t.sum(1)
    k = slots.shape[1]
    return o, UNIT[rows.dtype] * o.abs() + 1.01 * (k + 1) * E * t.abs().sum(1) + (2.0 ** -25 if rows.dtype == torch.float16 else 2.0 ** -140)


def scatter64(x, slots, N, capacity, weights=None):
    """(rows, their bound): rows[slot] = w x, zeros elsewhere"""
    D = x.shape[1]
    rows = torch.zeros(N * capacity, D, dtype=torch.float64)
    for j in range(slots.shape[1]):
        there = slots[:, j] >= 0
        v = x[there].double()
        if weights is not None:
            v = v * weights[there, j].double()[:, None]
        rows[slots[there, j].long()] = v
    u = 0.0 if weights is None else UNIT[x.dtype] * 1.01 + E
    tiny = 0.0 if weights is None else 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -134
    return rows.view(N, capacity, D), u * rows.abs().view(N, capacity, D) + tiny


def dot64(rows, x, slots):
    """(dw, its bound): <rows[slot], x>, 0 without a slot"""
    N, capacity, D = rows.shape
    flat = rows.double().reshape(-1, D)
    there = (slots >= 0)[..., None]
    r = torch.zeros(*slots.shape, D, dtype=torch.float64)
    if flat.numel():
        r = torch.where(there, flat[slots.long().clamp(min=0)], r)
    t = torch.where(there, r * x.double()[:, None], torch.zeros_like(r))
    return t.sum(2), 1.01 * (D + 8) * E * t.abs().sum(2) + 2.0 ** -140


def over(got, want, bound):
    """the largest excess over the bound, in bounds"""
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    if got.numel() == 0:
        return 0.0
    assert torch.isfinite(got).all()
    d = (got - want).abs()
    return torch.where(d == 0, torch.zeros_like(d), d / bound.clamp(min=1e-300)).max().item()
