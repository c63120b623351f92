"""The join of a block with its stream and its gradients in 64 bits, with elementwise error bounds (test
infrastructure only).

    n = o ro, ro = 1 / sqrt(mean(o^2) + eps), p = n w_post;  r' = r + s gate p
    m = r' rr, rr = 1 / sqrt(mean(r'^2) + eps);  y = m w_pre
    dm = dy w_pre, dr = dr' + rr (dm - m mean(dm m)), dw_pre = sum dy m
    dp = s gate dr, dgate = sum s dr p, dw_post = sum dp n, dn = dp w_post, do = ro (dn - n mean(dn n))

The kernels work in fp32 (a few roundings of 2^-24 a value, C or B terms a sum) and round the results
(unit roundoff u, the stream's ur); the backward of an fp32 stream, and of any where r is not given, reads r' as it was rounded, so its m is off by up
to ur |m| (stream_rounded); beside the row's mean it is always the rounded one.
"""
from __future__ import annotations

import torch

from .gated import UNIT


def join64(r, o, w_post, gate, w_pre, scale, eps, post, dr2, dy, stream_rounded=True):
    """All arguments on (B, C) rows; o, weights, gate, dr2 and dy may be None. Returns dicts of results and
    of their error bounds: r2, y, dr, do, dw_post, dgate, dw_pre."""
    u = UNIT[(o if o is not None else dy if dy is not None else r).dtype]
    ur = UNIT[r.dtype]
    up = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    r, o, w_post, gate, w_pre, dr2, dy = map(up, (r, o, w_post, gate, w_pre, dr2, dy))
    B, C = r.shape
    e = 2.0 ** -24
    k = (C + 32) * e  # a row's sum and what follows it, relative to the sum of absolute terms
    one = torch.ones(1, C, dtype=torch.float64)
    wq, wp = (one if w is None else w.view(1, C) for w in (w_post, w_pre))
    G = 1 if gate is None else gate.shape[0]
    gt = one if gate is None else gate.repeat_interleave(B // G, 0) if B else gate[:0]
    res, bound = {}, {}
    if o is not None:
        ro = torch.rsqrt(o.pow(2).mean(1, keepdim=True) + eps) if post else torch.ones(B, 1, dtype=torch.float64)
        n = o * ro
        p = n * wq
        r2 = r + scale * gt * p
        er2 = k * (r.abs() + (scale * gt * p).abs())
    else:
        r2, er2 = r, torch.zeros_like(r)
    res["r2"], bound["r2"] = r2, ur * r2.abs() + er2
    rr = torch.rsqrt(r2.pow(2).mean(1, keepdim=True) + eps)
    m = r2 * rr
    # er2 moves m by rr er2 and, through rr, by at most |m| rms(er2) rr
    em = rr * er2 + m.abs() * rr * er2.pow(2).mean(1, keepdim=True).sqrt() + 2 * k * m.abs()
    res["y"] = m * wp
    bound["y"] = u * res["y"].abs() + 1.01 * em * wp.abs() + k * res["y"].abs()
    if dr2 is None and dy is None:
        return res, bound
    zero = torch.zeros_like(r)
    d2 = zero if dr2 is None else dr2
    if dy is not None:
        em = em + ur * m.abs() if stream_rounded else em
        dm = dy * wp
        mean, amean = (dm * m).mean(1, keepdim=True), (dm * m).abs().mean(1, keepdim=True)
        dr = d2 + rr * (dm - m * mean)
        emean = (dm.abs() * em).mean(1, keepdim=True) + k * amean
        edr = rr * ((em + ur * m.abs()) * mean.abs() + m.abs() * emean) + 4 * k * (d2.abs() + rr * (dm.abs() + m.abs() * amean))
        edr = 1.01 * (edr + rr * er2.pow(2).mean(1, keepdim=True).sqrt() * (dr - d2).abs())
        t = (dy * m).sum(0)
        res["dw_pre"] = t
        bound["dw_pre"] = 1.01 * (u * t.abs() + (dy.abs() * em).sum(0) + (B + 32) * e * (dy * m).abs().sum(0))
    else:
        dr, edr = d2, k * d2.abs()
    res["dr"], bound["dr"] = dr, ur * dr.abs() + edr
    if o is not None:
        sd, esd = scale * dr, abs(scale) * edr + e * (scale * dr).abs()
        t, et = sd * p, esd * p.abs() + 4 * k * (sd * p).abs()
        fold = lambda v: v.reshape(G, -1, C).sum(1)  # noqa: E731
        res["dgate"] = fold(t)
        bound["dgate"] = 1.01 * (u * fold(t).abs() + fold(et) + (B + 32) * e * fold(t.abs()))
        dp, edp = sd * gt, esd * gt.abs() + k * (sd * gt).abs()
        t, et = dp * n, edp * n.abs() + 4 * k * (dp * n).abs()
        res["dw_post"] = t.sum(0)
        bound["dw_post"] = 1.01 * (u * t.sum(0).abs() + et.sum(0) + (B + 32) * e * t.abs().sum(0))
        dn, edn = dp * wq, edp * wq.abs() + k * (dp * wq).abs()
        if post:
            mean, amean = (dn * n).mean(1, keepdim=True), (dn * n).abs().mean(1, keepdim=True)
            do = ro * (dn - n * mean)
            edo = ro * (edn + n.abs() * ((edn * n.abs()).mean(1, keepdim=True) + 4 * k * amean)
                        + 4 * k * (dn.abs() + n.abs() * amean))
        else:
            do, edo = dn, edn
        res["do"], bound["do"] = do, u * do.abs() + 1.01 * edo
    return res, bound


def excess(got, want, bound, dtype):
    """How far `got` is beyond its bound, as a multiple of it."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    got = got.detach().double().cpu().reshape(want.shape)
    if got.numel() == 0:
        return 0.0
    assert torch.isfinite(got).all()
    return ((got - want).abs() / (1.01 * bound + tiny)).max().item()
