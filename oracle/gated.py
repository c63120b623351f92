"""The gated MLP and its gradients in 64 bits, with elementwise error bounds (test infrastructure only).

    G = X Wg, U = X Wu, a = act(G), h = a U, O = h W2
    dH = dO W2^T, dG = dH U act'(G), dU = dH a
    dX = dG Wg^T + dU Wu^T, dWg = X^T dG, dWu = X^T dU, dW2 = h^T dO

A kernel that sums in fp32 and rounds h, dG, dU and every result to the io type (unit roundoff u) is
off by at most
    u |h| |W2| + u |O|                          for O, and likewise for the gradients,
plus what fp32 sums add: a product sum of n terms is off by at most n 2^-24 sum |terms|, which `_D32`
carries through act and the later products with first-order terms only (everything is positive, so the
bound holds whatever the order of the sums).
"""
from __future__ import annotations

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def act64(name, z):
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if name == "leaky_relu":
        p = z > 0
        return torch.where(p, z, 0.01 * z), torch.where(p, 1.0, 0.01).to(z.dtype)
    return z, torch.ones_like(z)


def gated64(x, wg, wu, w2, do, act):
    """The five results and, for each, (rounded, summed): with unit roundoff u and results R, a kernel's
    error is at most  u (rounded + |R|) + summed."""
    x, wg, wu, w2, do = (t.double().cpu() for t in (x, wg, wu, w2, do))
    t = lambda m: m.transpose(1, 2)  # noqa: E731
    B, D, E = x.shape[1], x.shape[2], wg.shape[2]
    g, u = x @ wg, x @ wu
    a, f = act64(act, g)
    h = a * u
    dh = do @ t(w2)
    dg, du = dh * u * f, dh * a
    res = (h @ w2, dg @ t(wg) + du @ t(wu), t(x) @ dg, t(x) @ du, t(h) @ do)

    e32 = 2.0 ** -24
    n = lambda k: (k + 8) * e32  # noqa: E731  (a sum of k terms, and a few roundings beside it)
    ax, ag, au, a2, ado = x.abs(), wg.abs(), wu.abs(), w2.abs(), do.abs()
    eg, eu, eh = n(D) * (ax @ ag), n(D) * (ax @ au), n(D) * (ado @ t(a2))  # errors of g, u, dh
    # act, act' move by at most 1.1 and 0.6 per unit of g; leaky_relu's act' jumps where g may change sign
    ea = 1.1 * eg + 8 * e32 * a.abs()
    ef = (0.99 * (g.abs() <= eg).double() if act == "leaky_relu" else 0.6 * eg) + 8 * e32
    e_h = ea * u.abs() + a.abs() * eu + 4 * e32 * h.abs()
    e_dg = eh * (u * f).abs() + dh.abs() * (eu * f.abs() + u.abs() * ef) + 4 * e32 * dg.abs()
    e_du = eh * a.abs() + dh.abs() * ea + 4 * e32 * du.abs()
    h, dg, du = h.abs(), dg.abs(), du.abs()
    rounded = (h @ a2, dg @ t(ag) + du @ t(au), t(ax) @ dg, t(ax) @ du, t(h) @ ado)
    carried = (e_h @ a2, e_dg @ t(ag) + e_du @ t(au), t(ax) @ e_dg, t(ax) @ e_du, t(e_h) @ ado)
    terms = (E, 2 * E, B, B, B)
    # (1.01: products of two of these errors)
    summed = [1.01 * (c + n(k) * r) for c, r, k in zip(carried, rounded, terms)]
    return res, list(zip(rounded, summed))


def excess(got, want, bound, dtype):
    """How far `got` is beyond its bound, as a multiple of it (at most 1 is within)."""
    rounded, summed = bound
    u = UNIT[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134  # half the smallest subnormal
    stage = u if dtype != torch.float32 else 0.0  # fp32 io rounds no operand
    limit = 1.01 * stage * rounded + 1.01 * u * (want.abs() + stage * rounded) + summed + tiny
    if dtype == torch.float16:  # operands below the smallest normal number are rounded to its subnormals
        limit = limit + 2.0 ** -25 * (rounded > 0).double() * 4096
    got = got.detach().double().cpu()
    if got.numel() == 0:
        return 0.0
    assert torch.isfinite(got).all()
    return ((got - want).abs() / limit).max().item()
