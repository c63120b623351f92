"""Newton-Schulz orthogonalisation and the Muon step in 64 bits, with error bounds (test infrastructure only; CPU tensors).

    X = u / (|u| + eps), `steps` times X <- a X + b (X X^T) X + c (X X^T)^2 X

The kernels take the steps on the Gram matrix G in values of 22 bits and 32-bit sums. An error e of G at an eigenvalue l near 0 grows by
a^2 a step as l itself does, until l is of the size of one: by at most min(a^(2 (s - 1)), 1 / l) over the s steps that one Gram matrix
serves, and changes the polynomial's value there by b / a of it. Rounding gives e = 2^-22 of G's norm, which is at most 1: so a singular
value near one is off by 1.4 2^-22 min(...), and no element by more. Which steps share a Gram matrix: `stages`; in between, the
matrices themselves are rounded to 2^-24, twice (the products and their factor), which what follows multiplies by a a step.
"""
from __future__ import annotations

import math

import torch

from .gated import UNIT

COEFFICIENTS = (3.4445, -4.775, 2.0315)


def triples(coefficients, steps):
    return [tuple(coefficients)] * steps if not isinstance(coefficients[0], (tuple, list)) else [tuple(c) for c in coefficients]


def polynomials(steps, coefficients):
    """(largest |q(l)|, largest |(x q(x^2))'|, largest l q(l)^2) of each step, l = x^2 being the eigenvalues that the steps before
    it leave, [0, 1] at first"""
    r, out = 1.0, []
    for a, b, c in triples(coefficients, steps):
        def among(*inner):
            return [0.0, r] + [l for l in inner if 0 < l < r]

        q = max(abs(a + l * (b + l * c)) for l in among(*([-b / (2 * c)] if c else [])))
        slope = max(abs(a + l * (3 * b + l * 5 * c)) for l in among(*([-3 * b / (10 * c)] if c else [])))
        # (l q^2)' = q (a + 3 b l + 5 c l^2)
        d = max(9 * b * b - 20 * a * c, 0.0) ** 0.5
        roots = [(-3 * b + s * d) / (10 * c) for s in (1, -1)] if c else [-a / (3 * b)] if b else []
        r = max(l * (a + l * (b + l * c)) ** 2 for l in among(*roots))
        out.append((q, slope, r))
    return out


def orthogonal64(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = u.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    for a, b, c in triples(coefficients, steps):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def stages(steps, full, coefficients=COEFFICIENTS):
    """first steps of the Gram matrices, and the number of steps: for fp32 results two (one where the first grows an eigenvalue near 0
    more than 16 times), then one each; for others as few even ones as are of five at most and grow one by 2e4 at most before their last"""
    grow = [q * q for q, _, _ in polynomials(steps, coefficients)]
    if full:
        two = steps > 1 and grow[0] <= 16
        return [0, *range(1 + two, steps + 1)]
    for n in range((steps + 4) // 5, steps + 1):
        at = [(steps * i + n - 1) // n for i in range(n + 1)]
        if all(math.prod(grow[i:j - 1]) <= 2e4 for i, j in zip(at, at[1:])):
            return at


def bound(u, steps=5, coefficients=COEFFICIENTS, full=False):
    """of an element of the unrounded result; full: fp32 results"""
    if u.numel() == 0:
        return 0.0
    x = u.double()
    s = torch.linalg.svdvals(x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=1e-300))
    least = (s.reshape(-1, s.shape[-1])[:, -1].min() ** 2).item()  # the smallest eigenvalue of a G
    most = 1.0
    a = [abs(c[0]) for c in triples(coefficients, steps)]
    total, at = 0.0, stages(steps, full, coefficients)
    for first, end in zip(at, at[1:]):
        grow = 1.0
        for v in a[first:end - 1]:
            grow *= v * v
        total += 1.4 * min(grow, 1 / max(least, 1e-300))
        least = min(1.0, least * grow)
    after = 1.0
    for v in a:
        after *= v
    total += 2 * min(after, 1 / max(least, 1e-300) ** 0.5)
    return 2.0 ** -22 * (total + 8) * most


def step64(w, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
           kept=None):
    """dict of (value, bound) of w and m. kept: the momentum that the step has stored, which the update is made of; without it the
    update's bound allows for every element of it rounded the other way."""
    e = 2.0 ** -24
    wd, gd, md = w.double(), g.double(), m.double()
    m2 = momentum * md + (1 - momentum) * gd
    bm = UNIT[m.dtype] * m2.abs() + 3 * e * (md.abs() + gd.abs())
    k = (m2.to(torch.float32).to(m.dtype) if kept is None else kept).double()
    u = (1 - momentum) * gd + momentum * k if nesterov else k
    R, C = w.shape[-2:]
    s = max(1.0, R / C) ** 0.5 if scale is None else scale
    o = orthogonal64(u, steps, coefficients, eps)
    w2 = (1 - lr * weight_decay) * wd - lr * s * o
    # what moves u, by its place: the stored momentum's rounding, UNIT of it, or u's own two products and their sum
    moves = 2 * bm if kept is None else 3 * e * (gd.abs() + k.abs())
    move = 0.0
    if u.numel():
        norm = torch.linalg.matrix_norm(u, keepdim=True).clamp(min=1e-300)
        if kept is None:
            move = (moves / norm).amax().item() * 485
        else:  # (no element is above the norm; a step enlarges a change by at most its largest slope at the singular values)
            grow = 1.0
            for _, slope, _ in polynomials(steps, coefficients):
                grow *= slope
            move = (torch.linalg.matrix_norm(moves, keepdim=True) / norm).amax().item() * grow
    bw = UNIT[w.dtype] * w2.abs() + 4 * e * (wd.abs() + (lr * s * o).abs()) + lr * s * (bound(u, steps, coefficients) + move)
    return {"w": (w2, bw), "m": (m2, bm)}
