"""What the bounds of a Muon step (oracle/muon.py) can tell apart, with the momenta as they are stored: a step that leaves the
weights, the other rule of momentum, a step fewer, the other sign, for every mix of types."""
import ctypes
import itertools

import pytest
import torch

from flashmlp_amd import _lib
from oracle import muon as om

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
LR = 0.02


@pytest.mark.parametrize("types", list(itertools.product((BF, HF, FL), repeat=3)))
@pytest.mark.parametrize("shape", [(64, 100), (5, 16, 7), (100, 3), (2, 128, 130), (2, 40, 70)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_the_bound_rejects_other_steps(shape, types, nesterov):
    gen = torch.Generator().manual_seed(7)
    w = torch.randn(shape, generator=gen).div(shape[-2] ** 0.5).to(types[0])
    g = torch.randn(shape, generator=gen).to(types[1])
    m = (0.5 * torch.randn(shape, generator=gen)).to(types[2])
    kept = (0.95 * m.double() + 0.05 * g.double()).float().to(types[2])
    kw = dict(nesterov=nesterov, kept=kept)
    ref, tol = om.step64(w, g, m, LR, **kw)["w"]

    def seen(other):
        return ((other.to(types[0]).double() - ref).abs() > 1.01 * tol + 2.0 ** -25).any()

    assert not seen(ref)
    assert seen(w.double())
    assert seen(2 * w.double() - ref)
    assert seen(om.step64(w, g, m, LR, nesterov=not nesterov, kept=kept)["w"][0])
    assert seen(om.step64(w, g, m, LR, steps=4, **kw)["w"][0])


def test_largest_values_of_the_steps():
    """against many points of the interval"""
    for c in (om.COEFFICIENTS, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, 0.0, 0.0), (8.28721, -23.5959, 17.3004), (3.0, -9.0, 6.0)):
        r = 1.0
        for q, slope, after in om.polynomials(4, [c] * 4):
            x = torch.linspace(0, r ** 0.5, 20001, dtype=torch.float64)
            l, (a, b, d) = x * x, c
            v = a + l * (b + l * d)
            for got, want in ((q, v.abs()), (slope, (a + l * (3 * b + l * 5 * d)).abs()), (after, l * v * v)):
                assert want.max().item() * (1 - 1e-12) <= got <= want.max().item() * (1 + 1e-6) + 1e-9
            r = min(after, 100.0)
            if after > 100:
                break


@pytest.mark.parametrize("coefficients,steps,step", [((4.0, -4.0, 1.5), 5, 2), ((0.0, 0.0, 300.0), 2, 0), ((50.0, 0.0, 0.0), 3, 1),
                                                     ((1e4, 1e4, 1e4), 2, 0), ((3e4, 0.0, 0.0), 1, None)])
def test_refusal_of_coefficients(coefficients, steps, step):
    """whose values the steps' terms would not hold (300^2, 50^4 and 3e8 are above 2^16); on the host, as calls for no matrices show.
    step None: beyond the limit of a coefficient"""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    L = _lib.lib()
    abc = (ctypes.c_float * (3 * steps))(*coefficients * steps)
    for dtype in (0, 1, 2):
        assert L.fmlp_orthogonalize(None, None, 0, 8, 9, dtype, steps, abc, 1e-7, None, 0, None) != 0
        assert "coefficient" in L.fmlp_last_error().decode()
    t = (_lib.MuonTensor * 1)(_lib.MuonTensor(4096, 1 << 20, 2 << 20, 2, 8, 9, 2, 2, 2, 1.0))
    assert L.fmlp_muon_step(1, t, 0.1, 0.9, 1, 0.0, steps, abc, 1e-7, None, 0, None) != 0
    message = L.fmlp_last_error().decode()
    assert "coefficient" in message and (step is None or f"step {step}" in message)


def test_sizes_past_64_bits_are_refused():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    L = _lib.lib()
    abc = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    for H, R, C in ((1 << 62, 2, 2), (1 << 30, 256, 1 << 28), ((1 << 63) - 1, 1, 1), (1 << 40, 1, 1 << 30), (1, 200, 1 << 30)):
        assert L.fmlp_orthogonalize(4096, 1 << 20, H, R, C, 2, 1, abc, 1e-7, None, 0, None) == 1
        assert "too large" in L.fmlp_last_error().decode()
        assert L.fmlp_orthogonalize_workspace_bytes(H, R, C, 2, 1) == 0
