"""Workspaces of many matrices with small sides above 128, which go through them in batches: bounded, and each batch its own results."""
import ctypes

import pytest
import torch

from flashmlp_amd import _lib, muon_step, orthogonalize
from oracle import muon as om
from oracle.gated import UNIT

pytestmark = pytest.mark.gpu
BF, FL = torch.bfloat16, torch.float32


def test_bound():
    L = _lib.lib()
    abc = (ctypes.c_float * 15)(*[float(v) for v in om.COEFFICIENTS] * 5)
    few, many = (L.fmlp_orthogonalize_workspace_bytes_for(H, 256, 256, 1, 5, abc) for H in (1024, 12288))
    assert 0 < many <= few < 1 << 30
    stacks = (_lib.MuonTensor * 12)(*[_lib.MuonTensor(None, None, None, 1024, 256, 300, 2, 1, 2, 1.0)] * 12)
    assert 0 < L.fmlp_muon_workspace_bytes_for(12, stacks, 5, abc) < 1 << 30


@pytest.mark.parametrize("dtype,steps", [(BF, 5), (FL, 5), (BF, 6)])
@pytest.mark.parametrize("tall", [False, True])
def test_orthogonalize(dtype, steps, tall):
    H = 1101  # two batches: of 551 and 550
    x = torch.randn(H, 136, 150, generator=torch.Generator().manual_seed(0)).to(dtype)
    x = x.mT.contiguous() if tall else x
    buf = torch.full((x.numel() + 128,), 7.0, dtype=dtype, device="cuda")
    out = buf[64:-64].view(x.shape)
    orthogonalize(x.cuda(), out=out, steps=steps)
    assert (buf[:64] == 7).all() and (buf[-64:] == 7).all()
    at = [0, 1, 549, 550, 551, 552, H - 2, H - 1]
    want = om.orthogonal64(x[at], steps)
    tol = UNIT[dtype] * want.abs() + 1.01 * om.bound(x[at], steps, full=dtype == FL)
    assert ((out[at].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("steps", [5, 6])
def test_muon_step_across_stacks(steps):
    """batches end inside a stack and hold parts of several"""
    gen = torch.Generator().manual_seed(1)
    shapes = [(500, 140, 131), (3, 130, 137), (600, 150, 130), (20, 64, 70)]
    w, g, m = ([torch.randn(s, generator=gen) for s in shapes] for _ in range(3))
    g = [t.to(BF) for t in g]
    dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
    muon_step(dw, dg, dm, 0.1, steps=steps)
    for i, s in enumerate(shapes):
        at = sorted({0, 1, s[0] // 2, s[0] - 1, *([48, 49, 50, 51, 52] if i == 2 else [])} & set(range(s[0])))
        want = om.step64(w[i][at], g[i][at], m[i][at], 0.1, steps=steps, kept=dm[i][at].cpu())
        for t, got in (("w", dw[i][at]), ("m", dm[i][at])):
            ref, tol = want[t]
            assert ((got.double().cpu() - ref).abs() <= 1.01 * tol + 2.0 ** -130).all(), (i, t)
