"""How near the steps on Gram matrices come to the products of the matrices themselves: singular values that fall evenly in their
logarithm over one to five decades, noise around a low rank, the usual coefficients and a schedule that begins steeply.

An fp32 result is at most four times as far off, in norm, as the formula's products in fp32: the operands of the products are held
to 2^-22, those in fp32 to 2^-24, and there are as many."""
import ctypes

import pytest
import torch

from flashmlp_amd import _lib, muon_step, orthogonalize
from oracle import muon as om

pytestmark = pytest.mark.gpu
SCHEDULE = [(8.28721, -23.5959, 17.3004), (4.10706, -2.94785, 0.5448), (3.94869, -2.9089, 0.5518), (3.3184, -2.4885, 0.5100),
            (2.3007, -1.6689, 0.4188)]


def matrices(H, n, e, decades, seed):
    g = torch.Generator().manual_seed(seed)
    if decades is None:
        return torch.randn(H, n, 8, generator=g) @ torch.randn(H, 8, e, generator=g) / 8 ** 0.5 + 0.5 * torch.randn(H, n, e, generator=g)
    q = torch.linalg.qr(torch.randn(H, n, n, generator=g, dtype=torch.float64))[0]
    r = torch.linalg.qr(torch.randn(H, e, n, generator=g, dtype=torch.float64))[0]
    return ((q * 10.0 ** (-decades * torch.arange(n, dtype=torch.float64) / n)) @ r.mT).float()


def products(x, coefficients):
    """the formula in x's type"""
    y = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    for a, b, c in om.triples(coefficients, 5):
        t = y @ y.mT
        y = a * y + (b * t + c * (t @ t)) @ y
    return y


@pytest.mark.parametrize("coefficients", [om.COEFFICIENTS, SCHEDULE])
@pytest.mark.parametrize("decades", [None, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,e", [(24, 60), (64, 64), (64, 500), (128, 130), (128, 256), (128, 1024), (200, 256), (256, 256), (256, 1024)])
def test_full_precision(n, e, decades, coefficients):
    x = matrices(2, n, e, decades, n + e)
    want = om.orthogonal64(x, 5, coefficients)
    off = (products(x, coefficients).double() - want).norm().item()
    # two matrices in parts; the same two among as many as take a workgroup each
    for stack in (x, x.repeat(200, 1, 1)) if n <= 128 else (x,):
        for tall in (False, True):
            y = (stack.mT.contiguous() if tall else stack).cuda()
            o = orthogonalize(y, coefficients=coefficients)[:2].double().cpu()
            assert ((o.mT if tall else o) - want).norm().item() <= 4 * off, (len(stack), tall)


@pytest.mark.parametrize("coefficients", [om.COEFFICIENTS, SCHEDULE])
@pytest.mark.parametrize("decades", [None, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,e", [(24, 60), (64, 64), (64, 500), (128, 130), (128, 1024), (256, 256), (256, 1024)])
def test_updates_and_16_bit_results(n, e, decades, coefficients):
    """The update that weights take, from weights of zero at lr = 1, and a 16-bit result: off in norm by 2^-11 at most (the
    4e-4 that are documented), and a result's rounding"""
    x = matrices(2, n, e, decades, n + e)
    w, m = (torch.zeros(x.shape, device="cuda") for _ in range(2))
    muon_step(w, x.cuda(), m, 1.0, momentum=0.0, nesterov=False, scale=1.0, coefficients=coefficients)
    want = om.orthogonal64(x, 5, coefficients)
    assert (w.double().cpu() + want).norm() <= 2.0 ** -11 * want.norm()
    for dtype in (torch.bfloat16, torch.float16):
        y = x.to(dtype)
        want = om.orthogonal64(y, 5, coefficients)
        o = orthogonalize(y.cuda(), coefficients=coefficients).double().cpu()
        assert (o - want).norm() <= (want.to(dtype).double() - want).norm() + 2.0 ** -11 * want.norm()


def test_workspaces():
    """What a call with these coefficients needs, which a call runs with and one of less refuses; without coefficients what any
    need. Coefficients that take more Gram matrices hold the matrices in fp32 in between."""
    L = _lib.lib()
    steps, H, R, C = 5, 3, 64, 100
    usual, steep = ((ctypes.c_float * (3 * steps))(*[float(v) for c in om.triples(k, steps) for v in c]) for k in (om.COEFFICIENTS, SCHEDULE))
    fp32 = H * R * C * 4
    x = matrices(H, R, C, 2, 0).bfloat16().cuda()
    w, m = (torch.zeros(x.shape, device="cuda") for _ in range(2))
    stream = torch.cuda.current_stream().cuda_stream
    t = (_lib.MuonTensor * 1)(_lib.MuonTensor(w.data_ptr(), x.data_ptr(), m.data_ptr(), H, R, C, 2, 1, 2, 1.0))

    def ortho(abc, ws, n):
        return L.fmlp_orthogonalize(x.data_ptr(), out.data_ptr(), H, R, C, 1, steps, abc, 1e-7, ws.data_ptr(), n, stream)

    def muon(abc, ws, n):
        return L.fmlp_muon_step(1, t, 1.0, 0.0, 0, 0.0, steps, abc, 1e-7, ws.data_ptr(), n, stream)

    out = torch.empty_like(x)
    for call, query, any_ in ((ortho, lambda abc: L.fmlp_orthogonalize_workspace_bytes_for(H, R, C, 1, steps, abc),
                               L.fmlp_orthogonalize_workspace_bytes(H, R, C, 1, steps)),
                              (muon, lambda abc: L.fmlp_muon_workspace_bytes_for(1, t, steps, abc),
                               L.fmlp_muon_workspace_bytes(1, t, steps))):
        assert 0 < query(usual) == query(steep) - fp32 and any_ == query(steep)
        for abc in (usual, steep):
            n = query(abc)
            ws = torch.zeros(n + 16, dtype=torch.uint8, device="cuda")
            ws[n:] = 7
            assert call(abc, ws, n - 1) == 4 and call(abc, ws, n) == 0
            torch.cuda.synchronize()
            assert (ws[n:] == 7).all()
    assert torch.equal(out, orthogonalize(x, coefficients=SCHEDULE))
    for abc in (None, (ctypes.c_float * 15)(*[float("nan")] * 15)):
        assert (L.fmlp_orthogonalize_workspace_bytes_for(H, R, C, 1, steps, abc) > 0) == (abc is None)
