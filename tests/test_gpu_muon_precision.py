"""How near the steps on Gram matrices come to the products of the matrices themselves: singular values that fall evenly in their
logarithm over one to five decades, noise around a low rank, the usual coefficients and a schedule that begins steeply.

An fp32 result is at most four times as far off, in norm, as the formula's products in fp32: the operands of the products are held
to 2^-22, those in fp32 to 2^-24, and there are as many."""
import pytest
import torch

from flashmlp_amd import orthogonalize
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
