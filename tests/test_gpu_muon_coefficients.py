"""Coefficients other than the usual ones: a schedule whose polynomials end at the interval that the step before leaves and grow fast
behind it, singular values that come out above one, constant and vanishing polynomials."""
import pytest
import torch

from flashmlp_amd import muon_step, orthogonalize
from oracle import muon as om
from oracle.gated import UNIT

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
# each the best fit of one on the singular values that the steps before it leave
SCHEDULE = [(8.28721, -23.5959, 17.3004), (4.10706, -2.94785, 0.5448), (3.94869, -2.9089, 0.5518), (3.3184, -2.4885, 0.5100),
            (2.3007, -1.6689, 0.4188)]


def matrices(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def norm_off(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("shape", [(3, 24, 60), (2, 64, 500), (5, 200, 64), (3, 128, 300), (2, 256, 700), (40, 256, 300), (500, 40, 70),
                                   (300, 128, 150)])
def test_schedule(shape, dtype):
    """off in norm by the result's rounding, and 2^-12"""
    x = matrices(shape, dtype)
    want = om.orthogonal64(x, 5, SCHEDULE)
    assert norm_off(orthogonalize(x.cuda(), coefficients=SCHEDULE), want) <= UNIT[dtype] + 2.0 ** -12


@pytest.mark.parametrize("shape", [(3, 64, 200), (2, 130, 300), (300, 128, 150)])
def test_schedule_of_a_muon_step(shape):
    w, g, m = matrices(shape, FL, 1), matrices(shape, BF, 2), matrices(shape, FL, 3)
    dw, dm = w.cuda(), m.cuda()
    muon_step(dw, g.cuda(), dm, 0.5, coefficients=SCHEDULE)
    want = om.step64(w, g, m, 0.5, coefficients=SCHEDULE, kept=dm.cpu())["w"][0]
    # (weights of the size of one, an update of 0.5 times at most 2^-12 of its norm, and the weights' rounding)
    assert (dw.double().cpu() - want).norm() <= 2.0 ** -24 * want.norm() + 2.0 ** -12 * (want - w.double()).norm()


@pytest.mark.parametrize("coefficients", [(2.0, 0.0, 0.0), (0.0, 0.0, 0.0), (0.5, 0.0, 0.0), (1.5, -0.5, 0.0), (4.0, -4.0, 1.5), (0.0, 1.0, 0.0)])
@pytest.mark.parametrize("n", [50, 256])
def test_other_polynomials(n, coefficients):
    """Values are held to 2^-39 of what they may at most be, so within 2^-22 of one in the end (2^16 for the largest product of
    polynomials, n singular values a matrix), however small a result is; where singular values up to one may grow beyond what
    that holds for, the call is refused."""
    x = matrices((2, n, 300), FL)
    for steps in (1, 3, 5):
        if max(r for _, _, r in om.polynomials(steps, [coefficients] * steps)[:-1] or [(0, 0, 0)]) > 65536:
            with pytest.raises(RuntimeError, match="coefficients of step"):
                orthogonalize(x.cuda(), steps=steps, coefficients=coefficients)
            continue
        want = om.orthogonal64(x, steps, coefficients)
        got = orthogonalize(x.cuda(), steps=steps, coefficients=coefficients).double().cpu()
        assert torch.isfinite(got).all()
        assert (got - want).norm() <= 2.0 ** -18 * want.norm() + 2.0 ** -22 * (2 * n) ** 0.5, steps
