"""More matrices than one launch of a workgroup each has threads for."""
import pytest
import torch

from flashmlp_amd import muon_step
from oracle import muon as om

pytestmark = pytest.mark.gpu


def test_stacks_of_more_matrices_than_one_launch_has_workgroups():
    """65 stacks of 2^18 - 1 matrices of one element: 2^24 workgroups are 2^32 threads"""
    n, shape = 65, ((1 << 18) - 1, 1, 1)
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = [torch.randn(shape, generator=gen, device="cuda") for _ in range(n)]
    w, m = ([torch.zeros(shape, device="cuda") for _ in range(n)] for _ in range(2))
    muon_step(w, g, m, 1.0)
    for t, b in zip(w, g):
        u = 0.0975 * b.double()  # (0.05 g + 0.95 m, m = 0.05 g)
        x = u / (u.abs() + 1e-7)
        for a, c, d in om.triples(om.COEFFICIENTS, 5):
            x = x * (a + x * x * (c + x * x * d))
        assert ((t + x).abs() <= 1e-3).all()
