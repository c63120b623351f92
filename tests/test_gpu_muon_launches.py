"""More matrices than one launch of a workgroup each has threads for."""
import pytest
import torch

from flashmlp_amd import muon_step, orthogonalize
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


def usual(x):
    for a, c, d in om.triples(om.COEFFICIENTS, 5):
        x = x * (a + x * x * (c + x * x * d))
    return x


def test_a_stack_of_more_matrices_than_one_launch_has_workgroups():
    """matrices of one row, whose result is the row times a number; every launch's first and last matrices are among them"""
    H = (1 << 24) + 3
    x = torch.randn(H, 1, 2, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    n = x.double().norm(dim=(1, 2), keepdim=True)
    s = n / (n + 1e-7)
    want = x.double() / n * usual(s)
    assert ((orthogonalize(x) - want).abs() <= 1e-5).all()
    w, m = torch.zeros_like(x), torch.zeros_like(x)
    muon_step([w, w.new_zeros(5, 40, 50)], [x, x[:1000].view(1, 40, 50).expand(5, 40, 50)], [m, m.new_zeros(5, 40, 50)], 1.0, momentum=0.0,
              nesterov=False, scale=1.0)
    assert ((w + want).abs() <= 1e-3).all()
