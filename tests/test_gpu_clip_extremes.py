"""Finite gradients whose norm is beyond 32 bits' largest number are clipped to max_norm, not to zero; the norm that
is returned, an fp32 number, is infinite."""
import pytest
import torch

from flashmlp_amd import clip_grads

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dt", [BF, FL])
@pytest.mark.parametrize("odt", [BF, FL, HF, None])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e30])
@pytest.mark.parametrize("n", [100, 100003])
def test_norms_beyond_fp32(dt, odt, max_norm, n):
    g = torch.randn(n, generator=torch.Generator().manual_seed(n)).mul_(1e38).clamp_(-3e38, 3e38).to(dt).cuda()
    small = torch.full((9,), 1e-20, device="cuda").to(dt)
    before = [g.double(), small.double()]
    norm64 = torch.sqrt(before[0].square().sum()).item()
    assert norm64 > 3.5e38
    outs = None if odt is None else [torch.empty(t.shape, dtype=odt, device="cuda") for t in (g, small)]
    res, norm = clip_grads([g, small], max_norm, out=outs)
    assert norm.isinf()
    # the coefficient is one fp32 rounding off, a product two; the result's own rounding, and half of its type's
    # smallest subnormal (bf16's and fp32's: 2^-134, 2^-150)
    unit, tiny = {BF: (2.0 ** -8, 2.0 ** -134), FL: (2.0 ** -24, 2.0 ** -150), HF: (2.0 ** -11, 2.0 ** -25)}[res[0].dtype]
    for b, r in zip(before, res):
        w = b * (max_norm / norm64)
        top = torch.finfo(r.dtype).max
        fits, over = w.abs() < 0.99 * top, w.abs() > 1.01 * top  # (1e30 in fp16: infinite)
        e = (r.double() - w).abs() - 1.01 * (unit + 2.0 ** -22) * w.abs() - 1.01 * tiny
        assert (e[fits] <= 0).all() and torch.equal(r[over].double(), w[over].sign() * float("inf"))


def test_infinite_gradients_as_ever():
    g = torch.ones(100, device="cuda")
    g[3] = float("inf")
    out, norm = clip_grads([g], 1.0)
    assert norm.isinf() and g[3].isnan() and not g[:3].any()
