"""The join's arguments, refused before any GPU work: numbers that are tensors, row values of other sizes or types."""
import pytest
import torch

from flashmlp_amd import block_join, block_join_bwd, block_join_fwd, block_norm


@pytest.mark.parametrize("bad", [torch.tensor(0.5), torch.nn.Parameter(torch.tensor(0.5)), "0.5", None, 1j])
def test_scale_and_eps_are_numbers(bad):
    r, o, rs = torch.zeros(6, 64), torch.zeros(2, 6, 32), torch.ones(6)
    for call in (lambda: block_join(r, o, scale=bad), lambda: block_join(r, o, scale=bad, pre=False),
                 lambda: block_join_fwd(r, o, scale=bad), lambda: block_join(r, o, eps=bad), lambda: block_norm(r, eps=bad),
                 lambda: block_join_bwd(r, o, rs, rs, r, o, scale=bad), lambda: block_join_bwd(r, o, rs, rs, r, o, eps=bad)):
        with pytest.raises(TypeError, match="number"):
            call()


def test_row_values_are_checked():
    """(tensors that claim a GPU and hold nothing: what a call needs of them is their sizes, types and devices)"""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        e = lambda *s, dt=torch.float32, dev="cuda": torch.empty(s, dtype=dt, device=dev)  # noqa: E731
        r, o, rs = e(6, 64), e(2, 6, 32), e(6)
        bad = [(e(5), AssertionError), (e(7), AssertionError), (e(2, 6), AssertionError), (e(6, 1), AssertionError), (e(), AssertionError),
               (e(6, dt=torch.float64), TypeError), (e(6, dt=torch.bfloat16), TypeError), (e(6, dev="cpu"), TypeError)]
        for b, error in bad:
            with pytest.raises(error, match="rs_o"):
                block_join_bwd(r, o, b, rs, r, o)
            with pytest.raises(error, match="rs_r"):
                block_join_bwd(r, o, rs, b, r, o)
        h = e(6, 64, dt=torch.bfloat16)
        with pytest.raises(AssertionError, match="rs_o"):
            block_join_bwd(None, e(2, 6, 32, dt=torch.bfloat16), e(5), rs, h, None, residual=h)
        for kw in ({}, dict(residual=r)):
            with pytest.raises(AssertionError, match="stream"):
                block_join_bwd(None, o, rs, rs, r, o, **kw)
