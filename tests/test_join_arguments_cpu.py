"""block_join's scale and the norms' eps are numbers, refused before any GPU work."""
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
