"""block_join's scale and the norms' eps are numbers: a tensor, whose gradient would be lost, is refused."""
import numpy as np
import pytest
import torch

from flashmlp_amd import block_join, block_join_bwd, block_join_fwd, block_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dev", ["cpu", "cuda"])
def test_a_tensor_is_refused(strided, dev):
    r, o = torch.randn(8, 64, device="cuda"), torch.randn(2, 8, 32, device="cuda")
    if strided:
        r = torch.stack([r, r], -1).flatten(1)[:, ::2]
    rs = torch.ones(8, device="cuda")
    for grad in (False, True):
        s = torch.nn.Parameter(torch.tensor(0.5, device=dev), requires_grad=grad)
        for call in (lambda: block_join(r, o, None, None, s), lambda: block_join(r, o, scale=s, pre=False),
                     lambda: block_join_fwd(r, o, None, None, s), lambda: block_join(r, o, eps=s * 0 + 1e-6),
                     lambda: block_join_bwd(r, o, rs, rs, r, o, None, None, s), lambda: block_norm(r, eps=s * 0 + 1e-6)):
            with pytest.raises(TypeError, match="number"):
                call()


def test_numbers_of_every_kind():
    r, o = torch.randn(8, 64, device="cuda"), torch.randn(2, 8, 32, device="cuda")
    for a, b in ((2.0, 2), (2.0, np.float32(2)), (2.0, np.int64(2)), (1.0, True), (0.5, np.float64(0.5))):
        for x, y in zip(block_join(r, o, scale=a), block_join(r, o, scale=b)):
            assert torch.equal(x, y)
