"""GatedExperts with one expert a token: by default its weight is the softmax's probability, so that the router learns."""
import pytest
import torch

from flashmlp_amd import GatedExperts, expert_route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_the_router_learns(dtype):
    torch.manual_seed(0)
    m = GatedExperts(4, 32, 40, experts_per_token=1, dtype=dtype)
    x = torch.randn(50, 32, device="cuda").to(dtype)
    o = m(x)
    # each token's own expert, times its probability
    logits = x.double() @ m.router.detach().double()
    e = expert_route(x @ m.router, 1)[1][:, 0].long()
    p = torch.softmax(logits, 1).gather(1, e[:, None])[:, 0]
    wg, wu, w2 = (t.detach().double()[e] for t in (m.experts.wg, m.experts.wu, m.experts.w2))
    h = torch.nn.functional.silu((x.double()[:, None] @ wg)) * (x.double()[:, None] @ wu)
    want = (h @ w2)[:, 0] * p[:, None]
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -20}[dtype]
    # (logits rounded to the type move p by up to their size, 4, times its unit)
    assert (o.double() - want).norm() <= 8 * u * want.norm()
    o.float().square().sum().backward()
    assert m.router.grad.float().norm() > 1e-3
