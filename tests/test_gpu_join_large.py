"""A stream of more rows than one launch has threads for (a wave a row, fewer than 2^32 threads a launch: 2^26 rows)."""
import pytest
import torch

from flashmlp_amd import block_join_bwd, block_join_fwd, block_norm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("groups", [1, 3])
def test_rows_past_2_26(groups):
    B, C = (1 << 26) + 5, 16
    assert B % 3 == 0 and B * 64 > 1 << 32
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=BF)  # noqa: E731
    r, o, w, gate = n(B, C), n(1, B, C), n(C), n(groups, C)
    rows = torch.tensor([0, 1, 1 << 25, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, B - 1], device="cuda")
    p, q, g = r[rows], o[:, rows], gate[rows // (B // groups)]
    y = block_norm(r, w)
    assert torch.equal(y[rows], block_norm(p, w))
    del y
    r2, y, rs_o, rs_r = block_join_fwd(r, o, w, gate, 0.5, pre_weight=w, _save=True)
    s2, z, a, b = block_join_fwd(p, q, w, g, 0.5, pre_weight=w, _save=True)
    for got, want in ((r2[rows], s2), (y[:, rows], z), (rs_o[rows], a), (rs_r[rows], b)):
        assert torch.equal(got, want)
    dr, do, *_ = block_join_bwd(r2, o, rs_o, rs_r, r, o, w, gate, 0.5, pre_weight=w)
    er, eo, *_ = block_join_bwd(s2, q, a, b, p, q, w, g, 0.5, pre_weight=w)
    assert torch.equal(dr[rows], er) and torch.equal(do[:, rows], eo)
