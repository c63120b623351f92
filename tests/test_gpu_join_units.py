"""The join's backward where a unit (a workgroup or a wave) walks several rows: the row sums' buffers by turns, the next
row requested ahead, columns' sums over rows, gates kept over a part of a group, several whole groups a unit, ragged last
parts. On 256 CUs a workgroup's unit has more than one row past 512 rows, a wave's past 2048."""
import pytest
import torch

from flashmlp_amd import block_join_bwd, block_join_fwd
from test_gpu_join import check, make

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def test_row_values_of_any_stride():
    """rs_o and rs_r as columns of one array"""
    t = make(40, 3, 32, 1, BF, BF)
    args = (t["o"], t["w_post"], t["gate"], 0.5)
    r2, y, rs_o, rs_r = block_join_fwd(t["r"], *args, pre_weight=t["w_pre"], _save=True)
    both = torch.stack([rs_o, rs_r], 1)
    want = block_join_bwd(r2, t["o"], rs_o, rs_r, t["dr2"], t["dy"], *args[1:], pre_weight=t["w_pre"])
    got = block_join_bwd(r2, t["o"], both[:, 0], both[:, 1], t["dr2"], t["dy"], *args[1:], pre_weight=t["w_pre"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
