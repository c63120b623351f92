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


CASES = [
    # B, H, D, groups, dtype, stream's dtype
    # a workgroup a row, up to 512 threads: 16-bit stream (two workgroups a CU), fp32 stream (the next row ahead), by vectors
    # and element by element
    (1100, 16, 128, 1, BF, BF), (1100, 16, 128, 1, BF, FL), (1537, 16, 127, 1, HF, HF), (1100, 16, 127, 1, BF, FL),
    (1100, 9, 128, 1, FL, FL), (513, 32, 128, 1, HF, FL),
    # more than 512 threads, and two vectors a thread
    (1100, 64, 80, 1, BF, BF), (1030, 64, 128, 1, BF, FL), (1100, 64, 136, 1, BF, BF), (700, 64, 150, 1, HF, FL),
    (540, 64, 251, 1, BF, BF), (600, 64, 256, 1, FL, FL),
    # a wave a row, one and two vectors a lane
    (5003, 10, 100, 1, BF, BF), (4500, 15, 64, 1, HF, HF), (4100, 16, 64, 1, BF, FL), (6151, 7, 64, 1, BF, BF),
    (4097, 3, 50, 1, FL, FL),
    # parts of a gate's group, the last one ragged; groups of the rows of a unit
    (1203, 16, 128, 3, BF, BF), (1203, 16, 128, 3, BF, FL), (2206, 16, 129, 2, HF, HF), (1100, 64, 136, 5, BF, BF),
    (8207, 4, 64, 1, BF, FL), (9002, 12, 64, 2, BF, BF), (8400, 5, 50, 3, HF, FL), (2048, 16, 128, 512, BF, BF),
    # several whole groups a unit, and a last unit with fewer
    (3600, 16, 128, 1200, BF, BF), (3603, 16, 128, 1201, BF, FL), (2060, 16, 127, 1030, HF, HF), (1100, 64, 136, 1100, BF, BF),
    (9001, 4, 64, 9001, BF, BF), (9000, 4, 64, 4500, BF, FL), (8202, 12, 64, 2734, HF, HF), (8202, 5, 50, 4101, FL, FL),
]


@pytest.mark.parametrize("B,H,D,groups,dt,rdt", CASES)
def test_forward_and_gradients(B, H, D, groups, dt, rdt):
    print(f"[join] B={B} H={H} D={D} groups={groups} {dt} {rdt}", flush=True)
    check(make(B, H, D, groups, dt, rdt, seed=B + D))


@pytest.mark.parametrize("B,H,D,dt,rdt", [(1100, 16, 128, BF, BF), (1100, 16, 128, BF, FL), (1100, 64, 136, BF, BF),
                                          (5000, 10, 100, HF, HF), (1030, 64, 128, HF, FL)])
@pytest.mark.parametrize("drop", [("dy", "w_pre"), ("dr2",), ("gate", "w_post"), ("w_pre",), ("gate",)])
def test_parts_left_out(B, H, D, dt, rdt, drop):
    print(f"[join] B={B} H={H} D={D} {dt} {rdt} without {drop}", flush=True)
    t = make(B, H, D, 2, dt, rdt, seed=B + D)
    check({k: v for k, v in t.items() if k not in drop})
