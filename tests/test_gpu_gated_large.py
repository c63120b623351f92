"""Sizes past 32-bit offsets: rows and heads whose byte and element offsets exceed 2^32, against the same rows in a
small call (the kernels' sums do not depend on how many rows there are beside a row, up to the split of E)."""
import pytest
import torch

from flashmlp_amd import block_join_bwd, block_join_fwd, clip_grads, flashmlp_gated_bwd, flashmlp_gated_fwd

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=BF)


def close(a, b):
    # another order of the fp32 sums moves a bf16 result by at most one unit of its last place, 2^-7 of it
    return torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-3)


def test_gated_rows_past_2_32_bytes():
    H, B, D, E = 2, (1 << 25) + 300, 64, 40  # 2^31 elements a head
    x = normal(H, B, D)
    wg, wu, w2 = normal(H, D, E, seed=1) / 8, normal(H, D, E, seed=2) / 8, normal(H, E, D, seed=3) / 6
    o = flashmlp_gated_fwd(x, wg, wu, w2, "silu")
    pick = [0, 1 << 24, (1 << 25) + 299]
    ref = flashmlp_gated_fwd(x[:, pick].contiguous(), wg, wu, w2, "silu")
    assert close(o[:, pick], ref)
    dx, *dw = flashmlp_gated_bwd(x, wg, wu, w2, x, "silu")
    rx, *_ = flashmlp_gated_bwd(x[:, pick].contiguous(), wg, wu, w2, x[:, pick].contiguous(), "silu")
    assert close(dx[:, pick], rx)
    del o, dx
    # the weight gradients are sums over the rows: those of two halves
    half = B // 2
    a = flashmlp_gated_bwd(x[:, :half].contiguous(), wg, wu, w2, x[:, :half].contiguous(), "silu", _needs=(False, True))
    b = flashmlp_gated_bwd(x[:, half:].contiguous(), wg, wu, w2, x[:, half:].contiguous(), "silu", _needs=(False, True))
    for g, p, q in zip(dw, a[1:], b[1:]):
        s = p.double() + q.double()
        assert (g.double() - s).norm() <= 2.0 ** -7 * s.norm()


def test_join_rows_past_2_32_bytes():
    B, H, D = (1 << 23) + 5, 4, 64  # 2^31 elements
    r, o = normal(B, H * D), normal(H, B, D, seed=1)
    w = normal(H * D, seed=2)
    r2, y, rs_o, rs_r = block_join_fwd(r, o, w, None, 0.5, pre_weight=w, _save=True)
    dr, do, *_ = block_join_bwd(r2, o, rs_o, rs_r, r, o, w, None, 0.5, pre_weight=w)
    pick = [0, 1 << 22, (1 << 23) + 4]
    p = r[pick].contiguous(), o[:, pick].contiguous()
    q2, z, a, b = block_join_fwd(*p, w, None, 0.5, pre_weight=w, _save=True)
    eq, eo, *_ = block_join_bwd(q2, p[1], a, b, *p, w, None, 0.5, pre_weight=w)
    for got, want in ((r2[pick], q2), (y[:, pick], z), (dr[pick], eq), (do[:, pick], eo)):
        assert torch.equal(got, want)


def test_clipping_a_tensor_past_2_32_bytes():
    g = normal((1 << 31) + 77)
    g[-1] = 1000.0
    # in place: the last values too
    _, norm = clip_grads([g], 1.0)
    want = (float((1 << 31) + 76) + 1e6) ** 0.5  # N(0, 1): the sum of squares is the count up to 1e-4 of it
    assert abs(norm.item() - want) <= 1e-3 * want
    assert abs(g[-1].item() - 1000.0 / norm.item()) <= 2.0 ** -8 * 1000.0 / norm.item()
