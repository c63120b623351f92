"""The gated block's entry points without a GPU: what they refuse, on the host, before any GPU work."""
import ctypes

import pytest
import torch

from flashmlp_amd import (_lib, block_join, block_norm, clip_grad_norm_, clip_grads, flashmlp_gated_bwd,
                          flashmlp_gated_fwd, grad_norm)

INVALID, UNSUPPORTED = 1, 2


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    return _lib.lib()


def gated(H, B, D, E, **shapes):
    t = dict(x=(H, B, D), wg=(H, D, E), wu=(H, D, E), w2=(H, E, D))
    t.update(shapes)
    return [torch.zeros(s) for s in t.values()]


def test_gated_checks():
    for t, match in ((gated(2, 4, 64, 8, wu=(2, 64, 9)), "Gate and up"), (gated(2, 4, 64, 8, w2=(1, 8, 64)), "heads"),
                     (gated(2, 4, 64, 8, w2=(2, 9, 64)), "Intermediate"), (gated(2, 4, 64, 8, w2=(2, 8, 32)), "Output"),
                     (gated(2, 4, 32, 8, wg=(2, 64, 8), wu=(2, 64, 8)), "Hidden")):
        with pytest.raises(AssertionError, match=match):
            flashmlp_gated_fwd(*t)
    t = gated(2, 4, 64, 8)
    with pytest.raises(AssertionError, match="Gradient shape"):
        flashmlp_gated_bwd(*t, torch.zeros(2, 5, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        flashmlp_gated_fwd(*t)
    with pytest.raises(RuntimeError, match="GPU"):
        flashmlp_gated_bwd(*t, torch.zeros(2, 4, 64))


def test_fake_tensors_trace_the_registered_operators():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, wg, wu, w2 = (torch.empty(s, device="cuda", dtype=torch.bfloat16)
                         for s in ((2, 5, 32), (2, 32, 7), (2, 32, 7), (2, 7, 32)))
        assert torch.ops.flashmlp_amd.gated_fwd(x, wg, wu, w2, "silu").shape == x.shape
        g = torch.ops.flashmlp_amd.gated_bwd(x, wg, wu, w2, x, "silu")
        assert [t.shape for t in g] == [x.shape, wg.shape, wu.shape, w2.shape]
        with pytest.raises(RuntimeError, match="must match"):
            torch.ops.flashmlp_amd.gated_fwd(x, wg, wu[:, :, :5], w2, "silu")


def test_join_checks():
    r, o, w = torch.zeros(6, 64), torch.zeros(2, 6, 32), torch.zeros(64)
    for args, kw, match in (((r, o[:, :5]), {}, "rows"), ((r, o[:1]), {}, "Columns"), ((r[0], o), {}, "stream"),
                            ((r, o, w[:9]), {}, "Post norm"), ((r, o), dict(pre_weight=w[:9]), "Pre norm"),
                            ((r, o, None, torch.zeros(4, 64)), {}, "divide"), ((r, o, None, w[:8]), {}, "gate"),
                            ((r, o, w), dict(post=False), "post norm"), ((r, o), dict(pre_weight=w, pre=False), "pre norm"),
                            ((r, o.unsqueeze(0)), {}, "block's output")):
        with pytest.raises(AssertionError, match=match):
            block_join(*args, **kw)
    for heads in (0, 3):
        with pytest.raises(AssertionError, match="heads"):
            block_norm(r, heads=heads)
    with pytest.raises(RuntimeError, match="GPU"):
        block_join(r, o)
    with pytest.raises(RuntimeError, match="GPU"):
        block_norm(r)


def test_clip_checks():
    g = [torch.zeros(4), torch.zeros(5)]
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads(g, -1.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads(g, 1.0, out=g[:1])
    with pytest.raises(RuntimeError, match="GPU"):
        clip_grads(g, 1.0)
    with pytest.raises(RuntimeError, match="GPU"):
        grad_norm(g)
    assert grad_norm([]) == 0 and clip_grads([], 1.0)[1] == 0 and clip_grad_norm_([], 1.0) == 0


def test_library_refuses_gated_arguments(L):
    ok = dict(H=1, B=4, D=64, E=32, sx=256, dtype=1, act=1)

    def call(ptr=16, **kw):
        a = dict(ok, **kw)
        return L.fmlp_gated_fwd(ptr, 16, 16, 16, 16, a["H"], a["B"], a["D"], a["E"], a["sx"], a["dtype"], a["act"], None,
                                0, None)

    assert call(D=48) == UNSUPPORTED and call(E=0) == UNSUPPORTED and call(dtype=7) == UNSUPPORTED
    assert call(H=-1) == INVALID and call(B=1 << 40) == INVALID and call(act=9) == INVALID
    assert call(ptr=None) == INVALID and call(ptr=8) == INVALID
    assert call(H=2, sx=3) == INVALID and call(sx=-8) == INVALID
    assert call(dtype=1 | _lib.FMLP_BWD_NO_DX) == INVALID
    assert call(E=1 << 28) == UNSUPPORTED
    assert b"D*E" in L.fmlp_last_error()
    assert call(B=0, ptr=None) == 0 and call(H=0, ptr=None) == 0


def test_library_refuses_join_arguments(L):
    def call(bwd=False, **kw):
        j = _lib.Join()
        j.B, j.H, j.D, j.groups, j.dtype, j.r_dtype, j.post, j.eps = 4, 2, 32, 1, 1, 1, 1, 1e-6
        j.r = j.o = j.y = j.r_out = 16
        j.r_stride = j.o_row_stride = j.y_row_stride = 64
        for k, v in kw.items():
            setattr(j, k, v)
        if bwd:
            return L.fmlp_join_bwd(ctypes.byref(j), None, 0, None)
        return L.fmlp_join_fwd(ctypes.byref(j), None)

    assert call(B=-1) == INVALID and call(H=0) == INVALID and call(groups=3) == INVALID and call(D=0) == INVALID
    assert call(dtype=5) == UNSUPPORTED and call(r_dtype=0) == UNSUPPORTED and call(D=16384) == UNSUPPORTED
    assert call(r=None) == INVALID and call(r=17) == INVALID and call(eps=-1.0) == INVALID
    assert call(eps=float("nan")) == INVALID and call(r_stride=-64) == INVALID
    assert call(o=None, gate=16) == INVALID and call(post=0, w_post=16) == INVALID and call(y=None, w_pre=16) == INVALID
    assert call(y=None, r_out=None) == INVALID
    assert call(bwd=True, dy=16) == INVALID  # (without the rows' 1 / rms)
    assert call(bwd=True, o=None, dgate=16) == INVALID
    assert L.fmlp_join_fwd(None, None) == INVALID


def test_library_refuses_clip_arguments(L):
    def call(numel=4, dtype=1, odt=2, max_norm=1.0, g=16, o=16, norm=16, ws=16, n=1):
        gs, os_ = (ctypes.c_void_p * 1)(g), (ctypes.c_void_p * 1)(o)
        return L.fmlp_clip_grads(n, gs, os_, (ctypes.c_int64 * 1)(numel), (ctypes.c_int * 1)(dtype),
                                 (ctypes.c_int * 1)(odt), max_norm, norm, ws, 1 << 20, None)

    assert call(n=-1) == INVALID and call(numel=-1) == INVALID and call(numel=1 << 50) == INVALID
    assert call(dtype=9) == UNSUPPORTED and call(odt=3) == UNSUPPORTED
    assert call(g=None) == INVALID and call(g=15) == INVALID and call(o=18) == INVALID and call(norm=None) == INVALID
    assert call(max_norm=-1.0) == INVALID and call(max_norm=float("nan")) == INVALID


def test_a_parameter_listed_twice_is_clipped_once(monkeypatch):
    import flashmlp_amd.clip as clip

    p, q, r = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    p.grad, q.grad = torch.ones(3), torch.ones(3)
    seen = []
    monkeypatch.setattr(clip, "clip_grads", lambda grads, max_norm: (seen.append(list(grads)), 1.0))
    clip.clip_grad_norm_([p, q, r, p, q], 1.0)
    assert len(seen) == 1 and len(seen[0]) == 2 and seen[0][0] is p.grad and seen[0][1] is q.grad
