"""The gated MLP with less workspace than its plan would take: the library runs tiles whole, the wrappers ask again for the
least where the plan's does not fit on the device."""
import pytest
import torch

import flashmlp_amd.gated as gated
from flashmlp_amd import _lib, flashmlp_gated_bwd
from test_gpu_gated import both, check, make

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
CASES = [  # shapes whose plans split E or the rows, with and without padded weights
    (1, 5, 128, 2048, BF, "silu"), (1, 9000, 128, 100, BF, "sigmoid"), (1, 6049, 256, 33, HF, ""), (2, 2048, 64, 512, BF, "silu"),
    (1, 700, 256, 136, BF, "silu"), (2, 9000, 32, 64, FL, "silu"), (1, 260, 128, 95, FL, "sigmoid"), (1, 1000, 16, 640, HF, "silu"),
]


@pytest.mark.parametrize("H,B,D,E,dt,act", CASES)
def test_library_with_every_workspace(H, B, D, E, dt, act):
    print(f"[gated] H={H} B={B} D={D} E={E} {dt} act='{act}'", flush=True)
    L, t = _lib.lib(), make(H, B, D, E, dt, seed=B)
    code, a = gated._DTYPES[dt], gated._act_code(act)
    stream = torch.cuda.current_stream().cuda_stream
    least, fwd = L.fmlp_gated_min_workspace_bytes(H, D, E, code), L.fmlp_gated_fwd_workspace_bytes(H, B, D, E, code)
    bwd = L.fmlp_gated_bwd_workspace_bytes(H, B, D, E, code)
    assert (least > 0) == (E * t[0].element_size() % 16 != 0) and max(fwd, bwd) > least
    for nf, nb in ((least, least), (fwd, bwd), ((least + fwd) // 2, (least + bwd) // 2), (fwd + 4096, bwd + 4096)):
        out = [torch.full_like(v, float("nan")) for v in (t[0], *t[:4])]
        ws = torch.full((max(nf, nb) + 256,), 255, dtype=torch.uint8, device="cuda")  # (255s: NaNs)
        p = [v.data_ptr() for v in t]
        q = [v.data_ptr() for v in out]
        st = L.fmlp_gated_fwd(*p[:4], q[0], H, B, D, E, B * D, code, a, ws.data_ptr() if nf else None, nf, stream)
        assert st == 0, L.fmlp_last_error()
        assert ws[nf:].eq(255).all()
        ws.fill_(255)
        st = L.fmlp_gated_bwd(*p, *q[1:], H, B, D, E, B * D, B * D, code, a, 1.0, ws.data_ptr() if nb else None, nb, stream)
        assert st == 0, L.fmlp_last_error()
        assert ws[nb:].eq(255).all()
        check(out, t, act)
    if least:
        st = L.fmlp_gated_fwd(*p[:4], q[0], H, B, D, E, B * D, code, a, ws.data_ptr(), least - 1, stream)
        assert st == 4
        st = L.fmlp_gated_bwd(*p, *q[1:], H, B, D, E, B * D, B * D, code, a, 1.0, None, 0, stream)
        assert st == 4


@pytest.mark.parametrize("H,B,D,E,dt,act", CASES[:4])
def test_general_path(monkeypatch, H, B, D, E, dt, act):
    t, real, sizes = make(H, B, D, E, dt, seed=B), gated._alloc_ws, []
    least = _lib.lib().fmlp_gated_min_workspace_bytes(H, D, E, gated._DTYPES[dt])

    def tight(n, device):
        sizes.append(n)
        if n > least:
            raise torch.OutOfMemoryError("no room")
        return real(n, device)

    monkeypatch.setattr(gated, "_alloc_ws", tight)
    monkeypatch.setattr(gated, "_fast", None)
    check(both(*t, act), t, act)
    assert least in sizes and max(sizes) > least

    def none(n, device):
        raise torch.OutOfMemoryError("no room")

    monkeypatch.setattr(gated, "_alloc_ws", none)
    with pytest.raises(torch.OutOfMemoryError):
        both(*t, act)


def test_fast_path(monkeypatch):
    """a real allocation failure, with room for the outputs alone: the bits of the general path without a
    workspace"""
    H, B, D, E = 16, 4096, 128, 512
    t = [v.cuda() for v in make(H, B, D, E, BF)]
    L = _lib.lib()
    need = L.fmlp_gated_bwd_workspace_bytes(H, B, D, E, 1)
    out = 2 * (H * B * D + 3 * H * D * E)
    assert need > 32 << 20 and L.fmlp_gated_min_workspace_bytes(H, D, E, 1) == 0

    def none(n, device):
        if n:
            raise torch.OutOfMemoryError("no room")

    with monkeypatch.context() as m:
        m.setattr(gated, "_alloc_ws", none)
        m.setattr(gated, "_fast", None)
        want = flashmlp_gated_bwd(*t, "silu")
    split = flashmlp_gated_bwd(*t, "silu")  # (another order of the sums over rows)
    assert not all(torch.equal(a, b) for a, b in zip(split, want))
    del split
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    # no memory beyond what is reserved, all of it taken but room for the outputs
    room, hold = torch.empty(out + (12 << 20), dtype=torch.uint8, device="cuda"), []
    torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / torch.cuda.get_device_properties(0).total_memory)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            while True:
                hold.append(torch.empty(2 << 20, dtype=torch.uint8, device="cuda"))
        del room
        got = flashmlp_gated_bwd(*t, "silu")
        torch.cuda.synchronize()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
