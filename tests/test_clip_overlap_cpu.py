"""Clipping tensors that share memory: refused by the library on the host, counted once by clip_grad_norm_."""
import ctypes

import pytest
import torch

import flashmlp_amd.clip as clip
from flashmlp_amd import _lib

INVALID = 1
F16, BF16, F32 = 0, 1, 2


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    return _lib.lib()


def refused(L, *tensors):
    """(gradient, output, elements, dtype, output's dtype) of each tensor; addresses that nothing reads: a call that
    passes the check ends at the missing norm's workspace at the latest"""
    n = len(tensors)
    g, o, numel, dt, odt = zip(*tensors)
    st = L.fmlp_clip_grads(n, (ctypes.c_void_p * n)(*g), (ctypes.c_void_p * n)(*o), (ctypes.c_int64 * n)(*numel),
                           (ctypes.c_int * n)(*dt), (ctypes.c_int * n)(*odt), 1.0, 64, None, 0, None)
    assert st != 0
    return st == INVALID and b"overlap" in L.fmlp_last_error()


def test_library_refuses_overlapping_outputs(L):
    K = 1 << 12
    apart = [(K, 2 * K, 100, BF16, F32), (3 * K, 4 * K, 100, F32, F32)]
    assert not refused(L, *apart)
    assert not refused(L, (K, K, 100, F32, F32), (K + 400, K + 400, 100, F32, F32))  # in place, one behind the other
    assert not refused(L, (K, 2 * K, 100, F32, F32), (K, 3 * K, 100, F32, F32))  # one gradient, two outputs
    assert not refused(L, (K, 2 * K, 100, F32, F32), (0, 0, 0, F32, F32))
    assert refused(L, (K, K, 100, F32, F32), (K, K, 100, F32, F32))  # one tensor twice, in place
    assert refused(L, (K, 3 * K, 100, F32, F32), (2 * K, 3 * K, 100, F32, F32))  # one output twice
    assert refused(L, (K, 4 * K, 100, F32, F32), (2 * K, 4 * K + 396, 100, F32, F32))
    assert refused(L, (2 * K, 4 * K + 396, 100, F32, F32), (K, 4 * K, 100, F32, F32))  # in any order
    assert refused(L, (K, K + 4, 100, F32, F32))  # its own gradient, shifted
    assert refused(L, (K, K, 100, BF16, F32)) and refused(L, (K, K, 100, BF16, F16))  # in place in another type
    assert refused(L, (K, 2 * K, 100, F32, F32), (2 * K + 396, 3 * K, 100, F32, F32))  # another's gradient
    # a long one over many, whichever comes first in memory
    assert refused(L, (K, 9 * K, 10 * K, BF16, BF16), *((K, 9 * K + 64 * i, 4, F32, F32) for i in range(1, 5)))
    assert refused(L, (8, 9 * K, 2 * K, F32, F32), (7 * K, K, 4, F32, F32))


def test_a_gradient_that_parameters_share_is_clipped_once(monkeypatch):
    p, q, r, s = (torch.nn.Parameter(torch.zeros(3)) for _ in range(4))
    both = torch.ones(6)
    p.grad = q.grad = torch.ones(3)
    r.grad, s.grad = both[:3], both[3:]
    seen = []
    monkeypatch.setattr(clip, "clip_grads", lambda grads, max_norm: (seen.append(list(grads)), 1.0))
    clip.clip_grad_norm_([p, q, r, s], 1.0)
    assert [g.data_ptr() for g in seen[0]] == [g.data_ptr() for g in (p.grad, r.grad, s.grad)]
    r.grad, s.grad = both[:3], both[:3]  # two tensors over one memory
    clip.clip_grad_norm_([r, q, s], 1.0)
    assert [g.data_ptr() for g in seen[1]] == [both.data_ptr(), q.grad.data_ptr()]
