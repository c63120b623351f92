"""orthogonalize and muon_step without a GPU: what they refuse, on the host, before any GPU work; the oracle's own checks."""
import ctypes

import pytest
import torch

from flashmlp_amd import _lib, muon_step, orthogonalize
from flashmlp_amd.muon import _refuse_overlap
from oracle import muon as om

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


def places(t):
    """addresses of all bytes"""
    at = torch.zeros((), dtype=torch.int64)
    for stride, n in zip(t.stride(), t.shape):
        at = at.unsqueeze(-1) + stride * t.element_size() * torch.arange(n)
    return (at.unsqueeze(-1) + t.data_ptr() + torch.arange(t.element_size())).flatten().tolist()


def refused(ts):
    try:
        _refuse_overlap(ts)
    except RuntimeError:
        return True
    return False


def test_overlap_of_strided_tensors():
    """what shares memory is refused in any layout, views of one buffer side by side are not"""
    g = torch.Generator().manual_seed(0)
    buf = torch.zeros(4096)
    taken = 0
    for _ in range(3000):
        ts = []
        for _ in range(2):
            n = [int(v) for v in torch.randint(1, 5, (3,), generator=g)]
            stride = [int(v) for v in torch.tensor([1, 2, 3, 4, 8, 16, 32, 64])[torch.randint(0, 8, (3,), generator=g)]]
            ts.append(buf.as_strided(n, stride, int(torch.randint(0, 200, (), generator=g))))
        p = places(ts[0]) + places(ts[1])
        if not refused(ts):
            taken += 1
            assert len(set(p)) == len(p)
    assert taken > 100
    x, y = torch.zeros(3, 8, 12), torch.zeros(3, 8, 12).bfloat16()
    halves = [x[..., :6], x[..., 6:], y[:, :4], y[:, 4:], y.new_zeros(3, 5, 8).mT, torch.zeros(0, 4, 2).mT]
    assert not refused(halves) and not refused([x[..., 6:], x[:, 1:, :6]]) and not refused([x[:, :, ::2].mT, x[:, :, 1::2].mT])
    for bad in ([x.mT, x], [x[..., :6], x[..., 5:]], [x[..., 6:], x[:, 1:, :7]], [x[:, :1].expand(3, 8, 12)], halves + [x[0, :, 3:4]]):
        assert refused(bad)


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    return _lib.lib()


def test_orthogonalize_checks():
    x = torch.zeros(2, 8, 9)
    for kw in (dict(steps=0), dict(steps=11), dict(coefficients=(1.0, 2.0)), dict(coefficients=[(1.0, 2.0, 3.0)] * 4)):
        with pytest.raises(ValueError, match="steps|coefficients"):
            orthogonalize(x, **kw)
    with pytest.raises(ValueError, match="matrices"):
        orthogonalize(x[0, 0])
    with pytest.raises(TypeError, match="number"):
        orthogonalize(x, eps=torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="GPU"):
        orthogonalize(x)


def test_muon_checks():
    t = [torch.zeros(2, 8, 9) for _ in range(3)]
    for args in (([t[0]], [], [t[2]]), ([t[0]], [t[1][:1]], [t[2]]), ([t[0]], [t[1]], [t[2][0]]), ([t[0][0, 0]], [t[1][0, 0]], [t[2][0, 0]])):
        with pytest.raises(ValueError):
            muon_step(*args, 0.1)
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(lr=0.1, momentum=1.5), dict(lr=0.1, weight_decay=-1.0), dict(lr=0.1, steps=0)):
        with pytest.raises(ValueError):
            muon_step(*([v] for v in t), kw.pop("lr"), **kw)
    with pytest.raises(TypeError, match="number"):
        muon_step(*([v] for v in t), torch.tensor(0.1))
    with pytest.raises(RuntimeError, match="GPU"):
        muon_step(*([v] for v in t), 0.1)
    muon_step([], [], [], 0.1)


def test_abi_refusals(L):
    p, q = ctypes.c_void_p(4096), ctypes.c_void_p(1 << 20)  # (never read: every call is refused on the host)
    abc = (ctypes.c_float * 30)(*[1.0, -0.5, 0.1] * 10)
    nan = (ctypes.c_float * 3)(float("nan"), 0, 0)

    def ortho(**v):
        a = {**dict(x=p, o=q, H=2, R=8, C=9, d=2, s=5, abc=abc, eps=1e-7, ws=None, n=0, st=None), **v}
        return L.fmlp_orthogonalize(*a.values()), L.fmlp_last_error().decode()

    for v, st, match in ((dict(x=None), INVALID, "x of"), (dict(o=None), INVALID, "out of"), (dict(H=-1), INVALID, "negative"),
                         (dict(R=257, C=300), UNSUPPORTED, "256"), (dict(d=5), UNSUPPORTED, "dtype"), (dict(s=0), UNSUPPORTED, "steps"),
                         (dict(s=11), UNSUPPORTED, "steps"), (dict(abc=None), INVALID, "coefficients"), (dict(abc=nan, s=1), INVALID, "coefficient 0"),
                         (dict(eps=-1.0), INVALID, "eps"), (dict(o=ctypes.c_void_p(4096 + 16)), INVALID, "overlaps"),
                         (dict(x=ctypes.c_void_p(4097)), INVALID, "aligned")):
        got, msg = ortho(**v)
        assert got == st and match in msg, (v, msg)
    assert ortho(H=0, x=None, o=None)[0] == 0

    def step(n=1, lr=0.1, mu=0.9, wd=0.0, s=5, **v):
        a = {**dict(w=4096, g=1 << 20, m=2 << 20, H=2, R=8, C=9, wt=2, gt=2, mt=2, scale=1.0), **v}
        t = (_lib.MuonTensor * 1)(_lib.MuonTensor(*a.values()))
        return L.fmlp_muon_step(n, t, lr, mu, 1, wd, s, abc, 1e-7, None, 0, None), L.fmlp_last_error().decode()

    for v, st, match in ((dict(w=None), INVALID, "weights"), (dict(g=None), INVALID, "gradient"), (dict(m=None), INVALID, "momentum"),
                         (dict(n=-1), INVALID, "-1 stacks"), (dict(lr=-1.0), INVALID, "lr"), (dict(mu=1.5), INVALID, "momentum"),
                         (dict(wd=float("nan")), INVALID, "weight_decay"), (dict(gt=4), UNSUPPORTED, "dtype"), (dict(s=11), UNSUPPORTED, "steps"),
                         (dict(m=4096 + 64), INVALID, "overlap"), (dict(g=4096 + 64), INVALID, "overlap"), (dict(R=300, C=300), UNSUPPORTED, "256")):
        got, msg = step(**v)
        assert got == st and match in msg, (v, msg)


def test_oracle_against_singular_values():
    """every step is a polynomial of the singular values"""
    x = torch.randn(2, 7, 12, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    u, s, v = torch.linalg.svd(x, full_matrices=False)
    s = s / (torch.linalg.matrix_norm(x, keepdim=False)[:, None] + 1e-7)
    for a, b, c in om.triples(om.COEFFICIENTS, 5):
        s = a * s + b * s ** 3 + c * s ** 5
    want = (u * s[:, None]) @ v
    assert torch.allclose(om.orthogonal64(x), want, atol=1e-12)
    assert torch.allclose(om.orthogonal64(x.mT), want.mT, atol=1e-12)
