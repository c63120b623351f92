"""The experts' entry points without a GPU: what they refuse, on the host, before any GPU work; the oracle's own checks."""
import ctypes

import pytest
import torch

from flashmlp_amd import ExpertPlan, _lib, expert_combine, expert_dispatch, expert_plan, expert_route
from oracle import experts as ox

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libflashmlp.so not built (python -m flashmlp_amd.build)")
    return _lib.lib()


def plan(T=5, k=2, N=3, capacity=4):
    return ExpertPlan(torch.zeros(T, k, dtype=torch.int32), torch.zeros(N, dtype=torch.int32), N, capacity)


def test_checks():
    x = torch.zeros(5, 8)
    for args, match in (((x[0], 2), "Logits"), ((x, 0), "at least one"), ((x, 9), "at most all")):
        with pytest.raises(AssertionError, match=match):
            expert_route(*args)
    e = torch.zeros(5, 2, dtype=torch.int32)
    for args, match in (((e[0], 3), "Experts must"), ((e, 0), "counted"), ((e, 3, -1), "counted"), ((e[:, :0], 3), "counted")):
        with pytest.raises(AssertionError, match=match):
            expert_plan(*args)
    with pytest.raises(AssertionError, match="Tokens must"):
        expert_dispatch(x[0], plan())
    rows = torch.zeros(3, 4, 8)
    for args, match in (((rows[0], plan()), "Rows must be \\("), ((rows[:2], plan()), "the plan's"), ((rows[:, :3], plan()), "the plan's")):
        with pytest.raises(AssertionError, match=match):
            expert_combine(*args)
    for call in (lambda: expert_route(x, 2), lambda: expert_plan(e, 3), lambda: expert_dispatch(x, plan()),
                 lambda: expert_combine(rows, plan())):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def _call(L, name, *args):
    st = getattr(L, name)(*args)
    return st, L.fmlp_last_error().decode()


def test_abi_refusals(L):
    p = ctypes.c_void_p(4096)  # (never read: every call is refused on the host)
    route = lambda **v: _call(L, "fmlp_route_fwd", *{**dict(l=p, w=p, e=p, T=4, N=8, s=8, k=2, n=1, d=1, st=None), **v}.values())  # noqa: E731
    for v, st, match in ((dict(l=None), INVALID, "logits"), (dict(w=None), INVALID, "weights"), (dict(e=None), INVALID, "experts"),
                         (dict(T=-1), INVALID, "dimensions"), (dict(N=0), INVALID, "dimensions"), (dict(k=0), INVALID, "dimensions"),
                         (dict(k=9), INVALID, "of 8"), (dict(N=1025), UNSUPPORTED, "1024"), (dict(N=64, k=33), UNSUPPORTED, "32"),
                         (dict(d=3), UNSUPPORTED, "dtype"), (dict(s=-1), INVALID, "stride"), (dict(T=2 ** 31), INVALID, "many"),
                         (dict(l=ctypes.c_void_p(4097)), INVALID, "aligned")):
        got, msg = route(**v)
        assert got == st and match in msg, (v, msg)
    back = lambda **v: _call(L, "fmlp_route_bwd", *{**dict(l=None, w=p, e=p, g=p, o=p, T=4, N=8, s=8, k=2, n=0, d=1, st=None), **v}.values())  # noqa: E731
    for v, match in ((dict(), "logits"), (dict(l=p, g=None), "dweights"), (dict(l=p, o=None), "dlogits")):
        got, msg = back(**v)
        assert got == INVALID and match in msg, (v, msg)
    sort = lambda **v: _call(L, "fmlp_expert_plan", *{**dict(e=p, b=4, s=p, c=p, T=4, k=2, N=8, cap=3, ws=None, n=0, st=None), **v}.values())  # noqa: E731
    for v, st, match in ((dict(b=2), INVALID, "4 or 8"), (dict(e=None), INVALID, "experts"), (dict(s=None), INVALID, "slots"),
                         (dict(c=None), INVALID, "counts"), (dict(c=None, T=0), INVALID, "counts"), (dict(cap=-1), INVALID, "capacity"),
                         (dict(cap=2 ** 29), INVALID, "2\\^31".replace("\\", ""))):
        got, msg = sort(**v)
        assert got == st and match in msg, (v, msg)
    copy = lambda **v: _call(L, "fmlp_expert_scatter", *{**dict(x=p, xs=8, w=None, s=p, c=p, ri=None, ro=p, dw=None, T=4, k=2, N=3,  # noqa: E731
                                                                cap=4, D=8, d=1, st=None), **v}.values())
    for v, st, match in ((dict(x=None), INVALID, "x is"), (dict(s=None), INVALID, "slots"), (dict(c=None), INVALID, "counts"),
                         (dict(ro=None), INVALID, "no output"), (dict(dw=p), INVALID, "rows_in"), (dict(D=0), INVALID, "D=0"),
                         (dict(xs=-1), INVALID, "stride"), (dict(D=2 ** 25), UNSUPPORTED, "2^24"), (dict(d=7), UNSUPPORTED, "dtype")):
        got, msg = copy(**v)
        assert got == st and match in msg, (v, msg)
    back = lambda **v: _call(L, "fmlp_expert_gather", *{**dict(r=p, w=None, s=p, o=p, T=4, k=2, N=3, cap=4, D=8, d=1, st=None), **v}.values())  # noqa: E731
    for v, match in ((dict(r=None), "rows"), (dict(s=None), "slots"), (dict(o=None), "o is"), (dict(cap=-1), "capacity")):
        got, msg = back(**v)
        assert got == INVALID and match in msg, (v, msg)


def test_oracle_route_against_autograd():
    g = torch.Generator().manual_seed(0)
    logits, dw = torch.randn(9, 11, generator=g), torch.randn(9, 4, generator=g)
    for normalize in (True, False):
        w, _, e, dl, _ = ox.route64(logits, 4, normalize, dw)
        x = logits.double().requires_grad_(True)
        p = torch.softmax(x, 1).gather(1, e)
        p = p / p.sum(1, keepdim=True) if normalize else p
        assert torch.allclose(p, w, atol=1e-14) and torch.equal(torch.topk(x, 4).indices, e)
        assert torch.allclose(torch.autograd.grad(p, x, dw.double())[0], dl, atol=1e-14)


def test_oracle_plan_is_a_stable_sort():
    e = torch.tensor([[1, 0], [1, 2], [0, 1], [1, -1], [3, 1]], dtype=torch.int32)
    slots, counts = ox.plan(e, 3, 3)
    assert slots.tolist() == [[3, 0], [4, 6], [1, 5], [-1, -1], [-1, -1]] and counts.tolist() == [2, 5, 1]
