"""orthogonalize and muon_step in torch's hands: forward mode is refused, not left out."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from flashmlp_amd import muon, muon_step, orthogonalize

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["C++", "Python"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(muon, "_fast", None)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.enable_grad])
def test_forward_mode_is_refused(path, mode):
    x = torch.randn(2, 8, 12, device="cuda")
    three = [torch.randn(2, 8, 12, device="cuda") for _ in range(3)]
    kept = [t.clone() for t in three]
    with fwad.dual_level(), mode():
        d = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: orthogonalize(d), lambda: orthogonalize(x, out=d), lambda: orthogonalize(d, out=d)):
            with pytest.raises(RuntimeError, match="jvp"):
                call()
        for i in range(3):
            args = [fwad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(three)]
            with pytest.raises(RuntimeError, match="jvp"):
                muon_step(*args, 0.1)
        orthogonalize(x)
        muon_step(*three, 0.0, momentum=1.0)
    assert all(torch.equal(a, b) for a, b in zip(three, kept))


def test_under_compile(path):
    """the graph breaks at the calls, whose results are the eager ones"""
    x = torch.randn(2, 8, 12, device="cuda")
    w, g, m = (torch.randn(2, 8, 12, device="cuda") for _ in range(3))
    w2, m2 = w.clone(), m.clone()

    def step(x, w, g, m):
        y = orthogonalize(x * 2) + 1
        muon_step(w, g + 1, m, 0.1)
        return y - 1

    got = torch.compile(step, backend="eager")(x, w, g, m)
    want = step(x, w2, g, m2)
    assert torch.equal(got, want) and torch.equal(w, w2) and torch.equal(m, m2)
