"""Gradients that share memory: one tensor is clipped once, everything else that overlaps is refused before any launch."""
import pytest
import torch

from flashmlp_amd import clip_grad_norm_, clip_grads, grad_norm

pytestmark = pytest.mark.gpu


def test_refused_and_unchanged():
    buf = torch.ones(1000, device="cuda")
    out = torch.full((600,), 7.0, device="cuda")
    a, b = buf[:600], buf[400:]
    s = buf[::2]
    for grads, outs in (([a, a], None), ([a, b], None), ([a.view(2, 300), a], None), ([a, b], [out, out]),
                        ([a, b], [out, a]), ([a], [b]), ([a, b[:400]], [a, b[:400]]), ([s, s], None),
                        ([a.view(torch.int32).view(torch.float32), a], None),
                        ([a, a], [out.view(2, 300).t(), out.view(2, 300).t()])):
        if outs is not None and outs[0].dim() == 2:
            grads = [g.view(2, 300).t() for g in grads]
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads(grads, 0.1, out=outs)
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([buf.view(torch.bfloat16)], 0.1, out=[buf.view(torch.float16)])
    assert (buf == 1).all() and (out == 7).all()
    # beside one another, one gradient into two outputs, and a norm of one tensor twice
    clip_grads([buf[:400], buf[400:]], 1e9)
    o1, o2 = torch.empty_like(a), torch.empty_like(a)
    _, norm = clip_grads([a, a], 0.5, out=[o1, o2])
    assert torch.equal(o1, o2) and torch.equal(norm, grad_norm([a, a]))
    assert abs(norm.item() - 1200 ** 0.5) < 1e-4


def test_parameters_that_share_a_gradient():
    p, q = (torch.nn.Parameter(torch.zeros(100001, device="cuda")) for _ in range(2))
    g = torch.full((100001,), 2.0, device="cuda")
    for view in (False, True):
        p.grad, q.grad = g.clone(), None
        q.grad = p.grad[:] if view else p.grad
        want = 2.0 * 100001 ** 0.5
        norm = clip_grad_norm_([p, q], 1.0)
        assert abs(norm.item() - want) <= 1e-6 * want
        assert torch.allclose(p.grad, g / want, rtol=1e-6) and q.grad.data_ptr() == p.grad.data_ptr()
