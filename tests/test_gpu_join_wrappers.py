"""A tensor that has no memory of its own (a wrapper around other tensors) among the join's inputs: refused, not taken for
one that is not there."""
import pytest
import torch

import flashmlp_amd.block as block
from flashmlp_amd import block_join, block_join_bwd, block_norm
from test_gpu_join import make

pytestmark = pytest.mark.gpu


class Wrapper(torch.Tensor):
    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func in (torch.ops.aten.detach.default, torch.ops.aten.alias.default):
            return args[0]
        raise NotImplementedError(str(func))


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("grad", [True, False])
def test_refused(monkeypatch, fast, grad):
    if not fast:
        monkeypatch.setattr(block, "_fast", None)
    t = make(20, 3, 32, 1, torch.float32, torch.float32)
    r, o, w, g, p = (t[k] for k in ("r", "o", "w_post", "gate", "w_pre"))
    rs = torch.ones(20, device="cuda")
    with torch.set_grad_enabled(grad):
        q = r.clone().requires_grad_(grad)
        calls = [lambda: block_join(q, Wrapper(o), w, g, pre_weight=p), lambda: block_join(q, o, Wrapper(w), g),
                 lambda: block_join(q, o, w, Wrapper(g)), lambda: block_join(q, o, pre_weight=Wrapper(p)),
                 lambda: block_join(Wrapper(r), o), lambda: block_norm(q, Wrapper(p)), lambda: block_norm(Wrapper(r)),
                 lambda: block_join(q, o, w, pre=False, gate=Wrapper(g)),
                 lambda: block_join_bwd(r, o, rs, rs, Wrapper(r), o, w, g, pre_weight=p),
                 lambda: block_join_bwd(r, o, rs, rs, r, Wrapper(o), w, g, pre_weight=p),
                 lambda: block_join_bwd(r, o, rs, rs, r, o, Wrapper(w), g, pre_weight=p)]
        for i, call in enumerate(calls):
            with pytest.raises(TypeError, match="memory of its own"):
                call()
                pytest.fail(f"call {i} went through")
