"""FlashMLP for AMD Instinct MI355X (gfx950).

Fused multi-head MLP  O = act(X W1) W2  with a recomputing backward, as hand-written HIP
kernels behind a C ABI (include/flashmlp.h, libflashmlp.so). The Python API mirrors the
reference module `flashmlp`:

    from flashmlp_amd import flashmlp_fwd, flashmlp_bwd, FlashMLPFunction, FlashMLP, PyTorchMLP

`flashmlp_amd.flashmlp` (torch.ops.flashmlp_amd.fwd / .bwd) is the same computation as a
registered torch.library operator, for torch.compile and FakeTensor tracing.

A gated block built around it has the gated form  O = (act(X Wg) * (X Wu)) W2  (flashmlp_gated_fwd,
flashmlp_gated_bwd, GatedFlashMLPFunction, GatedFlashMLP), the norms, gate and residual
around it (block_norm, block_join) and the clipping of its gradients (grad_norm, clip_grads,
clip_grad_norm_). Its heads serve as experts that tokens choose (expert_route, expert_plan, expert_dispatch,
expert_combine, GatedExperts), and its stacks of weights are orthogonalised and stepped by orthogonalize and
muon_step.
"""
from .flashmlp import FlashMLP, FlashMLPFunction, flashmlp_bwd, flashmlp_fwd
from .baseline import PyTorchMLP, flashmlp_torch_bwd, flashmlp_torch_fwd
from .gated import GatedFlashMLP, GatedFlashMLPFunction, flashmlp_gated_bwd, flashmlp_gated_fwd
from .block import BlockJoinFunction, block_join, block_join_bwd, block_join_fwd, block_norm
from .clip import clip_grad_norm_, clip_grads, grad_norm
from .experts import ExpertPlan, GatedExperts, expert_combine, expert_dispatch, expert_plan, expert_route
from .muon import muon_step, orthogonalize
from . import ops
from .ops import flashmlp

__all__ = [
    "flashmlp_fwd",
    "flashmlp_bwd",
    "FlashMLPFunction",
    "FlashMLP",
    "PyTorchMLP",
    "flashmlp_torch_fwd",
    "flashmlp_torch_bwd",
    "flashmlp",
    "ops",
    "flashmlp_gated_fwd",
    "flashmlp_gated_bwd",
    "GatedFlashMLPFunction",
    "GatedFlashMLP",
    "block_norm",
    "block_join",
    "block_join_fwd",
    "block_join_bwd",
    "BlockJoinFunction",
    "grad_norm",
    "clip_grads",
    "clip_grad_norm_",
    "expert_route",
    "expert_plan",
    "ExpertPlan",
    "expert_dispatch",
    "expert_combine",
    "GatedExperts",
    "orthogonalize",
    "muon_step",
]
