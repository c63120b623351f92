"""A stack of mixtures of gated experts that learns: routing, the sort by expert, the experts' gated MLP, the norms, gate and
residual around it, the clipping of its gradients and Muon on its stacks of weights, as a training program uses them together.

    python examples/expert_stack.py [--layers 2 --heads 4 --dim 64 --hidden 128 --experts 8 --rows 1024 --steps 50]

Each layer is  x = x + scale * gate * norm(mixture(norm(x)))  on a stream of heads x dim columns; every head's part of a row is a
token that takes two experts of its own. The stack is fitted to a fixed random map with 16-bit weights, an fp32 stream, and
fp32 copies of the weights: matrices (routers and experts) by muon_step, vectors by plain momentum.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from flashmlp_amd import GatedExperts, block_join, block_norm, clip_grads, muon_step  # noqa: E402


class ExpertStack(torch.nn.Module):
    """L mixtures on rows of heads x dim columns; the output is the last block's normalised stream."""

    def __init__(self, layers, heads, dim, hidden, experts, dtype=torch.bfloat16, device="cuda", scale=1.0, capacity_factor=1.5):
        super().__init__()
        cols = heads * dim
        self.heads, self.scale = heads, scale

        def vector(value):
            return torch.nn.Parameter(torch.full((cols,), value, dtype=dtype, device=device))

        self.mixtures = torch.nn.ModuleList(GatedExperts(experts, dim, hidden, 2, capacity_factor, dtype=dtype, device=device)
                                            for _ in range(layers))
        self.pre = torch.nn.ParameterList(vector(1.0) for _ in range(layers + 1))  # the last one: the output's norm
        self.post = torch.nn.ParameterList(vector(1.0) for _ in range(layers))
        self.gate = torch.nn.ParameterList(vector(0.5) for _ in range(layers))

    def forward(self, x):
        """x (rows, heads x dim), fp32 or the weights' dtype -> (rows, heads x dim) in the weights' dtype"""
        y = block_norm(x, self.pre[0], heads=self.heads)
        for mixture, post, gate, pre in zip(self.mixtures, self.post, self.gate, self.pre[1:]):
            x, y = block_join(x, mixture(y), post, gate, self.scale, pre_weight=pre)
        return y.transpose(0, 1).reshape(x.shape)


class MuonAndMomentum:
    """fp32 copies of the parameters and of their clipped gradients: Muon on matrices, momentum on vectors."""

    def __init__(self, params, lr, lr_vectors, max_norm):
        self.params, self.lr, self.lr_vectors, self.max_norm = list(params), lr, lr_vectors, max_norm
        fp32 = lambda p: p.detach().float().clone()  # noqa: E731
        self.master = [fp32(p) for p in self.params]
        self.grads = [torch.empty_like(m) for m in self.master]
        self.momenta = [torch.zeros_like(m) for m in self.master]
        self.matrices = [i for i, p in enumerate(self.params) if p.dim() > 1]
        self.vectors = [i for i, p in enumerate(self.params) if p.dim() == 1]

    @torch.no_grad()
    def step(self):
        _, norm = clip_grads([p.grad for p in self.params], self.max_norm, out=self.grads)
        pick = lambda ts, at: [ts[i] for i in at]  # noqa: E731
        muon_step(pick(self.master, self.matrices), pick(self.grads, self.matrices), pick(self.momenta, self.matrices), self.lr)
        for i in self.vectors:
            self.momenta[i].mul_(0.9).add_(self.grads[i])
            self.master[i].sub_(self.momenta[i], alpha=self.lr_vectors)
        torch._foreach_copy_(self.params, self.master)
        for p in self.params:
            p.grad = None
        return norm


def train(model, rows, steps, lr=0.02, lr_vectors=0.1, max_norm=0.1, seed=0):
    """Losses and gradient norms of `steps` steps towards a fixed random map."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols = model.pre[0].numel()
    x = torch.randn(rows, cols, generator=g, device="cuda")
    mix = torch.randn(cols, cols, generator=g, device="cuda") / cols ** 0.5
    target = torch.tanh(x @ mix)
    opt = MuonAndMomentum(model.parameters(), lr, lr_vectors, max_norm)
    losses, norms = [], []
    for _ in range(steps):
        loss = (model(x).float() - target).square().mean()
        loss.backward()
        norms.append(opt.step())
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 2), ("heads", 4), ("dim", 64), ("hidden", 128), ("experts", 8), ("rows", 1024), ("steps", 50)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    torch.manual_seed(0)
    model = ExpertStack(a.layers, a.heads, a.dim, a.hidden, a.experts)
    losses, norms = train(model, a.rows, a.steps)
    for i in sorted({0, a.steps // 4, a.steps // 2, a.steps - 1}):
        print(f"step {i}: loss {losses[i]:.4f}, gradient norm {norms[i]:.4f}")
    with torch.no_grad():
        y = model(torch.randn(1, a.heads * a.dim, device="cuda"))
    print(f"one row alone: rms {y.float().square().mean().sqrt().item():.3f}")


if __name__ == "__main__":
    main()
