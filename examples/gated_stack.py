"""A stack of gated blocks that learns: the gated MLP, the norms, gate and residual around it, and the clipping
of its gradients, as a training program and a token-by-token one use them together.

    python examples/gated_stack.py [--layers 4 --heads 8 --dim 64 --hidden 256 --rows 2048 --steps 50]

Each layer is  x = x + scale * gate * norm(mlp(norm(x)))  on a stream of heads x dim columns; one block_join
joins a layer's output to the stream and takes the next layer's input from it. The stack is fitted to a fixed
random map with 16-bit weights, an fp32 stream, gradients clipped into one fp32 buffer and plain momentum on fp32
copies of the weights.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from flashmlp_amd import GatedFlashMLP, block_join, block_norm, clip_grads  # noqa: E402


class GatedStack(torch.nn.Module):
    """L gated blocks on rows of heads x dim columns; the output is the last block's normalised stream."""

    def __init__(self, layers, heads, dim, hidden, dtype=torch.bfloat16, device="cuda", scale=1.0):
        super().__init__()
        cols = heads * dim
        self.heads, self.scale = heads, scale

        def vector(value):
            return torch.nn.Parameter(torch.full((cols,), value, dtype=dtype, device=device))

        self.mlps = torch.nn.ModuleList(GatedFlashMLP(heads, dim, hidden, dtype=dtype, device=device)
                                        for _ in range(layers))
        self.pre = torch.nn.ParameterList(vector(1.0) for _ in range(layers + 1))  # the last one: the output's norm
        self.post = torch.nn.ParameterList(vector(1.0) for _ in range(layers))
        self.gate = torch.nn.ParameterList(vector(0.5) for _ in range(layers))

    def forward(self, x):
        """x (rows, heads x dim), fp32 or the weights' dtype -> (rows, heads x dim) in the weights' dtype"""
        y = block_norm(x, self.pre[0], heads=self.heads)
        for mlp, post, gate, pre in zip(self.mlps, self.post, self.gate, self.pre[1:]):
            x, y = block_join(x, mlp(y), post, gate, self.scale, pre_weight=pre)
        return y.transpose(0, 1).reshape(x.shape)


class Momentum:
    """Momentum on fp32 copies of the parameters, their gradients clipped into one fp32 buffer."""

    def __init__(self, params, lr, max_norm, beta=0.9):
        self.params, self.lr, self.max_norm, self.beta = list(params), lr, max_norm, beta
        sizes = [p.numel() for p in self.params]
        self.master = torch.cat([p.detach().float().flatten() for p in self.params])
        self.velocity = torch.zeros_like(self.master)
        self.buffer = torch.empty_like(self.master)
        self.views = [v.view(p.shape) for v, p in zip(self.buffer.split(sizes), self.params)]
        self.master_views = [v.view(p.shape) for v, p in zip(self.master.split(sizes), self.params)]

    @torch.no_grad()
    def step(self):
        _, norm = clip_grads([p.grad for p in self.params], self.max_norm, out=self.views)
        self.velocity.mul_(self.beta).add_(self.buffer)
        self.master.sub_(self.velocity, alpha=self.lr)
        torch._foreach_copy_(self.params, self.master_views)
        for p in self.params:
            p.grad = None
        return norm


def train(model, rows, steps, lr=1.0, max_norm=0.08, seed=0):
    """Losses and gradient norms of `steps` steps towards a fixed random map."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols = model.pre[0].numel()
    x = torch.randn(rows, cols, generator=g, device="cuda")
    mix = torch.randn(cols, cols, generator=g, device="cuda") / cols ** 0.5
    target = torch.tanh(x @ mix)
    opt = Momentum(model.parameters(), lr, max_norm)
    losses, norms = [], []
    for _ in range(steps):
        loss = (model(x).float() - target).square().mean()
        loss.backward()
        norms.append(opt.step())
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


@torch.no_grad()
def generate(model, x, steps):
    """Feeds each row's output back in, one row per request and call: the single-token forms."""
    out = []
    for _ in range(steps):
        x = model(x).float()
        out.append(x)
    return torch.stack(out)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("heads", 8), ("dim", 64), ("hidden", 256), ("rows", 2048), ("steps", 50)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    torch.manual_seed(0)
    model = GatedStack(a.layers, a.heads, a.dim, a.hidden)
    losses, norms = train(model, a.rows, a.steps)
    for i in sorted({0, a.steps // 4, a.steps // 2, a.steps - 1}):
        print(f"step {i}: loss {losses[i]:.4f}, gradient norm {norms[i]:.4f}")
    out = generate(model, torch.randn(4, a.heads * a.dim, device="cuda"), 8)
    print(f"8 tokens of 4 requests: {tuple(out.shape)}, rms {out.square().mean().sqrt().item():.3f}")


if __name__ == "__main__":
    main()
