"""Weights after muon_step against 64 bits, the update made of the momenta that the step has stored: their rounding, checked by
itself, then needs no room in the weights' bound, which is that of a step with fp32 momenta (oracle/muon.py)."""
import pytest
import torch

from flashmlp_amd import muon_step
from oracle import muon as om

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32

# gram and apply of each padded size, by tiles and whole; a workgroup a matrix from end to end; both orientations
LISTS = {
    "one": [(64, 100)],
    "layer": [(6, 64, 200), (6, 64, 200), (6, 200, 64)],
    "mixed": [(2, 32, 50), (3, 128, 130), (1, 256, 300), (2, 300, 256), (5, 16, 7), (2, 70, 64), (100, 3)],
    "many": [(300, 40, 70), (400, 70, 40), (350, 64, 33), (350, 128, 140), (513, 20, 30), (3, 140, 128)],
    "wide": [(30, 129, 200), (7, 200, 131), (8, 256, 512), (1, 256, 1)],
    "many wide": [(40, 256, 260), (30, 201, 150)],
}


def stacks(shapes, types, seed):
    g = torch.Generator().manual_seed(seed)
    w = [torch.randn(s, generator=g).div(s[-2] ** 0.5).to(types[0]) for s in shapes]
    gr = [(10.0 ** -(i % 3) * torch.randn(s, generator=g)).to(types[1]) for i, s in enumerate(shapes)]
    m = [(10.0 ** -(i % 3) * 0.5 * torch.randn(s, generator=g)).to(types[2]) for i, s in enumerate(shapes)]
    return w, gr, m


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("types", [(BF, BF, BF), (FL, BF, BF), (HF, FL, HF), (HF, FL, BF), (FL, FL, FL)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_weights_take_the_update_of_the_stored_momenta(name, types, nesterov):
    w, g, m = stacks(LISTS[name], types, 17)
    dw, dg, dm = ([t.cuda() for t in v] for v in (w, g, m))
    muon_step(dw, dg, dm, 0.02, nesterov=nesterov, weight_decay=0.1)
    for i in range(len(w)):
        kept = dm[i].cpu()
        want = om.step64(w[i], g[i], m[i], 0.02, nesterov=nesterov, weight_decay=0.1, kept=kept)
        for t, got in (("w", dw[i].cpu()), ("m", kept)):
            ref, tol = want[t]
            tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -130
            assert ((got.double() - ref).abs() <= 1.01 * tol + tiny).all(), (i, t, ((got.double() - ref).abs() / tol).max().item())
