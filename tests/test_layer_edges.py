"""The layer operators at the edges of their types.  The tolerances are those of the operators' own tests (test_layer_ops,
test_layer_moe), or derived where they stand."""
import pytest
import torch

import larql_b200
from test_layer_moe import Layer
from test_layer_ops import TYPES, U, gen, half_step

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = larql_b200.CudaBackend(0)
    yield b
    b.close()


# ------------------------------------------------------------------ MoE ----
@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("fmt,hidden,inter,experts,t", [
    ("mxfp4", 256, 64, 1, 1), ("mxfp4", 512, 96, 2, 16), ("nvfp4", 256, 160, 2, 12), ("fp8", 256, 800, 8, 30), ("fp8", 256, 64, 2, 64),
    ("mxfp4", 512, 2880, 2, 30), ("mxfp4", 512, 8192, 2, 20), ("nvfp4", 128, 64, 3, 64)])
def test_layer_keeps_its_activation(be, fmt, hidden, inter, experts, t, kind):
    """The activation between the two products is not rounded to the layer's type, nor to f16's 11 bits.  One element of a token,
    and one of a row of down, are not zero, so that the products are single terms: what is off before the output's own rounding
    is silu(gate) * up (8 U), the activation's two f16 terms (2 U), the weights' scales, a multiplication each (3 U) and the
    softmax of one expert (exact).  Beside the pair's largest activation, which is brought to [2^14, 2^15), a term is rounded to f16's
    smallest step, 2^-24: half of it is at most 2^-39 of that largest one."""
    layer = Layer(be, fmt, hidden, inter, experts, 1, kind, False, True, seed=t)
    g = gen(t + 1)
    for e in range(experts):
        codes = layer.keep[2 * (2 * experts + e)]
        at = torch.randint(0, inter, (hidden,), generator=g)
        one = torch.zeros(hidden, inter, dtype=torch.bool)
        one[torch.arange(hidden), at] = True
        keep = one.to(torch.uint8) * 255 if fmt == "fp8" else one[:, 0::2].to(torch.uint8) * 15 + one[:, 1::2].to(torch.uint8) * 240
        codes &= keep.cuda()
        layer.w[2][e] = (*layer.w[2][e][:3], layer.w[2][e][3] * one)
    x = torch.zeros(t, hidden, dtype=TYPES[kind][0])
    x[torch.arange(t), torch.randint(0, hidden, (t,), generator=g)] = (torch.randn(t, generator=g) * 8).to(x.dtype)
    out, idx, w = layer.run(be, x.cuda())
    assert (w == 1).all()
    for i in range(t):
        gate, up, down = (layer.w[m][int(idx[i])][3] for m in range(3))
        a = x[i].double() @ gate.t()
        act = a * torch.sigmoid(a) * (x[i].double() @ up.t())
        want, small = act @ down.t(), act.abs().max() * 2.0 ** -39 * down.abs().sum(1)
        assert ((out[i].cpu().double() - want).abs() <= half_step(kind, want) + (16 * U * want.abs() + small) * (1 + 2.0 ** -8)).all()
