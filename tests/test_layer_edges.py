"""The layer operators at the edges of their types.  The tolerances are those of the operators' own tests (test_layer_ops,
test_layer_moe), or derived where they stand."""
import copy

import pytest
import torch

import larql_b200
from test_layer_moe import Layer, check, tokens
from test_layer_ops import TYPES, U, check_norm, gen, half_step, norm_args, norm_case

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


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("mask", ["inf", "lowest"])
def test_masked_experts_weigh_nothing(be, kind, renorm, mask):
    """Experts switched off by a bias of minus infinity, or of the type's lowest value: weight 0, and the others as if they were
    alone, with fewer and with more experts a token than there are unmasked ones."""
    off = [1, 2, 4, 5, 6]
    on = [0, 3, 7]
    low = -float("inf") if mask == "inf" else torch.finfo(TYPES[kind][0]).min
    for top_e, t in [(2, 1), (2, 9), (6, 9), (8, 40)]:
        layer = Layer(be, "mxfp4", 64, 64, 8, top_e, kind, True, renorm, seed=3)
        layer.bias[off] = low
        x = tokens(gen(t), t, 64, kind)
        out, idx, w = layer.run(be, x)
        alone = copy.copy(layer)
        alone.w = [[per[e] for e in on] for per in layer.w]
        alone.router, alone.bias, alone.experts, alone.k = layer.router[on], layer.bias[on], 3, min(top_e, 3)
        want, widx, ww, w_off, o = alone.want(x)
        logits = (x.cpu().double() @ layer.router.cpu().double().t() + layer.bias.cpu().double()).float().double()
        assert torch.equal(idx.cpu().long(), torch.argsort(-logits, dim=1, stable=True)[:, :layer.k])
        assert torch.equal(idx[:, :alone.k].cpu().long(), torch.tensor(on)[widx])
        assert ((w[:, :alone.k].cpu().double() - ww).abs() <= w_off + U * ww).all()
        assert (w[:, alone.k:] == 0).all()
        err = (out[:t].cpu().double() - want).abs()
        assert (err <= half_step(kind, want) + o * (1 + 2.0 ** -8) + 1e-44).all()
        assert (out[t:] == 3).all()


@gpu
@pytest.mark.parametrize("renorm", [True, False])
def test_layer_with_every_expert_masked_is_nan(be, renorm):
    """softmax over minus infinities alone; a token with an infinity stays NaN beside masked experts."""
    layer = Layer(be, "mxfp4", 64, 64, 4, 2, "f32", True, renorm, seed=3)
    layer.bias[1:3] = -float("inf")
    x = tokens(gen(2), 3, 64, "f32")
    x[1, 7] = float("inf")
    out, _, w = layer.run(be, x)
    assert out[1].isnan().all() and w[1].isnan().all()
    assert out[[0, 2]].isfinite().all() and w[[0, 2]].isfinite().all()
    layer.bias[:] = -float("inf")
    out, _, w = layer.run(be, tokens(gen(2), 3, 64, "f32"))
    assert out[:3].isnan().all() and w.isnan().all()


@gpu
def test_graph_outlives_its_layer():
    """A graph that holds a layer's call is replayed after the handle was destroyed: the workspace it works in is still there,
    and its counters in order, until the context goes."""
    b = larql_b200.CudaBackend(0)
    try:
        layer = Layer(b, "mxfp4", 512, 96, 8, 2, "bf16", False, True, 5)
        x, out = tokens(gen(1), 20, 512, "bf16"), torch.empty(20, 512, dtype=torch.bfloat16, device="cuda")
        call = lambda: b.dev_moe_ffn(layer.layer, x.data_ptr(), larql_b200.T_BF16, 20, out.data_ptr())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(b.stream()), capture_error_mode="thread_local"):
            assert call()
        assert call()
        b.synchronize()
        want = out.clone()
        layer.layer.close()
        other = [Layer(b, "mxfp4", 512, 96, 8, 2, "bf16", False, True, 6) for _ in range(3)]  # (what was freed would be theirs)
        for o in other:
            o.run(b, x)
        out.zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del graph
    finally:
        b.close()


@gpu
@pytest.mark.parametrize("where,mode", [("library", "thread_local"), ("library", "global"), ("torch", "thread_local"), ("torch", "global")])
def test_layer_closed_during_a_capture(where, mode):
    """A handle destroyed while its own stream, or another one, is being captured (a garbage collector picks its time) neither
    ends the capture nor is lost."""
    b = larql_b200.CudaBackend(0)
    try:
        layer, other = (Layer(b, "mxfp4", 64, 96, 4, 2, "f32", False, True, 5 + i) for i in range(2))
        x = tokens(gen(1), 5, 64, "f32")
        want, out = layer.run(b, x)[0][:5], torch.zeros(5, 64, device="cuda")
        other.run(b, x)
        stream = torch.cuda.ExternalStream(b.stream()) if where == "library" else torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode=mode):
            if where == "library":
                assert b.dev_moe_ffn(layer.layer, x.data_ptr(), larql_b200.T_F32, 5, out.data_ptr())
            else:
                out.copy_(want)
            other.layer.close()
        again = Layer(b, "mxfp4", 64, 96, 4, 2, "f32", False, True, 6)
        check(again, x, again.run(b, x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        b.synchronize()
        del graph
    finally:
        b.close()


@gpu
@pytest.mark.parametrize("kind,t", [("f32", 1), ("f32", 9), ("bf16", 9)])
def test_moe_layer_scales_over_many_octaves(be, kind, t):
    """MXFP4 scales of 2^-43 to 2^29, as far as no f32 in between overflows (at most 64 x 6 x 4 x 2^29 a product, 2^117 an
    output): the formula's results, not only finite ones."""
    layer = Layer(be, "mxfp4", 64, 64, 3, 2, kind, False, True, 8, spread=36)
    x = tokens(gen(t), t, 64, kind).clamp_(-4, 4)
    check(layer, x, layer.run(be, x))


@gpu
@pytest.mark.parametrize("shift,down_shift,x_shift", [(101, 0, -94), (0, 101, 0), (-117, 0, 117), (0, -117, 0)])
def test_moe_layer_scales_at_the_ends(be, shift, down_shift, x_shift):
    """MXFP4 scales of 2^92 to 2^96, above which a sum may leave f32's range, and of 2^-126 to 2^-122, on tokens that keep the
    activation in range."""
    layer = Layer(be, "mxfp4", 64, 64, 3, 2, "f32", True, True, 8)
    layer.router.zero_()
    for i, s in enumerate((shift, shift, down_shift)):
        for e in range(3):
            layer.keep[2 * (3 * i + e) + 1] += s
            layer.w[i][e] = (*layer.w[i][e][:3], layer.w[i][e][3] * 2.0 ** s)
    scales = torch.stack([layer.keep[2 * m + 1] for m in range(9)]).cpu()
    assert 1 <= scales.min() and scales.max() <= 223
    x = tokens(gen(5), 7, 64, "f32").clamp_(-4, 4) * 2.0 ** x_shift
    check(layer, x, layer.run(be, x))


@gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "fp8"])
def test_layers_made_one_after_another_in_the_same_memory(be, fmt):
    """Layers made, run and destroyed in turn: the table and the tensor maps of each mostly lie where the last one's did, and
    describe other matrices of other sizes."""
    for i in range(12):
        hidden, inter = (256, 96) if i % 3 else (96, 256)
        layer = Layer(be, fmt, hidden, inter, 6, 2, "bf16", False, True, 40 + i)
        x = tokens(gen(i), 1 + 3 * (i % 4), hidden, "bf16")
        check(layer, x, layer.run(be, x))
        layer.layer.close()


# ----------------------------------------------------------- block norm ----
BIG = torch.finfo(torch.float32).max


def large_rows(cols, g):
    """f32 rows whose squares leave the type's range, up to the values at its end."""
    r = torch.randn(8, cols, generator=g)
    r[0] = torch.where(r[0] < 0, -BIG, BIG)      # the largest values throughout
    r[1, 0], r[1, 1:] = -BIG, 1.0                # the lowest value, as a mask writes it, beside ordinary ones
    r[2] = r[2].clamp(-3, 3) * 1e38
    r[3] *= 1e37
    r[3, cols // 2] = -BIG
    r[4] *= 1e30
    r[5] *= 1e20
    r[6] = r[6].abs() * 3.0e37 + 1.0e38          # 1 / rms subnormal
    return r


@gpu
@pytest.mark.parametrize("weight", [1.0, 1e-3, 1e-8, 1e3])
@pytest.mark.parametrize("rows,cols", [(8, 256), (300, 200), (8, 512), (8, 2885), (8, 4096), (1300, 4096), (8, 16384), (1300, 2880)])
@pytest.mark.parametrize("post", [True, False])
def test_block_norm_at_the_end_of_f32(be, rows, cols, weight, post):
    """Both norms, in every kernel (a warp a row, a block a row, blocks that walk many rows), of rows at the end of f32's range and
    with weights that a subnormal 1 / rms would lose bits with."""
    c = norm_case(rows, cols, "f32", "f32", post, "none", 0, 5, offset=0.0, y_scale=1.0)
    big, plain = ("y", "h") if post else ("h", "y")
    c[big][:8] = large_rows(cols, gen(cols)).cuda()
    c[plain].zero_()
    for k in ("post_w", "pre_w"):
        c[k].copy_(weight * (1 + 0.2 * torch.randn(cols, generator=gen(7))))
    h_out, n_out = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    check_norm(c, h_out, n_out)
    c[big][6, 3] = -float("inf")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    o = h_out if post else n_out
    assert o[6, 3].isnan() and (o[6, :3] == 0).all() and (o[6, 4:] == 0).all()


@gpu
@pytest.mark.parametrize("rows", [3, 1300])
def test_block_norm_n_beside_an_eps_beyond_f32(be, rows):
    """An eps of the size of squares that leave f32's range, in both norms: n to its bound."""
    c = norm_case(rows, 4096, "f32", "f32", True, "none", 0, 5, y_scale=1.0)
    c["h"].zero_()
    c["y"].mul_(1e18)  # sum of squares 4e39, mean 1e36
    c["eps"] = 1e36
    h_out, n_out = torch.empty(rows, 4096, device="cuda"), torch.empty(rows, 4096, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    check_norm(c, h_out, n_out)
