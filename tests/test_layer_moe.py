"""The whole mixture-of-experts layer (lq_moe_create, lq_dev_moe_ffn, lq_moe_ffn) against its formula in 64 bits, and
a decoder layer's tail made of the layer operators together.

The tolerance follows the arithmetic.  U = 2^-24.  A dot product: the activation as two f16 terms is off by at most
2^-23 of its value plus 2^-39 of the token's largest (bf16 activations fit one term: the 2^-39 alone); a block's 32 products
are summed in f32 by the tensor core, at most two U each, and the blocks and warps added in f32, one U each.  The
activation of a bf16 layer is rounded to f16 once (2^-12)."""
import ctypes as C

import numpy as np
import pytest
import torch

import larql_b200
from larql_b200 import build as lqbuild
from test_layer_ops import TYPES, U, check_norm, dev, fp8_matrix, fp8_tolerance, fp8_want, fp8_weight, gen, half_step, norm_args, norm_case, quantized

gpu = pytest.mark.gpu
FMTS = {"mxfp4": larql_b200.FMT_MXFP4, "nvfp4": larql_b200.FMT_NVFP4, "fp8": larql_b200.FMT_FP8_B128}
E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


@pytest.fixture(scope="module")
def be():
    b = larql_b200.CudaBackend(0)
    yield b
    b.close()


def random_weight(g, fmt, rows, cols, spread=2):
    """(codes, scales, tensor scale, the weight in f64): any code, scales over a few octaves."""
    if fmt == "fp8":
        q, s = fp8_weight(g, rows, cols)
        w = q.float().double() * s.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
        return q.view(torch.uint8), s, 1.0, w
    codes = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8)
    v = torch.stack((E2M1[(codes & 15).long()], E2M1[(codes >> 4).long()]), -1).view(rows, cols)
    if fmt == "mxfp4":
        s = torch.randint(120 - spread, 121 + spread, (rows, cols // 32), generator=g, dtype=torch.uint8)
        return codes, s, 1.0, v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    s = torch.randint(0, 0x7f, (rows, cols // 16), generator=g, dtype=torch.uint8)  # every positive e4m3 scale, zero too
    return codes, s, 2.0 ** -13, v * (s.view(torch.float8_e4m3fn).double() * 2.0 ** -13).repeat_interleave(16, 1)


class Layer:
    def __init__(self, be, fmt, hidden, inter, experts, top_e, kind="f32", bias=False, renorm=True, seed=0, spread=2):
        g = gen(seed)
        self.fmt, self.hidden, self.inter, self.experts, self.top_e, self.kind, self.renorm = fmt, hidden, inter, experts, top_e, kind, renorm
        self.w = [[random_weight(g, fmt, *((hidden, inter) if i == 2 else (inter, hidden)), spread) for _ in range(experts)] for i in range(3)]
        self.router = dev(torch.randn(experts, hidden, generator=g) * hidden ** -0.5, kind)
        self.bias = dev(torch.randn(experts, generator=g) * 0.3, kind) if bias else None
        self.mats, self.keep = [], []
        for per in self.w:
            self.mats.append([])
            for codes, scales, ts, _ in per:
                c, s = codes.cuda(), scales.cuda()
                self.keep += [c, s]
                self.mats[-1].append(larql_b200.DeviceMatrix(FMTS[fmt], c.shape[0], c.shape[1] * (1 if fmt == "fp8" else 2), c.data_ptr(),
                                                             c.numel(), s.data_ptr(), s.numel() * s.element_size(), ts))
        torch.cuda.synchronize()
        self.layer = be.moe_create(*self.mats, self.router.data_ptr(), TYPES[kind][1], self.bias.data_ptr() if bias else 0, top_e, renorm)
        assert self.layer is not None
        self.k = min(top_e, experts)

    def run(self, be, x, out=None):
        t = x.shape[0]
        out = torch.full((t + 1, self.hidden), 3.0, dtype=x.dtype, device="cuda") if out is None else out
        idx = torch.full((t + 1, self.k), -1, dtype=torch.int32, device="cuda")
        w = torch.full((t + 1, self.k), -1.0, device="cuda")
        torch.cuda.synchronize()
        assert be.dev_moe_ffn(self.layer, x.data_ptr(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype], t, out.data_ptr(),
                              idx.data_ptr(), w.data_ptr())
        be.synchronize()
        assert (idx[t:] == -1).all() and (w[t:] == -1).all()
        return out, idx[:t], w[:t]

    def want(self, x):
        """(out, idx, w) in f64 and the bound on |out - want| before the final rounding."""
        x = x.cpu().double()
        logits = x @ self.router.cpu().double().t()
        if self.bias is not None:
            logits = logits + self.bias.cpu().double()
        logits = logits.float().double()
        idx = torch.argsort(-logits, dim=1, stable=True)[:, :self.k]
        p = torch.softmax(logits, 1).gather(1, idx)
        w = p / p.sum(1, keepdim=True) if self.renorm else p
        # expf, the f32 sum over the experts, a division; the exponent's argument is off by U of its size
        w_off = w * U * (16 + self.experts + 2 * (logits.amax(1) - logits.amin(1)))[:, None]
        out, off = torch.zeros_like(x), torch.zeros_like(x)
        tx, ta = {"f32": (2.0 ** -23, 2.0 ** -23), "f16": (0.0, 2.0 ** -23), "bf16": (0.0, 2.0 ** -12)}[self.kind]

        def dot(a, a_off, m, t):
            """a . m^T for rows a with errors a_off; the bound on the result."""
            am = m.abs().t()
            big = a.abs().amax(1, keepdim=True) * 2.0 ** -39
            n = 64 + 2 * (m.shape[1] // 32) + 16
            return a @ m.t(), (a_off + t * a.abs() + big) @ am + n * U * (a.abs() @ am)

        for e in range(self.experts):
            t, j = torch.nonzero(idx == e, as_tuple=True)
            if t.numel():
                gate, up, down = (self.w[i][e][3] for i in range(3))
                g, g_off = dot(x[t], torch.zeros_like(x[t]), gate, tx)
                u, u_off = dot(x[t], torch.zeros_like(x[t]), up, tx)
                s = g * torch.sigmoid(g)
                a = s * u
                a_off = 1.1 * g_off * (u.abs() + u_off) + s.abs() * u_off + 8 * U * a.abs()
                d, d_off = dot(a, a_off, down, ta)
                wt = w[t, j][:, None]
                out.index_add_(0, t, wt * d)
                off.index_add_(0, t, wt * d_off + (w_off[t, j][:, None] + 2 * self.k * U * wt) * (a.abs() @ down.abs().t()))
        return out, idx, w, w_off, off


def check(layer, x, got):
    out, idx, w = got
    want, widx, ww, w_off, off = layer.want(x)
    assert torch.equal(idx.cpu().long(), widx)
    assert ((w.cpu().double() - ww).abs() <= w_off + U * ww).all()
    t = x.shape[0]
    err = (out[:t].cpu().double() - want).abs()
    assert (err <= half_step(layer.kind, want) + off * (1 + 2.0 ** -8) + 1e-44).all(), (err - off).max()
    if out.shape[0] > t:
        assert (out[t:] == 3).all()


def tokens(g, t, hidden, kind):
    return dev(torch.randn(t, hidden, generator=g), kind)


def test_null_context_is_an_argument_error():
    lqbuild.build()
    lib = larql_b200.load_library()
    m, h = larql_b200.LqMatrix(), C.c_void_p(5)
    assert lib.lq_moe_create(None, C.byref(m), C.byref(m), C.byref(m), 1, None, 0, None, 1, 1, C.byref(h)) == larql_b200.LQ_ERR_ARGUMENT
    assert h.value is None
    assert lib.lq_dev_moe_ffn(None, None, None, 0, 1, None, None, None) == larql_b200.LQ_ERR_ARGUMENT
    assert lib.lq_moe_ffn(None, None, None, 0, 1, None, None, None) == larql_b200.LQ_ERR_ARGUMENT
    lib.lq_moe_destroy(None, None)


CASES = [
    # fmt, hidden, inter, experts, top_e, kind, bias, renorm, tokens
    ("mxfp4", 32, 32, 1, 1, "f32", False, True, 1), ("mxfp4", 64, 96, 4, 2, "f32", True, False, 3), ("mxfp4", 2880, 320, 8, 4, "f32", True, True, 1),
    ("mxfp4", 320, 2880, 5, 2, "bf16", False, True, 7), ("mxfp4", 1056, 1120, 3, 3, "f16", True, True, 13),
    ("nvfp4", 32, 64, 3, 2, "f32", False, True, 2), ("nvfp4", 1024, 1056, 6, 3, "f32", True, True, 5), ("nvfp4", 2880, 160, 33, 6, "bf16", True, False, 20),
    ("nvfp4", 4128, 64, 4, 2, "f16", False, True, 9), ("fp8", 32, 32, 2, 2, "f32", False, False, 4), ("fp8", 544, 800, 7, 5, "bf16", True, True, 37),
    ("fp8", 1312, 160, 64, 6, "f32", False, True, 33), ("fp8", 160, 1312, 3, 1, "f16", True, True, 64), ("mxfp4", 256, 128, 256, 8, "f32", True, True, 11),
    ("fp8", 128, 64, 40, 32, "f32", False, True, 35), ("mxfp4", 96, 64, 4, 9, "bf16", True, True, 130), ("nvfp4", 64, 64, 2, 1, "f32", True, True, 65),
    ("mxfp4", 8192, 64, 3, 2, "f32", False, True, 6), ("fp8", 64, 8192, 2, 1, "bf16", False, True, 20), ("nvfp4", 4096, 32, 2, 2, "f32", False, True, 17),
]


@gpu
@pytest.mark.parametrize("case", CASES)
def test_moe_layer_matches_the_formula(be, case):
    *shape, t = case
    layer = Layer(be, *shape, seed=len(str(case)) + t)
    x = tokens(gen(t), t, layer.hidden, layer.kind)
    check(layer, x, layer.run(be, x))


@gpu
def test_moe_layer_repeats_bit_for_bit_and_in_place(be):
    layer = Layer(be, "mxfp4", 2880, 288, 16, 4, "f32", True, True, 3)
    x = tokens(gen(1), 19, 2880, "f32")
    first = layer.run(be, x)
    for _ in range(5):
        again = layer.run(be, x)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    y = x.clone()
    layer.run(be, y, out=y)
    assert torch.equal(y, first[0][:19])


@gpu
def test_moe_layer_ties_go_to_the_lower_expert(be):
    layer = Layer(be, "fp8", 64, 64, 40, 3, seed=2)
    layer.router[7] = layer.router[3]
    layer.router[39] = layer.router[3]
    layer.router[20] = layer.router[3]
    x = tokens(gen(3), 8, 64, "f32")
    x[0] = layer.router[3].float() * 50  # the four equal experts lead: 3, 7, 20
    got = layer.run(be, x)
    assert got[1][0].tolist() == [3, 7, 20]
    check(layer, x, got)


@gpu
def test_moe_layer_all_tokens_on_one_expert(be):
    """Many groups of one expert, none of the others: a router bias far above the rest."""
    layer = Layer(be, "nvfp4", 96, 160, 5, 1, "f32", True, True, 6)
    layer.bias.fill_(-50)
    layer.bias[4] = 50
    x = tokens(gen(9), 61, 96, "f32")
    got = layer.run(be, x)
    assert (got[1] == 4).all()
    check(layer, x, got)


@gpu
def test_moe_layer_extreme_values(be):
    """Tokens of zeros, very large and very small tokens, scales at the ends of their range, a NaN and an infinity that
    stay with their token."""
    layer = Layer(be, "mxfp4", 64, 64, 3, 2, "f32", False, True, 8)
    x = tokens(gen(4), 9, 64, "f32")
    x[0] = 0
    x[1] *= 1e12
    x[2] *= 1e-30
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    out, idx, w = layer.run(be, x)
    assert (out[0] == 0).all()
    assert out[3].isnan().all() and out[4].isnan().all() and w[3].isnan().all()
    good = [0, 2, 5, 6, 7, 8]
    check(layer, x[good], (out[good], idx[good], w[good]))
    # the large token: silu(gate) is gate or 0 to f32's precision; relative to its own size
    want, _, _, _, off = layer.want(x[[1]])
    assert ((out[[1]].cpu().double() - want).abs() <= half_step("f32", want) + off * 1.01).all()
    far = Layer(be, "mxfp4", 64, 64, 2, 2, "f32", False, True, 8, spread=60)
    x = tokens(gen(5), 3, 64, "f32")
    out, idx, w = far.run(be, x)
    want = far.want(x)[0]
    ok = want.abs() < 1e38
    assert ok.any() and torch.isfinite(out[:3].cpu()[ok]).all()


@gpu
def test_moe_layer_host_call_and_none(be):
    layer = Layer(be, "mxfp4", 128, 96, 6, 2, "f32", True, True, 12)
    x = tokens(gen(2), 5, 128, "f32")
    out, idx, w = be.moe_ffn(layer.layer, x.cpu().numpy())
    check(layer, x, (torch.from_numpy(out), torch.from_numpy(idx.astype(np.int64)), torch.from_numpy(w)))
    assert be.moe_ffn(layer.layer, np.zeros((2, 64), np.float32)) is None
    assert be.moe_ffn(layer.layer, np.zeros((0, 128), np.float32))[0].shape == (0, 128)
    none = Layer(be, "mxfp4", 128, 96, 6, 0, seed=12)
    out = torch.full((3, 128), 9.0, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_moe_ffn(none.layer, x.data_ptr(), 0, 3, out.data_ptr())
    be.synchronize()
    assert (out == 0).all()


@gpu
def test_moe_layer_in_a_captured_graph(be):
    layer = Layer(be, "fp8", 256, 128, 8, 2, "bf16", False, True, 5)
    x, out = torch.zeros(70, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(70, 256, dtype=torch.bfloat16, device="cuda")
    idx, w = torch.empty(70, 2, dtype=torch.int32, device="cuda"), torch.empty(70, 2, device="cuda")
    call = lambda: be.dev_moe_ffn(layer.layer, x.data_ptr(), larql_b200.T_BF16, 70, out.data_ptr(), idx.data_ptr(), w.data_ptr())
    torch.cuda.synchronize()
    assert call()
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream()), capture_error_mode="thread_local"):
        assert call()
    for i in range(3):
        x.copy_(tokens(gen(30 + i), 70, 256, "bf16"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(layer, x, (out, idx, w))


@gpu
def test_moe_refusals(be):
    a = Layer(be, "mxfp4", 64, 96, 2, 1, seed=1)
    r = a.router.data_ptr()
    g, u, d = a.mats
    assert be.moe_create(g, u, u, r, 0, 0, 1) is None                     # down is not [hidden, inter]
    assert be.moe_create(g, u[:1], d, r, 0, 0, 1) is None and be.moe_create([], [], [], r, 0, 0, 1) is None
    assert be.moe_create(g, u, d, r, 9, 0, 1) is None                     # router type
    n = Layer(be, "nvfp4", 64, 96, 2, 1, seed=1)
    assert be.moe_create(g, n.mats[1], d, r, 0, 0, 1) is None             # mixed formats
    q8 = larql_b200.DeviceMatrix(larql_b200.FMT_Q8_0, 96, 64, r, 96 * 68)
    assert be.moe_create([q8], [q8], [q8], r, 0, 0, 1) is None
    nan = a.keep[1].clone()
    nan[95, 1] = 255
    torch.cuda.synchronize()
    bad = larql_b200.DeviceMatrix(larql_b200.FMT_MXFP4, 96, 64, g[0].data_ptr, g[0].data_len, nan.data_ptr(), nan.numel())
    assert be.moe_create([g[0], bad], u, d, r, 0, 0, 1) is None           # an e8m0 NaN
    big = larql_b200.DeviceMatrix(larql_b200.FMT_MXFP4, 8224, 32, r & ~15, 8224 * 16, r & ~15, 8224)
    down = larql_b200.DeviceMatrix(larql_b200.FMT_MXFP4, 32, 8224, r & ~15, 8224 * 16, r & ~15, 8224)
    assert be.moe_create([big], [big], [down], r, 0, 0, 1) is None
    odd = larql_b200.DeviceMatrix(larql_b200.FMT_NVFP4, 48, 48, r & ~15, 48 * 24, r & ~15, 48 * 3)
    assert be.moe_create([odd], [odd], [odd], r, 0, 0, 1) is None
    many = Layer(be, "mxfp4", 32, 32, 64, 1, seed=1)
    assert be.moe_create(*many.mats, many.router.data_ptr(), 0, 0, 33) is None
    host = larql_b200.HostMatrix(larql_b200.FMT_MXFP4, 32, 32, np.zeros(32 * 16, np.uint8), np.zeros(32, np.uint8))
    for bad in [lambda: be.moe_create([host], [host], [host], r, 0, 0, 1), lambda: be.moe_create(g, u, d, 0, 0, 0, 1),
                lambda: be.moe_create(g, u, d, r + 2, 0, 0, 1),
                lambda: be.moe_create([larql_b200.DeviceMatrix(larql_b200.FMT_MXFP4, 96, 64, g[0].data_ptr + 8, 96 * 32, g[0].scales_ptr, 192)], u[:1], d[:1], r, 0, 0, 1)]:
        with pytest.raises(larql_b200.BackendError):
            bad()
    x = torch.zeros(2, 64, device="cuda")
    assert be.dev_moe_ffn(a.layer, x.data_ptr(), 3, 2, x.data_ptr()) is False
    assert be.dev_moe_ffn(a.layer, 0, 0, 0, 0)  # no tokens: nothing to do
    with pytest.raises(larql_b200.BackendError):
        be.dev_moe_ffn(a.layer, 0, 0, 2, x.data_ptr())
    other = larql_b200.CudaBackend(0)
    try:
        with pytest.raises(larql_b200.BackendError):
            other.dev_moe_ffn(a.layer, x.data_ptr(), 0, 2, x.data_ptr())
    finally:
        other.close()
    a.layer.close()
    a.layer.close()


@gpu
@pytest.mark.parametrize("t", [1, 6, 150])
def test_the_tail_of_a_decoder_runs_together(be, t):
    """norm -> mixture-of-experts layer -> norm behind it, gate, residual and the final norm -> FP8 LM head, enqueued back to
    back; every step is checked against its formula on the inputs it really had."""
    hidden, kind = 2880, "bf16"
    layer = Layer(be, "mxfp4", hidden, 160, 6, 2, kind, True, True, 21)
    c = norm_case(t, hidden, kind, "f32", False, "none", 0, 4)
    c["h"], c["y"] = dev(torch.randn(t, hidden, generator=gen(5)), kind), torch.zeros(t, hidden, dtype=torch.bfloat16, device="cuda")
    new = lambda n=hidden: torch.empty(t, n, dtype=torch.bfloat16, device="cuda")
    n1, y, h2, n2, logits = new(), new(), new(), new(), new(1000)
    idx, w = torch.empty(t, 2, dtype=torch.int32, device="cuda"), torch.empty(t, 2, device="cuda")
    wq, ws = fp8_weight(gen(6), 1000, hidden)
    head = fp8_matrix(wq.cuda(), ws.cuda())
    after = dict(norm_case(t, hidden, kind, "f32", True, "channel", 0, 7, y_scale=0.8), h=c["h"], y=y)
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, None, n1, use_y=False))
    assert be.dev_moe_ffn(layer.layer, n1.data_ptr(), larql_b200.T_BF16, t, y.data_ptr(), idx.data_ptr(), w.data_ptr())
    assert be.dev_block_norm(norm_args(after, h2, n2))
    assert be.dev_fp8_matmul(head, n2.data_ptr(), larql_b200.T_BF16, t, hidden, logits.data_ptr(), larql_b200.T_BF16, 1000)
    be.synchronize()
    check_norm(c, None, n1, use_y=False)
    check(layer, n1, (y, idx, w))
    check_norm(after, h2, n2)
    want, mag = fp8_want(*quantized(n2.float().cpu()), wq, ws)
    assert ((logits.cpu().double() - want).abs() <= fp8_tolerance(kind, want, mag, hidden)).all()
