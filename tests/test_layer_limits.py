"""The layer operators at the limits of what they take: every way a product can be cut up, the kernels for many rows, offsets
past 32 bits, workspaces across graphs, contexts at work side by side.  The tolerances are those of the operators' own tests
(test_layer_ops, test_layer_moe), whose derivation does not depend on the sizes here."""
import pytest
import torch

import larql_b200
from test_layer_moe import Layer, check, tokens
from test_layer_ops import TYPES, U, check_norm, dev, fp8_matrix, fp8_weight, gen, norm_args, norm_case, quantized, run_fp8

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = larql_b200.CudaBackend(0)
    yield b
    b.close()


# ----------------------------------------------------------- block norm ----
STREAM_CASES = [
    # rows, cols, kind, weights, post, gate, pad: enough rows for the kernel that copies them ahead, and odd ones beside it
    (1500, 4096, "bf16", "bf16", True, "full", 0), (1301, 2880, "f32", "f32", True, "full", 0), (1201, 6144, "f16", "f32", True, "channel", 8),
    (1333, 8192, "bf16", "f32", False, "row", 16), (1209, 4096, "f32", "bf16", True, "none", 4), (1205, 16384, "bf16", "bf16", True, "full", 0),
    (1203, 16384, "f32", "f32", True, "none", 0), (1300, 2885, "f32", "f32", True, "full", 3), (1207, 4104, "bf16", "bf16", True, "full", 1),
]


@gpu
@pytest.mark.parametrize("case", STREAM_CASES)
def test_block_norm_of_many_long_rows(be, case):
    c = norm_case(*case, seed=len(str(case)))
    h_out, n_out = (torch.empty(c["rows"], c["cols"], dtype=TYPES[c["kind"]][0], device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    check_norm(c, h_out, n_out)


@gpu
def test_block_norm_of_many_rows_in_place_with_every_second_output(be):
    """Many rows: h_out over h and n_out over y, a gate row per group, then either output alone."""
    c = norm_case(1400, 4096, "bf16", "bf16", True, "group", 0, 2, group=7)
    keep = {k: c[k].clone() for k in ("h", "y")}
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, c["h"], c["y"]))
    be.synchronize()
    h_out, n_out = c["h"], c["y"]
    c.update(keep)
    check_norm(c, h_out, n_out)
    h2, n2 = torch.full_like(h_out, 7.0), torch.full_like(n_out, 7.0)
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h2, None)) and be.dev_block_norm(norm_args(c, None, n2))
    be.synchronize()
    assert torch.equal(h2, h_out) and torch.equal(n2, n_out)


@gpu
def test_block_norm_extremes_among_many_rows(be):
    c = norm_case(1300, 4096, "f32", "f32", True, "none", 0, 5, y_scale=1.0)
    c["h"].zero_()
    c["y"][0] = 0
    c["y"][1] *= 1e30
    c["y"][2] *= 1e-30
    c["y"][600, 17] = float("nan")
    c["y"][1299, 4095] = float("inf")
    h_out, n_out = torch.empty(1300, 4096, device="cuda"), torch.empty(1300, 4096, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    assert (h_out[0] == 0).all() and (n_out[0] == 0).all()
    assert h_out[600].isnan().all() and n_out[600].isnan().all()
    assert h_out[1299, 4095].isnan() and (h_out[1299, :4095] == 0).all()
    good = [1, 2, *range(3, 600), *range(601, 1299)]
    check_norm(dict(c, h=c["h"][good], y=c["y"][good], rows=len(good)), h_out[good], n_out[good])


@gpu
def test_block_norm_offsets_past_32_bits(be):
    """Three rows whose strides put the last one past 2^31 elements and 2^32 bytes."""
    stride, cols = (1 << 30) + 64, 520
    big = {k: torch.empty(2 * stride + cols, dtype=torch.bfloat16, device="cuda") for k in ("h", "y", "h_out", "n_out")}
    rows = {k: v.as_strided((3, cols), (stride, 1)) for k, v in big.items()}
    c = norm_case(3, cols, "bf16", "f32", True, "none", 0, 8)
    rows["h"].copy_(c["h"])
    rows["y"].copy_(c["y"])
    c.update(h=rows["h"], y=rows["y"])
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, rows["h_out"], rows["n_out"]))
    be.synchronize()
    check_norm(c, rows["h_out"], rows["n_out"])


@gpu
@pytest.mark.parametrize("rows", [3, 1300])
def test_block_norm_eps_beside_values_beyond_f32(be, rows):
    """Rows whose squares leave f32's range, and an eps of their size."""
    c = norm_case(rows, 4096, "f32", "f32", True, "none", 0, 5, y_scale=1.0)
    c["h"].zero_()
    c["y"].mul_(1e18)  # sum of squares 4e39, mean 1e36
    c["eps"] = 1e36
    h_out, n_out = torch.empty(rows, 4096, device="cuda"), torch.empty(rows, 4096, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    check_norm(c, h_out, None)
    assert (n_out.abs().amax() < 1e-17) and (n_out != 0).any()  # h' is near 1, eps far above its square


@gpu
def test_block_norm_of_the_most_rows(be):
    """2^31 - 1 rows of one element: the last step of the walk over the rows leaves int's range."""
    rows = 2 ** 31 - 1
    h = torch.ones(rows, dtype=torch.float16, device="cuda")
    out = torch.zeros(rows, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(larql_b200.BlockNormArgs(type=larql_b200.T_F16, w_type=larql_b200.T_F16, h_scale=3.0, y_scale=1.0, eps=1e-6, rows=rows,
                                                      cols=1, h=h.data_ptr(), h_stride=1, gate_group=1, h_out=out.data_ptr(), h_out_stride=1))
    be.synchronize()
    assert bool((out == 3).all())


# ------------------------------------------------------------------ FP8 ----
@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_fp8_quantize_of_many_blocks(be, kind):
    x = dev(torch.randn(333, 8200, generator=gen(2)) * 3, kind)[:, :8192]
    x[5, :256] = 0
    x[6] *= 1e-6
    q, s = torch.empty(333, 8192, dtype=torch.uint8, device="cuda"), torch.empty(333, 64, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_fp8_quantize(x.data_ptr(), TYPES[kind][1], 333, 8192, x.stride(0), q.data_ptr(), s.data_ptr())
    be.synchronize()
    wq, ws = quantized(x.float().cpu())
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq.view(torch.uint8))


@gpu
def test_fp8_quantize_offsets_past_32_bits(be):
    """Codes past 2^32 bytes, activations past 2^32 elements: the first and the last tokens against the definition."""
    t, cols = 540_000, 8192
    x = torch.zeros(t, cols, dtype=torch.bfloat16, device="cuda")
    some = [0, 1, 262_143, 262_144, t // 2, t - 2, t - 1]
    x[some] = dev(torch.randn(len(some), cols, generator=gen(3)), "bf16")
    q, s = torch.full((t, cols), 0x55, dtype=torch.uint8, device="cuda"), torch.zeros(t, cols // 128, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_fp8_quantize(x.data_ptr(), larql_b200.T_BF16, t, cols, cols, q.data_ptr(), s.data_ptr())
    be.synchronize()
    wq, ws = quantized(x[some].float().cpu())
    assert torch.equal(s[some].cpu(), ws) and torch.equal(q[some].cpu(), wq.view(torch.uint8))
    rest = torch.ones(t, dtype=torch.bool, device="cuda")
    rest[some] = False
    assert (s[rest] == 2.0 ** -126).all() and int(q.sum(1, dtype=torch.int64)[rest].amax()) == 0


def check_fp8_on_device(be, tokens_, cols, rows, seed, x_stride=None, out_stride=None):
    """A bf16 -> f32 product against f64 on the GPU, with the tolerance of fp8_tolerance; returns the output."""
    g = gen(seed)
    x_stride, out_stride = x_stride or cols, out_stride or rows
    x = torch.empty((tokens_ - 1) * x_stride + cols, dtype=torch.bfloat16, device="cuda").as_strided((tokens_, cols), (x_stride, 1))
    x.copy_(torch.randn(tokens_, cols, generator=g))
    wq, ws = (v.cuda() for v in fp8_weight(g, rows, cols))
    out = torch.empty((tokens_ - 1) * out_stride + rows, device="cuda").as_strided((tokens_, rows), (out_stride, 1))
    torch.cuda.synchronize()
    assert be.dev_fp8_matmul(fp8_matrix(wq, ws), x.data_ptr(), larql_b200.T_BF16, tokens_, x_stride, out.data_ptr(), larql_b200.T_F32, out_stride)
    be.synchronize()
    xq, xs = (v.cuda() for v in quantized(x.float().cpu()))
    blocks = (cols + 127) // 128
    xv = xq.float().double() * xs.double().repeat_interleave(128, 1)[:, :cols]
    wv = wq.float().double() * ws.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    want, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    # fp8_tolerance, and cuBLAS's f64 sums (2^-53 a term)
    off = want.abs() * U + (min(cols, 128) * 2 + 4 * blocks) * U * mag + 1e-44 + cols * 2.0 ** -52 * mag
    assert ((out.double() - want).abs() <= off).all()
    return out


WAYS = [
    # tokens, cols, rows: tiles of 16, 32 and 64 tokens, whole and in pieces over the grid; the kernel for many tokens, ragged,
    # with more tiles than SMs; more tokens than one launch takes
    (64, 2880, 2880), (100, 2880, 2880), (250, 2880, 2880), (16, 16384, 8192), (128, 16384, 2048), (512, 16384, 1024),
    (1024, 2880, 2880), (300, 2896, 2885), (2000, 528, 5000), (33_000, 144, 260),
]


@gpu
@pytest.mark.parametrize("case", WAYS)
def test_fp8_matmul_every_way_of_cutting_it_up(be, case):
    a = check_fp8_on_device(be, *case, seed=sum(case))
    assert torch.equal(a, check_fp8_on_device(be, *case, seed=sum(case)))


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,pad", [(1221, 0), (1216, 3), (1216, 0), (1093, 8)])
def test_fp8_matmul_of_many_tokens_into_ragged_rows(be, kind, rows, pad):
    """The kernel for many tokens where a row of the output ends inside a tile or starts at any element: nothing beside the
    row is written (run_fp8 checks that too)."""
    run_fp8(be, kind, 1999, 528, rows, seed=rows + pad, out_pad=pad)


@gpu
def test_fp8_matmul_of_nothing(be):
    """No columns: zeros, for one token whatever its strides; no tokens, no rows: nothing."""
    for t, stride in ((1, 0), (1, 7), (3, 6)):
        out = torch.full((t, 6), 9.0, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        m = larql_b200.DeviceMatrix(larql_b200.FMT_FP8_B128, 5, 0, 0, 0)
        assert be.dev_fp8_matmul(m, 0, larql_b200.T_BF16, t, 0, out.data_ptr(), larql_b200.T_BF16, stride)
        be.synchronize()
        assert (out[:, :5] == 0).all() and (out[:, 5] == 9).all()
        assert be.dev_fp8_matmul(m, 0, larql_b200.T_BF16, 0, 0, 0, larql_b200.T_BF16, 0)
        assert be.dev_fp8_matmul(larql_b200.DeviceMatrix(larql_b200.FMT_FP8_B128, 0, 16, 0, 0), 0, larql_b200.T_BF16, t, 16, 0, larql_b200.T_BF16, 0)


@gpu
@pytest.mark.parametrize("tokens_", [3, 140])
def test_fp8_matmul_offsets_past_32_bits(be, tokens_):
    """Strides that put the last token's activations and outputs past 2^32 bytes."""
    stride = ((1 << 32) // (tokens_ - 1) + 64) // 16 * 16
    check_fp8_on_device(be, tokens_, 272, 300, 1, x_stride=stride, out_stride=stride // 2)


@gpu
def test_fp8_matmul_graph_outlives_its_workspace(be):
    """A graph captured with a small workspace, the workspace outgrown by a larger call, the graph replayed: what it holds is
    still there and still in order."""
    own = larql_b200.CudaBackend(0)
    try:
        g = gen(1)
        wq, ws = (v.cuda() for v in fp8_weight(g, 8192, 16384))
        m = fp8_matrix(wq, ws)
        x, out = torch.zeros(16, 16384, dtype=torch.bfloat16, device="cuda"), torch.empty(16, 8192, device="cuda")
        call = lambda b: b.dev_fp8_matmul(m, x.data_ptr(), larql_b200.T_BF16, 16, 16384, out.data_ptr(), larql_b200.T_F32, 8192)
        torch.cuda.synchronize()
        stream = torch.cuda.ExternalStream(own.stream())
        refused = torch.cuda.CUDAGraph()
        with torch.cuda.graph(refused, stream=stream, capture_error_mode="thread_local"):
            with pytest.raises(larql_b200.BackendError):  # no workspace yet: refused, and the capture goes on
                call(own)
        assert call(own)
        own.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            assert call(own)
        check_fp8_on_device(own, 700, 16384, 1024, 5)  # a larger workspace
        for i in range(2):
            x.copy_(torch.randn(16, 16384, generator=gen(50 + i)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert call(be)
            be.synchronize()
            assert torch.equal(got, out)
        del graph, refused
    finally:
        own.close()


# ------------------------------------------------------------------ MoE ----
@gpu
@pytest.mark.parametrize("fmt,kind,router", [("mxfp4", "f32", "bf16"), ("nvfp4", "bf16", "f32"), ("fp8", "f16", "bf16")])
def test_moe_layer_router_of_another_type_and_unaligned_tokens(be, fmt, kind, router):
    """The router's type is its own; x and out start at any element."""
    layer = Layer(be, fmt, 544, 96, 9, 3, kind, seed=4)
    layer.router = dev(layer.router, router)
    torch.cuda.synchronize()
    layer.layer = be.moe_create(*layer.mats, layer.router.data_ptr(), TYPES[router][1], 0, 3, True)
    for t in (1, 21):
        x = dev(torch.randn(t * 544 + 1, generator=gen(t)), kind)[1:].view(t, 544)
        out = torch.full(((t + 1) * 544 + 3,), 3.0, dtype=x.dtype, device="cuda")[3:].view(t + 1, 544)
        check(layer, x, layer.run(be, x, out))


MOE_SIZES = [
    # fmt, hidden, inter, experts, top_e, kind, tokens: odd numbers of scale blocks, both tiles of a down unit and one of them,
    # two tiles of columns, experts with several groups of tokens
    ("mxfp4", 736, 1504, 4, 2, "bf16", 50), ("mxfp4", 1504, 736, 2, 2, "f32", 30), ("nvfp4", 736, 1504, 4, 2, "bf16", 50),
    ("nvfp4", 1504, 736, 2, 1, "f32", 30), ("fp8", 736, 1504, 4, 2, "bf16", 50), ("fp8", 1504, 736, 2, 2, "f16", 30),
    ("mxfp4", 2880, 2880, 2, 1, "f32", 1), ("fp8", 8192, 96, 3, 2, "f32", 5), ("mxfp4", 96, 8192, 3, 2, "bf16", 64), ("nvfp4", 96, 6144, 3, 2, "f32", 9),
    ("nvfp4", 6144, 96, 3, 2, "bf16", 64), ("mxfp4", 8192, 8192, 1, 1, "f32", 2), ("fp8", 8192, 8192, 1, 1, "bf16", 3),
]


@gpu
@pytest.mark.parametrize("case", MOE_SIZES)
def test_moe_layer_at_the_ends_of_its_sizes(be, case):
    fmt, hidden, inter, experts, top_e, kind, t = case
    layer = Layer(be, fmt, hidden, inter, experts, top_e, kind, True, True, seed=t + hidden)
    x = tokens(gen(t), t, hidden, kind)
    check(layer, x, layer.run(be, x))


@gpu
def test_two_contexts_side_by_side(be):
    """Layers, products and norms of two contexts enqueued in turn without waiting: the same bits as one after another."""
    other = larql_b200.CudaBackend(0)
    try:
        side = []
        for k, b in enumerate((be, other)):
            layer = Layer(b, "mxfp4", 2880, 320, 8, 2, "bf16", seed=k)
            wq, ws = (v.cuda() for v in fp8_weight(gen(k), 2880, 2880))
            c = norm_case(20, 2880, "bf16", "f32", True, "none", 0, k)
            bufs = [torch.empty(20, 2880, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
            side.append((b, layer, fp8_matrix(wq, ws), c, bufs))
        torch.cuda.synchronize()

        def turn(s):
            b, layer, m, c, (n, y, z) = s
            assert b.dev_block_norm(norm_args(c, None, n))
            assert b.dev_moe_ffn(layer.layer, n.data_ptr(), larql_b200.T_BF16, 20, y.data_ptr())
            assert b.dev_fp8_matmul(m, y.data_ptr(), larql_b200.T_BF16, 20, 2880, z.data_ptr(), larql_b200.T_BF16, 2880)

        want = []
        for s in side:
            turn(s)
            s[0].synchronize()
            want.append([v.clone() for v in s[4]])
            for v in s[4]:
                v.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for s in side:
                turn(s)
        for s, w in zip(side, want):
            s[0].synchronize()
            assert all(torch.equal(a, b) for a, b in zip(s[4], w))
        side[1][1].layer.close()
    finally:
        other.close()


@gpu
def test_moe_handle_and_its_context():
    """A handle made during a capture is refused; one that outlives its context frees itself."""
    b = larql_b200.CudaBackend(0)
    layer = Layer(b, "mxfp4", 64, 96, 2, 1, seed=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(b.stream()), capture_error_mode="thread_local"):
        with pytest.raises(larql_b200.BackendError):
            b.moe_create(*layer.mats, layer.router.data_ptr(), 0, 0, 1)
    del graph
    x = tokens(gen(1), 3, 64, "f32")
    check(layer, x, layer.run(b, x))
    b.close()
    layer.layer.close()
    layer.layer.close()


@gpu
@pytest.mark.parametrize("t", [1, 40, 1400])
def test_a_captured_tail_of_a_decoder_replays_with_new_inputs(be, t):
    """norm -> layer -> norm -> quantisation -> coded product -> quantising product, captured once and replayed: the bits of
    the eager calls on the same inputs."""
    hidden, kind = 1024, "bf16"
    layer = Layer(be, "mxfp4", hidden, 96, 4, 2, kind, True, True, 3)
    before = norm_case(t, hidden, kind, kind, False, "none", 0, 4)
    new = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")
    n1, y, h2, n2, out1, out2 = (new(t, hidden) for _ in range(6))
    q, s = new(t, hidden, dt=torch.uint8), new(t, hidden // 128, dt=torch.float32)
    after = dict(norm_case(t, hidden, kind, kind, True, "channel", 0, 7, y_scale=0.8), h=before["h"], y=y)
    wq, ws = (v.cuda() for v in fp8_weight(gen(6), hidden, hidden))
    m = fp8_matrix(wq, ws)
    bf16, e4m3 = larql_b200.T_BF16, larql_b200.T_E4M3

    def calls():
        assert be.dev_block_norm(norm_args(before, None, n1, use_y=False))
        assert be.dev_moe_ffn(layer.layer, n1.data_ptr(), bf16, t, y.data_ptr())
        assert be.dev_block_norm(norm_args(after, h2, n2))
        assert be.dev_fp8_quantize(n2.data_ptr(), bf16, t, hidden, hidden, q.data_ptr(), s.data_ptr())
        assert be.dev_fp8_matmul(m, q.data_ptr(), e4m3, t, hidden, out1.data_ptr(), bf16, hidden, s.data_ptr())
        assert be.dev_fp8_matmul(m, out1.data_ptr(), bf16, t, hidden, out2.data_ptr(), bf16, hidden)

    torch.cuda.synchronize()
    calls()
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream()), capture_error_mode="thread_local"):
        calls()
    for i in range(3):
        before["h"].copy_(torch.randn(t, hidden, generator=gen(60 + i)))
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (n1, y, h2, n2, q, s, out1, out2)]
        torch.cuda.synchronize()
        calls()
        be.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (n1, y, h2, n2, q, s, out1, out2)))
        assert out2.isfinite().all() and (out2 != 0).any()
