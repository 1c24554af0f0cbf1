"""The layer operators beside the walk, against plain implementations in 64 bits: the norms around a block
(lq_dev_block_norm) and the FP8 product with its quantisation (lq_dev_fp8_quantize, lq_dev_fp8_matmul).

Tolerances are bounds, not measurements.  A result is rounded once to its type: half a step, eps / 2 of the value
(plus half the smallest subnormal for f16).  Before that the arithmetic is f32: every operation adds at most 2^-24 of
the magnitude it works on, and the bounds below count the operations on the magnitudes (sums of absolute values)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import larql_b200
from larql_b200 import build as lqbuild

ROOT = Path(__file__).resolve().parent.parent
gpu = pytest.mark.gpu
TYPES = {"f32": (torch.float32, larql_b200.T_F32), "bf16": (torch.bfloat16, larql_b200.T_BF16),
         "f16": (torch.float16, larql_b200.T_F16)}
U = 2.0 ** -24


def half_step(kind, want):
    """Half a rounding step of `want` in the type, as an absolute error."""
    dt = TYPES[kind][0]
    return want.abs() * (torch.finfo(dt).eps / 2) * (1 + 1e-6) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


@pytest.fixture(scope="module")
def be():
    b = larql_b200.CudaBackend(0)
    yield b
    b.close()


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def dev(t, kind=None):
    return t.to(device="cuda", dtype=TYPES[kind][0] if kind else t.dtype)


# ------------------------------------------------------------------ CPU ----
def test_null_context_is_an_argument_error():
    lqbuild.build()
    lib = larql_b200.load_library()
    args, m = larql_b200.BlockNormArgs(), larql_b200.LqMatrix()
    assert lib.lq_dev_block_norm(None, C.byref(args)) == larql_b200.LQ_ERR_ARGUMENT
    assert lib.lq_dev_fp8_quantize(None, None, 0, 1, 128, 128, None, None) == larql_b200.LQ_ERR_ARGUMENT
    assert lib.lq_dev_fp8_matmul(None, C.byref(m), None, 0, None, 1, 128, None, 0, 128) == larql_b200.LQ_ERR_ARGUMENT
    assert lib.lq_fp8_matmul(None, C.byref(m), None, 0, 0, None, 0) == larql_b200.LQ_ERR_ARGUMENT


def test_argument_record_has_the_header_layout(tmp_path):
    """Field offsets of lq_block_norm_args as the C compiler sees them and as the ctypes mirror lays them out."""
    fields = [n for n, _ in larql_b200.BlockNormArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "larql_cuda.h"\nint main(void) {\n' +
                   "".join(f'  printf("{f} %zu\\n", offsetof(lq_block_norm_args, {f}));\n' for f in fields) +
                   '  printf("size %zu\\n", sizeof(lq_block_norm_args));\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for f in fields:
        assert int(got[f]) == getattr(larql_b200.BlockNormArgs, f).offset, f
    assert int(got["size"]) == C.sizeof(larql_b200.BlockNormArgs)


# ----------------------------------------------------------- block norm ----
def norm_case(rows, cols, kind, w_kind, post, gate, pad, seed, offset=1.0, h_scale=1.0, y_scale=0.5, group=None, scale=1.0):
    g = gen(seed)
    mk = lambda *s, k=kind: dev(torch.randn(*s, generator=g) * scale, k)
    wide = cols + pad
    c = {"h": mk(rows, wide)[:, :cols], "y": mk(rows, wide)[:, :cols], "post_w": dev(torch.randn(cols, generator=g) * 0.3, w_kind),
         "pre_w": dev(torch.randn(cols, generator=g) * 0.3, w_kind), "gate": None, "gate_cols": 0, "gate_group": 1}
    if gate == "channel":
        c["gate"], c["gate_cols"], c["gate_group"] = dev(torch.randn(1, cols, generator=g), kind), cols, max(rows, 1)
    elif gate == "row":
        c["gate"], c["gate_cols"] = dev(torch.randn(rows, 1, generator=g), kind), 1
    elif gate == "full":
        c["gate"], c["gate_cols"] = dev(torch.randn(rows, cols, generator=g), kind), cols
    elif gate == "group":
        n = (rows + group - 1) // group
        c["gate"], c["gate_cols"], c["gate_group"] = dev(torch.randn(n, cols, generator=g), kind), cols, group
    c.update(rows=rows, cols=cols, kind=kind, w_kind=w_kind, post=post, offset=offset, h_scale=h_scale, y_scale=y_scale, eps=1e-6)
    return c


def norm_args(c, h_out, n_out, use_post_w=True, use_pre_w=True, use_y=True):
    p = lambda t: 0 if t is None else t.data_ptr()
    return larql_b200.BlockNormArgs(
        type=TYPES[c["kind"]][1], w_type=TYPES[c["w_kind"]][1], post_norm=int(c["post"]), w_offset=c["offset"],
        h_scale=c["h_scale"], y_scale=c["y_scale"], eps=c["eps"], rows=c["rows"], cols=c["cols"], h=p(c["h"]),
        h_stride=c["h"].stride(0), y=p(c["y"]) if use_y else 0, y_stride=c["y"].stride(0),
        post_w=p(c["post_w"]) if use_post_w else 0, pre_w=p(c["pre_w"]) if use_pre_w else 0, gate=p(c["gate"]),
        gate_cols=c["gate_cols"], gate_stride=c["gate"].stride(0) if c["gate"] is not None else 0, gate_group=c["gate_group"],
        h_out=p(h_out), h_out_stride=h_out.stride(0) if h_out is not None else 0, n_out=p(n_out),
        n_out_stride=n_out.stride(0) if n_out is not None else 0)


def norm_want(c, use_post_w=True, use_pre_w=True, use_y=True):
    """(h', n) in f64 and the magnitudes their f32 evaluation works on."""
    d = lambda t: t.cpu().double()
    h = c["h_scale"] * d(c["h"])
    mag = h.abs()
    if use_y:
        z = d(c["y"])
        if c["post"]:
            z = z / (z.square().mean(1, keepdim=True) + c["eps"]).sqrt()
            if use_post_w:
                z = z * (c["offset"] + d(c["post_w"]))
                mag = mag + 0
        g = 1.0
        if c["gate"] is not None:
            g = d(c["gate"]).repeat_interleave(c["gate_group"], 0)[:c["rows"]]
        z = c["y_scale"] * g * z
        h, mag = h + z, mag + z.abs()
    inv = 1.0 / (h.square().mean(1, keepdim=True) + c["eps"]).sqrt()
    w = c["offset"] + d(c["pre_w"]) if use_pre_w else torch.ones(c["cols"], dtype=torch.float64)
    # (offset + w is one f32 rounding of a sum that may cancel: its absolute error is U of the larger magnitudes)
    return h, h * inv * w, mag, mag * inv * (w.abs() + U)


def check_norm(c, h_out, n_out, **use):
    h, n, mh, mn = norm_want(c, **use)
    if h_out is not None:  # h_scale h; inv, z inv, off + w, product, gate scale, product; the sum: at most 8 roundings
        assert ((h_out.cpu().double() - h).abs() <= half_step(c["kind"], h) + 8 * U * mh + 1e-45).all()
    if n_out is not None:  # h' as above; its rms moves by at most the same share of rms; inv, off + w, two products
        rms_share = 8 * U * mh.square().mean(1, keepdim=True).sqrt() / (h.square().mean(1, keepdim=True) + c["eps"]).sqrt()
        assert ((n_out.cpu().double() - n).abs() <= half_step(c["kind"], n) + 12 * U * mn + rms_share * n.abs() + 1e-45).all()


NORM_CASES = [
    # rows, cols, kind, weights, post, gate, pad
    (1, 1, "f32", "f32", True, "none", 0), (1, 3840, "bf16", "bf16", True, "none", 0), (3, 7, "f16", "f32", True, "full", 2),
    (5, 512, "bf16", "f32", True, "channel", 0), (9, 513, "f32", "bf16", False, "row", 0), (8, 520, "bf16", "f16", True, "full", 8),
    (2, 2885, "f32", "f32", False, "channel", 3), (33, 2880, "f16", "f16", True, "row", 0), (2, 8192, "bf16", "bf16", True, "full", 0),
    (3, 16384, "f32", "f32", True, "channel", 0), (2, 16383, "bf16", "bf16", True, "none", 1), (300, 256, "f32", "f32", True, "full", 0),
    (1000, 1024, "bf16", "bf16", True, "none", 0), (17, 4096, "f16", "bf16", False, "none", 5),
]


@gpu
@pytest.mark.parametrize("case", NORM_CASES)
def test_block_norm_matches_the_formula(be, case):
    c = norm_case(*case, seed=sum(map(ord, str(case))))
    h_out, n_out = (torch.empty(c["rows"], c["cols"], dtype=TYPES[c["kind"]][0], device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    check_norm(c, h_out, n_out)


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_block_norm_optional_operands(be, kind):
    """Each of y, the weights and the outputs left out; a gate row per group of rows; rows behind the last kept."""
    c = norm_case(10, 640, kind, "f32", True, "group", 0, 3, offset=0.0, group=4)
    new = lambda: torch.full((12, 648), 7.0, dtype=TYPES[kind][0], device="cuda")
    for use, keep in [({}, "both"), ({"use_post_w": False}, "both"), ({"use_pre_w": False}, "n"), ({}, "h")]:
        h_out, n_out = new(), new()
        torch.cuda.synchronize()
        assert be.dev_block_norm(norm_args(c, h_out if keep != "n" else None, n_out if keep != "h" else None, **use))
        be.synchronize()
        check_norm(c, h_out[:10, :640] if keep != "n" else None, n_out[:10, :640] if keep != "h" else None, **use)
        for o in (h_out, n_out):  # rows behind the last and the padding behind each row are left as they were
            assert (o[10:] == 7).all() and (o[:, 640:] == 7).all()
        if keep == "n":
            assert (h_out == 7).all()
    c.update(post=False, gate=None, gate_cols=0)
    h_out, n_out = new(), new()
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out, use_y=False))
    be.synchronize()
    check_norm(c, h_out[:10, :640], n_out[:10, :640], use_y=False)


@gpu
def test_block_norm_in_place(be):
    """h_out over h and n_out over y, the rows of one residual stream updated where they lie."""
    c = norm_case(6, 3840, "bf16", "bf16", True, "full", 0, 11)
    h, n, _, _ = norm_want(c)
    keep = {k: c[k].clone() for k in ("h", "y")}
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, c["h"], c["y"]))
    be.synchronize()
    h_out, n_out = c["h"], c["y"]
    c.update(keep)
    check_norm(c, h_out, n_out)


@gpu
def test_block_norm_extremes(be):
    """Rows of zeros, rows whose squares leave f32's range, NaN and infinity kept to their row."""
    c = norm_case(5, 1024, "f32", "f32", True, "none", 0, 5, y_scale=1.0)
    c["h"].zero_()
    c["y"][0] = 0
    c["y"][1] *= 1e30
    c["y"][2] *= 1e-30
    c["y"][3, 17] = float("nan")
    h_out, n_out = torch.empty(5, 1024, device="cuda"), torch.empty(5, 1024, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    assert (h_out[0] == 0).all() and (n_out[0] == 0).all()
    assert h_out[3].isnan().all() and n_out[3].isnan().all()
    good = [0, 1, 2, 4]
    sub = dict(c, h=c["h"][good], y=c["y"][good], rows=4)
    check_norm(sub, h_out[good], n_out[good])
    c["y"][3, 17] = float("inf")
    torch.cuda.synchronize()
    assert be.dev_block_norm(norm_args(c, h_out, n_out))
    be.synchronize()
    assert h_out[3, 17].isnan() and (h_out[3, :17] == 0).all()  # inf / inf, finite / inf
    check_norm(sub, h_out[good], n_out[good])


@gpu
def test_block_norm_refusals(be):
    c = norm_case(4, 256, "f32", "f32", True, "full", 0, 1)
    out = torch.empty(4, 256, device="cuda")

    def a(**kw):
        args = norm_args(c, out, out)
        for k, v in kw.items():
            setattr(args, k, v)
        return args

    for kw in [{"type": 3}, {"w_type": 9}, {"cols": 16385}, {"rows": 1 << 32}, {"h_stride": 255}, {"y_stride": 8},
               {"gate_cols": 2}, {"gate_group": 0}, {"gate_stride": 10}, {"n_out_stride": 255}]:
        assert be.dev_block_norm(a(**kw)) is False, kw
    for kw in [{"eps": 0.0}, {"eps": float("nan")}, {"eps": -1.0}, {"eps": float("inf")}, {"h": 0}, {"h_out": 0, "n_out": 0},
               {"y": 0}, {"h": c["h"].data_ptr() + 2}]:
        with pytest.raises(larql_b200.BackendError):
            be.dev_block_norm(a(**kw))
    assert be.dev_block_norm(a(rows=0)) and be.dev_block_norm(a(cols=0))
    be.synchronize()


# ------------------------------------------------------------------ FP8 ----
def quantized(x):
    """The definition on the CPU: (codes as e4m3, scales) of f32 values [tokens, cols]."""
    t, c = x.shape
    nb = (c + 127) // 128
    b = torch.nn.functional.pad(x, (0, nb * 128 - c)).view(t, nb, 128)
    s = torch.clamp((b.abs().amax(-1).double() / 448).float(), min=2.0 ** -126)
    q = (b.double() / s.double()[..., None]).float().to(torch.float8_e4m3fn)
    return q.view(t, nb * 128)[:, :c].contiguous(), s


def fp8_weight(g, rows, cols, std=0.02):
    w = torch.randn(rows, cols, generator=g) * std
    rb, cb = (rows + 127) // 128, (cols + 127) // 128
    p = torch.nn.functional.pad(w, (0, cb * 128 - cols, 0, rb * 128 - rows)).view(rb, 128, cb, 128)
    s = torch.clamp(p.abs().amax((1, 3)) / 448, min=2.0 ** -126)
    q = (p / s[:, None, :, None]).reshape(rb * 128, cb * 128)[:rows, :cols].to(torch.float8_e4m3fn).contiguous()
    return q, s.contiguous()


def fp8_matrix(q, s):
    """The device matrix over (codes, scales) tensors on the GPU."""
    return larql_b200.DeviceMatrix(larql_b200.FMT_FP8_B128, q.shape[0], q.shape[1], q.data_ptr(), q.numel(), s.data_ptr(),
                                   s.numel() * 4, keepalive=(q, s))


def fp8_want(xq, xs, wq, ws):
    """(product in f64, sum of the absolute terms)."""
    x = xq.float().double() * xs.double().repeat_interleave(128, 1)[:, :xq.shape[1]]
    w = wq.float().double() * ws.double().repeat_interleave(128, 0)[:wq.shape[0]].repeat_interleave(128, 1)[:, :wq.shape[1]]
    return x @ w.t(), x.abs() @ w.abs().t()


def fp8_tolerance(kind, want, mag, cols):
    # a block: 128 exact products summed in f32 in an order of the tensor core's, each step rounded or cut (2 U);
    # per block the scale product, the fused multiply-add, and the joining of pieces: 4 roundings
    blocks = (cols + 127) // 128
    return half_step(kind, want) + (min(cols, 128) * 2 + 4 * blocks) * U * mag + 1e-44


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,cols,pad", [(1, 128, 0), (1, 1, 0), (3, 200, 0), (17, 2880, 0), (5, 1003, 4), (40, 256, 8), (2, 16384, 0)])
def test_fp8_quantize_is_the_definition(be, kind, tokens, cols, pad):
    x = dev(torch.randn(tokens, cols + pad, generator=gen(cols + tokens)) * 3, kind)[:, :cols]
    x[0, :min(cols, 128)] = 0          # a block of zeros
    if tokens > 1:
        x[1, :min(cols, 128)] *= 1e-6  # (subnormal or zero in f16)
    if kind == "f32" and tokens > 2:
        x[2, :min(cols, 128)] *= 1e-41  # the smallest scale
    guard = 64
    q = torch.full((tokens * cols + guard,), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.empty(tokens, (cols + 127) // 128, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_fp8_quantize(x.data_ptr(), TYPES[kind][1], tokens, cols, x.stride(0), q.data_ptr(), s.data_ptr())
    be.synchronize()
    wq, ws = quantized(x.float().cpu())
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q[:tokens * cols].cpu().view(tokens, cols), wq.view(torch.uint8))
    assert (q[tokens * cols:] == 0x55).all()


@gpu
def test_fp8_quantize_ties_and_non_finite(be):
    """Quotients on the borders between codes go to the even one; a NaN or infinity reaches its block's codes or scale."""
    grid = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (grid[1:] + grid[:-1]) / 2  # exact in f32; with 448 in the block the scale is 1 and these are ties
    x = torch.zeros(4, 128)
    x[0, :126], x[0, 126] = mid, 448
    x[1, :126], x[1, 127] = -mid, -448
    x[2, 5], x[3, 5] = float("nan"), float("inf")
    xd = x.cuda()
    q, s = torch.empty(4, 128, dtype=torch.uint8, device="cuda"), torch.empty(4, 1, device="cuda")
    torch.cuda.synchronize()
    assert be.dev_fp8_quantize(xd.data_ptr(), larql_b200.T_F32, 4, 128, 128, q.data_ptr(), s.data_ptr())
    be.synchronize()
    wq, ws = quantized(x[:2])
    assert torch.equal(s[:2].cpu(), ws) and torch.equal(q[:2].cpu(), wq.view(torch.uint8))
    v = q.cpu().view(torch.float8_e4m3fn).float() * s.cpu()
    assert v[2].isnan().any() and v[3].isnan().any()


def run_fp8(be, kind, tokens, cols, rows, seed, x_pad=0, out_pad=0, std=1.0, coded=False):
    g = gen(seed)
    x = dev(torch.randn(tokens, cols + x_pad, generator=g) * std, kind)[:, :cols]
    wq, ws = fp8_weight(g, rows, cols)
    wq_d, ws_d = wq.cuda(), ws.cuda()
    m = fp8_matrix(wq_d, ws_d)
    out = torch.full((tokens + 1, rows + out_pad), 5.0, dtype=TYPES[kind][0], device="cuda")
    xq, xs = quantized(x.float().cpu())
    if coded:
        xqd, xsd = xq.cuda(), xs.cuda()
        torch.cuda.synchronize()
        ok = be.dev_fp8_matmul(m, xqd.data_ptr(), larql_b200.T_E4M3, tokens, cols, out.data_ptr(), TYPES[kind][1], rows + out_pad,
                               xsd.data_ptr())
    else:
        torch.cuda.synchronize()
        ok = be.dev_fp8_matmul(m, x.data_ptr(), TYPES[kind][1], tokens, x.stride(0), out.data_ptr(), TYPES[kind][1], rows + out_pad)
    assert ok
    be.synchronize()
    assert (out[tokens:] == 5).all() and (out[:, rows:] == 5).all()  # nothing behind the last token or row
    want, mag = fp8_want(xq, xs, wq, ws)
    got = out[:tokens, :rows].cpu().double()
    assert ((got - want).abs() <= fp8_tolerance(kind, want, mag, cols)).all()
    return out[:tokens, :rows].clone()


FP8_CASES = [
    # tokens, cols, rows: both kernels, every column count, ragged blocks, pieces of tiles over several SMs
    (1, 16, 1), (1, 128, 128), (1, 2880, 2880), (2, 4096, 130), (7, 144, 300), (16, 1024, 1000), (17, 2880, 257), (32, 512, 128),
    (33, 640, 129), (64, 1040, 1024), (65, 256, 384), (100, 2880, 640), (128, 384, 100), (129, 384, 100), (130, 2880, 300),
    (200, 1040, 513), (257, 128, 700), (1, 16384, 64), (130, 16384, 256),
]


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", FP8_CASES)
def test_fp8_matmul_matches_the_formula(be, kind, case):
    run_fp8(be, kind, *case, seed=sum(case))


@gpu
@pytest.mark.parametrize("tokens", [1, 5, 40, 200])
def test_fp8_matmul_strides_types_and_coded_input(be, tokens):
    """Rows of wider buffers, unaligned starts of an output row, f16, activations quantised beforehand: the codes being
    the same, the coded call gives the same bits as the quantising one."""
    run_fp8(be, "f16", tokens, 272, 333, 1, x_pad=3, out_pad=7, std=0.1)
    a = run_fp8(be, "bf16", tokens, 1056, 200, 2, x_pad=8, out_pad=1)
    b = run_fp8(be, "bf16", tokens, 1056, 200, 2, x_pad=8, out_pad=1, coded=True)
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("tokens", [3, 150])
def test_fp8_matmul_repeats_bit_for_bit(be, tokens):
    a = run_fp8(be, "f32", tokens, 2880, 1000, 9)
    for _ in range(5):
        assert torch.equal(a, run_fp8(be, "f32", tokens, 2880, 1000, 9))


@gpu
def test_fp8_matmul_keeps_non_finite_to_its_token(be):
    g = gen(4)
    wq, ws = fp8_weight(g, 300, 512)
    wq, ws = wq.cuda(), ws.cuda()
    for tokens in (4, 140):
        x = torch.randn(tokens, 512, generator=g).cuda()
        x[1, 300] = float("nan")
        x[2, 3] = float("inf")
        out = torch.empty(tokens, 300, device="cuda")
        torch.cuda.synchronize()
        assert be.dev_fp8_matmul(fp8_matrix(wq, ws), x.data_ptr(), 0, tokens, 512, out.data_ptr(), 0, 300)
        be.synchronize()
        assert out[1].isnan().all() and out[2].isnan().all()
        rest = [0] + list(range(3, tokens))
        xq, xs = quantized(x.cpu()[rest])
        want, mag = fp8_want(xq, xs, wq.cpu(), ws.cpu())
        assert ((out.cpu().double()[rest] - want).abs() <= fp8_tolerance("f32", want, mag, 512)).all()


@gpu
def test_fp8_matmul_host_call(be):
    g = gen(8)
    wq, ws = fp8_weight(g, 200, 320)
    hm = larql_b200.HostMatrix(larql_b200.FMT_FP8_B128, 200, 320, wq.view(torch.uint8).numpy(), ws.numpy())
    for tokens in (1, 30):
        x = torch.randn(tokens, 320, generator=g)
        got = be.fp8_matmul(hm, x.numpy())
        want, mag = fp8_want(*quantized(x), wq, ws)
        assert ((torch.from_numpy(got).double() - want).abs() <= fp8_tolerance("f32", want, mag, 320)).all()
    assert be.fp8_matmul(hm, np.zeros((2, 319), np.float32)) is None
    assert be.fp8_matmul(hm, np.zeros((0, 320), np.float32)).shape == (0, 200)


@gpu
def test_fp8_matmul_in_a_captured_graph(be):
    """Both kernels captured on the context's stream and replayed with other inputs in place."""
    g = gen(6)
    wq, ws = fp8_weight(g, 640, 512)
    m = fp8_matrix(wq.cuda(), ws.cuda())
    for tokens in (6, 150):
        x, out = torch.zeros(tokens, 512, device="cuda"), torch.empty(tokens, 640, device="cuda")
        call = lambda: be.dev_fp8_matmul(m, x.data_ptr(), 0, tokens, 512, out.data_ptr(), 0, 640)
        torch.cuda.synchronize()
        assert call()  # the workspace grows here and not in the capture
        be.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream()), capture_error_mode="thread_local"):
            assert call()
        for _ in range(3):
            x.copy_(torch.randn(tokens, 512, generator=g))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want, mag = fp8_want(*quantized(x.cpu()), wq, ws)
            assert ((out.cpu().double() - want).abs() <= fp8_tolerance("f32", want, mag, 512)).all()
        be.synchronize()


@gpu
def test_fp8_refusals(be):
    q, s = torch.zeros(256, 256, dtype=torch.uint8, device="cuda"), torch.ones(2, 2, device="cuda")
    x, out = torch.zeros(4, 512, device="cuda"), torch.zeros(4, 256, device="cuda")

    def mat(rows=256, cols=256, off=0, n=256 * 256, sn=16, fmt=larql_b200.FMT_FP8_B128):
        return larql_b200.DeviceMatrix(fmt, rows, cols, q.data_ptr() + off, n, s.data_ptr(), sn)

    def mm(m=None, xp=None, xt=0, t=4, xs=256, ot=0, os_=256, sc=0):
        return be.dev_fp8_matmul(m or mat(), x.data_ptr() if xp is None else xp, xt, t, xs, out.data_ptr(), ot, os_, sc)

    for bad in [mat(cols=250), mat(n=100), mat(sn=15), mat(fmt=larql_b200.FMT_MXFP4)]:
        assert mm(bad) is False
    assert mm(xt=7) is False and mm(ot=larql_b200.T_E4M3) is False and mm(xs=255) is False and mm(os_=255) is False
    assert mm(t=1 << 31) is False
    for kw in [dict(m=mat(rows=255, off=8)), dict(xt=larql_b200.T_E4M3), dict(sc=s.data_ptr()), dict(xp=0),
               dict(xt=larql_b200.T_E4M3, sc=s.data_ptr(), xs=264), dict(xt=larql_b200.T_E4M3, sc=s.data_ptr(), xp=x.data_ptr() + 8)]:
        with pytest.raises(larql_b200.BackendError):
            mm(**kw)
    assert mm(t=0) and mm(mat(rows=0, n=0))
    assert mm(mat(cols=0, n=0, sn=0))
    be.synchronize()
    assert (out == 0).all()
    assert be.dev_fp8_quantize(x.data_ptr(), larql_b200.T_E4M3, 4, 128, 128, q.data_ptr(), s.data_ptr()) is False
    assert be.dev_fp8_quantize(x.data_ptr(), 0, 4, 128, 127, q.data_ptr(), s.data_ptr()) is False
    with pytest.raises(larql_b200.BackendError):
        be.dev_fp8_quantize(x.data_ptr() + 1, 0, 4, 128, 128, q.data_ptr(), s.data_ptr())
    # the walk and the other formats' entry points do not take the format
    h = larql_b200.HostMatrix(larql_b200.FMT_FP8_B128, 4, 256, np.zeros((4, 256), np.uint8), np.ones((1, 2), np.float32))
    assert be.gemv(h, np.zeros(256, np.float32)) is None and be.dequantize(h) is None
    assert be.walk_ffn(h, h, h, np.zeros((1, 256), np.float32), 2) is None
