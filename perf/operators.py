"""Cases of the layer operators that stand beside the vindex walk: the norms around a block, the 8-bit
floating-point matrix product, and the whole mixture-of-experts layer for a few tokens.

`listed()` names fixed cases, `draw(rng)` makes more of the same ranges, `prepare(case, seed)` builds the inputs
on the GPU, `run(state)` is one pass (the plain torch form, or the library's kernels when `own` is set),
`exact(case, seed)` is the operator's definition evaluated in 64 bits, and `work(case)` what a pass has to move
and compute.

Operators and their formulas

block_norm      z = y / rms(y) * (offset + post_w)   (z = y without the post norm)
                h' = h_scale * h + y_scale * gate * z
                n = h' / rms(h') * (offset + pre_w),  rms(v) = sqrt(mean(v^2) + eps)
fp8_quantize    per token and 128 columns: s = max(amax / 448, 2^-126), q = e4m3(x / s)
fp8_matmul      out[t, r] = sum_b sx[t, b] * sw[r / 128, b] * sum_{k in block b} qx[t, k] * qw[r, k], the activation
                quantised as above, the weight held as e4m3 with one f32 scale per 128 x 128 block
moe_ffn         logits = x . router^T + bias; the top_e experts by logit (ties to the lower index), softmax weights
                (renormalised over the selected); out = sum_j w_j * down_j . (silu(gate_j . x) * (up_j . x))
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_EPS = 1e-6


def listed():
    return [
        # one token between two layers of a decoder with norms on both sides of the block: latency
        {"name": "norm_1x3840_bf16", "op": "block_norm", "rows": 1, "cols": 3840, "type": "bf16", "post": True, "gate": "none",
         "h_scale": 1.0, "y_scale": 1.0, "offset": 1.0, "pad": 0},
        # a ragged batch of odd width with a learned gate per channel and a residual scale, rows of a wider buffer
        {"name": "norm_77x2885_f32", "op": "block_norm", "rows": 77, "cols": 2885, "type": "f32", "post": False, "gate": "channel",
         "h_scale": 1.0, "y_scale": 0.22, "offset": 0.0, "pad": 3},
        # a long prompt: both norms, one gate per token and channel
        {"name": "norm_4096x8192_bf16", "op": "block_norm", "rows": 4096, "cols": 8192, "type": "bf16", "post": True, "gate": "full",
         "h_scale": 1.0, "y_scale": 1.0, "offset": 0.0, "pad": 0},
        # a small batch of activations quantised once for several products (last block of 64 columns)
        {"name": "quant_16x2880_bf16", "op": "fp8_quantize", "tokens": 16, "cols": 2880, "type": "bf16"},
        # a prompt's activations
        {"name": "quant_4096x8192_bf16", "op": "fp8_quantize", "tokens": 4096, "cols": 8192, "type": "bf16"},
        # one token through an up projection: the weights' bytes are all there is
        {"name": "fp8_1x3840x15360_bf16", "op": "fp8_matmul", "tokens": 1, "cols": 3840, "rows": 15360, "type": "bf16"},
        # a decode batch through a down projection
        {"name": "fp8_16x28672x8192_bf16", "op": "fp8_matmul", "tokens": 16, "cols": 28672, "rows": 8192, "type": "bf16"},
        # a short prompt, sizes that are no multiple of the block, f32 in and out
        {"name": "fp8_250x2880x2880_f32", "op": "fp8_matmul", "tokens": 250, "cols": 2880, "rows": 2880, "type": "f32"},
        # a long prompt through an up projection: a matrix product bound by the tensor cores
        {"name": "fp8_4096x8192x28672_bf16", "op": "fp8_matmul", "tokens": 4096, "cols": 8192, "rows": 28672, "type": "bf16"},
        # one token through a layer of 32 MXFP4 experts, four chosen: decode latency
        {"name": "moe_1_mxfp4_f32", "op": "moe_ffn", "tokens": 1, "hidden": 2880, "inter": 2880, "experts": 32, "top_e": 4,
         "fmt": "mxfp4", "type": "f32", "bias": True, "renorm": True},
        # a decode batch: most experts are read, a few tokens each
        {"name": "moe_16_mxfp4_bf16", "op": "moe_ffn", "tokens": 16, "hidden": 2880, "inter": 2880, "experts": 32, "top_e": 4,
         "fmt": "mxfp4", "type": "bf16", "bias": True, "renorm": True},
        # many small experts in 8-bit blocks, an odd batch
        {"name": "moe_37_fp8_bf16", "op": "moe_ffn", "tokens": 37, "hidden": 3840, "inter": 800, "experts": 64, "top_e": 6,
         "fmt": "fp8", "type": "bf16", "bias": False, "renorm": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["block_norm", "fp8_quantize", "fp8_matmul", "fp8_matmul", "moe_ffn", "moe_ffn"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "block_norm":
        return {"op": op, "rows": _log_int(rng, 1, 4096), "cols": rng.choice([8, 1]) * _log_int(rng, 32, 1000) + rng.choice([0, 0, 1]),
                "type": kind, "post": rng.random() < 0.6, "gate": rng.choice(["none", "channel", "row", "full"]),
                "h_scale": rng.choice([1.0, 0.5]), "y_scale": rng.choice([1.0, 0.22]), "offset": rng.choice([0.0, 1.0]),
                "pad": rng.choice([0, 0, 5, 8])}
    if op == "fp8_quantize":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "cols": 16 * _log_int(rng, 4, 512), "type": kind}
    if op == "fp8_matmul":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "cols": 16 * _log_int(rng, 16, 900), "rows": _log_int(rng, 100, 15000),
                "type": kind}
    fmt = rng.choice(["mxfp4", "nvfp4", "fp8"])
    experts = rng.choice([4, 8, 16, 32, 60])
    return {"op": op, "tokens": _log_int(rng, 1, 64), "hidden": 32 * _log_int(rng, 8, 90), "inter": 32 * _log_int(rng, 6, 80),
            "experts": experts, "top_e": rng.randint(1, min(8, experts)), "fmt": fmt, "type": kind,
            "bias": rng.random() < 0.5, "renorm": rng.random() < 0.7}


# ---------------------------------------------------------------- inputs ----
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, tokens, cols):
    """Normed activations as a decoder layer sees them: unit variance, a few channels twenty times as large."""
    x = _randn(gen, tokens, cols)
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.004
    return torch.where(loud, x * 20, x)


def _encode_fp8(w):
    """[..., r, c] f32 -> e4m3 codes as bytes, one f32 scale per 128 x 128 block (ragged at the ends)."""
    r, c = w.shape[-2:]
    rb, cb = (r + 127) // 128, (c + 127) // 128
    p = torch.nn.functional.pad(w, (0, cb * 128 - c, 0, rb * 128 - r))
    p = p.unflatten(-2, (rb, 128)).unflatten(-1, (cb, 128))
    s = torch.clamp(p.abs().amax(dim=(-3, -1)) / 448, min=2.0 ** -126)
    q = (p / s[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :r, :c]
    return q.to(torch.float8_e4m3fn).contiguous().view(torch.uint8), s.contiguous()


def _encode_e2m1(v):
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=v.device)
    code = torch.bucketize(v.abs(), edges) + torch.where(v < 0, 8, 0)
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _encode(fmt, w):
    """(codes, scales, tensor scale) of a [..., r, c] f32 weight."""
    if fmt == "fp8":
        return (*_encode_fp8(w), 1.0)
    if fmt == "mxfp4":
        b = w.unflatten(-1, (-1, 32))
        e = torch.clamp(torch.floor(torch.log2(b.abs().amax(-1).clamp(min=1e-30))) - 2, -127, 127)
        return _encode_e2m1((b / torch.exp2(e)[..., None]).flatten(-2)), (e + 127).to(torch.uint8), 1.0
    ts = float(2.0 ** -11)
    b = w.unflatten(-1, (-1, 16))
    s = (b.abs().amax(-1) / (6 * ts)).to(torch.float8_e4m3fn)
    d = torch.clamp(s.float() * ts, min=1e-30)
    return _encode_e2m1((b / d[..., None]).flatten(-2)), s.view(torch.uint8), ts


def _strided(x, pad):
    """The rows of x inside a buffer whose rows are `pad` elements longer."""
    return torch.nn.functional.pad(x, (0, pad))[:, :x.shape[1]] if pad else x.contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, s = _TYPES[case["type"]], {"case": dict(case)}
    if case["op"] == "block_norm":
        r, c = case["rows"], case["cols"]
        s["h"] = _strided((_randn(gen, r, c) * 3).to(kind), case["pad"])
        s["y"] = _strided((_randn(gen, r, c) * 0.7).to(kind), case["pad"])
        near = 0.0 if case["offset"] else 1.0
        s["post_w"] = (near + 0.2 * _randn(gen, c)).to(kind) if case["post"] else None
        s["pre_w"] = (near + 0.2 * _randn(gen, c)).to(kind)
        shape = {"none": None, "channel": (1, c), "row": (r, 1), "full": (r, c)}[case["gate"]]
        s["gate"] = None if shape is None else (0.5 + 0.3 * _randn(gen, *shape)).to(kind)
    elif case["op"] == "fp8_quantize":
        s["x"] = _activations(gen, case["tokens"], case["cols"]).to(kind)
    elif case["op"] == "fp8_matmul":
        s["x"] = _activations(gen, case["tokens"], case["cols"]).to(kind)
        s["codes"], s["scales"] = _encode_fp8(_randn(gen, case["rows"], case["cols"]) * 0.02)
    else:
        t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
        x = _activations(gen, t, h)
        s["x"] = (x / x.square().mean(-1, keepdim=True).sqrt()).to(kind)
        s["router"] = (_randn(gen, e, h) * h ** -0.5).to(kind)
        s["bias"] = (_randn(gen, e) * 0.1).to(kind) if case["bias"] else None
        s["gate"] = _encode(case["fmt"], _randn(gen, e, i, h) * 0.02)
        s["up"] = _encode(case["fmt"], _randn(gen, e, i, h) * 0.02)
        s["down"] = _encode(case["fmt"], _randn(gen, e, h, i) * 0.02)
    return s


# ------------------------------------------------- the library's operators ----
_backend = _stream = None


def _library():
    """The library's module, its backend, and the backend's stream, on which its calls are enqueued."""
    global _backend, _stream
    import larql_b200
    if _backend is None:
        _backend = larql_b200.CudaBackend(0)
        _stream = torch.cuda.ExternalStream(_backend.stream())
    return larql_b200, _backend, _stream


def _matrix(lib, fmt, codes, scales, ts):
    """A resident matrix of the library over torch memory: codes [r, bytes], scales of its format."""
    tag = {"fp8": lib.FMT_FP8_B128, "mxfp4": lib.FMT_MXFP4, "nvfp4": lib.FMT_NVFP4}[fmt]
    cols = codes.shape[1] * (1 if fmt == "fp8" else 2)
    return lib.DeviceMatrix(tag, codes.shape[0], cols, codes.data_ptr(), codes.numel(), scales.data_ptr(),
                            scales.numel() * scales.element_size(), ts)


def _own_state(s):
    """What a program that uses the library keeps between calls: argument records, the layer's handle, outputs."""
    lib, be, _ = _library()
    case = s["case"]
    tag = {"f32": lib.T_F32, "bf16": lib.T_BF16, "f16": lib.T_F16}[case["type"]]
    if case["op"] == "block_norm":
        r, c = case["rows"], case["cols"]
        h, y, g = s["h"], s["y"], s["gate"]
        s["h_out"], s["n_out"] = torch.empty(r, c, dtype=h.dtype, device="cuda"), torch.empty(r, c, dtype=h.dtype, device="cuda")
        s["args"] = lib.BlockNormArgs(
            type=tag, w_type=tag, rows=r, cols=c, h=h.data_ptr(), h_stride=h.stride(0), y=y.data_ptr(), y_stride=y.stride(0),
            post_norm=case["post"], post_w=s["post_w"].data_ptr() if case["post"] else 0, pre_w=s["pre_w"].data_ptr(),
            w_offset=case["offset"], eps=_EPS, gate=0 if g is None else g.data_ptr(),
            gate_cols=0 if g is None else g.shape[1], gate_stride=0 if g is None else g.stride(0),
            gate_group=r if case["gate"] == "channel" else 1, h_scale=case["h_scale"], y_scale=case["y_scale"],
            h_out=s["h_out"].data_ptr(), h_out_stride=c, n_out=s["n_out"].data_ptr(), n_out_stride=c)
    elif case["op"] == "fp8_quantize":
        t, c = case["tokens"], case["cols"]
        s["q"] = torch.empty(t, c, dtype=torch.float8_e4m3fn, device="cuda")
        s["s"] = torch.empty(t, (c + 127) // 128, dtype=torch.float32, device="cuda")
        s["tag"] = tag
    elif case["op"] == "fp8_matmul":
        s["w"] = _matrix(lib, "fp8", s["codes"], s["scales"], 1.0)
        s["out"] = torch.empty(case["tokens"], case["rows"], dtype=s["x"].dtype, device="cuda")
        s["tag"] = tag
    else:
        t, n = case["tokens"], case["experts"]
        experts = [[_matrix(lib, case["fmt"], s[k][0][e], s[k][1][e], s[k][2]) for e in range(n)] for k in ("gate", "up", "down")]
        s["layer"] = be.moe_create(*experts, s["router"].data_ptr(), tag, 0 if s["bias"] is None else s["bias"].data_ptr(),
                                   case["top_e"], case["renorm"])
        s["out"] = torch.empty_like(s["x"])
        s["idx"] = torch.empty(t, case["top_e"], dtype=torch.int32, device="cuda")
        s["w"] = torch.empty(t, case["top_e"], dtype=torch.float32, device="cuda")
        s["tag"] = tag
    return s


def _own_run(s):
    _, be, stream = _library()
    if torch._C._cuda_getCurrentRawStream(0) == stream.cuda_stream:  # (torch.cuda.current_stream() takes 3 us, as long as a norm)
        return _own_call(s, be)
    # on another stream: the call behind what made its inputs, what reads its outputs behind the call
    current = torch.cuda.current_stream()
    stream.wait_stream(current)
    out = _own_call(s, be)
    current.wait_stream(stream)
    return out


def _own_call(s, be):
    op = s["case"]["op"]
    if op == "block_norm":
        be.dev_block_norm(s["args"])
        return {"h": s["h_out"], "n": s["n_out"]}
    if op == "fp8_quantize":
        x = s["x"]
        be.dev_fp8_quantize(x.data_ptr(), s["tag"], x.shape[0], x.shape[1], x.shape[1], s["q"].data_ptr(), s["s"].data_ptr())
        return {"q": s["q"], "s": s["s"]}
    if op == "fp8_matmul":
        x = s["x"]
        be.dev_fp8_matmul(s["w"], x.data_ptr(), s["tag"], x.shape[0], x.shape[1], s["out"].data_ptr(), s["tag"], s["out"].shape[1])
        return s["out"]
    be.dev_moe_ffn(s["layer"], s["x"].data_ptr(), s["tag"], s["x"].shape[0], s["out"].data_ptr(), s["idx"].data_ptr(), s["w"].data_ptr())
    return {"out": s["out"], "idx": s["idx"], "w": s["w"]}


# -------------------------------------------------------- the plain forms ----
def _rms(v):
    return torch.sqrt(v.square().mean(-1, keepdim=True) + _EPS)


def _quantize(x):
    t, c = x.shape
    nb = (c + 127) // 128
    b = torch.nn.functional.pad(x.float(), (0, nb * 128 - c)).view(t, nb, 128)
    amax = b.abs().amax(-1)
    s = torch.clamp(amax / torch.full_like(amax, 448), min=2.0 ** -126)  # (a number would be multiplied by its inverse)
    return (b / s[..., None]).to(torch.float8_e4m3fn).view(t, nb * 128)[:, :c], s


def _spread(scales, shape):
    """One scale per 128 x 128 block -> one per element."""
    return scales.repeat_interleave(128, -2)[..., :shape[-2], :].repeat_interleave(128, -1)[..., :shape[-1]]


def _decode(fmt, codes, scales, ts):
    if fmt == "fp8":
        return codes.view(torch.float8_e4m3fn).float() * _spread(scales, codes.shape)
    lut = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack((lut[(codes & 15).int()], lut[(codes >> 4).int()]), -1).flatten(-2)
    if fmt == "mxfp4":
        return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)
    return (v.unflatten(-1, (-1, 16)) * (scales.view(torch.float8_e4m3fn).float() * ts)[..., None]).flatten(-2)


def _plain_run(s):
    case = s["case"]
    if case["op"] == "block_norm":
        h, y = s["h"].float(), s["y"].float()
        if case["post"]:
            y = y / _rms(y) * (case["offset"] + s["post_w"].float())
        if s["gate"] is not None:
            y = y * s["gate"].float()
        h = case["h_scale"] * h + case["y_scale"] * y
        n = h / _rms(h) * (case["offset"] + s["pre_w"].float())
        return {"h": h.to(s["h"].dtype), "n": n.to(s["h"].dtype)}
    if case["op"] == "fp8_quantize":
        q, sc = _quantize(s["x"])
        return {"q": q.contiguous(), "s": sc}
    if case["op"] == "fp8_matmul":
        q, sc = _quantize(s["x"])
        x = q.float() * sc.repeat_interleave(128, 1)[:, :q.shape[1]]
        return (x @ _decode("fp8", s["codes"], s["scales"], 1.0).t()).to(s["x"].dtype)
    t, k, n = case["tokens"], case["top_e"], case["experts"]
    x = s["x"].float()
    # the choice of experts compares neighbouring logits: 64-bit sums, so that rounding does not decide it
    logits = x.double() @ s["router"].double().t()
    if s["bias"] is not None:
        logits = logits + s["bias"].double()
    logits = logits.float()
    idx = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :k]
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    chosen = e.gather(1, idx)
    w = chosen / (chosen if case["renorm"] else e).sum(-1, keepdim=True)
    if t * k <= n:  # few pairs: the chosen experts' weights alone
        gate, up, down = (_decode(case["fmt"], s[m][0][idx], s[m][1][idx], s[m][2]) for m in ("gate", "up", "down"))
        g, u = torch.einsum("th,tkih->tki", x, gate), torch.einsum("th,tkih->tki", x, up)
        out = torch.einsum("tki,tkhi,tk->th", g / (1 + torch.exp(-g)) * u, down, w)
    else:  # every expert for every token, unchosen ones weighted zero
        every = torch.zeros(t, n, device=x.device).scatter_(1, idx, w)
        gate, up, down = (_decode(case["fmt"], *s[m]) for m in ("gate", "up", "down"))
        g, u = torch.matmul(x, gate.transpose(1, 2)), torch.matmul(x, up.transpose(1, 2))  # [experts, tokens, inter]
        a = g / (1 + torch.exp(-g)) * u * every.t()[:, :, None]
        out = torch.bmm(a, down.transpose(1, 2)).sum(0)
    return {"out": out.to(s["x"].dtype), "idx": idx.int(), "w": w}


def prepare(case, seed):
    if not own:
        return _inputs(case, seed)
    # a program that works with the library runs its own GPU work on the library's stream: one order for both
    torch.cuda.set_stream(_library()[2])
    return _own_state(_inputs(case, seed))


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ---------------------------------------- the definitions, in 64 bits ----
def _to_e4m3(v):
    """The nearest e4m3 value of each f64, ties to the even code, up to the largest finite value."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(v) * torch.clamp(torch.round(a / step) * step, max=448.0)


def _exact_quantized(x):
    """(code values, scales) of the activation, both f64, by the definition's roundings."""
    x = x.double()
    t, c = x.shape
    q, scales = torch.empty_like(x), torch.empty(t, (c + 127) // 128, dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, 128 * b:128 * b + 128]
        sc = torch.clamp((part.abs().max(1).values / 448).float().double(), min=2.0 ** -126)
        scales[:, b] = sc
        q[:, 128 * b:128 * b + 128] = _to_e4m3((part / sc[:, None]).float().double())
    return q, scales


def _exact_weight(fmt, codes, scales, ts):
    """One matrix, in f64."""
    if fmt == "fp8":
        w = codes.view(torch.float8_e4m3fn).double()
        for i in range(scales.shape[0]):
            for j in range(scales.shape[1]):
                w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= scales[i, j].double()
        return w
    values = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2], w[:, 1::2] = values[codes.long() % 16], values[codes.long() // 16]
    if fmt == "mxfp4":
        return w * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, 1)
    return w * (scales.view(torch.float8_e4m3fn).double() * ts).repeat_interleave(16, 1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "block_norm":
        h, z = s["h"].double() * case["h_scale"], s["y"].double()
        if case["post"]:
            z = z * (s["post_w"].double() + case["offset"]) / ((z * z).sum(1, keepdim=True) / case["cols"] + _EPS) ** 0.5
        z = z * case["y_scale"]
        h = h + (z if s["gate"] is None else z * s["gate"].double())
        return {"h": h, "n": h * (s["pre_w"].double() + case["offset"]) / ((h * h).sum(1, keepdim=True) / case["cols"] + _EPS) ** 0.5}
    if case["op"] == "fp8_quantize":
        q, sc = _exact_quantized(s["x"])
        return {"q": q, "s": sc}
    if case["op"] == "fp8_matmul":
        q, sc = _exact_quantized(s["x"])
        x = q * sc.repeat_interleave(128, 1)[:, :q.shape[1]]
        return x @ _exact_weight("fp8", s["codes"], s["scales"], 1.0).t()
    x = s["x"].double()
    logits = torch.einsum("th,eh->te", x, s["router"].double())
    if s["bias"] is not None:
        logits = logits + s["bias"].double()
    logits = logits.float().double()
    out, k = torch.zeros_like(x), case["top_e"]
    rank = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    p = torch.softmax(logits, 1)
    w = torch.gather(p, 1, rank)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    for e in range(case["experts"]):
        t, j = torch.nonzero(rank == e, as_tuple=True)
        if t.numel():
            gate, up, down = (_exact_weight(case["fmt"], s[m][0][e], s[m][1][e], s[m][2]) for m in ("gate", "up", "down"))
            g = x[t] @ gate.t()
            out.index_add_(0, t, (g * torch.sigmoid(g) * (x[t] @ up.t())) @ down.t() * w[t, j][:, None])
    return {"out": out, "idx": rank.int(), "w": w}


def work(case):
    z = _SIZE[case["type"]]
    if case["op"] == "block_norm":
        r, c = case["rows"], case["cols"]
        gate = {"none": 0, "channel": c, "row": r, "full": r * c}[case["gate"]]
        return {"bytes": z * (4 * r * c + gate + c * (2 if case["post"] else 1)), "flops": 12 * r * c}
    if case["op"] == "fp8_quantize":
        t, c = case["tokens"], case["cols"]
        return {"bytes": t * (c * (z + 1) + 4 * ((c + 127) // 128)), "flops": 3 * t * c}
    if case["op"] == "fp8_matmul":
        t, c, r = case["tokens"], case["cols"], case["rows"]
        return {"bytes": z * t * (c + r) + r * c + 4 * ((r + 127) // 128) * ((c + 127) // 128), "flops": 2 * t * c * r}
    t, h, i, n, k = (case[m] for m in ("tokens", "hidden", "inter", "experts", "top_e"))
    read = n * (1 - (1 - k / n) ** t)  # experts that at least one token chooses, on average
    per = {"mxfp4": 17 / 32, "nvfp4": 9 / 16, "fp8": 1 + 4 / 16384}[case["fmt"]]
    return {"bytes": 3 * read * h * i * per + z * (n * h + 2 * t * h) + 8 * t * k, "flops": 2 * t * (n * h + 3 * k * h * i)}
