"""What is measured of the transformer-block operators: the residual join with its norms (`block_norm` and its backward pass), rotary
positions over several axes (`rotary_axes`) and the 4-bit microscaled Linear layer (`mxfp4_quantize`, `mxfp4_dequantize`,
`mxfp4_linear`).

`listed()` are the cases, `draw(rng)` gives more of the same ranges, `prepare(case, seed)` what a program has in hand before the call,
`run(state)` one pass, `work(case)` what a pass cannot do without, `exact(case, seed)` the outputs from the definition in 64 bits.
With `own` false a pass is elementary torch operations, with `own` true the calls of `onedc_amd.kernels`.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------------------------------------------
def _norm(name, batch, tokens, channels, type, stream="same", kind="layer", post=False, gate=True, mod=True, affine=False, alpha=1.0,
          back=False):
    return {"name": name, "op": "norm_back" if back else "norm", "type": type, "stream": stream, "batch": batch, "tokens": tokens,
            "channels": channels, "kind": kind, "post": post, "gate": gate, "mod": mod, "affine": affine, "alpha": alpha}


def _rotary(name, batch, t, h, w, heads, kv_heads, dim, type, axes="thw", layout="halves", shared=False, positions="int", offset=0,
            inverse=False):
    return {"name": name, "op": "rotary", "type": type, "batch": batch, "t": t, "h": h, "w": w, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "axes": axes, "layout": layout, "shared": shared, "positions": positions, "offset": offset, "inverse": inverse}


def _mx(name, op, rows, k, n, type, epi="linear", bias=True, res=False):
    return {"name": name, "op": op, "type": type, "rows": rows, "k": k, "n": n, "epi": epi, "bias": bias, "res": res}


def listed():
    return [
        # one token of a serving step: the join between attention and the feed-forward part, 1280 channels; latency
        _norm("norm-token", 1, 1, 1280, "bf16", kind="rms", post=True, gate=False, mod=False, affine=True),
        # sixteen 768 x 768 pictures at the first level of the denoiser (96 x 96 tokens of 320 channels), gated and modulated per picture
        _norm("norm-level0", 16, 9216, 320, "f16"),
        # three sequences of an odd length, norms on both sides of the block, the residual stream kept in 32 bits, residuals scaled down
        _norm("norm-sandwich", 3, 1031, 1000, "bf16", stream="f32", kind="rms", post=True, mod=False, affine=True, alpha=0.25),
        # training step at the second level (48 x 48 tokens of 640 channels), every parameter's gradient
        _norm("norm-back-level1", 16, 2304, 640, "f16", post=True, affine=True, back=True),
        # the same with an odd channel count (nothing is aligned), few rows, a 32-bit stream
        _norm("norm-back-odd", 2, 333, 1283, "bf16", stream="f32", kind="rms", back=True),
        # one token of a sequence far along its time axis: query heads share key heads; latency
        _rotary("rotary-token", 1, 1, 1, 1, 16, 4, 128, "bf16", offset=1000003),
        # a clip of 16 frames of 48 x 64 latents, 16 heads of 80 dims
        _rotary("rotary-video", 1, 16, 48, 64, 16, 16, 80, "f16"),
        # backward pass over sixteen 48 x 48 maps, neighbouring pairs, one spectrum for both axes, positions between the grid's points
        _rotary("rotary-back-image", 16, 1, 48, 48, 8, 8, 80, "bf16", axes="hw", layout="neighbours", shared=True, positions="real",
                inverse=True),
        # activations of the third level (24 x 24 tokens of 1280 channels, sixteen pictures) held in 4 bits and read back
        _mx("mx-hold", "mx_hold", 9216, 1280, 0, "f16"),
        # one token against a weight of 8192 x 8192: bound by the weight's bytes
        _mx("mx-token", "mx_linear", 1, 8192, 8192, "bf16"),
        # gated feed-forward projection 1280 -> 2 x 5120 over fifteen ragged sequences
        _mx("mx-geglu", "mx_linear", 8655, 1280, 10240, "f16", epi="geglu"),
        # a large layer with its residual: bound by the matrix cores
        _mx("mx-large", "mx_linear", 16384, 8192, 8192, "bf16", res=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "norm_back", "norm_back", "rotary", "rotary", "mx_hold", "mx_linear", "mx_linear", "mx_linear"))
    type = rng.choice(("f16", "bf16"))
    if op.startswith("norm"):
        channels = _log(rng, 64, 4096)
        channels -= rng.choice((channels % 8, channels % 8, 0))
        batch = rng.randint(1, 16)
        tokens = _log(rng, 1, max(1, min(9216, 47185920 // (batch * channels))))
        return dict(_norm("", batch, tokens, channels, type, rng.choice(("same", "f32")), rng.choice(("layer", "rms")), rng.random() < 0.5,
                          rng.random() < 0.7, rng.random() < 0.7, rng.random() < 0.7, rng.choice((1.0, 0.25, 0.7071)), op == "norm_back"))
    if op == "rotary":
        dim = rng.choice((40, 64, 72, 80, 96, 128, 160))
        heads = _log(rng, 1, 32)
        kv_heads = rng.choice([d for d in range(1, heads + 1) if heads % d == 0])
        batch = rng.randint(1, 4)
        most = max(1, 62914560 // (batch * (heads + kv_heads) * dim))
        w = _log(rng, 1, max(1, min(96, most)))
        h = _log(rng, 1, max(1, min(96, most // w)))
        t = _log(rng, 1, max(1, min(32, most // (w * h))))
        return dict(_rotary("", batch, t, h, w, heads, kv_heads, dim, type, rng.choice(("thw", "hw")), rng.choice(("halves", "neighbours")),
                            rng.random() < 0.5, rng.choice(("int", "real")), rng.choice((0, 17, 100003)), rng.random() < 0.4))
    k = _log(rng, 32, 8192)
    k -= rng.choice((k % 32, k % 32, k % 8, 0))
    rows = _log(rng, 1, 16384)
    if op == "mx_hold":
        return dict(_mx("", op, rows, k, 0, type))
    epi = rng.choice(("linear", "linear", "silu", "geglu"))
    n = _log(rng, 32, 8192)
    n -= n % 32 if epi == "geglu" else rng.choice((n % 8, 0))
    return dict(_mx("", op, rows, k, n, type, epi, rng.random() < 0.7, rng.random() < 0.4))


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _sections(case):
    """Dims of a head that each axis turns, even numbers; what is left over at the end passes through."""
    d, a = case["dim"], len(case["axes"])
    if a == 2:
        part = d // 4 * 2
        return (part, part)
    part = d // 6 * 2
    return (d - 2 * part - (d - 2 * part) % 2, part, part)


def _stream_type(case):
    return torch.float32 if case["stream"] == "f32" else TYPES[case["type"]]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    type = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device=DEV) * scale + shift

    s = {"case": case}
    if case["op"].startswith("norm"):
        B, N, C = case["batch"], case["tokens"], case["channels"]
        spread = torch.exp(normal(C, scale=0.5)) * torch.where(torch.rand(C, generator=g, device=DEV) < 0.01, 8.0, 1.0)
        s["x"] = (normal(B, N, C) * spread + normal(C, scale=0.3)).to(_stream_type(case))
        s["f"] = normal(B, N, C, scale=0.7, shift=0.1).to(type)
        mod = normal(B, 3 * C, scale=0.3)                          # one projection of the conditioning: scale | shift | gate
        s["scale"], s["shift"] = (mod[:, :C], mod[:, C:2 * C]) if case["mod"] else (None, None)
        s["gate"] = mod[:, 2 * C:].add_(0.5) if case["gate"] else None
        s["w"] = normal(C, scale=0.1, shift=1.0) if case["affine"] else None
        s["b"] = normal(C, scale=0.1) if case["affine"] and case["kind"] == "layer" else None
        s["post_w"] = normal(C, scale=0.1, shift=1.0) if case["post"] else None
        if case["op"] == "norm_back":
            s["dy"] = normal(B, N, C, scale=0.1).to(type)
            s["dxo"] = normal(B, N, C, scale=0.1).to(_stream_type(case))
        return s
    if case["op"] == "rotary":
        T, H, W, D = case["t"], case["h"], case["w"], case["dim"]
        N, hq, hk = T * H * W, case["heads"], case["kv_heads"]
        s["qk"] = normal(case["batch"], N, (hq + hk) * D).to(type)      # one projection: queries | keys
        grid = torch.meshgrid(*(torch.arange(n, device=DEV) for n in (T, H, W)), indexing="ij")
        pos = torch.stack([v.reshape(-1) for v in grid], 1) + case["offset"]
        pos = pos[:, 3 - len(case["axes"]):]
        if case["positions"] == "real":                              # a grid of another resolution, stretched onto the trained one
            s["pos"] = (pos.float() + 0.5) * 0.73
        else:
            s["pos"] = pos.to(torch.int32)
        sec = _sections(case)
        rot = sum(sec)
        axis = torch.cat([torch.full((n // 2,), a) for a, n in enumerate(sec)])
        if case["shared"]:
            freq = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
        else:
            freq = torch.cat([10000.0 ** (-2.0 * torch.arange(n // 2, dtype=torch.float64) / n) for n in sec])
        s["axis"], s["freq"] = axis.to(DEV), freq.to(DEV)
        if own:
            from onedc_amd import kernels
            s["plan"] = kernels.RotaryAxes(D, sec, theta=10000.0, neighbours=case["layout"] == "neighbours",
                                           shared_spectrum=case["shared"], device=torch.device("cuda", torch.cuda.current_device()))
        return s
    rows, k, n = case["rows"], case["k"], case["n"]
    spread = torch.exp(normal(k, scale=0.7)) * torch.where(torch.rand(k, generator=g, device=DEV) < 0.01, 16.0, 1.0)
    s["x"] = (normal(rows, k) * spread).to(type)
    if case["op"] == "mx_linear":
        w = normal(n, k, scale=k ** -0.5) * torch.exp(normal(n, 1, scale=0.3))
        s["codes"], s["scales"] = _codes(w)
        s["bias"] = normal(n, scale=0.1) if case["bias"] else None
        s["res"] = normal(rows, n // 2 if case["epi"] == "geglu" else n).to(type) if case["res"] else None
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------
def _normed(v, kind):
    """(normalised rows, reciprocal deviation) in 32 bits."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * r, r


def _per_picture(v):
    return v[:, None, :]


def _plain_norm(s, kind, alpha, out, stream):
    branch = s["f"].float()
    if s["post_w"] is not None:
        branch = _normed(branch, kind)[0] * s["post_w"]
    if s["gate"] is not None:
        branch = branch * _per_picture(s["gate"])
    t = s["x"].float() + alpha * branch
    y = _normed(t, kind)[0]
    if s["w"] is not None:
        y = y * s["w"]
    if s["b"] is not None:
        y = y + s["b"]
    if s["scale"] is not None:
        y = y * (1 + _per_picture(s["scale"])) + _per_picture(s["shift"])
    return {"stream": t.to(stream), "y": y.to(out)}


def _through(u, hat, r, kind):
    """Gradient through a norm: u is the gradient of the normalised rows."""
    u = u - hat * (u * hat).mean(-1, keepdim=True) - (u.mean(-1, keepdim=True) if kind == "layer" else 0)
    return u * r


def _total(v, dims):
    return v.sum(dims, dtype=torch.float64).float()


def _plain_norm_back(s, kind, alpha, out, stream):
    got = {}
    dy, hat_r = s["dy"].float(), _normed(s["x"].float(), kind)
    hat, u = hat_r[0], dy
    if s["scale"] is not None:
        affine = hat if s["w"] is None else hat * s["w"]
        affine = affine if s["b"] is None else affine + s["b"]
        got["d_shift"], got["d_scale"] = _total(dy, 1), _total(dy * affine, 1)
        u = u * (1 + _per_picture(s["scale"]))
    if s["b"] is not None:
        got["d_b"] = _total(u, (0, 1))
    if s["w"] is not None:
        got["d_w"] = _total(u * hat, (0, 1))
        u = u * s["w"]
    dt = s["dxo"].float() + _through(u, *hat_r, kind)
    branch = f_hat = s["f"].float()
    if s["post_w"] is not None:
        f_hat, f_r = _normed(f_hat, kind)
        branch = f_hat * s["post_w"]
    v = alpha * dt
    if s["gate"] is not None:
        got["d_gate"] = _total(v * branch, 1)
        v = v * _per_picture(s["gate"])
    if s["post_w"] is not None:
        got["d_post_w"] = _total(v * f_hat, (0, 1))
        v = _through(v * s["post_w"], f_hat, f_r, kind)
    return {"dx": dt.to(stream), "df": v.to(out), **got}


def _plain_rotary(s, case):
    D, pairs = case["dim"], s["freq"].numel()
    angle = s["pos"].double()[:, s["axis"]] * s["freq"]                # far positions: the angle in 64 bits
    c, n = torch.cos(angle).float()[None, :, None], torch.sin(angle).float()[None, :, None]
    if case["inverse"]:
        n = -n
    v = s["qk"].float().unflatten(-1, (-1, D))
    if case["layout"] == "halves":
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat([a * c - b * n, b * c + a * n, v[..., 2 * pairs:]], -1)
    else:
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.cat([torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2), v[..., 2 * pairs:]], -1)
    return {"qk": turned.flatten(-2).to(s["qk"].dtype)}


def _held(v):
    """Blocks of 32 along the last axis as 4-bit floats (0 .5 1 1.5 2 3 4 6) with a power of two each: (q, exponent), v ~ q 2^exponent."""
    k = v.shape[-1]
    v = torch.nn.functional.pad(v.float(), (0, -k % 32)).unflatten(-1, (-1, 32))
    e = (torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 3).clamp_min(-127)      # floor(log2 amax) - 2
    e = torch.where(v.abs().amax(-1, keepdim=True) > 0, e, -127)
    v = torch.ldexp(v, -e)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return (torch.round(v / step) * step).clamp(-6, 6), e                          # round half to even


def _values(v):
    q, e = _held(v)
    return torch.ldexp(q, e).flatten(-2)[..., :v.shape[-1]]


def _codes(w):
    """What a checkpoint in 4 bits holds: two codes a byte (the lower half first), rows padded with zeros to 128, and a biased exponent
    byte per block of 32."""
    q, e = _held(torch.nn.functional.pad(w, (0, -w.shape[-1] % 128)))
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), (e[..., 0] + 127).to(torch.uint8).contiguous()


def _weight(codes, scales, k):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()].unflatten(-1, (-1, 32))
    return torch.ldexp(v, scales.int()[..., None] - 127).flatten(-2)[:, :k]


def _pairs(v):
    """Columns in blocks of 16, a block of values in front of each block of gates."""
    v = v.unflatten(-1, (-1, 2, 16))
    return v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)


def _plain_linear(s, case):
    y = _values(s["x"]) @ _weight(s["codes"], s["scales"], case["k"]).T
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["epi"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["epi"] == "geglu":
        a, b = _pairs(y)
        y = a * (0.5 * b * (1 + torch.erf(b * math.sqrt(0.5))))
    if s["res"] is not None:
        y = y + s["res"].float()
    return {"y": y.to(s["x"].dtype)}


# ---- one pass -----------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    type = TYPES[case["type"]]
    if case["op"] == "norm":
        return _plain_norm(s, case["kind"], case["alpha"], type, s["x"].dtype)
    if case["op"] == "norm_back":
        return _plain_norm_back(s, case["kind"], case["alpha"], type, s["x"].dtype)
    if case["op"] == "rotary":
        return _plain_rotary(s, case)
    if case["op"] == "mx_hold":
        return {"values": _values(s["x"]).to(type)}
    return _plain_linear(s, case)


def _own(s, case):
    from onedc_amd import kernels as K
    with K.act_format(case["type"]):
        if case["op"].startswith("norm"):
            return _own_norm(K, s, case)
        if case["op"] == "rotary":
            qk = s["qk"]
            B, N, C = qk.shape
            nq = case["heads"] * case["dim"]
            out = torch.empty_like(qk)
            v, o = K.View(qk, B, 1, N, C), K.View(out, B, 1, N, C)
            K.rotary_axes(s["plan"], s["pos"], v.slice(0, nq), o.slice(0, nq), v.slice(nq, C - nq), o.slice(nq, C - nq),
                          inverse=case["inverse"])
            return {"qk": out}
        rows, k = s["x"].shape
        x = K.View(s["x"], 1, 1, rows, k)
        if case["op"] == "mx_hold":
            out = torch.empty_like(s["x"])
            K.mxfp4_dequantize(K.mxfp4_quantize(x), K.View(out, 1, 1, rows, k))
            return {"values": out}
        n = case["n"] // 2 if case["epi"] == "geglu" else case["n"]
        y = torch.empty(rows, n, dtype=s["x"].dtype, device=s["x"].device)
        K.mxfp4_linear(x, K.MxFp4(s["codes"], s["scales"], case["n"], k), s["bias"], K.View(y, 1, 1, rows, n),
                       epi={"linear": K.EPI_LINEAR, "silu": K.EPI_SILU, "geglu": K.EPI_GEGLU}[case["epi"]],
                       res=K.View(s["res"], 1, 1, rows, n) if s["res"] is not None else None)
        return {"y": y}


def _own_norm(K, s, case):
    B, N, C = s["x"].shape

    def view(t):
        return K.View(t, B, 1, N, C)

    kind = K.NORM_LAYER if case["kind"] == "layer" else K.NORM_RMS
    given = dict(kind=kind, eps=EPS, alpha=case["alpha"], post=s["post_w"] is not None, post_w=s["post_w"], gate=s["gate"], w=s["w"],
                 b=s["b"], scale=s["scale"], shift=s["shift"])
    if case["op"] == "norm":
        xo, y = torch.empty_like(s["x"]), torch.empty_like(s["f"])
        K.block_norm(view(s["x"]), view(y), f=view(s["f"]), xo=view(xo), **given)
        return {"stream": xo, "y": y}
    out = {"dx": torch.empty_like(s["x"]), "df": torch.empty_like(s["f"])}
    grads = {"d_" + p: torch.empty_like(s[p], memory_format=torch.contiguous_format)
             for p in ("shift", "scale", "b", "w", "gate", "post_w") if s[p] is not None}
    K.block_norm_backward(view(s["x"]), view(s["dy"]), view(out["dx"]), dxo=view(s["dxo"]), f=view(s["f"]), df=view(out["df"]), **given,
                          **grads)
    return {**out, **grads}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    if case["op"].startswith("norm"):
        n = case["batch"] * case["tokens"] * case["channels"]
        wide = 4 if case["stream"] == "f32" else 2
        if case["op"] == "norm":
            return {"bytes": n * (2 * wide + 2 * 2), "flops": 20 * n}
        return {"bytes": n * (3 * wide + 3 * 2), "flops": 45 * n}
    if case["op"] == "rotary":
        tokens = case["t"] * case["h"] * case["w"]
        n = case["batch"] * tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * 2 * n + 4 * tokens * len(case["axes"]), "flops": 3 * n}
    rows, k, n = case["rows"], case["k"], case["n"]
    if case["op"] == "mx_hold":
        return {"bytes": 2 * 2 * rows * k, "flops": 4 * rows * k}
    out = n // 2 if case["epi"] == "geglu" else n
    return {"bytes": 2 * rows * k + n * k * 17 // 32 + 2 * rows * out * (2 if case["res"] else 1) + (4 * n if case["bias"] else 0),
            "flops": 2 * rows * n * k}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["op"].startswith("norm"):
        return _exact_norm(s, case)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    if case["op"] == "mx_hold":
        return {"values": _exact_held(s["x"])}
    return _exact_linear(s, case)


def _exact_norm(s, case):
    back = case["op"] == "norm_back"
    names = ["x", "f"] + [p for p in ("shift", "scale", "b", "w", "gate", "post_w") if s[p] is not None]
    leaf = {p: s[p].detach().clone().requires_grad_(back) for p in names}

    def norm(v):
        if case["kind"] == "layer":
            var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
            return (v - mean) / (var + EPS).sqrt()
        return v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()

    def after(t):
        y = norm(t) * leaf.get("w", 1.0) + leaf.get("b", 0.0)
        if case["mod"]:
            y = y + y * leaf["scale"].unsqueeze(1) + leaf["shift"].unsqueeze(1)
        return y

    branch = norm(leaf["f"]) * leaf["post_w"] if case["post"] else leaf["f"]
    if case["gate"]:
        branch = leaf["gate"].unsqueeze(1) * branch
    branch = branch * case["alpha"]
    if not back:
        t = s["x"] + branch
        return {"stream": t, "y": after(t)}
    # the stored stream is given: it is the join's own output, and x's gradient is the stream's
    names.remove("f")
    first = torch.autograd.grad(after(leaf["x"]), [leaf[p] for p in names if p not in ("gate", "post_w")], s["dy"])
    got = dict(zip([p for p in names if p not in ("gate", "post_w")], first))
    dt = got.pop("x") + s["dxo"]
    second = ["f"] + [p for p in ("gate", "post_w") if p in leaf]
    got.update(zip(second, torch.autograd.grad(branch, [leaf[p] for p in second], dt)))
    return {"dx": dt, "df": got.pop("f"), **{"d_" + p: got[p] for p in ("shift", "scale", "b", "w", "gate", "post_w") if p in got}}


def _exact_rotary(s, case):
    pairs = s["freq"].numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       (-1 if case["inverse"] else 1) * torch.index_select(s["pos"].double(), 1, s["axis"]) * s["freq"]).unsqueeze(1)
    v = s["qk"].reshape(*s["qk"].shape[:2], -1, case["dim"]).clone()
    first, second = ((slice(0, pairs), slice(pairs, 2 * pairs)) if case["layout"] == "halves" else
                     (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)))
    z = torch.complex(v[..., first], v[..., second]) * turn
    v[..., first], v[..., second] = z.real, z.imag
    return {"qk": v.reshape(s["qk"].shape)}


def _exact_held(v):
    rows, k = v.shape
    x = torch.zeros(rows, -(-k // 32) * 32, dtype=torch.float64, device=DEV)
    x[:, :k] = v
    x = x.reshape(rows, -1, 32)
    top = x.abs().amax(2, keepdim=True)
    unit = torch.where(top > 0, 2.0 ** (torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2), 1.0)
    a = x.abs() / unit
    held = torch.zeros_like(a)
    # halfway points go to the code with an even last bit: 0, 1, 2, 4
    for value, over, with_tie in ((.5, .25, False), (1., .75, True), (1.5, 1.25, False), (2., 1.75, True), (3., 2.5, False), (4., 3.5, True),
                                  (6., 5., False)):
        held = torch.where(a >= over if with_tie else a > over, value, held)
    return (held * torch.sign(x) * unit).reshape(rows, -1)[:, :k]


def _exact_linear(s, case):
    rows, k = s["x"].shape
    x = _exact_held(s["x"])
    byte = s["codes"].int()
    code = torch.empty(byte.shape[0], byte.shape[1] * 2, dtype=torch.int32, device=DEV)
    code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
    mant, ex = code % 2, code // 2 % 4
    w = torch.where(ex > 0, (1 + 0.5 * mant) * 2.0 ** (ex.double() - 1), 0.5 * mant) * (1 - 2 * (code // 8))
    w = w * (2.0 ** (s["scales"].double() - 127)).repeat_interleave(32, 1)
    y = x @ w[:, :k].T
    if s["bias"] is not None:
        y += s["bias"]
    if case["epi"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["epi"] == "geglu":
        column = torch.arange(case["n"] // 2, device=DEV)
        at = column // 16 * 32 + column % 16
        y = y[:, at] * y[:, at + 16] * torch.special.ndtr(y[:, at + 16])
    if s["res"] is not None:
        y = y + s["res"]
    return {"y": y}
