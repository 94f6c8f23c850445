"""Transformer-block operators on the GPU against plain implementations in 64 bits: block_norm and its backward pass, rotary_axes,
mxfp4_quantize / _dequantize / _linear, and a transformer block made of them.

Tolerances, derived before any run.  u(t) = finfo(t).eps / 2 is half a step of the output type, eps32 = 2^-24 half a step of f32.
 * one rounding to the output type: u |value| (and half of the type's smallest subnormal);
 * the f32 arithmetic in front of it: every operation rounds once.  A row's mean and mean square are sums of C terms in some order:
   relative to the sum of magnitudes at most C eps32, in a tree of the kind a wave uses far less; n eps32 times the largest
   magnitude of a row's terms, n = C + 32, is what is allowed;
 * a sum over n rows: n eps32 times the sum of the terms' magnitudes, plus what the terms themselves were off;
 * sine and cosine: the fraction of a turn is rounded to f32 (2^-26 of a turn = 2^-23.3 rad at the half turn), the functions to
   2^-23, the two products and the sum to eps32 each: together under 2^-21 (|a| + |b|);
 * codes and scales of MXFP4 are exact: equality;
 * a product of K terms: every product is exact in f32, sums in any order are K eps32 sum |x w|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from onedc_amd import kernels as K
from onedc_amd import pack
from onedc_amd.kernels import KernelError, MxFp4, RotaryAxes, View, new_view

DEV = "cuda:0"
F32 = torch.float32
EPS32 = 2.0 ** -24
FORMATS = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(params=["f16", "bf16"])
def fmt(request):
    with K.act_format(request.param):
        yield FORMATS[request.param]


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, ref, tol, what=""):
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = tol.cpu() if isinstance(tol, torch.Tensor) else tol
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what + ": NaN in other places"
    bad = ~(((got - ref).abs() <= tol) | torch.isnan(ref) | (got == ref))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - ref).abs() / tol)[bad].max()):.2f} x tolerance"


def rand(gen, *shape, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=gen) * scale + shift


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tokens(t, cs=None, co=0, fill=7.0):
    """[B, N, C] CPU tensor (already of its final type) -> View on the GPU, inside rows of cs channels filled with `fill`."""
    B, N, Cc = t.shape
    cs = cs or Cc
    buf = torch.full((B * N, cs), fill, dtype=t.dtype)
    buf[:, co:co + Cc] = t.reshape(-1, Cc)
    return View(buf.reshape(-1).to(DEV), B, 1, N, Cc, cs, co)


def empty(B, N, Cc, dtype, cs=None, co=0, fill=7.0):
    return tokens(torch.full((B, N, Cc), 3.0, dtype=dtype), cs, co, fill)


def back(v):
    return v.t[:v.B * v.H * v.W * v.cs].view(v.B, v.H * v.W, v.cs)[..., v.co:v.co + v.C].cpu()


def untouched(v, fill=7.0):
    rows = v.t[:v.B * v.H * v.W * v.cs].view(-1, v.cs)
    rest = torch.cat([rows[:, :v.co], rows[:, v.co + v.C:]], 1)
    return bool((rest == fill).all()) and bool((v.t[v.B * v.H * v.W * v.cs:] == fill).all())


# ---- block_norm -------------------------------------------------------------------------------------------------------------------
def norm64(v, kind, eps):
    if kind == K.NORM_LAYER:
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def join64(x, f, a, eps):
    """(t, y) of the definition in 64 bits; a: the options, tensors in 64 bits."""
    t = x
    if f is not None:
        v = f
        if a.get("post"):
            v = norm64(f, a["kind"], eps) * a.get("post_w", 1.0) + a.get("post_b", 0.0)
        g = a.get("gate", 1.0)
        t = x + a.get("alpha", 1.0) * (g.unsqueeze(-2) if isinstance(g, torch.Tensor) and g.dim() == 2 else g) * v
    y = norm64(t, a["kind"], eps) * a.get("w", 1.0) + a.get("b", 0.0)
    for name in ("scale", "shift"):
        if name in a:
            m = a[name].unsqueeze(-2) if a[name].dim() == 2 else a[name]
            y = y * (1 + m) if name == "scale" else y + m
    return t, y


def options(g, B, Cc, kind, post, gate, mod, affine, alpha=1.0):
    """gate / mod: None, "one" ([C]), "each" ([B, C], a slice of wider rows)."""
    def row(how, shift=0.0):
        return rand(g, Cc, scale=0.4, shift=shift) if how == "one" else rand(g, B, 3 * Cc, scale=0.4, shift=shift)[:, Cc:2 * Cc]
    a = dict(kind=kind, alpha=alpha)
    if post:
        a.update(post=True, post_w=rand(g, Cc, scale=0.2, shift=1.0))
        if affine:
            a["post_b"] = rand(g, Cc, scale=0.2)
    if gate:
        a["gate"] = row(gate, 0.6)
    if mod:
        a["scale"], a["shift"] = row(mod), row(mod)
    if affine:
        a["w"], a["b"] = rand(g, Cc, scale=0.2, shift=1.0), rand(g, Cc, scale=0.2)
    return a


def on_gpu(a):
    # (a slice stays a slice: its row stride is part of what is tested)
    out = {}
    for k, v in a.items():
        if isinstance(v, torch.Tensor) and v.dim() == 2 and not v.is_contiguous():
            wide = torch.zeros(v.shape[0], v.stride(0))
            wide[:, v.shape[1]:2 * v.shape[1]] = v
            v = wide.to(DEV)[:, v.shape[1]:2 * v.shape[1]]
        elif isinstance(v, torch.Tensor):
            v = v.to(DEV)
        out[k] = v
    return out


def in64(a):
    return {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in a.items()}


def tol_y(t, y, a, out):
    """Tolerance of y: f32 arithmetic on a normalised row, one rounding to `out`."""
    Cc = t.shape[-1]
    r = 1 / torch.sqrt(((t - (t.mean(-1, keepdim=True) if a["kind"] == K.NORM_LAYER else 0)) ** 2).mean(-1, keepdim=True) + 1e-12)
    gain = (a.get("w", torch.ones(1)).abs().max() * (1 + (a["scale"].abs().max() if "scale" in a else 0))).double()
    top = t.abs().amax(-1, keepdim=True) * r * gain + sum(a[n].abs().max().double() for n in ("b", "shift") if n in a) * (1 + gain)
    return half_step(out) * y.abs() + tiny(out) + (Cc + 32) * EPS32 * top


CASES = [
    # B, N, C, kind, post, gate, mod, affine, alpha
    (1, 1, 1280, "rms", True, None, None, True, 1.0),
    (2, 5, 320, "layer", False, "each", "each", False, 1.0),
    (3, 7, 1000, "rms", True, "one", None, True, 0.25),
    (2, 9, 640, "layer", True, "each", "each", True, 1.0),
    (2, 3, 1283, "rms", False, "each", "one", False, 0.7),
    (1, 4, 1, "layer", False, None, "each", True, 1.0),
    (1, 4, 1, "rms", True, "one", None, True, 1.0),
    (4, 33, 64, "layer", False, None, None, True, 1.0),
    (1, 2, 4096, "layer", True, "one", "each", True, 1.0),
    (1, 3, 8200, "rms", True, "each", "each", True, 1.0),
    (2, 2, 20001, "layer", True, "each", "each", True, 1.0),
    (5, 1, 100, "layer", False, "each", "each", True, -2.0),
    (2, 131, 72, "rms", False, "each", None, True, 1.0),
    (1, 17, 2048, "layer", False, "one", "one", True, 1.0),
    (2, 6, 1536, "rms", True, "each", "each", True, 1.0),
    (1, 5, 2500, "layer", False, "one", None, True, 1.0),
    (1, 2, 5001, "rms", True, "each", "each", True, 1.0),
    (70000, 1, 8, "layer", False, "each", "each", False, 1.0),
    (1, 70000, 3, "layer", False, "one", None, True, 1.0),
    (2, 40, 7, "rms", True, "each", "each", True, 1.0),
]


@pytest.mark.parametrize("types", ["16", "32/16", "32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_block_norm(case, types, fmt):
    B, N, Cc, kind, post, gate, mod, affine, alpha = case
    xt, ft = (F32 if types != "16" else fmt), (F32 if types == "32" else fmt)
    g = gen(Cc + N)
    kind = K.NORM_LAYER if kind == "layer" else K.NORM_RMS
    a = options(g, B, Cc, kind, post, gate, mod, affine, alpha)
    x, f = rand(g, B, N, Cc, scale=2.0, shift=0.5).to(xt), rand(g, B, N, Cc, shift=0.2).to(ft)
    cs = Cc + (8 if N % 2 else 3)                        # even and odd pitches
    xo, y = empty(B, N, Cc, xt, cs, 1 if N % 2 == 0 else 8), empty(B, N, Cc, ft, cs + 5, 5)
    K.block_norm(tokens(x, cs, 2), y, f=tokens(f), xo=xo, eps=1e-6, **on_gpu(a))
    t, ref = join64(x.double(), f.double(), in64(a), 1e-6)
    step = (t - x.double()).abs() + x.double().abs()
    within(back(xo), t, half_step(xt) * t.abs() + tiny(xt) + (Cc + 32) * EPS32 * step.amax(-1, keepdim=True) * (1 if post else 0.2), "xo")
    within(back(y), ref, tol_y(t, ref, a, ft), "y")
    assert untouched(xo) and untouched(y)
    # the parts of it: the join alone, the norm alone, the stream in place
    alone = empty(B, N, Cc, xt)
    K.block_norm(tokens(x), f=tokens(f), xo=alone, eps=1e-6, **{k: v for k, v in on_gpu(a).items() if k not in ("w", "b", "scale", "shift")})
    within(back(alone), t, half_step(xt) * t.abs() + tiny(xt) + (Cc + 32) * EPS32 * step.amax(-1, keepdim=True), "join alone")
    pre = {k: v for k, v in on_gpu(a).items() if k in ("kind", "w", "b", "scale", "shift")}
    yn = empty(B, N, Cc, ft)
    K.block_norm(tokens(x), yn, eps=1e-6, **pre)
    _, ref = join64(x.double(), None, in64(a), 1e-6)
    within(back(yn), ref, tol_y(x.double(), ref, a, ft), "norm alone")
    xv, y2 = tokens(x, cs, 2), empty(B, N, Cc, ft, cs + 5, 5)
    K.block_norm(xv, y2, f=tokens(f), xo=xv, eps=1e-6, **on_gpu(a))
    assert torch.equal(back(xv), back(xo)) and torch.equal(back(y2), back(y)) and untouched(xv)


def test_block_norm_rows_of_one_value_and_rows_that_are_not_numbers():
    Cc = 320
    x = torch.randn(1, 6, Cc, generator=gen(1)).half()
    x[0, 1], x[0, 2], x[0, 3, 7], x[0, 4, 9] = 0.0, 3.0, float("nan"), float("inf")
    w, b = rand(gen(2), Cc, shift=1.0), rand(gen(3), Cc)
    with K.act_format("f16"):
        for kind in (K.NORM_LAYER, K.NORM_RMS):
            y = empty(1, 6, Cc, torch.float16)
            K.block_norm(tokens(x), y, kind=kind, eps=1e-6, w=w.to(DEV), b=b.to(DEV))
            got = back(y)[0]
            _, ref = join64(x.double(), None, dict(kind=kind, w=w.double(), b=b.double()), 1e-6)
            within(got[[0, 5]], ref[0, [0, 5]], tol_y(x[0, [0, 5]].double(), ref[0, [0, 5]], dict(kind=kind, w=w, b=b), torch.float16), "others")
            assert torch.equal(got[1], b.half())                             # zeros: the shift alone
            if kind == K.NORM_LAYER:
                assert torch.equal(got[2], b.half())                         # a constant has no variance, and its mean is exact
            assert got[3].isnan().all() and got[4].isnan().any()


def test_block_norm_has_nothing_to_do_for_no_rows(fmt):
    x, y = View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 4, 64), View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 4, 64)
    K.block_norm(x, y)
    dw = torch.full((64,), 3.0, device=DEV)
    K.block_norm_backward(x, y, View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 4, 64), w=torch.ones(64, device=DEV), d_w=dw)
    assert float(dw.abs().max()) == 0.0
    none = View(torch.empty(0, dtype=fmt, device=DEV), 3, 1, 0, 64)              # three pictures without a token: gradients of their gates too
    for B in (1, 3):
        none.B = B
        dg, dw, gate = torch.full((B, 64), 3.0, device=DEV), torch.full((64,), 3.0, device=DEV), torch.ones(B, 64, device=DEV)
        K.block_norm_backward(none, none, f=none, gate=gate, w=torch.ones(64, device=DEV), d_gate=dg, d_w=dw)
        assert float(dg.abs().max()) == 0.0 and float(dw.abs().max()) == 0.0


@pytest.mark.parametrize("Cc", [64, 320, 1280, 2048])
def test_block_norm_with_no_epsilon(Cc, fmt):
    """eps = 0 and a row count that leaves lanes of the last turn without a row: nothing of theirs reaches the sums."""
    B, N = 1, 5
    g = gen(30)
    a = options(g, B, Cc, K.NORM_LAYER, True, "each", "each", True)
    x, f, dy = (rand(g, B, N, Cc).to(fmt) for _ in range(3))
    p, dx, df = on_gpu(a), empty(B, N, Cc, fmt), empty(B, N, Cc, fmt)
    out = {"d_" + n: torch.empty(p[n].shape, device=DEV) for n in ("post_w", "post_b", "gate", "w", "b", "scale", "shift")}
    K.block_norm_backward(tokens(x), tokens(dy), dx, f=tokens(f), df=df, eps=0.0, **p, **out)
    ref = grads64(x.double(), f.double(), dy.double(), None, in64(a), 0.0)
    for name, got in {"dx": back(dx), "df": back(df), **out}.items():
        # terms of order 10 in 16-bit outputs and sums of five of them
        got, want = got.cpu().double(), ref[name]
        assert float((got.reshape(want.shape) - want).norm() / want.norm()) < (2 * half_step(fmt) if name in ("dx", "df") else 2e-5), name


@pytest.mark.parametrize("Cc", [8, 11, 643, 1027, 1542, 1283, 2051, 4103, 8193])
def test_block_norm_in_place_with_a_ragged_end(Cc, fmt):
    """A row's last channels are read together with those in front of them, which in place other lanes store over (widths around whole
    waves of a row): the same bits as out of place, forward and backward, without a norm in between that would hold the lanes together."""
    B, N = 2, 700
    g = torch.Generator(device=DEV).manual_seed(Cc)

    def mk(dt):
        return View(torch.randn(B * N * Cc, generator=g, device=DEV).to(dt), B, 1, N, Cc)
    gate = torch.randn(B, Cc, generator=g, device=DEV)
    for xt in (fmt, F32):
        x, f, xo, dxo, dx, df = mk(xt), mk(fmt), mk(xt), mk(xt), mk(xt), mk(fmt)
        K.block_norm(x, f=f, xo=xo, gate=gate, alpha=0.5)
        part = (0.5 * gate[:, None] * f.t.float().view(B, N, Cc)).reshape(-1)
        want = x.t.float() + part                     # (f32 too: four roundings here and there of what is added)
        assert bool(((xo.t.float() - want).abs() <= half_step(xt) * want.abs() + tiny(xt) + 4 * EPS32 * (x.t.float().abs() + part.abs())).all())
        keep = x.t.clone()
        K.block_norm(x, f=f, xo=x, gate=gate, alpha=0.5)
        assert torch.equal(x.t, xo.t)
        x.t.copy_(keep)
        K.block_norm_backward(xo, None, dx, dxo=dxo, f=f, df=df, gate=gate, alpha=0.5)
        assert torch.equal(dx.t, dxo.t)
        df2 = mk(fmt)
        K.block_norm_backward(xo, None, dxo, dxo=dxo, f=f, df=df2, gate=gate, alpha=0.5)
        assert torch.equal(dx.t, dxo.t) and torch.equal(df.t, df2.t)
        y, y2, dy = mk(fmt), mk(fmt), mk(fmt)
        K.block_norm(x, y, f=f, xo=xo, post=True)
        K.block_norm(x, y2, f=f, xo=x, post=True)
        assert torch.equal(x.t, xo.t) and torch.equal(y.t, y2.t)
        K.block_norm_backward(x, dy, dx, dxo=dxo, f=f, df=df, post=True)
        K.block_norm_backward(x, dy, dxo, dxo=dxo, f=f, df=dy, post=True)
        assert torch.equal(dx.t, dxo.t) and torch.equal(df.t, dy.t)


def test_block_norm_addresses_past_32_bits():
    """Rows 2^30 channels apart: the third begins 2^31 values into the buffer."""
    pitch, Cc = 1 << 30, 320
    buf = torch.empty((2 << 30) + Cc, dtype=torch.float16, device=DEV)
    x = torch.randn(3, Cc, generator=gen(4)).half()
    for i in range(3):
        buf[i * pitch:i * pitch + Cc] = x[i].to(DEV)
    with K.act_format("f16"):
        y = empty(1, 3, Cc, torch.float16)
        K.block_norm(View(buf, 1, 1, 3, Cc, pitch), y, eps=1e-6)
        small = empty(1, 3, Cc, torch.float16)
        K.block_norm(tokens(x[None]), small, eps=1e-6)
    assert torch.equal(back(y), back(small))


def grads64(x, f, dy, dxo, a, eps):
    """Gradients of sum(y dy) + sum(t dxo) through the definition, the norm taken of the given stream x."""
    leaf = {k: v.clone().requires_grad_() for k, v in a.items() if isinstance(v, torch.Tensor)}
    opt = {**a, **leaf}
    t = x.clone().requires_grad_()
    names = [n for n in ("w", "b", "scale", "shift") if n in leaf] if dy is not None else []
    out, dt = {}, torch.zeros_like(x) if dxo is None else dxo
    if dy is not None:
        _, y = join64(t, None, opt, eps)
        got = torch.autograd.grad((y * dy).sum(), [t] + [leaf[n] for n in names])
        dt = dt + got[0]
        out.update({"d_" + n: v for n, v in zip(names, got[1:])})
    out["dx"] = dt
    if f is not None:
        fl = f.clone().requires_grad_()
        names = [n for n in ("post_w", "post_b", "gate") if n in leaf]
        joined, _ = join64(torch.zeros_like(x), fl, opt, eps)
        got = torch.autograd.grad((joined * dt).sum(), [fl] + [leaf[n] for n in names])
        out["df"] = got[0]
        out.update({"d_" + n: v for n, v in zip(names, got[1:])})
    return out


@pytest.mark.parametrize("types", ["16", "32/16", "32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_block_norm_backward(case, types, fmt):
    B, N, Cc, kind, post, gate, mod, affine, alpha = case
    xt, ft = (F32 if types != "16" else fmt), (F32 if types == "32" else fmt)
    g = gen(Cc + 2 * N)
    kind = K.NORM_LAYER if kind == "layer" else K.NORM_RMS
    a = options(g, B, Cc, kind, post, gate, mod, affine, alpha)
    x, f = rand(g, B, N, Cc, scale=2.0, shift=0.5).to(xt), rand(g, B, N, Cc, shift=0.2).to(ft)
    dy, dxo = rand(g, B, N, Cc).to(ft), rand(g, B, N, Cc, scale=0.5).to(xt)
    if Cc == 1:                                          # one channel: a LayerNorm's gradient is 0, an RMSNorm's cancels to eps
        x, f = x * 0 + 0.5, f * 0 + 0.5
    cs = Cc + (8 if N % 2 else 3)
    dx, df = empty(B, N, Cc, xt, cs, 2), empty(B, N, Cc, ft, cs + 1, 1)
    p = on_gpu(a)
    out = {"d_" + n: torch.full(p[n].shape, 9.0, device=DEV) for n in ("post_w", "post_b", "gate", "w", "b", "scale", "shift") if n in p}
    args = dict(dxo=tokens(dxo), f=tokens(f, cs, 3), eps=1e-6, **p)
    K.block_norm_backward(tokens(x, cs, 1), tokens(dy), dx, df=df, **args, **out)
    ref = grads64(x.double(), f.double(), dy.double(), dxo.double(), in64(a), 1e-6)

    def row_top(v, r, *m):                               # the largest magnitude that a row's terms have
        return v.abs().amax(-1, keepdim=True) * r * torch.stack([torch.as_tensor(q, dtype=torch.float64).abs().max() for q in m] +
                                                               [torch.ones((), dtype=torch.float64)]).prod()
    r = 1 / torch.sqrt(((x.double() - (x.double().mean(-1, keepdim=True) if kind == K.NORM_LAYER else 0)) ** 2).mean(-1, keepdim=True) + 1e-6)
    rf = 1 / torch.sqrt(((f.double() - (f.double().mean(-1, keepdim=True) if kind == K.NORM_LAYER else 0)) ** 2).mean(-1, keepdim=True) + 1e-6)
    hat = norm64(x.double(), kind, 1e-6)
    fh = norm64(f.double(), kind, 1e-6) if post else f.double()
    n = (Cc + 32) * EPS32
    # u = dy (1 + s) w; its two means carry n eps32 of u's largest magnitude, times r and the largest normalised value; a normalised
    # value itself is off by n eps32 (|t| r), which the products with u see too
    gain = (a.get("w", torch.ones(1)).abs().max() * (1 + (a["scale"].abs().max() if "scale" in a else 0))).double()
    lift = 1 + x.double().abs().amax(-1, keepdim=True) * r
    e_dt = 4 * n * dy.double().abs().amax(-1, keepdim=True) * gain * r * lift * (1 + hat.abs().amax(-1, keepdim=True)) + 4 * EPS32 * dxo.double().abs()
    within(back(dx), ref["dx"], half_step(xt) * ref["dx"].abs() + tiny(xt) + e_dt, "dx")
    dt = ref["dx"]
    mult = abs(alpha) * (a["gate"].abs().max().double() if "gate" in a else 1.0)
    pw = a["post_w"].abs().max().double() if post else 1.0
    if post:
        flift = 1 + f.double().abs().amax(-1, keepdim=True) * rf
        e_df = (4 * n * dt.abs().amax(-1, keepdim=True) * flift * (1 + fh.abs().amax(-1, keepdim=True)) + e_dt.amax(-1, keepdim=True) * (
            2 + fh.abs().amax(-1, keepdim=True) ** 2)) * mult * pw * rf
    else:
        e_df = (e_dt + 8 * EPS32 * dt.abs()) * mult
    within(back(df), ref["df"], half_step(ft) * ref["df"].abs() + tiny(ft) + e_df, "df")
    assert untouched(dx) and untouched(df)
    # parameter gradients: sums over the rows of a picture (or of all), every term's own error and the sum's
    e_hat, e_fh = n * (x.double().abs().amax(-1, keepdim=True) * r + hat.abs()), n * (f.double().abs().amax(-1, keepdim=True) * (rf if post else 0) + fh.abs())
    m_s = 1 + (a["scale"].abs().max().double() if "scale" in a else 0.0)
    m_w, m_b = (a[k].abs().max().double() if k in a else torch.tensor(d).double() for k, d in (("w", 1.0), ("b", 0.0)))
    m_pb = a["post_b"].abs().max().double() if "post_b" in a else 0.0
    rows = (N + 8) * EPS32
    S1 = dy.double().abs()
    E2 = S1 * (e_hat + rows * hat.abs())
    T1, T1e = dt.abs(), e_dt.expand_as(dt) + rows * dt.abs()
    T2e = T1 * e_fh + T1e * (fh.abs() + 1e-30)
    err = {"d_shift": rows * S1, "d_scale": m_w * E2 + m_b * rows * S1 + 4 * EPS32 * (m_w * hat.abs() + m_b) * S1, "d_w": m_s * (E2 + 4 * EPS32 * hat.abs() * S1),
           "d_b": m_s * rows * S1, "d_gate": abs(alpha) * (pw * T2e + m_pb * T1e) + 4 * EPS32 * abs(alpha) * (pw * fh.abs() + m_pb) * T1,
           "d_post_w": mult * (T2e + 4 * EPS32 * fh.abs() * T1), "d_post_b": mult * (T1e + 4 * EPS32 * T1)}
    for name, got in out.items():
        e = err[name].sum(1)
        if got.dim() == 1:
            e = e.sum(0)
        within(got, ref[name], e + EPS32 * ref[name].abs() + 1e-37, name)
    # the same bits again, and in place
    dxv, dyv = tokens(dxo, cs, 2), tokens(dy, cs + 1, 1)
    again = {k: torch.empty_like(v) for k, v in out.items()}
    K.block_norm_backward(tokens(x, cs, 1), dyv, dxv, df=dyv, **{**args, "dxo": dxv}, **again)
    assert torch.equal(back(dxv), back(dx)) and torch.equal(back(dyv), back(df)) and untouched(dxv) and untouched(dyv)
    assert all(torch.equal(again[k], out[k]) for k in out)


@pytest.mark.parametrize("with_f", [False, True])
@pytest.mark.parametrize("which", ["dy", "dxo"])
def test_block_norm_backward_parts(which, with_f, fmt):
    """One of the two gradients alone, with and without a branch, some outputs not asked for."""
    B, N, Cc = 2, 21, 320
    g = gen(5)
    a = options(g, B, Cc, K.NORM_LAYER, with_f, "each" if with_f else None, "each" if which == "dy" else None, which == "dy")
    if which == "dxo":
        a.pop("post_b", None)
    if not with_f:
        a = {k: v for k, v in a.items() if k in ("kind", "w", "b", "scale", "shift")}
    x, f, d = (rand(g, B, N, Cc).to(fmt) for _ in range(3))
    ref = grads64(x.double(), f.double() if with_f else None, d.double() if which == "dy" else None, d.double() if which == "dxo" else None,
                  in64(a), 1e-6)
    p, dx = on_gpu(a), empty(B, N, Cc, fmt)
    df = empty(B, N, Cc, fmt) if with_f else None
    out = {"d_" + n: torch.empty(p[n].shape, device=DEV) for n in ("gate", "scale") if n in p}
    K.block_norm_backward(tokens(x), tokens(d) if which == "dy" else None, dx, dxo=tokens(d) if which == "dxo" else None,
                          f=tokens(f) if with_f else None, df=df, eps=1e-6, **p, **out)
    n = (Cc + 32) * EPS32
    within(back(dx), ref["dx"], half_step(fmt) * ref["dx"].abs() + tiny(fmt) + 64 * n, "dx")
    if with_f:
        within(back(df), ref["df"], half_step(fmt) * ref["df"].abs() + tiny(fmt) + 512 * n, "df")
    for name, got in out.items():
        within(got, ref[name], 512 * n * N, name)
    only = {k: torch.empty_like(v) for k, v in out.items()}
    if only:                                             # the parameter gradients without dx and df
        K.block_norm_backward(tokens(x), tokens(d) if which == "dy" else None, None, dxo=tokens(d) if which == "dxo" else None,
                              f=tokens(f) if with_f else None, eps=1e-6, **p, **only)
        assert all(torch.equal(only[k], out[k]) for k in out)


def test_block_norm_backward_against_differences():
    """dx, df and the parameters' gradients as the slope of a loss of block_norm itself, in f32: central differences of step h along a
    random direction agree to h^2 times the third derivative plus the loss's own error over h: 2e-3 relative at h = 1/64 for loss
    values of order 1 made of 3 x 5 x 64 terms."""
    B, N, Cc, h = 3, 5, 64, 2.0 ** -6
    g = gen(6)
    a = options(g, B, Cc, K.NORM_LAYER, True, "each", "each", True, 0.5)
    x, f, cy, cx = (rand(g, B, N, Cc) for _ in range(4))

    def loss(x, f, a):
        xo, y = empty(B, N, Cc, F32), empty(B, N, Cc, F32)
        K.block_norm(tokens(x), y, f=tokens(f), xo=xo, eps=1e-3, **on_gpu(a))
        return float((back(y).double() * cy.double()).sum() + (back(xo).double() * cx.double()).sum()), xo
    _, xo = loss(x, f, a)
    p, dx, df = on_gpu(a), empty(B, N, Cc, F32), empty(B, N, Cc, F32)
    out = {"d_" + n: torch.empty(p[n].shape, device=DEV) for n in ("post_w", "post_b", "gate", "w", "b", "scale", "shift")}
    K.block_norm_backward(xo, tokens(cy), dx, dxo=tokens(cx), f=tokens(f), df=df, eps=1e-3, **p, **out)
    grads = {"x": back(dx), "f": back(df), **{k[2:]: v.cpu() for k, v in out.items()}}
    for name, grad in grads.items():
        base = {"x": x, "f": f, **a}[name]
        d = rand(gen(7), *base.shape)
        d = d / d.norm()

        def moved(s):
            v = base + s * d
            return loss(v if name == "x" else x, v if name == "f" else f, {**a, name: v} if name in a else a)[0]
        slope = (moved(h) - moved(-h)) / (2 * h)
        want = float((grad.double().reshape(d.shape) * d.double()).sum())
        assert abs(slope - want) <= 2e-3 * (1 + abs(want)), (name, slope, want)


def test_block_norm_many_rows_and_sums(fmt):
    """More rows than a run of partial sums holds, several pictures: sums over runs, pictures and a shared gate."""
    B, N, Cc = 3, 1000, 64
    g = gen(8)
    a = options(g, B, Cc, K.NORM_RMS, False, "one", "each", True)
    x, f, dy, dxo = (rand(g, B, N, Cc).to(fmt) for _ in range(4))
    p, dx, df = on_gpu(a), empty(B, N, Cc, fmt), empty(B, N, Cc, fmt)
    out = {"d_" + n: torch.empty(p[n].shape, device=DEV) for n in ("gate", "w", "b", "scale", "shift")}
    K.block_norm_backward(tokens(x), tokens(dy), dx, dxo=tokens(dxo), f=tokens(f), df=df, eps=1e-6, **p, **out)
    ref = grads64(x.double(), f.double(), dy.double(), dxo.double(), in64(a), 1e-6)
    for name, got in out.items():
        # terms of order 10 at most, N (or B N) of them, each off by 256 eps32, and their sum by a random walk over the run
        within(got, ref[name], B * N * 10 * 64 * EPS32, name)
        assert float((got.cpu().double() - ref[name]).norm() / ref[name].norm()) < 2e-6, name


# ---- rotary -----------------------------------------------------------------------------------------------------------------------
def rotary64(x, heads, D, sections, pos, theta, neighbours, shared, inverse):
    """x [B, N, heads D] in 64 bits; pos [N, A] or [B, N, A]."""
    rot = sum(sections)
    out = x.reshape(*x.shape[:2], heads, D).clone()
    src = out.clone()
    pos = pos.double() if pos.dim() == 3 else pos.double()[None]
    i = 0
    for a, n in enumerate(sections):
        for j in range(n // 2):
            fr = theta ** (-2.0 * i / rot) if shared else theta ** (-2.0 * j / n)
            ang = (pos[..., a] * fr).unsqueeze(-1) * (-1 if inverse else 1)
            ia, ib = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
            out[..., ia] = src[..., ia] * ang.cos() - src[..., ib] * ang.sin()
            out[..., ib] = src[..., ib] * ang.cos() + src[..., ia] * ang.sin()
            i += 1
    return out.reshape(x.shape)


def tol_rot(x, ref, heads, D, dtype):
    top = x.double().reshape(*x.shape[:2], heads, D).abs().amax(-1, keepdim=True).expand(*x.shape[:2], heads, D).reshape(x.shape)
    return half_step(dtype) * ref.abs() + tiny(dtype) + 2.0 ** -20 * top


ROT = [
    # B, N, q heads, k heads, D, sections
    (1, 1, 16, 4, 128, (44, 42, 42)),
    (2, 7, 3, 3, 80, (28, 26, 26)),
    (1, 33, 8, 0, 40, (20, 20)),
    (2, 5, 2, 1, 160, (160,)),
    (1, 6, 5, 5, 72, (24, 22, 22)),                       # 4 dims of a head pass through
    (3, 4, 1, 1, 10, (4, 2)),
    (1, 9, 2, 2, 64, (0, 0)),                             # nothing turns
    (1, 3, 1, 1, 7, (2, 2, 2)),
    (1, 130, 4, 2, 96, (32, 32, 32)),
]


@pytest.mark.parametrize("dtype", ["16", "32"])
@pytest.mark.parametrize("neighbours,shared,inverse,real", [(False, False, False, False), (True, True, True, True), (True, False, False, True),
                                                           (False, True, True, False)])
@pytest.mark.parametrize("case", ROT, ids=lambda c: "-".join(str(v) for v in c))
def test_rotary_axes(case, neighbours, shared, inverse, real, dtype, fmt):
    B, N, hq, hk, D, sections = case
    t = F32 if dtype == "32" else fmt
    g = gen(N + D)
    q, k = rand(g, B, N, hq * D).to(t), rand(g, B, N, max(hk, 1) * D).to(t)
    pos = torch.randint(0, 4000, (B, N, len(sections)), generator=g, dtype=torch.int32)
    pos = (pos.float() * 0.37 - 100) if real else pos
    if not neighbours:
        pos = pos[0]                                      # the same for every picture
    plan = RotaryAxes(D, sections, 10000.0, neighbours, shared, DEV)
    wide = (hq + hk) * D + 3
    buf = torch.full((B * N, wide), 7.0, dtype=t)
    buf[:, 1:1 + hq * D] = q.reshape(B * N, -1)
    if hk:
        buf[:, 2 + hq * D:2 + (hq + hk) * D] = k.reshape(B * N, -1)
    v = View(buf.reshape(-1).to(DEV), B, 1, N, wide)
    qv, kv = v.slice(1, hq * D), v.slice(2 + hq * D, hk * D) if hk else None
    qo, ko = empty(B, N, hq * D, t, hq * D + 8, 8), empty(B, N, hk * D, t) if hk else None
    K.rotary_axes(plan, pos.to(DEV), qv, qo, kv, ko, inverse=inverse)
    ref = rotary64(q.double(), hq, D, sections, pos, 10000.0, neighbours, shared, inverse)
    within(back(qo), ref, tol_rot(q, ref, hq, D, t), "q")
    assert untouched(qo) and torch.equal(v.t.cpu(), buf.reshape(-1))
    if hk:
        ref = rotary64(k.double(), hk, D, sections, pos, 10000.0, neighbours, shared, inverse)
        within(back(ko), ref, tol_rot(k, ref, hk, D, t), "k")
    K.rotary_axes(plan, pos.to(DEV), qv, None, kv, None, inverse=inverse)                       # in place: the same bits
    assert torch.equal(back(qv), back(qo)) and (not hk or torch.equal(back(kv), back(ko)))
    rest = v.t.cpu().view(B * N, wide)
    assert bool((rest[:, [0, 1 + hq * D, wide - 1]] == 7.0).all())


def test_rotary_far_positions():
    """Whole positions up to 2^31 - 1 and 32-bit ones of 1e6: the reference angle is reduced exactly (position times frequency in turns
    carries 2^-53 of 2^31 turns = 2^-22 of a turn at most)."""
    D = 64
    plan = RotaryAxes(D, (32, 32), device=DEV)
    pos = torch.tensor([[2 ** 31 - 1, 0], [-(2 ** 31), 5], [10 ** 6, 10 ** 9]], dtype=torch.int32)
    q = torch.ones(1, 3, D)
    with K.act_format("f16"):
        qo = empty(1, 3, D, F32)
        K.rotary_axes(plan, pos.to(DEV), tokens(q), qo)
        ref = rotary64(q.double(), 1, D, (32, 32), pos, 10000.0, False, False, False)
        within(back(qo), ref, 2.0 ** -19 + torch.zeros(1, 3, D, dtype=torch.float64), "far")
        rp = torch.tensor([[1e6 + 0.5, -123456.75], [0.0, float("nan")], [float("inf"), 1.0]])
        K.rotary_axes(plan, rp.to(DEV), tokens(q), qo)
    got = back(qo)[0].view(3, 2, 32)
    ref = rotary64(q.double(), 1, D, (32, 32), rp, 10000.0, False, False, False)[0].view(3, 2, 32)
    within(got[0], ref[0], 2.0 ** -19 + torch.zeros(2, 32, dtype=torch.float64), "real")
    # a position that is no number spoils its own axis' pairs only
    assert got[1][:, :16].isfinite().all() and got[1][:, 16:].isnan().all() and got[2][:, :16].isnan().all() and got[2][:, 16:].isfinite().all()


def test_rotary_is_undone_by_its_inverse_and_addresses_past_32_bits(fmt):
    D, heads, pitch = 40, 2, 1 << 30
    plan = RotaryAxes(D, (20, 20), device=DEV)
    pos = torch.tensor([[3, 5], [7, 1], [100, 200]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 3, heads * D, generator=gen(9)).to(fmt)
    buf = torch.empty((2 << 30) + heads * D, dtype=fmt, device=DEV)
    for i in range(3):
        buf[i * pitch:i * pitch + heads * D] = q[0, i].to(DEV)
    far, near = View(buf, 1, 1, 3, heads * D, pitch), tokens(q)
    K.rotary_axes(plan, pos, far)
    K.rotary_axes(plan, pos, near)
    assert all(torch.equal(buf[i * pitch:i * pitch + heads * D].cpu(), back(near)[0, i]) for i in range(3))
    K.rotary_axes(plan, pos, near, inverse=True)
    # two roundings to the format, a turn keeps a pair's length: each rounding is at most half a step of the pair's length
    top = q.double().view(1, 3, heads, D).abs().amax(-1, keepdim=True).expand(1, 3, heads, D).reshape(q.shape)
    within(back(near), q.double(), 4 * half_step(fmt) * top * 2 ** 0.5, "round trip")


def test_rotary_gradient_is_the_inverse():
    """<turn(q), c> as a function of q has the gradient turn back(c): both sides of the identity, f32."""
    D, sections = 24, (8, 8, 8)
    plan = RotaryAxes(D, sections, neighbours=True, device=DEV)
    g = gen(10)
    pos = torch.randint(0, 50, (11, 3), generator=g, dtype=torch.int32)
    q, c = rand(g, 2, 11, 3 * D), rand(g, 2, 11, 3 * D)
    leaf = q.double().requires_grad_()
    (rotary64(leaf, 3, D, sections, pos, 10000.0, True, False, False) * c.double()).sum().backward()
    with K.act_format("f16"):
        d = empty(2, 11, 3 * D, F32)
        K.rotary_axes(plan, pos.to(DEV), tokens(c), d, inverse=True)
    within(back(d), leaf.grad, tol_rot(c, leaf.grad, 3, D, F32), "gradient")


# ---- mxfp4 ------------------------------------------------------------------------------------------------------------------------
GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def held64(x):
    """(codes, scales, values) of x [rows, K], blocks of 32 padded with zeros to whole 128s, from the definition, in 64 bits."""
    rows, k = x.shape
    v = torch.zeros(rows, -(-k // 128) * 128, dtype=torch.float64)
    v[:, :k] = x.double()
    v = v.view(rows, -1, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.where((top > 0) & ~bad, torch.frexp(torch.where(bad, 1.0, top))[1].double() - 3, -127.0).clamp_min(-127.0)
    unit = torch.where(bad[..., None], 0.0, v / 2.0 ** e[..., None]).nan_to_num()
    # nearest code; of two as near, the even one
    d = (unit.abs()[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    code = torch.where(near & (torch.arange(8) % 2 == 0), torch.arange(8), torch.where(near, torch.arange(8) + 8, 99)).amin(-1) % 8
    code = code | (torch.signbit(unit).long() << 3)
    code = torch.where(bad[..., None], 0, code)
    val = GRID[code & 7] * torch.where(code > 7, -1.0, 1.0) * 2.0 ** e[..., None]
    val = torch.where(bad[..., None], float("nan"), val).view(rows, -1)[:, :k]
    code = code.view(rows, -1)
    return (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8), val


def rows_view(x, cs=None, co=0):
    return tokens(x[None], cs, co)


@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 128), (7, 129), (4, 320), (33, 1000), (130, 257), (1, 8192)])
def test_mxfp4_quantize_and_back(rows, k, fmt):
    g = gen(rows + k)
    spread = 2.0 ** torch.randint(-9, 6, (1, k), generator=g)
    for t in (fmt, F32):
        x = (rand(g, rows, k) * spread).to(t)
        for cs, co in ((None, 0), (k + 8, 8), (k + 3, 1)):
            q = K.mxfp4_quantize(rows_view(x, cs, co))
            codes, scales, val = held64(x)
            assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
        for yt in (fmt, F32):
            for cs, co in ((None, 0), (k + 8, 8), (k + 3, 2)):
                y = empty(1, rows, k, yt, cs, co)
                K.mxfp4_dequantize(q, y)
                assert torch.equal(back(y)[0], val.to(yt)) and untouched(y)


def test_mxfp4_borders():
    """Halves between codes, saturation, the lowest scales, blocks that are zero or not numbers."""
    halves = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.5, 7.0, 7.5, 7.99, .2499, .2501, 0, .5, 1, 1.5, 2, 3, 4, 6])
    blocks = [torch.cat([halves, -halves])[:32], torch.cat([-halves, halves])[:32] * 2.0 ** 40, torch.cat([halves, torch.zeros(11)]) * 2.0 ** -100,
              torch.zeros(32), -torch.zeros(32), torch.full((32,), 2.0 ** -126), torch.full((32,), 2.0 ** -149), torch.full((32,), 1.5 * 2.0 ** -127),
              torch.full((32,), torch.finfo(F32).max), torch.cat([torch.full((31,), 1.0), torch.tensor([float("nan")])]),
              torch.cat([torch.tensor([float("inf")]), torch.full((31,), 1.0)]), torch.cat([torch.tensor([-float("inf")]), torch.zeros(31)]),
              torch.cat([torch.full((31,), 1e-30), torch.tensor([1e30])])]
    x = torch.stack(blocks).reshape(1, -1).repeat(3, 1)
    x = torch.cat([x, x[:, 32:64]], 1)
    with K.act_format("f16"):
        q = K.mxfp4_quantize(rows_view(x))
        codes, scales, val = held64(x)
        assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
        y = empty(1, 3, x.shape[1], F32)
        K.mxfp4_dequantize(q, y)
        got = back(y)[0]
        assert torch.equal(got.isnan(), val.isnan()) and torch.equal(got.nan_to_num(7.0), val.float().nan_to_num(7.0))


def linear64(xv, wv, bias, epi, alpha, slope, res):
    y = alpha * (xv @ wv.T) + (0 if bias is None else bias.double())
    size = abs(alpha) * (xv.abs() @ wv.abs().T) + (0 if bias is None else bias.double().abs())
    k = xv.shape[1]
    err = (k + 8) * EPS32 * size
    if epi == K.EPI_SILU:
        y, err = y * torch.sigmoid(y), err * 1.2 + 2.0 ** -20 * y.abs()
    elif epi == K.EPI_LEAKY:
        y = torch.where(y >= 0, y, y * slope)
    elif epi == K.EPI_GEGLU:
        y, err = y.unflatten(1, (-1, 2, 16)), err.unflatten(1, (-1, 2, 16))
        a, b, ea, eb = y[:, :, 0].flatten(1), y[:, :, 1].flatten(1), err[:, :, 0].flatten(1), err[:, :, 1].flatten(1)
        # gelu: |error| <= 0.5 |b| 1.5e-7 from its erf, a slope of at most 1.13
        y, err = a * torch.nn.functional.gelu(b), ea * b.abs() + a.abs() * (1.2 * eb + 2.0 ** -21 * b.abs())
    if res is not None:
        y = y + res.double()
        err = err + EPS32 * y.abs()
    return y, err + 4 * EPS32 * y.abs()


LIN = [
    # M, N, K, epi, bias, res
    (1, 1, 1, "linear", True, False),
    (1, 320, 1280, "linear", True, True),
    (2, 33, 31, "silu", True, False),
    (3, 8, 130, "leaky", False, True),
    (15, 640, 320, "geglu", True, False),
    (16, 100, 256, "linear", False, False),
    (17, 100, 256, "linear", True, True),
    (1, 2048, 8192, "linear", True, False),
    (16, 288, 4000, "geglu", True, True),
    (64, 64, 128, "silu", True, True),
    (100, 257, 1000, "linear", True, True),
    (129, 320, 96, "geglu", False, False),
    (257, 640, 640, "geglu", True, True),
    (300, 520, 1312, "linear", True, True),
    (513, 264, 2080, "leaky", True, False),
    (1031, 1280, 384, "linear", True, False),
    (2500, 96, 5120, "silu", False, True),
    (50, 3, 100, "linear", True, False),
    (33, 65, 4097, "silu", True, False),
    (70, 160, 8191, "geglu", True, True),
    (40, 1, 300, "linear", False, True),
]
EPI = {"linear": K.EPI_LINEAR, "leaky": K.EPI_LEAKY, "silu": K.EPI_SILU, "geglu": K.EPI_GEGLU}


@pytest.mark.parametrize("M,N,k,epi,bias,res", LIN)
def test_mxfp4_linear(M, N, k, epi, bias, res, fmt):
    g = gen(M + N + k)
    x = (rand(g, M, k) * 2.0 ** torch.randint(-3, 4, (1, k), generator=g)).to(fmt)
    w = rand(g, N, k, scale=k ** -0.5) * 2.0 ** torch.randint(-2, 3, (N, 1), generator=g)
    b = rand(g, N) if bias else None
    wq = pack.pack_mxfp4(w, DEV)
    xv, wv = held64(x)[2], held64(w)[2]
    assert torch.equal(wq.codes.cpu(), held64(w)[0])
    out = N // 2 if epi == "geglu" else N
    for yt, cs, co in ((fmt, out, 0), (F32, out + 3, 1), (fmt, out + 8, 8)):
        r = rand(g, M, out).to(yt) if res else None
        ref, err = linear64(xv, wv, b, EPI[epi], 0.5, 0.1, r)
        y = empty(1, M, out, yt, cs, co)
        args = dict(epi=EPI[epi], alpha=0.5, slope=0.1, res=rows_view(r, out + 5, 5) if res else None)
        K.mxfp4_linear(rows_view(x, k + 8, 8), wq, b.to(DEV) if bias else None, y, **args)
        within(back(y)[0], ref, half_step(yt) * ref.abs() + tiny(yt) + err, f"raw rows, {yt}")
        assert untouched(y)
        # the same operand held in 4 bits already: the same bits; unaligned rows too
        again = empty(1, M, out, yt, cs, co)
        K.mxfp4_linear(K.mxfp4_quantize(rows_view(x, k + 3, 1)), wq, b.to(DEV) if bias else None, again, **args)
        assert torch.equal(back(again), back(y))
        K.mxfp4_linear(rows_view(x, k + 3, 3), wq, b.to(DEV) if bias else None, again, **args)
        assert torch.equal(back(again), back(y))
    if res:                                               # the residual in place
        yr = rows_view(r, cs, co)
        K.mxfp4_linear(rows_view(x), wq, b.to(DEV) if bias else None, yr, epi=EPI[epi], alpha=0.5, slope=0.1, res=yr)
        assert torch.equal(back(yr), back(y)) and untouched(yr)


@pytest.mark.parametrize("M,N,k,epi,res", [
    (2100, 2100, 520, "linear", True),         # 128 x 128, two stages; an odd number of steps
    (4200, 2624, 260, "geglu", False),         # 128 x 128, one stage
    (6001, 5664, 300, "geglu", True),          # 128 x 256
    (2600, 4200, 200, "silu", True),           # 256 x 256; two steps, ragged both ways
    (2600, 4224, 4500, "geglu", True),         # 256 x 256, gated; 36 steps
    (2601, 4195, 1150, "leaky", False),        # 256 x 256, nothing aligned; nine steps: a group of scales with one step
])
def test_mxfp4_linear_large_tiles(M, N, k, epi, res, fmt):
    """The tiles of large layers, against the product of the values that the operands stand for (read back: their own tests) in 64 bits on the
    GPU, a row and a column that are no numbers among them."""
    g = torch.Generator(device=DEV).manual_seed(M + k)

    def rnd(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * scale
    x, w, b = rnd(M, k).to(fmt), rnd(N, k, scale=k ** -0.5), rnd(N)
    x[M - 1, k - 1], w[N - 33, 0] = float("nan"), float("inf")
    out = N // 2 if epi == "geglu" else N
    r = rnd(M, out).to(fmt) if res else None
    xq, wq = K.mxfp4_quantize(View(x, 1, 1, M, k)), pack.pack_mxfp4(w, DEV)
    xv, wv = torch.empty(M, k, device=DEV), torch.empty(N, k, device=DEV)
    K.mxfp4_dequantize(xq, View(xv, 1, 1, M, k))
    K.mxfp4_dequantize(wq, View(wv, 1, 1, N, k))
    ref, err = linear64(xv.double(), wv.double(), b, EPI[epi], 1.0, 0.1, r)
    y = torch.full((M + 1, out), 7.0, dtype=fmt, device=DEV)
    K.mxfp4_linear(xq, wq, b, View(y, 1, 1, M, out), epi=EPI[epi], slope=0.1, res=None if r is None else View(r, 1, 1, M, out))
    assert bool((y[M] == 7.0).all())
    got = y[:M].double()
    assert torch.equal(got.isnan(), ref.isnan()) and bool(ref[M - 1].isnan().all()) and not bool(ref[:M - 1, :(N - 40) // 2].isnan().any())
    bad = ~(((got - ref).abs() <= half_step(fmt) * ref.abs() + tiny(fmt) + err) | ref.isnan())
    assert not bool(bad.any()), (int(bad.sum()), float((got - ref).abs()[bad].max()))


def test_mxfp4_linear_from_f32_rows(fmt):
    g = gen(11)
    for M in (4, 40):
        x, w = rand(g, M, 200), rand(g, 48, 200, scale=0.1)
        ref, err = linear64(held64(x)[2], held64(w)[2], None, K.EPI_LINEAR, 1.0, 0.0, None)
        y = empty(1, M, 48, F32)
        K.mxfp4_linear(rows_view(x, 203, 2), pack.pack_mxfp4(w, DEV), None, y)
        within(back(y)[0], ref, EPS32 * ref.abs() + err, "f32 rows")


@pytest.mark.parametrize("M", [5, 300])
def test_mxfp4_linear_keeps_what_is_no_number_in_its_row_and_column(M, fmt):
    g = gen(12)
    k, N = 384, 320
    x, w = rand(g, M, k).to(fmt), rand(g, N, k, scale=0.05)
    x[2, 130], w[7, 383] = float("nan"), float("inf")
    y = empty(1, M, N, F32)
    K.mxfp4_linear(rows_view(x), pack.pack_mxfp4(w, DEV), None, y)
    got = back(y)[0]
    want = torch.zeros(M, N, dtype=torch.bool)
    want[2], want[:, 7] = True, True
    assert torch.equal(got.isnan(), want) and got[~want].isfinite().all()


def test_mxfp4_linear_row_is_the_same_alone_and_among_others(fmt):
    """A token's bits do not depend on how many rows it shares the launch with, wherever one kernel runs both."""
    g = gen(13)
    x, w = rand(g, 700, 640).to(fmt), pack.pack_mxfp4(rand(g, 320, 640, scale=0.05), DEV)
    whole, some = empty(1, 700, 320, F32), empty(1, 300, 320, F32)
    K.mxfp4_linear(rows_view(x), w, None, whole)
    K.mxfp4_linear(rows_view(x[200:500]), w, None, some)
    assert torch.equal(back(whole)[0, 200:500], back(some)[0])
    many, one = empty(1, 16, 320, F32), empty(1, 1, 320, F32)
    K.mxfp4_linear(rows_view(x[:16]), w, None, many)
    K.mxfp4_linear(rows_view(x[9:10]), w, None, one)
    assert torch.equal(back(many)[0, 9:10], back(one)[0])


def test_mxfp4_no_rows(fmt):
    q = K.mxfp4_quantize(View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 1, 64))
    assert q.rows == 0
    w = pack.pack_mxfp4(torch.ones(32, 64), DEV)
    y = View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 1, 32)
    K.mxfp4_linear(q, w, None, y)
    K.mxfp4_dequantize(q, View(torch.empty(0, dtype=fmt, device=DEV), 0, 1, 1, 64))


def test_mxfp4_addresses_past_32_bits():
    """Output and residual rows 2^30 values apart."""
    pitch, N, k = 1 << 30, 64, 128
    g = gen(14)
    x, w = rand(g, 3, k).half(), pack.pack_mxfp4(rand(g, N, k, scale=0.1), DEV)
    buf = torch.empty((2 << 30) + N, dtype=torch.float16, device=DEV)
    with K.act_format("f16"):
        y, far = empty(1, 3, N, torch.float16), View(buf, 1, 1, 3, N, pitch)
        K.mxfp4_linear(rows_view(x), w, None, y)
        K.mxfp4_linear(rows_view(x), w, None, far)
        assert all(torch.equal(buf[i * pitch:i * pitch + N].cpu(), back(y)[0, i]) for i in range(3))
        for i in range(3):
            buf[i * pitch:i * pitch + k // 2] = x[i, :k // 2].to(DEV)
        qa, qb = K.mxfp4_quantize(View(buf, 1, 1, 3, k // 2, pitch)), K.mxfp4_quantize(rows_view(x[:, :k // 2].contiguous()))
        assert torch.equal(qa.codes, qb.codes) and torch.equal(qa.scales, qb.scales)


# ---- streams, graphs, a run of them together ------------------------------------------------------------------------------------------
def block_weights(Cc, seed, device=DEV):
    g = gen(seed)

    def mat(n, k):
        return rand(g, n, k, scale=k ** -0.5)
    perm = pack.glu_perm(2 * Cc)
    return {"qk": mat(2 * Cc, Cc), "v": mat(Cc, Cc), "o": mat(Cc, Cc), "up": mat(4 * Cc, Cc)[perm], "down": mat(Cc, 2 * Cc),
            "mod": rand(g, 2, 6 * Cc, scale=0.3), "pw1": rand(g, Cc, scale=0.1, shift=1.0), "pw2": rand(g, Cc, scale=0.1, shift=1.0)}


def run_block(x, wts, plan, pos, B, H, W, heads, D):
    """One transformer block over image tokens: modulated norm, 4-bit projections, rotary, flash attention, gated joins with a norm of the
    branch, a gated feed-forward part; x, out: Views."""
    Cc, N = heads * D, H * W
    fmt = x.t.dtype
    mod = wts["mod"]
    s1, h1, g1, s2, h2, g2 = (mod[:, i * Cc:(i + 1) * Cc] for i in range(6))
    y = new_view(B, H, W, Cc, DEV)
    K.block_norm(x, y, scale=s1, shift=h1)
    yq = K.mxfp4_quantize(y)
    qk = new_view(B, H, W, 2 * Cc, DEV)
    K.mxfp4_linear(yq, wts["qk"], None, qk)
    K.rotary_axes(plan, pos, qk.slice(0, Cc), k=qk.slice(Cc, Cc))
    vt = torch.empty(B, Cc, N, dtype=K.flash_vt_dtype(D, D, N), device=DEV)
    for b in range(B):                                    # V^T of a picture: the weights' rows times its tokens
        t = torch.empty(Cc, N, dtype=fmt, device=DEV)
        K.mxfp4_linear(wts["v"], MxFp4(yq.codes[b * N:(b + 1) * N], yq.scales[b * N:(b + 1) * N], N, Cc), None, View(t, 1, 1, Cc, N))
        vt[b] = t
    o = new_view(B, H, W, Cc, DEV)
    K.flash_attn(qk.t, qk.t[Cc:], vt, o.t, B, heads, N, N, N, D, D, D ** -0.5, q_rs=2 * Cc, k_rs=2 * Cc)
    f, xo = new_view(B, H, W, Cc, DEV), new_view(B, H, W, Cc, DEV)
    K.mxfp4_linear(o, wts["o"], None, f)
    K.block_norm(x, y, f=f, xo=xo, post=True, post_w=wts["pw1"], gate=g1, scale=s2, shift=h2)
    u = new_view(B, H, W, 2 * Cc, DEV)
    K.mxfp4_linear(y, wts["up"], None, u, epi=K.EPI_GEGLU)
    K.mxfp4_linear(u, wts["down"], None, f)
    out = new_view(B, H, W, Cc, DEV)
    K.block_norm(xo, f=f, xo=out, post=True, post_w=wts["pw2"], gate=g2, alpha=0.5)
    return out


def block64(x, wts, sections, pos, heads, D, fmt):
    """The same block from the operators' definitions in 64 bits, rounded where the run stores."""
    B, N, Cc = x.shape

    def store(v):
        return v.to(fmt).double()

    def held(v):
        return held64(v.reshape(-1, v.shape[-1]))[2].reshape(v.shape)
    s1, h1, g1, s2, h2, g2 = (wts["mod"].double()[:, i * Cc:(i + 1) * Cc] for i in range(6))
    w = {k: held64(wts[k])[2] for k in ("qk", "v", "o", "up", "down")}
    y = held(store(join64(x, None, dict(kind=K.NORM_LAYER, scale=s1, shift=h1), 1e-5)[1]))
    qk = store(y @ w["qk"].T)
    q, k = (store(rotary64(t, heads, D, sections, pos, 10000.0, False, False, False)).view(B, N, heads, D).transpose(1, 2)
            for t in qk.split(Cc, -1))
    v = store(y @ w["v"].T).view(B, N, heads, D).transpose(1, 2)
    o = store((torch.softmax(q @ k.transpose(-1, -2) * D ** -0.5, -1) @ v).transpose(1, 2).reshape(B, N, Cc))
    f = store(held(o) @ w["o"].T)
    a = dict(kind=K.NORM_LAYER, post=True, post_w=wts["pw1"].double(), gate=g1, scale=s2, shift=h2)
    t, y = join64(x, f, a, 1e-5)
    t, y = store(t), store(y)
    u = (held(y) @ w["up"].T).unflatten(-1, (-1, 2, 16))
    u = store(u[..., 0, :].flatten(-2) * torch.nn.functional.gelu(u[..., 1, :].flatten(-2)))
    f = store(held(u) @ w["down"].T)
    return join64(t, f, dict(kind=K.NORM_LAYER, post=True, post_w=wts["pw2"].double(), gate=g2, alpha=0.5), 1e-5)[0]


def block_setup(fmt, seed=15):
    B, H, W, heads, D = 2, 8, 16, 8, 40
    Cc, sections = heads * D, (20, 20)
    wts = block_weights(Cc, seed)
    dev = {k: (pack.pack_mxfp4(v, DEV) if k in ("qk", "v", "o", "up", "down") else v.to(DEV)) for k, v in wts.items()}
    pos = torch.stack(torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij"), -1).reshape(-1, 2).to(torch.int32)
    x = rand(gen(seed + 1), B, H * W, Cc).to(fmt)
    return B, H, W, heads, D, sections, wts, dev, pos, x, RotaryAxes(D, sections, device=DEV)


def test_a_transformer_block_of_them(fmt):
    """The whole run against the definitions.  A value that lies within the run's own rounding of a border between two codes may fall on
    the other side of it, a quarter of its magnitude away; that happens to a share of about 8 u of the values (the rounding's width over
    the distance of two borders), so that a product's relative error is of order 0.25 sqrt(8 u), three times in a row.  u is bf16's in
    either format: flash attention at this head size multiplies bf16 P and V^T (onedc_flash_attn_vt_is_bf16), so that what the output
    projection quantises is bf16-rounded in the f16 library too (with f16's own u, 0.04, the bound left that out; measured 0.043).
    0.25 sqrt(8 / 256) = 0.044 a product; under 0.1 of the branches' sum."""
    B, H, W, heads, D, sections, wts, dev, pos, x, plan = block_setup(fmt)
    out = run_block(tokens(x), dev, plan, pos.to(DEV), B, H, W, heads, D)
    ref = block64(x.double(), wts, sections, pos, heads, D, fmt)
    got = out.t[:ref.numel()].view(ref.shape).cpu().double()
    rel = float((got - ref).norm() / (ref - x.double()).norm())
    assert rel < 0.1, rel


def test_a_captured_block_replays(fmt):
    """Two graphs of the block, captured on one stream, replayed in turn with eager work and new inputs between: every replay is the eager
    result, bit for bit (the workspaces inside a graph are its own)."""
    B, H, W, heads, D, sections, wts, dev, pos, x, plan = block_setup(fmt)
    pos = pos.to(DEV)
    xs, eager = [tokens(x), tokens(rand(gen(20), *x.shape).to(fmt))], []
    for v in xs:
        eager.append(run_block(v, dev, plan, pos, B, H, W, heads, D).t.clone())
    torch.cuda.synchronize()
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for v in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=stream):
            outs.append(run_block(v, dev, plan, pos, B, H, W, heads, D))
        graphs.append(gr)
    n = x.numel()
    for turn in range(3):
        for i in (0, 1):
            outs[i].t.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i].t[:n], eager[i][:n]), (turn, i)
            run_block(xs[1 - i], dev, plan, pos, B, H, W, heads, D)                     # eager work between the replays
    xs[0].t.copy_(xs[1].t)                                                            # the graph reads what its input holds now
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0].t[:n], eager[1][:n])


def test_captured_backward_replays(fmt):
    """The backward pass in a graph while eager passes over the same tensors go on."""
    B, N, Cc = 2, 300, 320
    g = gen(21)
    a = on_gpu(options(g, B, Cc, K.NORM_LAYER, True, "each", "each", True))
    x, f, dy, dxo = (tokens(rand(g, B, N, Cc).to(fmt)) for _ in range(4))

    def go():
        out = {"d_" + n: torch.empty(a[n].shape, device=DEV) for n in ("post_w", "post_b", "gate", "w", "b", "scale", "shift")}
        dx, df = empty_like(x), empty_like(f)
        K.block_norm_backward(x, dy, dx, dxo=dxo, f=f, df=df, **a, **out)
        return [dx.t, df.t, *out.values()]
    want = [t.clone() for t in go()]
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = go()
    for _ in range(3):
        for t in got:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert all(torch.equal(p, q) for p, q in zip(go(), want))


def empty_like(v):
    return View(torch.empty_like(v.t), v.B, v.H, v.W, v.C)


def test_on_another_stream(fmt):
    """Launches go to the current stream: a chain on a side stream behind a long piece of work there sees that work's result."""
    B, H, W, heads, D, sections, wts, dev, pos, x, plan = block_setup(fmt)
    pos = pos.to(DEV)
    want = run_block(tokens(x), dev, plan, pos, B, H, W, heads, D).t.clone()
    src, xv = tokens(x), tokens(torch.zeros_like(x))
    busy = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-3
        xv.t.copy_(src.t)
        out = run_block(xv, dev, plan, pos, B, H, W, heads, D)
    side.synchronize()
    assert torch.equal(out.t[:x.numel()], want[:x.numel()])


def test_cpu_tensors_among_gpu_tensors_are_refused(fmt):
    x, y = tokens(torch.zeros(1, 4, 64, dtype=fmt)), empty(1, 4, 64, fmt)
    with pytest.raises(KernelError, match="is on cpu"):
        K.block_norm(x, y, w=torch.ones(64))
    with pytest.raises(KernelError, match="is on cpu"):
        K.rotary_axes(RotaryAxes(64, (32, 32), device="cpu"), torch.zeros(4, 2, dtype=torch.int32, device=DEV), x)
    with pytest.raises(KernelError, match="is on cpu"):
        K.mxfp4_linear(x, K.mxfp4_empty(64, 64, "cpu"), None, y)
