"""Transformer-block operators on the GPU, at the sizes and values where a bound per element says little: norms of the error of every output
of block_norm and its backward pass, rotary_axes as large calls run it, infinities and subnormals.

half_step(t) = finfo(t).eps / 2 relative to a value is one rounding to t; EPS32 = 2^-24 is half a step of f32.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from onedc_amd import kernels as K
from onedc_amd.kernels import KernelError, RotaryAxes, View
from test_gpu_token_ops import (CASES, DEV, EPS32, F32, FORMATS, back, block_setup, empty, gen, grads64, half_step, held64, in64, join64, linear64,
                                norm64, on_gpu, options, rand, rotary64, rows_view, run_block, tiny, tokens, tol_rot, tol_y, within)


@pytest.fixture(params=["f16", "bf16"])
def fmt(request):
    with K.act_format(request.param):
        yield FORMATS[request.param]


# ---- block_norm: the error of a whole output -----------------------------------------------------------------------------------------
# A sum over a row is at most 24 additions in a lane (three pieces of eight, or 20001 / 1024 channels a thread), 6 exchanges and 16 waves: relative to
# the sum of magnitudes 46 EPS32.  So a mean is off by 46 EPS32 mean|v|, a normalised value by 75 EPS32 (1 + top r) times its row's size (top: the
# row's largest magnitude, r: its reciprocal deviation), and the gradient through a norm, r (u - mean u - h mean(u h)), by that twice, two such means
# and its own roundings: SUM = 300 EPS32 (1 + top r) r |u| in the row's norm.  A parameter's gradient adds its terms' errors and those of a run of
# rows, of which there are at least 256 where there are rows enough (N / 256 + 64 additions).
SUM = 300 * EPS32


def rows_norm(v):
    return v.norm(dim=-1, keepdim=True)


@pytest.mark.parametrize("types", ["16", "32/16", "32"])
@pytest.mark.parametrize("case", [c for c in CASES if c[2] > 1], ids=lambda c: "-".join(str(v) for v in c))
def test_block_norm_norms_of_the_error(case, types, fmt):
    B, N, Cc, kind, post, gate, mod, affine, alpha = case
    xt, ft = (F32 if types != "16" else fmt), (F32 if types == "32" else fmt)
    g = gen(3 * Cc + N)
    kind, eps = K.NORM_LAYER if kind == "layer" else K.NORM_RMS, 1e-3
    a = options(g, B, Cc, kind, post, gate, mod, affine, alpha)
    x, f = rand(g, B, N, Cc, scale=2.0, shift=0.5).to(xt), rand(g, B, N, Cc, shift=0.2).to(ft)
    dy, dxo = rand(g, B, N, Cc).to(ft), rand(g, B, N, Cc, scale=0.5).to(xt)
    p, wide, xo, y = on_gpu(a), in64(a), empty(B, N, Cc, xt), empty(B, N, Cc, ft)
    K.block_norm(tokens(x), y, f=tokens(f), xo=xo, eps=eps, **p)
    dx, df = empty(B, N, Cc, xt), empty(B, N, Cc, ft)
    grads = {"d_" + n: torch.full(p[n].shape, 9.0, device=DEV) for n in ("post_w", "post_b", "gate", "w", "b", "scale", "shift") if n in p}
    K.block_norm_backward(tokens(x), tokens(dy), dx, dxo=tokens(dxo), f=tokens(f), df=df, eps=eps, **p, **grads)

    x, f, dy, dxo = (v.double() for v in (x, f, dy, dxo))
    ref = grads64(x, f, dy, dxo, wide, eps)
    ref["xo"], ref["y"] = join64(x, f, wide, eps)

    def spread(v):                                       # (reciprocal deviation, 1 + largest magnitude times it) of every row
        c = v - v.mean(-1, keepdim=True) if kind == K.NORM_LAYER else v
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        return r, 1 + v.abs().amax(-1, keepdim=True) * r

    def each(v):                                         # a parameter per picture against [B, N, C]
        return v[:, None] if v.dim() == 2 else v

    def of(name, none):
        return each(wide[name]) if name in wide else torch.tensor(none, dtype=torch.float64)
    (rx, lx), (rf, lf), (_, lt) = spread(x), spread(f), spread(ref["xo"])
    pw, ga, w, sc, b = of("post_w", 1.0), alpha * of("gate", 1.0), of("w", 1.0), 1 + of("scale", 0.0), of("b", 0.0)
    branch = f * 1.0 if not post else norm64(f, kind, eps)
    # rows: the norm of what a row may be off by, in front of the rounding to the output's type
    e_xo = SUM * (rows_norm(ga * pw * branch) * (lf if post else 1) + rows_norm(x) + rows_norm(ref["xo"]))
    hat_t = norm64(ref["xo"], kind, eps)
    e_y = (SUM * lt * rows_norm(hat_t) + 2 * spread(ref["xo"])[0] * e_xo) * (w * sc).abs().amax() + SUM * rows_norm(ref["y"])
    u = dy * sc * w
    e_dx = SUM * lx * rx * rows_norm(u) + 4 * EPS32 * rows_norm(dxo)
    v = ref["dx"] * ga * pw
    top = (ga * pw).abs().amax()
    e_df = (SUM * lf * rf * rows_norm(v) + 3 * rf * top * e_dx) if post else top * e_dx + 4 * EPS32 * rows_norm(v)
    off = {"xo": e_xo, "y": e_y, "dx": e_dx, "df": e_df}
    got = {"xo": back(xo), "y": back(y), "dx": back(dx), "df": back(df), **{k: t.cpu() for k, t in grads.items()}}
    for name, t in (("xo", xt), ("y", ft), ("dx", xt), ("df", ft)):
        full, size = ref[name], float(ref[name].norm())
        allowed = half_step(t) * size + float(off[name].norm()) + tiny(t) * full.numel() ** 0.5
        assert allowed < 0.05 * size, (name, allowed / size)               # (the bound says something: no gradient at all would be off by 1)
        assert float((got[name].double() - full).norm()) <= allowed, (name, float((got[name].double() - full).norm()) / size, allowed / size)
    # sums over rows: magnitudes of the terms, with their errors spread evenly over a row's channels
    hat, run = norm64(x, kind, eps), (N / 256 + 64) * EPS32
    n1, n2 = dy.abs() * run, dy.abs() * (SUM * lx * (hat.abs() + 1) + run * hat.abs())
    flat = e_dx / Cc ** 0.5
    m1, m2 = ref["dx"].abs() * run + flat, ref["dx"].abs() * (run * branch.abs() + (SUM * lf * (branch.abs() + 1) if post else 0)) + flat * branch.abs()
    pb = of("post_b", 0.0)
    terms = {"d_shift": n1, "d_scale": w.abs() * n2 + b.abs() * n1, "d_w": sc.abs() * n2, "d_b": sc.abs() * n1,
             "d_gate": abs(alpha) * (pw.abs() * m2 + pb.abs() * m1), "d_post_w": ga.abs() * m2, "d_post_b": ga.abs() * m1}
    for name in grads:
        e, full = terms[name].expand(B, N, Cc).sum(1), ref[name]
        allowed, size = float((e if got[name].dim() == 2 else e.sum(0)).norm()) + EPS32 * float(full.norm()), float(full.norm())
        assert allowed < 0.15 * size, (name, allowed / size)
        assert float((got[name].double() - full).norm()) <= allowed, (name, float((got[name].double() - full).norm()) / size, allowed / size)


WIDTHS = [5, 64, 100, 320, 643, 1280, 1283, 2048, 4096, 8200, 20001]          # every shape that a row has in registers, with and without a ragged end


@pytest.mark.parametrize("types", ["16", "32"])
@pytest.mark.parametrize("Cc", WIDTHS)
def test_block_norm_of_an_infinite_value(Cc, types, fmt):
    """RMSNorm of a row with an infinity: v / sqrt(inf) is 0 for every finite value and no number at the infinity itself.  The same where the
    squares leave f32's range, in which they are summed.  LayerNorm: nothing is a number (inf - inf)."""
    t = F32 if types == "32" else fmt
    x = rand(gen(Cc), 1, 4, Cc).to(t)
    x[0, 1, Cc // 2], x[0, 2, Cc - 1] = float("inf"), -float("inf")
    if t != torch.float16:
        x[0, 3] = 2.0 ** 70
    w, b = rand(gen(1), Cc, shift=1.0), rand(gen(2), Cc)
    y, xo = empty(1, 4, Cc, t), empty(1, 4, Cc, t)
    K.block_norm(tokens(x), y, kind=K.NORM_RMS, eps=1e-6, w=w.to(DEV), b=b.to(DEV))
    got, want = back(y)[0], b.to(t)
    lost = torch.isinf(x[0])
    assert torch.equal(got.isnan(), lost)
    assert all(torch.equal(got[i][~lost[i]], want[~lost[i]]) for i in ((1, 2) if t == torch.float16 else (1, 2, 3)))
    K.block_norm(tokens(x), y, kind=K.NORM_LAYER, eps=1e-6, w=w.to(DEV), b=b.to(DEV))
    assert back(y)[0][1:3].isnan().all()
    # the infinity comes from a gate: of the last channel, whose combined vector is read on behind the row
    gate, f = torch.ones(Cc), rand(gen(3), 1, 4, Cc).to(t)
    gate[Cc - 1] = float("inf")
    x = rand(gen(4), 1, 4, Cc).to(t)
    K.block_norm(tokens(x), y, f=tokens(f), xo=xo, kind=K.NORM_RMS, eps=1e-6, gate=gate.to(DEV), w=w.to(DEV), b=b.to(DEV))
    got, last = back(y)[0], torch.arange(Cc) == Cc - 1
    assert got[:, last].isnan().all() and torch.equal(got[:, ~last], want[~last].expand(4, -1))
    assert torch.equal(back(xo)[0][:, last].double(), f[0][:, last].double().sign() * float("inf"))


# ---- rotary: as large calls run it ------------------------------------------------------------------------------------------------
def turned64(x, heads, plan, pos, theta, inverse):
    """[B, N, heads D] on the GPU in 64 bits, from the definition: a pair is a complex number, turned."""
    sections, rot = plan.sections, sum(plan.sections)
    freq = [theta ** (-2.0 * j / n) for n in sections for j in range(n // 2)]
    if plan.shared_spectrum:
        freq = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    freq = torch.tensor(freq, dtype=torch.float64, device=x.device)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n // 2)], device=x.device)
    angle = pos.double()[..., axis] * freq * (-1.0 if inverse else 1.0)
    turn = torch.polar(torch.ones_like(angle), angle)
    turn = turn[:, :, None] if turn.dim() == 3 else turn[None, :, None]
    v = x.double().reshape(*x.shape[:2], heads, plan.D).clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if plan.neighbours else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(v[..., a], v[..., b]) * turn
    v[..., a], v[..., b] = z.real, z.imag
    return v.reshape(x.shape)


def close_turns(got, x, ref, heads, D, t):
    """One rounding to t, and of the pair's largest magnitude 2^-20 (sine and cosine to 2^-21, two products and a sum)."""
    top = x.double().view(-1, heads, D).abs().amax(-1, keepdim=True).expand(-1, heads, D).reshape(x.shape)
    off = (got.double() - ref).abs() - half_step(t) * ref.abs() - tiny(t) - 2.0 ** -20 * top
    assert float(off.max()) <= 0, float(off.max())


LARGE = [
    # B, N, q heads, k heads, D, sections: rows enough for several tokens a workgroup; N no multiple of any number of them
    (3, 2741, 2, 2, 64, (24, 20, 20)),                     # 16-byte pieces of 16-bit halves
    (2, 4099, 4, 1, 80, (28, 26, 26)),
    (3, 1501, 3, 3, 72, (24, 24, 24)),                     # halves: 8-byte pieces, neighbours: 16
    (2, 2999, 2, 2, 72, (24, 22, 22)),                     # four dims pass through; neighbours: 8-byte pieces, halves single values
    (1, 5003, 2, 1, 128, (32, 32, 32)),                    # 32 dims pass through
    (2, 2503, 2, 0, 40, (20, 20)),
    (5, 1013, 1, 1, 160, (64, 48, 48)),
    (2, 3001, 2, 2, 96, (16, 16, 16)),
]


@pytest.mark.parametrize("dtype", ["16", "32"])
@pytest.mark.parametrize("neighbours,shared,inverse,real,own", [(False, False, False, False, True), (True, True, True, True, True),
                                                               (True, False, False, False, False), (False, True, True, True, False)])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "-".join(str(v) for v in c))
def test_rotary_of_many_tokens(case, neighbours, shared, inverse, real, own, dtype, fmt):
    """Aligned heads; own: positions per picture, so that a workgroup's tokens lie in two of them."""
    check_rotary(*case, neighbours, shared, inverse, real, own, F32 if dtype == "32" else fmt)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dtype", ["16", "32"])
def test_rotary_of_more_than_a_cache(dtype, neighbours, fmt):
    """Over 32 MB read and written: four pieces of a thread in flight, a last turn that has fewer."""
    check_rotary(2, 9007, 7, 2, 64, (24, 20, 20), neighbours, False, False, False, True, F32 if dtype == "32" else fmt)
    check_rotary(1, 17011, 3, 3, 88, (20, 20, 20), neighbours, False, True, True, False, F32 if dtype == "32" else fmt)


@pytest.mark.parametrize("qh,kh,D,N", [(1, 1, 128, 70001), (1, 0, 128, 66000), (1, 1, 64, 131077)])
def test_rotary_with_the_largest_table(qh, kh, D, N, fmt):
    """Few heads of many tokens: sines and cosines fill the 64 KB of LDS that a launch may have."""
    check_rotary(1, N, qh, kh, D, (D // 2, D // 4, D // 4), False, False, False, False, False, fmt)


def check_rotary(B, N, hq, hk, D, sections, neighbours, shared, inverse, real, own, t):
    g = torch.Generator(device=DEV).manual_seed(N + D)
    heads = hq + hk
    buf = torch.randn(B, N, heads * D + 8, generator=g, device=DEV).to(t)        # 16 bytes of another operand in front of the queries
    buf[..., :8] = 7.0
    out = torch.full_like(buf, 5.0)
    pos = torch.randint(0, 4000, (B, N, len(sections)), generator=g, device=DEV, dtype=torch.int32)
    pos = pos.float() * 0.37 - 100 if real else pos
    pos = pos if own else pos[0].contiguous()
    plan = RotaryAxes(D, sections, 10000.0, neighbours, shared, DEV)
    v, o = (View(b.view(-1), B, 1, N, heads * D + 8) for b in (buf, out))
    keep = buf.clone()

    def parts(w):
        return w.slice(8, hq * D), w.slice(8 + hq * D, hk * D) if hk else None
    (q, k), (qo, ko) = parts(v), parts(o)
    K.rotary_axes(plan, pos, q, qo, k, ko, inverse=inverse)
    assert torch.equal(buf, keep) and bool((out[..., :8] == 5.0).all())
    x = buf[..., 8:].contiguous()
    ref = turned64(x, heads, plan, pos, 10000.0, inverse)
    close_turns(out[..., 8:], x, ref, heads, D, t)
    K.rotary_axes(plan, pos, q, None, k, None, inverse=inverse)                  # in place: the same bits
    assert torch.equal(buf[..., 8:], out[..., 8:]) and bool((buf[..., :8] == 7.0).all())


# ---- mxfp4 ------------------------------------------------------------------------------------------------------------------------
def test_mxfp4_of_subnormal_blocks(fmt):
    """Blocks whose largest magnitude is a subnormal of the 16-bit type, down to its smallest, and blocks that reach from there to normal values."""
    small = torch.finfo(fmt).smallest_normal * torch.finfo(fmt).eps
    g = gen(40)
    rows = [torch.randint(-n, n + 1, (96,), generator=g).double() * small for n in (1, 2, 3, 7, 100, 127)]
    if fmt == torch.float16:
        rows += [torch.randint(-1023, 1024, (96,), generator=g).double() * small]
    rows += [rows[-1].clone(), torch.zeros(96, dtype=torch.float64)]
    rows[-2][::32] = torch.finfo(fmt).smallest_normal * 1.5
    x = torch.stack(rows).to(fmt)
    q = K.mxfp4_quantize(rows_view(x))
    codes, scales, val = held64(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    y = empty(1, x.shape[0], 96, F32)
    K.mxfp4_dequantize(q, y)
    assert torch.equal(back(y)[0], val.float())


# ---- operands in each other's memory: refused before a launch ------------------------------------------------------------------------
def shared(fn, *a, **k):
    with pytest.raises(KernelError, match="shares memory"):
        fn(*a, **k)


def test_mxfp4_outputs_in_operands(fmt):
    M, N, k = 40, 64, 256
    x, w = rows_view(rand(gen(50), M, k).to(fmt)), K.mxfp4_quantize(rows_view(rand(gen(51), N, k)))
    q = K.mxfp4_quantize(x)
    bias = torch.ones(M * N, device=DEV)
    keep = [t.clone() for t in (q.codes, q.scales, w.codes, w.scales)]

    def over(t, rows, Cc, dtype=fmt):                     # a View of rows in t's memory
        return View(t.view(-1).view(dtype), 1, 1, rows, Cc)
    for t in (q.codes, w.codes):
        shared(K.mxfp4_linear, q, w, None, over(t, 40, 64))
    big = torch.zeros(M * N * 8, dtype=torch.uint8, device=DEV)                  # scales of a matrix inside the output's memory
    for held in (q, w):
        scales = big[64:64 + held.scales.numel()].view(held.scales.shape).copy_(held.scales)
        inside = K.MxFp4(held.codes, scales, held.rows, k)
        shared(K.mxfp4_linear, inside if held is q else q, inside if held is w else w, None, over(big, M, N, F32))
    shared(K.mxfp4_linear, q, w, bias[:N], View(bias, 1, 1, M, N))
    assert all(torch.equal(a, b) for a, b in zip((q.codes, q.scales, w.codes, w.scales), keep))
    room = torch.zeros(M * k * 4, dtype=torch.uint8, device=DEV)                 # x, and in its memory the codes or the scales
    y = View(room.view(F32), 1, 1, M, k)
    shared(K.mxfp4_quantize, y, K.MxFp4(room[:M * k // 2].view(M, k // 2), q.scales, M, k))
    shared(K.mxfp4_quantize, y, K.MxFp4(q.codes, room[-M * k // 32:].view(M, k // 32), M, k))
    shared(K.mxfp4_quantize, x, K.MxFp4(room[:M * k // 2].view(M, k // 2), room[64:64 + M * k // 32].view(M, k // 32), M, k))
    shared(K.mxfp4_dequantize, K.MxFp4(room[:M * k // 2].view(M, k // 2), q.scales, M, k), y)
    shared(K.mxfp4_dequantize, K.MxFp4(q.codes, room[-M * k // 32:].view(M, k // 32), M, k), y)


def test_block_norm_outputs_in_vectors_and_gradients_in_rows(fmt):
    B, N, Cc = 2, 6, 64
    g = gen(52)
    x, f, dy, dxo = (tokens(rand(g, B, N, Cc).to(F32)) for _ in range(4))
    xo, y, dx, df = (empty(B, N, Cc, F32) for _ in range(4))
    mod = torch.ones(B, 3 * Cc, device=DEV)
    gate, scale, shift = mod[:, :Cc], mod[:, Cc:2 * Cc], mod[:, 2 * Cc:]
    w, flat = torch.ones(Cc, device=DEV), torch.ones(B * N * Cc, device=DEV)
    inside = View(flat, B, 1, N, Cc)
    for p in (dict(gate=flat[Cc:2 * Cc]), dict(scale=flat[-Cc:]), dict(shift=flat[:B * Cc].view(B, Cc)), dict(w=flat[5:5 + Cc]),
              dict(post=True, post_b=flat[:Cc])):
        shared(K.block_norm, x, inside, f=f, xo=xo, **p)
        shared(K.block_norm, x, y, f=f, xo=inside, **p)
        shared(K.block_norm_backward, x, dy, inside, dxo=dxo, f=f, df=df, **p)
        shared(K.block_norm_backward, x, dy, dx, dxo=dxo, f=f, df=inside, **p)
    given = dict(dxo=dxo, f=f, df=df, gate=gate, scale=scale, shift=shift, w=w, b=w)
    buf = torch.empty(4 * Cc, device=DEV)
    shared(K.block_norm_backward, x, dy, dx, **given, d_w=buf[:Cc], d_b=buf[8:8 + Cc])
    shared(K.block_norm_backward, x, dy, dx, **given, d_gate=buf[:B * Cc].view(B, Cc), d_w=buf[B * Cc - 1:(B + 1) * Cc - 1])
    for v in (x, f, dy, dxo, dx, df):
        shared(K.block_norm_backward, x, dy, dx, **given, d_w=v.t[-Cc:])
        shared(K.block_norm_backward, x, dy, dx, **given, d_scale=v.t[:B * Cc].view(B, Cc))
    shared(K.block_norm_backward, x, dy, dx, **given, d_w=w)
    shared(K.block_norm_backward, x, dy, dx, **given, d_b=mod.view(-1)[Cc - 1:2 * Cc - 1])
    # end to end is apart
    K.block_norm_backward(x, dy, dx, **given, d_w=buf[:Cc], d_b=buf[Cc:2 * Cc], d_gate=buf[2 * Cc:].view(B, Cc))
    alone = [torch.empty(Cc, device=DEV), torch.empty(Cc, device=DEV), torch.empty(B, Cc, device=DEV)]
    K.block_norm_backward(x, dy, dx, **given, d_w=alone[0], d_b=alone[1], d_gate=alone[2])
    assert torch.equal(buf, torch.cat([t.flatten() for t in alone]))


def test_rotary_outputs_in_positions(fmt):
    D, N = 16, 8
    plan, q, k = RotaryAxes(D, (8, 8), device=DEV), tokens(rand(gen(53), 1, N, 2 * D).to(fmt)), tokens(rand(gen(54), 1, N, D).to(fmt))
    buf = torch.zeros(N * 2 * D, dtype=torch.int32, device=DEV)
    inside = View(buf.view(fmt)[:N * 2 * D], 1, 1, N, 2 * D)
    for at in (0, N * D - 2 * N):
        pos = buf[at:at + 2 * N].view(N, 2)
        shared(K.rotary_axes, plan, pos, q, inside, k)
        shared(K.rotary_axes, plan, pos, inside)
        shared(K.rotary_axes, plan, pos, q, None, k, View(inside.t, 1, 1, N, D, 2 * D, D if at else 0))
    K.rotary_axes(plan, buf[N * D:N * D + 2 * N].view(N, 2), q, inside)          # behind it
    assert torch.equal(back(inside), back(q))                                    # position 0


def test_two_threads_in_their_own_format_and_stream():
    """Calls of two threads at once, each on a stream of its own, one with either format's library: workspaces are the calls' own, the format and the
    current stream the threads'."""
    import threading
    B, N, Cc = 2, 700, 320
    turns, plan = 30, RotaryAxes(40, (20, 20), device=DEV)
    pos = torch.randint(0, 100, (N, 2), dtype=torch.int32, device=DEV)

    def work(name):
        t = FORMATS[name]
        g = torch.Generator(device=DEV).manual_seed(60)
        x, f, dy, dxo = (torch.randn(B * N * Cc, generator=g, device=DEV).to(t) for _ in range(4))
        gate, scale, w = torch.randn(B, Cc, generator=g, device=DEV), torch.randn(B, Cc, generator=g, device=DEV), torch.randn(Cc, Cc, generator=g, device=DEV)
        held = K.mxfp4_quantize(View(w, 1, 1, Cc, Cc))

        def v(buf):
            return View(buf, B, 1, N, Cc)

        def once():
            xo, y, z, dx, df = (torch.empty_like(x) for _ in range(5))
            dg, ds = torch.empty_like(gate), torch.empty_like(scale)
            K.block_norm(v(x), v(y), f=v(f), xo=v(xo), post=True, gate=gate, scale=scale)
            K.mxfp4_linear(v(y), held, None, v(z))
            K.rotary_axes(plan, pos, v(z))
            K.block_norm_backward(v(xo), v(dy), v(dx), dxo=v(dxo), f=v(f), df=v(df), post=True, gate=gate, scale=scale, d_gate=dg, d_scale=ds)
            return [xo, z, dx, df, dg, ds]
        return once
    fns, want, got, failed = {}, {}, {"f16": [], "bf16": []}, []
    for name in FORMATS:
        with K.act_format(name):
            fns[name] = work(name)
            want[name] = fns[name]()
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def run(name):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream), K.act_format(name):
                start.wait(30)
                for _ in range(turns):
                    got[name].append(fns[name]())
                stream.synchronize()
        except Exception as e:                           # noqa: BLE001 (shown by the thread that waits)
            failed.append(e)
    threads = [threading.Thread(target=run, args=(name,)) for name in FORMATS]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for name in FORMATS:
        assert len(got[name]) == turns and all(torch.equal(a, b) for r in got[name] for a, b in zip(r, want[name])), name


def test_every_operator_of_a_block_on_the_inputs_it_got(fmt, monkeypatch):
    """The block of test_gpu_token_ops, each of its operators compared with its definition in 64 bits on what the run itself handed it, to that
    operator's own tolerance: a small wrong term has nowhere to hide behind the block's other roundings."""
    B, H, W, heads, D, sections, wts, dev, pos, x, plan = block_setup(fmt)
    calls, real = [], {n: getattr(K, n) for n in ("block_norm", "mxfp4_linear", "rotary_axes", "mxfp4_quantize")}

    def values(v):                                        # what rows of a View or codes stand for, [rows, K] in 64 bits
        if isinstance(v, K.MxFp4):
            y = torch.empty(v.rows, v.K, device=DEV)
            K.mxfp4_dequantize(v, View(y, 1, 1, v.rows, v.K))
            return y.cpu().double()
        return held64(back(v).flatten(0, 1))[2]

    def block_norm(xv, y=None, f=None, xo=None, **a):
        given, branch = back(xv).double(), back(f).double() if f is not None else None
        real["block_norm"](xv, y, f=f, xo=xo, **a)
        a = {k: v.cpu().double() if isinstance(v, torch.Tensor) else v for k, v in {"kind": K.NORM_LAYER, **a}.items()}
        t, ref = join64(given, branch, a, 1e-5)
        if xo is not None:
            step = (t - given).abs() + given.abs()
            within(back(xo), t, half_step(fmt) * t.abs() + tiny(fmt) + 64 * EPS32 * step.amax(-1, keepdim=True), "xo")
        if y is not None:
            within(back(y), ref, tol_y(t, ref, a, fmt), "y")
        calls.append("block_norm")

    def mxfp4_linear(xv, w, bias, y, epi=K.EPI_LINEAR):
        ref, err = linear64(values(xv), values(w), None, epi, 1.0, 0.0, None)
        real["mxfp4_linear"](xv, w, bias, y, epi=epi)
        within(back(y).flatten(0, 1), ref, half_step(fmt) * ref.abs() + tiny(fmt) + err, "linear")
        calls.append("mxfp4_linear")

    def rotary_axes(p, at, q, k=None):
        given = [back(v) for v in (q, k)]
        real["rotary_axes"](p, at, q, k=k)
        for v, was in zip((q, k), given):
            ref = rotary64(was.double(), heads, D, sections, at.cpu(), 10000.0, False, False, False)
            within(back(v), ref, tol_rot(was, ref, heads, D, fmt), "rotary")
        calls.append("rotary_axes")

    def mxfp4_quantize(v, q=None):
        q = real["mxfp4_quantize"](v, q)
        codes, scales, _ = held64(back(v).flatten(0, 1))
        assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
        calls.append("mxfp4_quantize")
        return q
    for fn in (block_norm, mxfp4_linear, rotary_axes, mxfp4_quantize):
        monkeypatch.setattr(K, fn.__name__, fn)
    out = run_block(tokens(x), dev, plan, pos.to(DEV), B, H, W, heads, D)
    assert sorted(calls) == ["block_norm"] * 3 + ["mxfp4_linear"] * (4 + B) + ["mxfp4_quantize", "rotary_axes"]
    monkeypatch.undo()
    assert torch.equal(back(out), back(run_block(tokens(x), dev, plan, pos.to(DEV), B, H, W, heads, D)))
