"""Transformer-block operators (block_norm, rotary_axes, mxfp4_*): what is refused, before anything reaches a GPU; plans and layouts."""
import ctypes as C
import os

import pytest
import torch

from onedc_amd import build, kernels as K
from onedc_amd.kernels import KernelError, MxFp4, RotaryAxes, View

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def _hip():
    build.build_hip()


def view(B, N, Cc, dtype=None, cs=None, co=0, rows=None):
    cs = cs or Cc + co
    return View(torch.zeros((rows if rows is not None else B * N) * cs, dtype=dtype or K.a16()), B, 1, N, Cc, cs, co)


def vec(*shape):
    return torch.ones(*shape)


F32 = torch.float32


def test_struct_sizes_and_constants_match_the_header(tmp_path):
    src = tmp_path / "sizes.cpp"
    src.write_text('#include "onedc_hip.h"\n#include <cstdio>\nint main() { printf("%zu %zu %zu %zu %d %d %d", sizeof(onedc_block_norm_params), '
                   "sizeof(onedc_block_norm_grad), sizeof(onedc_rotary_params), sizeof(onedc_mxfp4_params), ONEDC_MXFP4_ROWS_RAW, "
                   "ONEDC_NORM_LAYER, ONEDC_NORM_RMS); }\n")
    import subprocess
    exe = str(tmp_path / "sizes")
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(K.BlockNormParams), C.sizeof(K.BlockNormGrad), C.sizeof(K.RotaryParams), C.sizeof(K.MxFp4Params), K.MXFP4_ROWS_RAW,
                   K.NORM_LAYER, K.NORM_RMS]


# ---- block_norm -------------------------------------------------------------------------------------------------------------------
def refused(match, fn, *a, **k):
    with pytest.raises(KernelError, match=match):
        fn(*a, **k)


def test_block_norm_refusals():
    B, N, Cc = 2, 5, 24
    x, f, y, xo = (view(B, N, Cc) for _ in range(4))
    bn = K.block_norm
    refused("nothing to compute", bn, x)
    refused("come together", bn, x, y, f=f)
    refused("come together", bn, x, y, xo=xo)
    refused("kind", bn, x, y, kind=2)
    refused("needs f", bn, x, y, post=True)
    refused("needs f", bn, x, y, gate=vec(Cc))
    refused("need post=True", bn, x, y, f=f, xo=xo, post_w=vec(Cc))
    refused("belong to the norm", bn, x, f=f, xo=xo, w=vec(Cc))
    refused("belong to the norm", bn, x, f=f, xo=xo, shift=vec(B, Cc))
    refused("y has 2 x 4 rows", bn, x, view(B, 4, Cc))
    refused("y has 16 channels", bn, x, view(B, N, 16))
    refused("f has 16 channels", bn, x, y, f=view(B, N, 16), xo=xo)
    refused("x is torch.bfloat16" if K.a16() == torch.float16 else "x is torch.float16", bn,
            view(B, N, Cc, torch.bfloat16 if K.a16() == torch.float16 else torch.float16), y)
    refused("f is torch.float32", bn, x, y, f=view(B, N, Cc, F32), xo=xo)                     # a 32-bit branch into a 16-bit stream
    refused("one type", bn, view(B, N, Cc, F32), view(B, N, Cc, F32), f=f, xo=view(B, N, Cc, F32))
    refused("xo is", bn, x, y, f=f, xo=view(B, N, Cc, F32))
    refused("outside its buffer", bn, view(B, N, Cc, rows=B * N - 1), y)
    refused("outside its buffer", bn, View(torch.zeros(B * N * Cc, dtype=K.a16()), B, 1, N, Cc, Cc, 1), y)
    refused("outside its buffer", bn, x, View(torch.zeros(B * N, 2 * Cc, dtype=K.a16())[:, :Cc], B, 1, N, Cc))
    for name in ("w", "b"):
        refused(f"{name} must be", bn, x, y, **{name: vec(Cc + 1)})
        refused(f"{name} must be", bn, x, y, **{name: vec(Cc).double()})
    for name in ("scale", "shift"):
        refused(f"{name} must be", bn, x, y, **{name: vec(3, Cc)})
        refused(f"{name} must be", bn, x, y, **{name: vec(Cc, B).t()})
        refused(f"{name} must be", bn, x, y, **{name: vec(1, Cc).expand(B, Cc)})                # its gradient would have no place
        refused(f"{name} must be", bn, x, y, **{name: vec(B, Cc).half()})
    refused("gate must be", bn, x, y, f=f, xo=xo, gate=vec(B, Cc + 8))
    # memory that two operands share
    refused("y shares memory", bn, x, x)
    refused("y shares memory", bn, x, f, f=f, xo=xo)
    refused("xo shares memory", bn, x, y, f=f, xo=f)
    wide = view(B, N, 2 * Cc)
    refused("shares memory", bn, wide.slice(0, Cc), wide.slice(8, Cc))
    # nothing wrong but the device: different channel slices of one buffer, the stream in place
    refused("is on cpu", bn, wide.slice(0, Cc), wide.slice(Cc, Cc))
    refused("is on cpu", bn, x, y, f=f, xo=x)
    refused("is on cpu", bn, view(B, N, Cc, F32), y, f=f, xo=view(B, N, Cc, F32), gate=vec(B, 3 * Cc)[:, Cc:2 * Cc], scale=vec(1, Cc),
            shift=vec(Cc))


def test_block_norm_backward_refusals():
    B, N, Cc = 2, 5, 24
    x, f, dy, dxo, dx, df = (view(B, N, Cc) for _ in range(6))
    bw = K.block_norm_backward
    refused("no gradient to pass on", bw, x, None, dx)
    refused("need f", bw, x, dy, dx, df=df)
    refused("belong to the norm", bw, x, None, dx, dxo=dxo, f=f, w=vec(Cc))
    refused("parameter that the call has not", bw, x, dy, dx, d_w=vec(Cc))
    refused("d_scale must be 48", bw, x, dy, dx, scale=vec(B, Cc), d_scale=vec(Cc))
    refused("d_scale must be 24", bw, x, dy, dx, scale=vec(Cc), d_scale=vec(B, Cc))
    refused("d_gate must be", bw, x, dy, dx, f=f, df=df, gate=vec(B, Cc), d_gate=vec(B, 2 * Cc)[:, :Cc])
    refused("dx shares memory", bw, x, dy, x)
    refused("dx shares memory", bw, x, dy, dy)
    refused("dx shares memory", bw, x, dy, dx, f=f, df=dx)
    refused("df shares memory", bw, x, dy, dx, dxo=dxo, f=f, df=f)
    refused("dxo is torch.float32", bw, x, dy, dx, dxo=view(B, N, Cc, F32))
    once = vec(Cc)
    refused("gradients share memory", bw, x, dy, dx, w=vec(Cc), b=vec(Cc), d_w=once, d_b=once)
    refused("is on cpu", bw, x, dy, dxo, dxo=dxo, f=f, df=dy)


def block_norm_c(**over):
    """Status of the C entry for a call that something in `over` makes it refuse (or that has no rows): no launch."""
    p = K.BlockNormParams(x=4096, y=8192, B=1, N=4, C=8, x_cs=8, y_cs=8, f_cs=8, xo_cs=8, alpha=1.0, eps=1e-5)
    for k, v in over.items():
        setattr(p, k, v)
    return K.lib().onedc_block_norm(C.byref(p), None)


def test_block_norm_c_statuses():
    assert block_norm_c(B=0) == 0 and block_norm_c(N=0, x=None, y=None) == 0
    assert block_norm_c(x=None) == -1 and block_norm_c(y=None) == -1
    for bad in (dict(C=0), dict(x_cs=7), dict(x_co=1), dict(x_co=-1), dict(y_cs=4), dict(B=-1), dict(B=1 << 20, N=1 << 20),
                dict(N=(1 << 30) + 1), dict(x_cs=-2 ** 31), dict(scale=64, scale_rs=-8)):
        assert block_norm_c(**bad) == -2, bad
    for bad in (dict(kind=2), dict(f_f32=1), dict(post=1), dict(gate=64), dict(post_w=64), dict(f=64), dict(xo=64)):
        assert block_norm_c(**bad) == -3, bad
    p = K.BlockNormParams(x=4096, w=64, B=2, N=4, C=8, x_cs=8, alpha=1.0, eps=1e-5)
    g = K.BlockNormGrad(dy=4096, dy_cs=8, dx=8192, dx_cs=8, d_w=64)
    assert K.lib().onedc_block_norm_backward_ws_bytes(C.byref(p), C.byref(g)) > 0
    assert K.lib().onedc_block_norm_backward(C.byref(p), C.byref(g), None) == -15
    g.d_w, g.d_b = None, 64
    assert K.lib().onedc_block_norm_backward(C.byref(p), C.byref(g), None) == -3
    g.d_b, g.dx_cs = None, 7
    assert K.lib().onedc_block_norm_backward_ws_bytes(C.byref(p), C.byref(g)) == 0
    assert K.lib().onedc_block_norm_backward(C.byref(p), C.byref(g), None) == -2


# ---- rotary -----------------------------------------------------------------------------------------------------------------------
def test_rotary_plan():
    plan = RotaryAxes(16, (4, 6, 2), theta=(100.0, 1000.0, 10.0), device="cpu")
    assert (plan.pairs, plan.axes) == (6, 3) and plan.axis[:6].tolist() == [0, 0, 1, 1, 1, 2]
    want = [1, 100 ** -0.5, 1, 1000 ** (-1 / 3), 1000 ** (-2 / 3), 1]
    assert torch.allclose(plan.turns[:6] * 2 * torch.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15, atol=0)
    plan = RotaryAxes(16, (8, 4), shared_spectrum=True, device="cpu")
    assert torch.allclose(plan.turns[:6] * 2 * torch.pi, 10000.0 ** (-torch.arange(6, dtype=torch.float64) / 6), rtol=1e-15, atol=0)
    assert RotaryAxes(8, (0, 0), device="cpu").pairs == 0
    for bad in (dict(sections=(3,)), dict(sections=(6, 4)), dict(sections=()), dict(sections=(-2,)), dict(sections=(4,), theta=(1.0, 2.0)),
                dict(sections=(4,), theta=0.0), dict(sections=(4, 4), theta=(1.0, 2.0), shared_spectrum=True)):
        with pytest.raises(KernelError):
            RotaryAxes(8, device="cpu", **bad)


def test_rotary_refusals():
    B, N, D = 2, 6, 16
    plan = RotaryAxes(D, (8, 8), device="cpu")
    q, k = view(B, N, 4 * D), view(B, N, 2 * D)
    pos = torch.zeros(N, 2, dtype=torch.int32)
    ra = K.rotary_axes
    refused("not 1 to 4096 heads", ra, plan, pos, view(B, N, 3 * D + 2))
    refused("k has 2 x 5 rows", ra, plan, pos, q, k=view(B, 5, D))
    refused("k is torch.float32", ra, plan, pos, q, k=view(B, N, D, F32))
    refused("ko without k", ra, plan, pos, q, ko=k)
    refused("qo has", ra, plan, pos, q, k)
    for bad in (pos.long(), pos[:5], torch.zeros(N, 3, dtype=torch.int32), torch.zeros(3, N, 2, dtype=torch.int32),
                torch.zeros(2, N, dtype=torch.int32).t(), pos.double()):
        refused("pos must be", ra, plan, bad, q)
    wide = view(B, N, 6 * D)
    refused("qo shares memory", ra, plan, pos, wide.slice(0, 4 * D), wide.slice(D, 4 * D))
    refused("qo shares memory", ra, plan, pos, q, k=View(q.t, B, 1, N, 4 * D))
    refused("shares memory", ra, plan, pos, wide.slice(0, 4 * D), k=wide.slice(4 * D, D), ko=wide.slice(3 * D, D))
    refused("is on cpu", ra, plan, pos, wide.slice(0, 4 * D), k=wide.slice(4 * D, 2 * D))
    refused("is on cpu", ra, plan, torch.zeros(B, N, 2), q, view(B, N, 4 * D), k, view(B, N, 2 * D))


def test_rotary_c_statuses():
    def status(**over):
        p = K.RotaryParams(q=64, qo=64, k=128, ko=128, pos=256, turns=512, axis=1024, B=0, N=3, D=8, pairs=4, axes=2, qh=2, kh=1, q_cs=24,
                           qo_cs=24, k_cs=24, k_co=16, ko_cs=24, ko_co=16)
        for k, v in over.items():
            setattr(p, k, v)
        return K.lib().onedc_rotary_axes(C.byref(p), None)
    assert status() == 0 and status(kh=0, k=None, ko=None) == 0
    for name in ("q", "qo", "k", "ko", "pos", "turns", "axis"):
        assert status(**{name: None}) == -1
    for bad in (dict(pairs=5), dict(pairs=-1), dict(D=0), dict(axes=0), dict(qh=0), dict(kh=-1), dict(q_cs=15), dict(k_co=17), dict(ko_co=-1),
                dict(B=1 << 20, N=1 << 20), dict(pos_bs=-1), dict(q_cs=-2 ** 31), dict(ko_cs=-2 ** 31)):
        assert status(**bad) == -2, bad


# ---- mxfp4 ------------------------------------------------------------------------------------------------------------------------
def held(rows, k):
    return K.mxfp4_empty(rows, k, "cpu")


def test_mxfp4_refusals():
    with pytest.raises(KernelError, match="codes must be"):
        MxFp4(torch.zeros(4, 63, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 4, 100)
    with pytest.raises(KernelError, match="scales must be"):
        MxFp4(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.int8), 4, 100)
    with pytest.raises(KernelError, match="codes must be"):
        MxFp4(torch.zeros(4, 128, dtype=torch.uint8)[:, :64], torch.zeros(4, 4, dtype=torch.uint8), 4, 100)
    with pytest.raises(KernelError, match="aligned"):
        MxFp4(torch.zeros(4 * 64 + 8, dtype=torch.uint8)[8:].view(4, 64), torch.zeros(4, 4, dtype=torch.uint8), 4, 128)
    with pytest.raises(KernelError, match="no matrix"):
        MxFp4(torch.zeros(4, 0, dtype=torch.uint8), torch.zeros(4, 0, dtype=torch.uint8), 4, 0)
    x, w, y = view(1, 40, 100), held(64, 100), view(1, 40, 64)
    refused("q holds", K.mxfp4_quantize, x, held(40, 96))
    refused("is on cpu", K.mxfp4_quantize, x)
    refused("y has 99 channels", K.mxfp4_dequantize, held(40, 100), view(1, 40, 99))
    refused("y has 39 rows", K.mxfp4_dequantize, held(40, 100), view(1, 39, 100))
    refused("is on cpu", K.mxfp4_dequantize, held(40, 100), view(1, 40, 100))
    ln = K.mxfp4_linear
    refused("not one of", ln, x, w, None, y, epi=K.EPI_GLU_LEAKY)
    refused("blocks of 16", ln, x, held(48, 100), None, view(1, 40, 24), epi=K.EPI_GEGLU)
    refused("x has 96 values", ln, view(1, 40, 96), w, None, y)
    refused("x has 96 values", ln, held(40, 96), w, None, y)
    refused("y has 32 channels", ln, x, w, None, view(1, 40, 32))
    refused("y has 64 channels, not 32", ln, x, w, None, y, epi=K.EPI_GEGLU)
    refused("y has 39 rows", ln, x, w, None, view(1, 39, 64))
    refused("bias must be", ln, x, w, vec(63), y)
    refused("res is", ln, x, w, None, y, res=view(1, 40, 64, F32))
    refused("res has", ln, x, w, None, y, res=view(1, 40, 32))
    wide = view(1, 40, 164)
    refused("y shares memory", ln, wide.slice(0, 100), w, None, wide.slice(90, 64))
    later = _one_row_later(y := view(1, 41, 64))
    refused("y shares memory", ln, x, w, None, View(y.t, 1, 1, 40, 64), res=later)
    refused("is on cpu", ln, wide.slice(0, 100), w, vec(64), wide.slice(100, 64))
    y = view(1, 40, 64)
    refused("is on cpu", ln, held(40, 100), w, None, y, res=y)


def _one_row_later(y):
    """y's buffer from its second row on: as a residual, what another row of the same launch writes."""
    return View(y.t[y.cs:], 1, 1, y.W - 1, y.C)


def test_mxfp4_c_statuses():
    def status(**over):
        p = K.MxFp4Params(xc=4096, xs=4096, wc=4096, ws=4096, y=4096, M=0, N=64, K=100, y_cs=64, r_cs=64, alpha=1.0)
        for k, v in over.items():
            setattr(p, k, v)
        return K.lib().onedc_mxfp4_linear(C.byref(p), None)
    assert status() == 0 and status(epi=K.EPI_GEGLU, y_cs=32) == 0
    for bad in (dict(xc=None), dict(xs=None), dict(wc=None), dict(ws=None), dict(y=None)):
        assert status(**bad) == -1, bad
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(y_cs=63), dict(y_co=1), dict(wc=4104), dict(xs=4098), dict(res=64, r_co=1),
                dict(y_cs=-2 ** 31), dict(res=64, r_cs=-2 ** 31), dict(xc=None, xr=64, xr_cs=-2 ** 31)):
        assert status(**bad) == -2, bad
    for bad in (dict(epi=K.EPI_GLU_LEAKY), dict(epi=9), dict(epi=K.EPI_GEGLU, N=48, y_cs=64)):
        assert status(**bad) == -3, bad
    assert status(xc=None, xr=64, xr_cs=100, M=K.MXFP4_ROWS_RAW + 1) == -4
    assert status(xc=None, xr=64, xr_cs=99, M=1) == -2
    lib = K.lib()
    assert lib.onedc_mxfp4_quantize(64, 0, 8, 0, 64, 64, 0, 8, None) == 0
    assert lib.onedc_mxfp4_quantize(None, 0, 8, 0, 64, 64, 1, 8, None) == -1
    assert lib.onedc_mxfp4_quantize(64, 0, 7, 0, 64, 64, 1, 8, None) == -2
    assert lib.onedc_mxfp4_quantize(64, 0, 8, 0, 72, 64, 1, 8, None) == -2
    assert lib.onedc_mxfp4_quantize(64, 0, -2 ** 31, 0, 64, 64, 0, 8, None) == -2
    assert lib.onedc_mxfp4_dequantize(64, 64, 64, 0, -2 ** 31, 0, 0, 8, None) == -2
    assert lib.onedc_mxfp4_dequantize(64, 64, 64, 0, 8, 1, 1, 8, None) == -2
    assert lib.onedc_mxfp4_dequantize(64, 64, None, 0, 8, 0, 1, 8, None) == -1
