"""Operands of the transformer-block operators that lie in each other's memory: what the C entries refuse (on the host, nothing is launched).

Addresses are made up.  The comparison itself (csrc/apart.h) is compiled for the host."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

from onedc_amd import build, kernels as K
from test_launch_limits import launches  # noqa: F401  (a fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHARED = -17


@pytest.fixture(scope="module", autouse=True)
def _hip():
    build.build_hip()


def test_the_status_is_the_headers(tmp_path):
    src = tmp_path / "status.cpp"
    src.write_text('#include "onedc_hip.h"\n#include <cstdio>\nint main() { printf("%d", ONEDC_SHARED_MEMORY); }\n')
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "status"), str(src)], check=True)
    got = int(subprocess.run([str(tmp_path / "status")], check=True, capture_output=True, text=True).stdout)
    assert got == SHARED == K.SHARED_MEMORY
    with pytest.raises(K.KernelError, match="shares memory"):
        K._ok(SHARED, "onedc_mxfp4_linear")


def test_rows_that_meet_or_do_not(tmp_path):
    """Against the bytes themselves, over small operands: nothing shared is missed; what is apart is called shared only for rows of different pitches."""
    src = tmp_path / "apart.cpp"
    src.write_text('#include "apart.h"\nextern "C" int shared(long a, long n, long cs, long w, long b, long m, long ds, long v) {\n'
                   "    return onedc_mem_shared(onedc_mem_rows((void *)a, n, cs, 0, w, 1), onedc_mem_rows((void *)b, m, ds, 0, v, 1)); }\n")
    so = str(tmp_path / "apart.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onedc_amd", "csrc"), "-o", so, str(src)], check=True)
    shared = C.CDLL(so).shared
    shared.argtypes = [C.c_long] * 8

    def bytes_of(at, rows, pitch, width):
        return {at + r * pitch + i for r in range(rows) for i in range(width)}
    over = 0
    for n, cs, w, m, ds, v in itertools.product((1, 2, 3), (3, 4, 8), (1, 2, 3), (1, 2, 4), (2, 4, 12), (1, 2)):
        for b in range(970, 1040):
            meet = bool(bytes_of(1000, n, cs, w) & bytes_of(b, m, ds, v))
            got = bool(shared(1000, n, cs, w, b, m, ds, v))
            assert got or not meet, (n, cs, w, b, m, ds, v)
            if got and not meet:
                over += 1
                assert n > 1 and m > 1 and cs != ds or w > cs or v > ds or n == 1 or m == 1, (n, cs, w, b, m, ds, v)
    assert over
    assert not shared(0, 3, 8, 2, 1, 1, 8, 1)             # NULL: no operand


# ---- block_norm -------------------------------------------------------------------------------------------------------------------
B, TOKENS, CH = 3, 5, 24
ROWS = dict(x=0x100000, f=0x200000, xo=0x300000, y=0x400000)
VECTORS = dict(post_w=0x500000, post_b=0x510000, gate=0x520000, w=0x530000, b=0x540000, scale=0x550000, shift=0x560000)
PER_PICTURE = dict(gate_rs=CH + 8, scale_rs=CH, shift_rs=3 * CH)


def norm_params(**over):
    p = dict(B=B, N=TOKENS, C=CH, x_cs=CH, f_cs=CH, xo_cs=CH, y_cs=CH, post=1, alpha=1.0, eps=1e-5, **ROWS, **VECTORS, **PER_PICTURE)
    return {**p, **over}


def norm(**over):
    return K.lib().onedc_block_norm(C.byref(K.BlockNormParams(**norm_params(**over))), None)


def last_of(name):
    """The first byte of a vector's last value."""
    return VECTORS[name] + 4 * ((CH if name in ("post_w", "post_b", "w", "b") else (B - 1) * PER_PICTURE[name + "_rs"] + CH) - 1)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("name", sorted(VECTORS))
def test_block_norm_outputs_in_a_vector(name, f32):
    size = B * TOKENS * CH * (4 if f32 else 2)
    for out in ("xo", "y"):
        for at in (VECTORS[name], last_of(name), VECTORS[name] - size + 4):
            assert norm(**{out: at}, x_f32=f32, f_f32=f32) == SHARED, (out, hex(at))
    # a row of the stream that has the parameters behind its channels, whatever picture's they are
    if name == "gate":
        assert norm(gate=ROWS["xo"] + 4 * CH - 4, gate_rs=TOKENS * 64, xo_cs=64, x_f32=1) == SHARED


GRADS = dict(d_post_w=0x600000, d_post_b=0x610000, d_gate=0x620000, d_w=0x630000, d_b=0x640000, d_scale=0x650000, d_shift=0x660000)
GRAD_ROWS = dict(dy=0x700000, dxo=0x710000, dx=0x720000, df=0x730000)


def norm_back(p=None, **over):
    g = dict(**GRADS, **GRAD_ROWS, dy_cs=CH, dxo_cs=CH, dx_cs=CH, df_cs=CH, ws=0x900000, ws_bytes=1 << 20)
    params, grad = K.BlockNormParams(**norm_params(**(p or {}))), K.BlockNormGrad(**{**g, **over})
    return K.lib().onedc_block_norm_backward(C.byref(params), C.byref(grad), None)


def grad_bytes(name):
    return 4 * CH * (B if name in ("d_gate", "d_scale", "d_shift") else 1)


@pytest.mark.parametrize("name", sorted(GRADS))
def test_block_norm_gradients_in_other_memory(name):
    size = grad_bytes(name)
    places = [v for o, v in GRADS.items() if o != name] + [v + grad_bytes(o) - 4 for o, v in GRADS.items() if o != name]
    places += [v - size + 4 for o, v in GRADS.items() if o != name]
    places += list(VECTORS.values()) + [last_of(v) for v in VECTORS] + [VECTORS["scale"] - size + 4]
    places += list(GRAD_ROWS.values()) + [v + B * TOKENS * CH * 2 - 4 for v in GRAD_ROWS.values()] + [ROWS["x"], ROWS["f"] + 48, 0x900000, 0x900040]
    for at in places:
        assert norm_back(**{name: at}) == SHARED, hex(at)
    # one row for all pictures: C values, not B C
    if size > 4 * CH:
        one = {name[2:] + "_rs": 0}
        assert norm_back(one, **{name: GRADS["d_w"] - 4 * CH + 4}) == SHARED
        # no rows: gradients are written all the same (zeros), and parameters are not theirs to write
        assert norm_back(dict(N=0), **{name: VECTORS["w"]}) == SHARED


def test_block_norm_backward_outputs_and_workspace_in_other_memory():
    for out in ("dx", "df"):
        for name in VECTORS:
            assert norm_back(**{out: VECTORS[name]}) == norm_back(**{out: last_of(name) - 2}) == SHARED
    for at in [*VECTORS.values(), *GRAD_ROWS.values(), *GRADS.values(), ROWS["x"], ROWS["f"]]:
        assert norm_back(ws=at) == SHARED, hex(at)


def test_what_block_norm_still_takes(launches):
    p = norm_params()
    g = dict(**GRADS, **GRAD_ROWS, dy_cs=CH, dxo_cs=CH, dx_cs=CH, df_cs=CH)
    stream = 0x100000                                    # one buffer: f32 rows of 128 values, a picture one token; parameters behind the channels
    rows = dict(B=B, N=1, x=stream, xo=stream, x_cs=128, xo_cs=128, x_f32=1, gate=stream + 4 * CH, gate_rs=128, scale=stream + 8 * CH, scale_rs=128)
    packed = {n: 0x600000 + 4 * CH * i for i, n in enumerate(("d_w", "d_b", "d_post_w", "d_post_b"))}        # end to end
    calls = [["onedc_block_norm", p], ["onedc_block_norm", {**p, "xo": p["x"]}], ["onedc_block_norm", {**p, **rows}],
             ["onedc_block_norm", {**p, "scale": p["gate"], "shift": p["gate"], "scale_rs": p["gate_rs"], "shift_rs": p["gate_rs"]}],
             ["onedc_block_norm_backward", [p, g]], ["onedc_block_norm_backward", [p, {**g, "dx": g["dxo"], "df": g["dy"]}]],
             ["onedc_block_norm_backward", [{**p, **rows}, {**g, **packed}]], ["onedc_block_norm_backward", [{**p, "N": 0}, g]]]
    assert [rc for rc, _ in launches(calls)] == [0] * len(calls)


# ---- rotary -----------------------------------------------------------------------------------------------------------------------
ROT = dict(q=0x100000, qo=0x200000, k=0x300000, ko=0x400000, pos=0x500000, turns=0x510000, axis=0x520000, B=2, N=6, D=16, pairs=7, axes=3, qh=4, kh=2,
           q_cs=64, qo_cs=64, k_cs=32, ko_cs=32, pos_bs=18)


def rotary(**over):
    return K.lib().onedc_rotary_axes(C.byref(K.RotaryParams(**{**ROT, **over})), None)


@pytest.mark.parametrize("f32", [0, 1])
def test_rotary_outputs_in_the_plan_or_the_positions(f32):
    size = 4 if f32 else 2
    for out, heads in (("qo", 4), ("ko", 2)):
        rows = 12 * heads * 16 * size
        for name, n in (("pos", 2 * 18 * 4), ("turns", 7 * 8), ("axis", 7 * 4)):
            for at in (ROT[name], ROT[name] + n - size, ROT[name] - rows + size):
                assert rotary(**{out: at}, x_f32=f32) == SHARED, (out, name, hex(at))
    assert rotary(qo=0x500000 + 18 * 4 - size, pos_bs=0, x_f32=f32) == SHARED               # one picture's positions for all


def test_what_rotary_still_takes(launches):
    same = dict(ROT, qo=ROT["q"], ko=ROT["k"])
    calls = [["onedc_rotary_axes", ROT], ["onedc_rotary_axes", same], ["onedc_rotary_axes", dict(ROT, qo=ROT["pos"] + 2 * 18 * 4, ko=ROT["axis"] + 28)],
             ["onedc_rotary_axes", dict(ROT, pos_bs=0, qo=ROT["pos"] + 18 * 4)], ["onedc_rotary_axes", dict(ROT, kh=0, k=None, ko=None)]]
    assert [rc for rc, _ in launches(calls)] == [0] * len(calls)


# ---- mxfp4 ------------------------------------------------------------------------------------------------------------------------
M, N, KV = 40, 64, 200                                    # two steps of 128: 128 bytes of codes and 8 of scales a row
AT = dict(xc=0x100000, xs=0x200000, wc=0x300000, ws=0x400000, bias=0x500000, y=0x600000)
SIZE = dict(xc=M * 128, xs=M * 8, wc=N * 128, ws=N * 8, bias=N * 4)


def linear(**over):
    p = K.MxFp4Params(**{**AT, **dict(M=M, N=N, K=KV, y_cs=N, alpha=1.0), **over})
    return K.lib().onedc_mxfp4_linear(C.byref(p), None)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("name", sorted(SIZE))
def test_mxfp4_linear_over_what_it_reads(name, f32):
    rows = ((M - 1) * N + N) * (4 if f32 else 2)
    for y in (AT[name], AT[name] + SIZE[name] - (4 if f32 else 2), AT[name] - rows + 4, AT[name] - rows // 2 // 4 * 4):
        assert linear(y=y, y_f32=f32) == SHARED, (name, hex(y))
    if name == "bias":                                   # (the end of a row lies on it, and it does not fit between the rows)
        assert linear(y=AT[name] - 128 * 4, y_cs=256, y_f32=1, y_co=96) == SHARED


def test_what_stays_allowed(launches):
    """Other columns of one buffer's rows, and memory that begins where another operand ends."""
    p = dict(M=16, N=N, K=KV, alpha=1.0, wc=AT["wc"], ws=AT["ws"])
    calls = [["onedc_mxfp4_linear", dict(**p, xr=0x100000, xr_cs=300, y=0x100000, y_cs=300, y_co=KV)],
             ["onedc_mxfp4_linear", dict(**p, xr=0x100000, xr_cs=300, xr_co=100, y=0x100000, y_cs=300, y_co=36, res=0x100000, r_cs=300, r_co=36)],
             ["onedc_mxfp4_linear", dict(**p, xr=0x100000, xr_cs=KV, y=AT["wc"] + N * 128, y_cs=N, bias=AT["wc"] - 4 * N)],
             ["onedc_mxfp4_quantize", [0x100000, 0, KV, 0, 0x100000 + 8 * KV * 2, 0x100000 - 64, 8, KV]],
             ["onedc_mxfp4_dequantize", [0x100000, 0x100000 + 8 * 128, 0x100000 + 8 * 136, 0, KV, 0, 8, KV]]]
    assert [rc for rc, _ in launches(calls)] == [0] * len(calls)


def test_mxfp4_linear_over_raw_rows():
    raw = dict(xc=None, xs=None, xr=0x100000, xr_cs=KV, M=16)
    assert linear(**raw, y=0x100000) == SHARED
    assert linear(**{**raw, "xr_cs": 300}, y=0x100000, y_cs=300, y_co=KV - 1) == SHARED
    assert linear(**{**raw, "xr_f32": 1}, y=0x100000 + 4 * (16 * KV - 1)) == SHARED


def test_mxfp4_quantize_and_back_over_their_operands():
    lib, x, c, s = K.lib(), 0x100000, 0x200000, 0x300000

    def quantize(x, c, s, rows=8, f32=0):
        return lib.onedc_mxfp4_quantize(x, f32, KV, 0, c, s, rows, KV, None)

    def back(c, s, y, rows=8, f32=0, cs=KV, co=0):
        return lib.onedc_mxfp4_dequantize(c, s, y, f32, cs, co, rows, KV, None)
    assert quantize(x, x, s) == quantize(x, x + 8 * KV * 2 - 16, s) == quantize(x + 8 * 128 - 2, x, s) == SHARED
    assert quantize(x, c, x) == quantize(x, c, x + 8 * KV * 2 - 4) == SHARED
    assert quantize(x, c, x + 8 * KV * 4 - 4, f32=1) == SHARED
    assert quantize(x, c, c) == quantize(x, c, c + 8 * 128 - 4) == quantize(x, c + 32, c) == SHARED
    assert back(c, s, c) == back(c, s, c + 8 * 128 - 2) == back(c, s, s) == back(c, s, s + 8 * 8 - 2) == SHARED
    assert back(c, s, c - 4 * KV, f32=1) == back(c, s, c, cs=KV + 8, co=8) == SHARED
