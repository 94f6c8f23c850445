"""What the transformer-block operators ask of a launch, on the host: the runtime's launch calls are replaced by ones that write down grid, block
and dynamic LDS, and nothing reaches a GPU."""
import json
import os
import subprocess
import sys

import pytest

from onedc_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# (the kernels' opt-in for more LDS than the default 64 KB is noted per kernel; device and last error are what a working one gives)
SHIM = r"""
#include <cstdio>
#include <cstddef>
#include <map>
struct dim { unsigned x, y, z; };
static std::map<const void *, int> opted;
static FILE *out() { static FILE *f = fopen(OUT, "a"); return f; }
static dim G, B;
static size_t L;
extern "C" {
int __hipPushCallConfiguration(dim g, dim b, size_t lds, void *) { G = g, B = b, L = lds; return 0; }
int __hipPopCallConfiguration(dim *g, dim *b, size_t *lds, void **s) { *g = G, *b = B, *lds = L, *s = nullptr; return 0; }
int hipLaunchKernel(const void *f, dim g, dim b, void **, size_t lds, void *) {
    fprintf(out(), "[%u, %u, %u, %u, %u, %u, %zu, %d]\n", g.x, g.y, g.z, b.x, b.y, b.z, lds, opted.count(f) ? opted[f] : 65536);
    fflush(out());
    return 0;
}
int hipFuncSetAttribute(const void *f, int, int v) { opted[f] = v; return 0; }
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipGetLastError() { return 0; }
}
"""

CHILD = r"""
import ctypes, json, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)            # in front of the runtime, which the kernel library brings
from onedc_amd import kernels as K
structs = {"onedc_block_norm": K.BlockNormParams, "onedc_rotary_axes": K.RotaryParams, "onedc_mxfp4_linear": K.MxFp4Params}
lib = ctypes.CDLL(K._native.HIP_F16_SO)
K.attach_signatures(lib)
read = open(sys.argv[2], "a+")
for name, args in json.load(sys.stdin):
    if name == "onedc_block_norm_backward":
        p, g = K.BlockNormParams(**args[0]), K.BlockNormGrad(**args[1])
        g.ws, g.ws_bytes = 1 << 54, 1 << 62
        rc = lib.onedc_block_norm_backward(ctypes.byref(p), ctypes.byref(g), None)
    elif name in structs:
        rc = getattr(lib, name)(ctypes.byref(structs[name](**args)), None)
    else:
        rc = getattr(lib, name)(*args, None)
    read.write(json.dumps(rc) + "\n")
    read.flush()
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """calls -> per call (status, [launches]); a launch is grid x y z, block x y z, dynamic LDS, its limit."""
    build.build_hip()
    d = tmp_path_factory.mktemp("shim")
    log, so = str(d / "log"), str(d / "shim.so")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", f'-DOUT="{log}"', "-o", so, str(d / "shim.cpp")], check=True)

    def run(calls):
        open(log, "w").close()
        subprocess.run([sys.executable, "-c", CHILD, so, log], input=json.dumps(calls), text=True, check=True, cwd=ROOT, timeout=300)
        got, open_ = [], []
        for line in open(log):
            v = json.loads(line)
            if isinstance(v, list):
                open_.append(v)
            else:
                got.append((v, open_))
                open_ = []
        assert len(got) == len(calls)
        return got
    return run


def inside_limits(calls, got):
    """Fewer than 2^32 work items along x, as the runtime demands, and no more LDS than the kernel may ask for."""
    for call, (rc, ls) in zip(calls, got):
        for gx, gy, gz, bx, by, bz, lds, most in ls:
            assert 0 < gx * bx < 1 << 32 and gy == gz == by == bz == 1 and bx <= 1024, (call, gx, bx)
            assert lds <= most <= 160 * 1024, (call, lds, most)


FAR = 1 << 43                                             # operands far from each other


def rotary(rows, qh, kh, D, pairs, x_f32=0, neighbours=0, B=1):
    c = (qh + kh) * D
    return ["onedc_rotary_axes", dict(q=FAR, qo=2 * FAR, k=FAR, ko=2 * FAR, pos=3 * FAR, turns=4 * FAR, axis=5 * FAR, B=B, N=rows, D=D, pairs=pairs,
                                      axes=3, qh=qh, kh=kh, q_cs=c, qo_cs=c, k_cs=c, k_co=qh * D, ko_cs=c, ko_co=qh * D, x_f32=x_f32,
                                      neighbours=neighbours)]


def test_rotary_asks_for_no_more_than_64_kb(launches):
    """The table of a workgroup's tokens: few heads and many rows make it largest."""
    calls = [rotary(rows, qh, kh, D, pairs, f32, nb) for rows in (1, 511, 513, 20000, 70000, 140000, 300000, 1 << 22)
             for qh, kh in ((1, 0), (1, 1), (2, 1), (8, 8), (32, 32)) for D, pairs in ((128, 64), (64, 32), (80, 40), (2, 1), (40, 16), (4096, 2048),
                                                                                      (4095, 2047), (7, 3), (64, 0))
             for f32 in (0, 1) for nb in (0, 1)]
    got = launches(calls)
    assert [(c, rc, ls) for c, (rc, ls) in zip(calls, got) if rc or len(ls) != 1] == []
    inside_limits(calls, got)


def norm(B, C, *, picture, N=1, **over):
    p = dict(x=FAR, f=2 * FAR, xo=3 * FAR, y=4 * FAR, gate=5 * FAR, B=B, N=N, C=C, x_cs=C, f_cs=C, xo_cs=C, y_cs=C, gate_rs=C if picture else 0,
             alpha=1.0, eps=1e-5)
    return ["onedc_block_norm", {**p, **over}]


def norm_back(B, C, *, picture, sums, N=1):
    p = dict(x=FAR, f=2 * FAR, gate=5 * FAR, w=9 * FAR, B=B, N=N, C=C, x_cs=C, f_cs=C, gate_rs=C if picture else 0, alpha=1.0, eps=1e-5)
    g = dict(dy=6 * FAR, dy_cs=C, dx=7 * FAR, dx_cs=C, df=8 * FAR, df_cs=C)
    if sums:
        g.update(d_gate=10 * FAR, d_w=11 * FAR)
    return ["onedc_block_norm_backward", [p, g]]


def linear(M, N, K_, epi=0):
    out = N // 2 if epi == 4 else N
    return ["onedc_mxfp4_linear", dict(xc=FAR, xs=2 * FAR, wc=3 * FAR, ws=4 * FAR, y=5 * FAR, M=M, N=N, K=K_, y_cs=out, alpha=1.0, epi=epi)]


M31 = 0x7fffffff
FITS = [
    # the last call that a launch holds, and the first that it does not
    (norm((1 << 24) - 1, 64, picture=True), norm(1 << 24, 64, picture=True)),
    (norm((1 << 23) - 1, 4000, picture=True), norm(1 << 23, 4000, picture=True)),
    (norm((1 << 22) - 1, 8200, picture=True), norm(1 << 22, 8200, picture=True)),
    (norm_back((1 << 24) - 1, 64, picture=True, sums=False), norm_back(1 << 24, 64, picture=True, sums=False)),
    (norm_back((1 << 23) - 1, 64, picture=True, sums=True), norm_back(1 << 23, 64, picture=True, sums=True)),
    (norm_back(((1 << 24) - 1) // 10, 320, picture=True, sums=True), norm_back(((1 << 24) - 1) // 10 + 1, 320, picture=True, sums=True)),
    (norm_back((1 << 22) - 1, 20000, picture=True, sums=False), norm_back(1 << 22, 20000, picture=True, sums=False)),
    (["onedc_mxfp4_quantize", [FAR, 0, 1, 0, 2 * FAR, 3 * FAR, (1 << 30) - 64, 1]], ["onedc_mxfp4_quantize", [FAR, 0, 1, 0, 2 * FAR, 3 * FAR, 1 << 30, 1]]),
    (["onedc_mxfp4_dequantize", [FAR, 2 * FAR, 3 * FAR, 1, 1, 0, (1 << 30) - 64, 1]], ["onedc_mxfp4_dequantize", [FAR, 2 * FAR, 3 * FAR, 1, 1, 0, 1 << 30, 1]]),
    (linear((1 << 26) - 16, 1, 1), linear(1 << 26, 1, 1)),
    (linear(M31 - 128, 128, 128), linear(M31, 128, 128)),
    (linear((1 << 28) - 128, 1024, 128, epi=4), linear(1 << 29, 1024, 128, epi=4)),
    (rotary((1 << 24) - 1, 16, 1, 128, 0, x_f32=1), rotary(1 << 24, 128, 1, 128, 0, x_f32=1)),
]


def test_what_a_launch_does_not_hold_is_refused(launches):
    calls = [c for pair in FITS for c in pair]
    got = launches(calls)
    inside_limits(calls, got)
    for i, (fits, not_) in enumerate(FITS):
        assert got[2 * i][0] == 0 and got[2 * i][1], fits
        assert got[2 * i + 1] == (-2, []), not_


def test_rows_without_a_parameter_per_picture_are_one_picture(launches):
    """2^30 rows, however they are cut into pictures."""
    calls = [norm(1 << 30, 64, picture=False), norm(1, 320, picture=False, N=1 << 30), norm(1 << 20, 5, picture=False, N=1 << 10),
             norm_back(1 << 30, 64, picture=False, sums=True), norm_back(1 << 15, 1283, picture=False, sums=True, N=1 << 15)]
    got = launches(calls)
    assert [rc for rc, _ in got] == [0] * len(calls)
    inside_limits(calls, got)


def test_launches_over_the_range_of_sizes(launches):
    sizes = [1, 2, 15, 17, 100, 513, 4097, 36864]
    calls = [linear(M, N, K_, epi) for M in sizes for N in (32, 96, 320, 2048, 10240) for K_ in (1, 129, 640, 8192) for epi in (0, 4)]
    calls += [norm(B, C, picture=pic, N=N) for B in (1, 3, 16) for N in (1, 7, 9216) for pic in (False, True)
              for C in (1, 7, 8, 64, 65, 512, 1024, 1025, 1280, 1536, 1537, 2048, 4096, 8192, 8193, 16384, 16385, 100000)]
    calls += [norm_back(B, C, picture=pic, sums=s, N=N) for B in (1, 16) for N in (1, 9216) for pic in (False, True) for s in (False, True)
              for C in (1, 8, 64, 512, 1024, 1025, 2048, 4096, 8192, 8193, 100000)]
    got = launches(calls)
    assert [(c, rc) for c, (rc, ls) in zip(calls, got) if rc or not ls] == []
    inside_limits(calls, got)
