// mxfp4.hip — 4-bit microscaled floating point (OCP MX v1.0, MXFP4): quantise, read back, and the product of two such matrices.
//
// A block of 32 consecutive values of a row is 2^e * q, q in e2m1: e = max(floor(log2 amax) - 2, -127), so amax * 2^-e lies in [4, 8)
// and is the only place where the largest code, 6, saturates.  v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 rows over
// 128 values: lane l holds row l % 16, values 32 (l / 16) .. + 31 (16 bytes of codes) and that block's scale byte -- the memory
// layout itself, no shuffle.  Its products are exact, the sums f32.
#include <type_traits>

#include "conv_common.h"
#include "elem.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// scale byte of a block from the bits of its largest magnitude (255: a NaN or an infinity in it)
__device__ __forceinline__ uint32_t block_scale(uint32_t amax_bits) {
    const int ex = (int)(amax_bits >> 23);           // biased exponent; 0 (zero, subnormal) lands on the lowest scale too
    return amax_bits >= 0x7f800000u ? 255u : (uint32_t)(ex > 2 ? ex - 2 : 0);
}
// largest magnitude of two pairs of 16-bit values, as pairs of magnitude bits (ordered as integers are)
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t pair) {
    const uint32_t lo = pair & 0xffffu, hi = pair >> 16;
    return __float_as_uint(a2f((a16_t)(lo > hi ? lo : hi)));
}
// eight values as codes, round half to even, magnitudes over 6 to 6; scale: the block's power of two
__device__ __forceinline__ uint32_t codes8(uint4 v, float scale) {
    uint32_t w = 0;
#ifdef ONEDC_ACT_F16
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v.x), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v.y), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v.z), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v.w), scale, 3);
#else
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v.x), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v.y), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v.z), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v.w), scale, 3);
#endif
    return w;
}
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}
// v_cvt_scalef32_* take the exponent field of the f32 scale; the field 0 is 2^-127 in a scale byte
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

// Eight consecutive values of a row, from k on; values from K on are 0.  VEC: whole aligned 16-byte pieces.
template <bool F32, bool VEC>
struct Eight {
    float f[8];
    uint4 h;
    __device__ __forceinline__ void load(const void *x, int64_t at, int left) {
        if (F32) {
            const float *src = (const float *)x + at;
            if (VEC) {
                const float4 a = left > 0 ? *(const float4 *)src : make_float4(0, 0, 0, 0), b = left > 0 ? *(const float4 *)(src + 4) : make_float4(0, 0, 0, 0);
                f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = j < left ? src[j] : 0.f;
        } else {
            const a16_t *src = (const a16_t *)x + at;
            if (VEC) {
                h = left > 0 ? *(const uint4 *)src : make_uint4(0, 0, 0, 0);
            } else {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = j < left ? src[j] : 0u;
                h = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
        }
    }
    __device__ __forceinline__ uint32_t amax_bits() const {
        if (F32) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
            return m;
        }
        constexpr uint32_t MAG = 0x7fff7fffu;
        return magnitude_bits(max_pair(max_pair(h.x & MAG, h.y & MAG), max_pair(h.z & MAG, h.w & MAG)));
    }
    __device__ __forceinline__ uint32_t codes(uint32_t s) const { return s == 255u ? 0u : F32 ? codes8(f, scale_of(s)) : codes8(h, scale_of(s)); }
};

template <int CTRL>
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
}

// Four neighbouring lanes hold a block, eight values each: a wave reads 1 KB (16-bit) in a row and writes 256 bytes of codes.  HBM bound.
// A workgroup takes QN consecutive groups of 256 pieces of eight values, the pieces of all rows counted through.
constexpr int QN = 4;
template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, int x_cs, int x_co, uint32_t *codes, uint8_t *scales, int64_t rows, int K,
                                                       int per, OnedcFastDiv div) {
    const int64_t first = (int64_t)blockIdx.x * (256 * QN);
    const int64_t row0 = first / per;
    const int rest = (int)(first - row0 * per) + threadIdx.x;
    const int64_t total = rows * per;
    Eight<F32, VEC> v[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int at = rest + i * 256, dr = div.div(at), k = (at - dr * per) * 8;
        v[i].load(x, (row0 + dr) * x_cs + x_co + k, first + threadIdx.x + i * 256 < total ? K - k : 0);
    }
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int64_t piece = first + threadIdx.x + i * 256;
        const uint32_t s = block_scale(quad_max<0x4e>(quad_max<0xb1>(v[i].amax_bits())));
        if (piece >= total) continue;
        codes[piece] = v[i].codes(s);
        if ((threadIdx.x & 3) == 0) scales[piece >> 2] = (uint8_t)s;
    }
}

template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint32_t *codes, const uint8_t *scales, void *y, int y_cs, int y_co, int64_t rows,
                                                         int K, int per, OnedcFastDiv div) {
    const int64_t first = (int64_t)blockIdx.x * (256 * QN);
    const int64_t row0 = first / per;
    const int rest = (int)(first - row0 * per) + threadIdx.x;
    const int64_t total = rows * per;
    uint32_t w[QN], s[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int64_t piece = first + threadIdx.x + i * 256;
        w[i] = piece < total ? codes[piece] : 0u;
        s[i] = piece < total ? scales[piece >> 2] : 0u;
    }
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int at = rest + i * 256, dr = div.div(at), k = (at - dr * per) * 8;
        if (first + threadIdx.x + i * 256 >= total || k >= K) continue;
        const float sc = scale_of(s[i]), nan = __uint_as_float(0x7fc00000u);
        f32x2_t q[4];
        q[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 0);
        q[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 1);
        q[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 2);
        q[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 3);
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = s[i] == 255u ? nan : q[j >> 1][j & 1];
        const int64_t to = (row0 + dr) * y_cs + y_co + k;
        if (F32) {
            float *dst = (float *)y + to;
            if (VEC) {
                *(float4 *)dst = make_float4(o[0], o[1], o[2], o[3]);
                *(float4 *)(dst + 4) = make_float4(o[4], o[5], o[6], o[7]);
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j < K) dst[j] = o[j];
        } else {
            a16_t *dst = (a16_t *)y + to;
            if (VEC) {
                *(uint4 *)dst = make_uint4(pack_a2(o[0], o[1]), pack_a2(o[2], o[3]), pack_a2(o[4], o[5]), pack_a2(o[6], o[7]));
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j < K) dst[j] = f2a(o[j]);
        }
    }
}

// J: which byte of the lane's scale words holds the scale of its 32 values
template <int J>
__device__ __forceinline__ f32x4 mfma_fp4(uint4 a, uint4 b, f32x4 c, uint32_t sa, uint32_t sb) {
    const i32x8 va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, J, (int)sa, J, (int)sb);
}

__device__ __forceinline__ float activation(const onedc_mxfp4_params &p, float v) {
    return p.epi == ONEDC_EPI_SILU ? silu_f(v) : p.epi == ONEDC_EPI_LEAKY ? leaky(v, p.slope) : v;
}
__device__ __forceinline__ float bias_of(const onedc_mxfp4_params &p, int n) { return p.bias && n < p.N ? p.bias[n] : 0.f; }

// eight outputs of a row, n on: residual, rounding, store.  whole: 16-byte accesses are allowed (sizes, strides and pointers)
__device__ __forceinline__ void store8(const onedc_mxfp4_params &p, int64_t m, int n, int out, const float (&v0)[8], bool whole) {
    float v[8];
    const int64_t ry = m * p.y_cs + p.y_co + n, rr = m * p.r_cs + p.r_co + n;
    if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v0[j];
        if (p.y_f32) {
            if (p.res) {
                const float4 a = *(const float4 *)((const float *)p.res + rr), b = *(const float4 *)((const float *)p.res + rr + 4);
                v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
            }
            *(float4 *)((float *)p.y + ry) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4 *)((float *)p.y + ry + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            if (p.res) {
                const uint4 r = *(const uint4 *)((const a16_t *)p.res + rr);
                v[0] += a2f_lo(r.x), v[1] += a2f_hi(r.x), v[2] += a2f_lo(r.y), v[3] += a2f_hi(r.y);
                v[4] += a2f_lo(r.z), v[5] += a2f_hi(r.z), v[6] += a2f_lo(r.w), v[7] += a2f_hi(r.w);
            }
            *(uint4 *)((a16_t *)p.y + ry) = make_uint4(pack_a2(v[0], v[1]), pack_a2(v[2], v[3]), pack_a2(v[4], v[5]), pack_a2(v[6], v[7]));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (n + j >= out) continue;
        float t = v0[j];
        if (p.y_f32) {
            if (p.res) t += ((const float *)p.res)[rr + j];
            ((float *)p.y)[ry + j] = t;
        } else {
            if (p.res) t += a2f(((const a16_t *)p.res)[rr + j]);
            ((a16_t *)p.y)[ry + j] = f2a(t);
        }
    }
}

// ---- few rows: the weights' bytes bound it -------------------------------------------------------------------------------------------
// A workgroup computes 32 weight rows x 16 FM activation rows; its eight waves take every eighth 128-value step of K straight from
// memory (each weight byte is read once, 64 bytes of 16 rows an instruction) and their sums are added through LDS in wave order.  Raw rows
// are quantised by the lane that multiplies them, once per workgroup: 70 instructions a step against 2 KB of weights.
constexpr int SKW = 8;
template <int FM, bool RAW, bool VEC>
__global__ __launch_bounds__(64 * SKW) void skinny_kernel(onedc_mxfp4_params p, int steps, int whole) {
    __shared__ __attribute__((aligned(16))) float red[SKW][FM][2][16][20];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kb = lane >> 4;
    const int nt = (p.N + 31) / 32;
    const int n0 = (int)(blockIdx.x % nt) * 32;
    const int64_t m0 = (int64_t)(blockIdx.x / nt) * (16 * FM);
    const int na = min(n0 + r, p.N - 1), nc = min(n0 + 16 + r, p.N - 1);
    const uint4 *wa = (const uint4 *)p.wc + (int64_t)na * steps * 4 + kb, *wb = (const uint4 *)p.wc + (int64_t)nc * steps * 4 + kb;
    const uint8_t *sa = (const uint8_t *)p.ws + (int64_t)na * steps * 4 + kb, *sb = (const uint8_t *)p.ws + (int64_t)nc * steps * 4 + kb;
    int64_t m[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) m[i] = m0 + i * 16 + r < p.M ? m0 + i * 16 + r : p.M - 1;
    f32x4 acc[FM][2];
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = FM == 1 ? 4 : 2;               // steps whose loads are in flight together
    for (int s0 = wave; s0 < steps; s0 += SKW * U) {
        uint4 a[U], c[U], x[FM][U];
        uint32_t xa[U], xc[U], sx[FM][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u * SKW, steps - 1);
            a[u] = wa[s * 4], c[u] = wb[s * 4];
            xa[u] = sa[s * 4], xc[u] = sb[s * 4];
            if (!RAW)
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    x[i][u] = ((const uint4 *)p.xc)[(m[i] * steps + s) * 4 + kb];
                    sx[i][u] = ((const uint8_t *)p.xs)[(m[i] * steps + s) * 4 + kb];
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * SKW;
            if (s >= steps) break;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (RAW) {
                    const int k0 = s * 128 + kb * 32;
                    const int64_t at = m[i] * p.xr_cs + p.xr_co + k0;
                    uint32_t top = 0;
                    if (p.xr_f32) {
                        Eight<true, VEC> v[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j].load(p.xr, at + j * 8, p.K - k0 - j * 8), top = max(top, v[j].amax_bits());
                        sx[i][u] = block_scale(top);
                        x[i][u] = make_uint4(v[0].codes(sx[i][u]), v[1].codes(sx[i][u]), v[2].codes(sx[i][u]), v[3].codes(sx[i][u]));
                    } else {
                        Eight<false, VEC> v[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j].load(p.xr, at + j * 8, p.K - k0 - j * 8), top = max(top, v[j].amax_bits());
                        sx[i][u] = block_scale(top);
                        x[i][u] = make_uint4(v[0].codes(sx[i][u]), v[1].codes(sx[i][u]), v[2].codes(sx[i][u]), v[3].codes(sx[i][u]));
                    }
                }
                acc[i][0] = mfma_fp4<0>(a[u], x[i][u], acc[i][0], xa[u], sx[i][u]);
                acc[i][1] = mfma_fp4<0>(c[u], x[i][u], acc[i][1], xc[u], sx[i][u]);
            }
        }
    }
    // lane: activation row r, weight rows 4 kb + e of each half
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) *(f32x4 *)&red[wave][i][h][r][kb * 4] = acc[i][h];
    __syncthreads();
    const bool glu = p.epi == ONEDC_EPI_GEGLU;
    const int out = glu ? p.N / 2 : p.N, pieces = glu ? 2 : 4;             // eight outputs each
    for (int t = threadIdx.x; t < 16 * FM * pieces; t += 64 * SKW) {
        const int row = t / pieces, piece = t - row * pieces;
        if (m0 + row >= p.M) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int n = piece * 8 + j;
            float a = 0.f, g = 0.f;
#pragma unroll
            for (int w = 0; w < SKW; ++w) a += red[w][row >> 4][n >> 4][row & 15][n & 15];
            if (glu) {
#pragma unroll
                for (int w = 0; w < SKW; ++w) g += red[w][row >> 4][1][row & 15][n];
                v[j] = (p.alpha * a + bias_of(p, n0 + n)) * gelu_f(p.alpha * g + bias_of(p, n0 + 16 + n));
            } else {
                v[j] = activation(p, p.alpha * a + bias_of(p, n0 + n));
            }
        }
        const int n = (glu ? n0 / 2 : n0) + piece * 8;
        if (n < out) store8(p, m0 + row, n, out, v, whole && n + 8 <= out);
    }
}

// ---- tiles: the matrix cores and what feeds them bound it ---------------------------------------------------------------------------------
// A workgroup of 2 x 2 waves computes 32 FN weight rows x 32 FM activation rows.  A stage is one 128-value step of both operands, 64 bytes
// of codes a row, LDS-DMA'd into a ring of NST; the 16-byte chunks of a row are placed at chunk ^ (row / 2 % 4), which puts the eight
// rows that a fragment read touches together on different banks.  Scales come four steps (16 bytes a row) at a time, one such group ahead;
// two byte permutes collect a lane's four scales into the word that the matrix instruction picks from.
// The DMA is written as instructions (it has no destination register): behind the builtin the compiler drains every DMA in flight
// before each LDS read.
#define MX_VMCNT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")

typedef __attribute__((ext_vector_type(4))) int i32x4;
__device__ __forceinline__ i32x4 raw_rsrc(const void *base, int64_t bytes) {
    const uint64_t a = (uint64_t)base;
    return i32x4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), (int)(uint32_t)(bytes < 0xfffff000ll ? bytes : 0xfffff000ll), 0x00020000};
}
// 16 bytes a lane from base + voff + soff to lds + 16 lane; a lane whose voff lies behind the descriptor's end writes zeros
// (m0 is reserved: nothing else in these kernels reads it)
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned voff, unsigned soff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory");
}

template <int FN, int FM, int NST, int OCC>
__global__ __launch_bounds__(256, OCC) void tile_kernel(onedc_mxfp4_params p, int steps, int tiles_n, int tiles_m, int whole) {
    constexpr int TN = 32 * FN, TM = 32 * FM, STAGE = (TN + TM) * 64, WN = TN / 64, WM = TM / 64, NI = WN + WM;
    constexpr int GROUP = (TN + TM) * 16, NSC = (TN + TM + 255) / 256, RING = NST * STAGE;     // scales of four steps, behind the ring
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, kb = lane >> 4;
    const int wn = wave >> 1, wm = wave & 1;
    // tiles that run at the same time on one XCD share operands: eight rows of tiles deep, then along n
    const int logical = xcd_logical_tile(blockIdx.x, tiles_n * tiles_m);
    const int band = 8 * tiles_n, b0 = logical / band, in = logical - b0 * band, deep = min(8, tiles_m - b0 * 8);
    const int tn = in / deep, tm = b0 * 8 + in - tn * deep;
    const int n0 = tn * TN;
    const int64_t m0 = (int64_t)tm * TM;

    // codes: rows past the last read zeros (their byte offset lies behind the descriptor's end)
    const unsigned row_bytes = (unsigned)steps * 64;
    const i32x4 w_rsrc = raw_rsrc((const char *)p.wc + (int64_t)n0 * row_bytes, (int64_t)(p.N - n0) * row_bytes);
    const i32x4 x_rsrc = raw_rsrc((const char *)p.xc + m0 * row_bytes, (p.M - m0) * (int64_t)row_bytes);
    const int srow = wave * 16 + (lane >> 2);
    const unsigned schunk = ((lane & 3) ^ ((lane >> 3) & 3)) << 4;
    const unsigned voff = (unsigned)srow * row_bytes + schunk;
    unsigned wv[WN], xv[WM];
#pragma unroll
    for (int q = 0; q < WN; ++q) wv[q] = voff + (unsigned)(q * 64) * row_bytes;
#pragma unroll
    for (int q = 0; q < WM; ++q) xv[q] = voff + (unsigned)(q * 64) * row_bytes;
    auto stage = [&](int s, int slot) {
        const unsigned dst = lds0 + slot * STAGE + wave * 1024;
#pragma unroll
        for (int q = 0; q < WN; ++q) dma16(w_rsrc, wv[q], (unsigned)s * 64, dst + q * 4096);
#pragma unroll
        for (int q = 0; q < WM; ++q) dma16(x_rsrc, xv[q], (unsigned)s * 64, dst + TN * 64 + q * 4096);
    };

    // scales: four bytes a step and row.  A group of a last row may end behind the matrix: such a read moves back by `over`
    const unsigned srb = (unsigned)steps * 4;
    const int64_t sw_all = (int64_t)(p.N - n0) * srb - 16, sx_all = (p.M - m0) * (int64_t)srb - 16;
    const int sw_max = (int)(sw_all < 0x7ffffff0ll ? sw_all : 0x7ffffff0ll), sx_max = (int)(sx_all < 0x7ffffff0ll ? sx_all : 0x7ffffff0ll);
    // (the descriptors begin at the matrix, so that moving back from a tile's first row stays inside)
    const int64_t sw_base = (int64_t)n0 * srb, sx_base = m0 * (int64_t)srb;
    const int64_t sw_lo = sw_base < 16 ? sw_base : 16, sx_lo = sx_base < 16 ? sx_base : 16;
    const i32x4 sw_rsrc = raw_rsrc((const char *)p.ws + sw_base - sw_lo, sw_all + 16 + sw_lo);
    const i32x4 sx_rsrc = raw_rsrc((const char *)p.xs + sx_base - sx_lo, sx_all + 16 + sx_lo);
    auto stage_scales = [&](int g) {
#pragma unroll
        for (int q = 0; q < NSC; ++q) {
            const int first = min(q * 256 + wave * 64, TN + TM - 64);           // (a wave without rows of its own repeats the last ones)
            const bool w = first < TN;                                          // wave-uniform
            const int row = (w ? first : first - TN) + lane;
            const int off = min(row * (int)srb + g * 16, w ? sw_max : sx_max) + (int)(w ? sw_lo : sx_lo);
            dma16(w ? sw_rsrc : sx_rsrc, (unsigned)off, 0, lds0 + RING + (g & 1) * GROUP + first * 16);
        }
    };
    uint32_t sc[FN + FM];
    const uint32_t pick = (uint32_t)kb * 0x0101u + 0x0400u;
    auto take_scales = [&](int g) {
        const char *at = smem + RING + (g & 1) * GROUP;
#pragma unroll
        for (int i = 0; i < FN + FM; ++i) {
            const int row = i < FN ? wn * 16 * FN + i * 16 + r : wm * 16 * FM + (i - FN) * 16 + r;
            const uint4 raw = *(const uint4 *)(at + ((i < FN ? 0 : TN) + row) * 16);
            const uint32_t lo = __builtin_amdgcn_perm(raw.y, raw.x, pick), hi = __builtin_amdgcn_perm(raw.w, raw.z, pick);
            const int over = max(row * (int)srb + g * 16 - (i < FN ? sw_max : sx_max), 0);
            sc[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u) >> ((over * 2) & 31);
        }
    };

    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int frag = r * 64 + ((kb ^ ((r >> 1) & 3)) << 4);

    const int groups = (steps + 3) >> 2;
    stage_scales(0);
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
        if (i < steps) stage(i, i);
    int slot = 0, fill = NST - 1;
    auto step = [&](auto jc, int s, bool more) {
        constexpr int J = decltype(jc)::value;
        // this step's codes (and a new group's scales) have landed: what was issued behind them are the next NST - 2 steps' and, up to the
        // step that was issued together with them, the next group's scales
        if (s + NST - 2 < steps) {
            if (J > 0 && J < NST && more) MX_VMCNT((NST - 2) * NI + NSC);
            else MX_VMCNT((NST - 2) * NI);
        } else {
            MX_VMCNT(0);
        }
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (s + NST - 1 < steps) stage(s + NST - 1, fill);       // into the slot that every wave left behind at this barrier
        if (J == 0) {
            if (more) stage_scales((s >> 2) + 1);
            take_scales(s >> 2);
        }
        const char *a = smem + slot * STAGE + wn * FN * 1024 + frag, *b = smem + slot * STAGE + TN * 64 + wm * FM * 1024 + frag;
        uint4 fa[FN], fb[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j) fb[j] = *(const uint4 *)(b + j * 1024);
#pragma unroll
        for (int i = 0; i < FN; ++i) fa[i] = *(const uint4 *)(a + i * 1024);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = mfma_fp4<J>(fa[i], fb[j], acc[i][j], sc[i], sc[FN + j]);
        fill = slot;
        slot = slot + 1 == NST ? 0 : slot + 1;
    };
    for (int g = 0; g < groups; ++g) {
        const bool more = g + 1 < groups;
        const int s = g * 4;
        step(std::integral_constant<int, 0>(), s, more);
        if (s + 1 < steps) step(std::integral_constant<int, 1>(), s + 1, more);
        if (s + 2 < steps) step(std::integral_constant<int, 2>(), s + 2, more);
        if (s + 3 < steps) step(std::integral_constant<int, 3>(), s + 3, more);
    }
    __syncthreads();                                 // the ring is free: the waves' own scratch from here

    // epilogue: 16 activation rows at a time through LDS, so that a row's outputs leave as whole lines
    constexpr int PITCH = FN * 16 + 4;
    float *my = (float *)smem + wave * 16 * PITCH;
    const bool glu = p.epi == ONEDC_EPI_GEGLU;
    const int out = glu ? p.N / 2 : p.N, nw = n0 + wn * FN * 16, no = glu ? nw / 2 : nw;
    f32x4 bias[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[i][e] = bias_of(p, nw + i * 16 + kb * 4 + e);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t mt = m0 + (wm * FM + j) * 16;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if (glu && (i & 1)) continue;
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float t = p.alpha * acc[i][j][e] + bias[i][e];
                if (glu) v[e] = t * gelu_f(p.alpha * acc[i | 1][j][e] + bias[i | 1][e]);
                else v[e] = activation(p, t);
            }
            *(f32x4 *)(my + r * PITCH + (glu ? i / 2 : i) * 16 + kb * 4) = v;
        }
        const int pieces = glu ? FN : 2 * FN;                             // eight outputs each, per row
        for (int t = lane; t < 16 * pieces; t += 64) {
            const int row = t / pieces, n = no + (t - row * pieces) * 8;
            const f32x4 lo = *(const f32x4 *)(my + row * PITCH + n - no), hi = *(const f32x4 *)(my + row * PITCH + n - no + 4);
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (mt + row < p.M && n < out) store8(p, mt + row, n, out, v, whole && n + 8 <= out);
        }
    }
}

bool held_ok(const void *codes, const void *scales) { return ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0; }
// whole 16-byte pieces of eight (16-bit) or four (f32) values at every row
bool whole_ok(const void *t, int cs, int co, bool f32) { return ((uintptr_t)t & 15) == 0 && ((cs | co) & (f32 ? 3 : 7)) == 0; }

template <bool F32, bool VEC>
int launch_quantize(const void *x, int x_cs, int x_co, void *codes, void *scales, int64_t rows, int K, void *stream) {
    const int per = (K + 127) / 128 * 16;
    hipLaunchKernelGGL((quantize_kernel<F32, VEC>), dim3((unsigned)((rows * per + 256 * QN - 1) / (256 * QN))), dim3(256), 0, as_stream(stream), x,
                       x_cs, x_co, (uint32_t *)codes, (uint8_t *)scales, rows, K, per, OnedcFastDiv(per));
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <bool F32, bool VEC>
int launch_dequantize(const void *codes, const void *scales, void *y, int y_cs, int y_co, int64_t rows, int K, void *stream) {
    const int per = (K + 127) / 128 * 16;
    hipLaunchKernelGGL((dequantize_kernel<F32, VEC>), dim3((unsigned)((rows * per + 256 * QN - 1) / (256 * QN))), dim3(256), 0, as_stream(stream),
                       (const uint32_t *)codes, (const uint8_t *)scales, y, y_cs, y_co, rows, K, per, OnedcFastDiv(per));
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <int FM, bool RAW, bool VEC>
int launch_skinny(const onedc_mxfp4_params *p, int steps, int whole, void *stream) {
    const int64_t wgs = (int64_t)((p->N + 31) / 32) * ((p->M + 16 * FM - 1) / (16 * FM));
    hipLaunchKernelGGL((skinny_kernel<FM, RAW, VEC>), dim3((unsigned)wgs), dim3(64 * SKW), 0, as_stream(stream), *p, steps, whole);
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <int FN, int FM, int NST, int OCC>
int launch_tiles(const onedc_mxfp4_params *p, int steps, int whole, void *stream) {
    constexpr int ring = 32 * (FN + FM) * (NST * 64 + 2 * 16), scratch = 4 * 16 * (FN * 16 + 4) * 4, lds = ring > scratch ? ring : scratch;
    static OnedcLdsAttrOnce once;
    once.ensure({{(const void *)tile_kernel<FN, FM, NST, OCC>, lds}});
    const int64_t tn = (p->N + 32 * FN - 1) / (32 * FN), tm = (p->M + 32 * FM - 1) / (32 * FM);
    if (tn * tm > 0x7fffffff) return -2;
    hipLaunchKernelGGL((tile_kernel<FN, FM, NST, OCC>), dim3((unsigned)(tn * tm)), dim3(256), lds, as_stream(stream), *p, steps, (int)tn, (int)tm, whole);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" {

int onedc_mxfp4_quantize(const void *x, int x_f32, int x_cs, int x_co, void *codes, void *scales, int64_t rows, int K, void *stream) {
    if (!x || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > ONEDC_MXFP4_MAX_K || x_co < 0 || x_cs - K < x_co || !held_ok(codes, scales) ||
        rows * ((K + 127) / 128) > (1ll << 36))
        return -2;
    if (!rows) return 0;
    const bool vec = K % 8 == 0 && whole_ok(x, x_cs, x_co, x_f32);
    if (x_f32) return vec ? launch_quantize<true, true>(x, x_cs, x_co, codes, scales, rows, K, stream) : launch_quantize<true, false>(x, x_cs, x_co, codes, scales, rows, K, stream);
    return vec ? launch_quantize<false, true>(x, x_cs, x_co, codes, scales, rows, K, stream) : launch_quantize<false, false>(x, x_cs, x_co, codes, scales, rows, K, stream);
}

int onedc_mxfp4_dequantize(const void *codes, const void *scales, void *y, int y_f32, int y_cs, int y_co, int64_t rows, int K, void *stream) {
    if (!y || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > ONEDC_MXFP4_MAX_K || y_co < 0 || y_cs - K < y_co || !held_ok(codes, scales) ||
        rows * ((K + 127) / 128) > (1ll << 36))
        return -2;
    if (!rows) return 0;
    const bool vec = K % 8 == 0 && whole_ok(y, y_cs, y_co, y_f32);
    if (y_f32) return vec ? launch_dequantize<true, true>(codes, scales, y, y_cs, y_co, rows, K, stream) : launch_dequantize<true, false>(codes, scales, y, y_cs, y_co, rows, K, stream);
    return vec ? launch_dequantize<false, true>(codes, scales, y, y_cs, y_co, rows, K, stream) : launch_dequantize<false, false>(codes, scales, y, y_cs, y_co, rows, K, stream);
}

int onedc_mxfp4_linear(const onedc_mxfp4_params *p, void *stream) {
    if (!p || !p->wc || !p->ws || !p->y || (!p->xr && (!p->xc || !p->xs))) return -1;
    if (p->epi != ONEDC_EPI_LINEAR && p->epi != ONEDC_EPI_LEAKY && p->epi != ONEDC_EPI_SILU && p->epi != ONEDC_EPI_GEGLU) return -3;
    if (p->epi == ONEDC_EPI_GEGLU && p->N % 32) return -3;
    const int out = p->epi == ONEDC_EPI_GEGLU ? p->N / 2 : p->N;
    if (p->M < 0 || p->M > 0x7fffffff || p->N < 1 || p->N > (1 << 24) || p->K < 1 || p->K > ONEDC_MXFP4_MAX_K || p->y_co < 0 ||
        p->y_cs - out < p->y_co || (p->res && (p->r_co < 0 || p->r_cs - out < p->r_co)) || !held_ok(p->wc, p->ws))
        return -2;
    if (p->xc ? !held_ok(p->xc, p->xs) : (p->xr_co < 0 || p->xr_cs - p->K < p->xr_co)) return -2;
    if (!p->xc && p->M > ONEDC_MXFP4_ROWS_RAW) return -4;
    if (!p->M) return 0;
    const int steps = (p->K + 127) / 128;
    const int whole = whole_ok(p->y, p->y_cs, p->y_co, p->y_f32) && (!p->res || whole_ok(p->res, p->r_cs, p->r_co, p->y_f32));
    if (((int64_t)(p->N + 31) / 32) * ((p->M + 15) / 16) > 0x7fffffff) return -2;
    if (!p->xc) {
        if (p->K % 8 == 0 && whole_ok(p->xr, p->xr_cs, p->xr_co, p->xr_f32)) return launch_skinny<1, true, true>(p, steps, whole, stream);
        return launch_skinny<1, true, false>(p, steps, whole, stream);
    }
    if (p->M <= 16) return launch_skinny<1, false, true>(p, steps, whole, stream);
    if (p->M <= 32 || (int64_t)p->N * steps < 4) return launch_skinny<2, false, true>(p, steps, whole, stream);
    const int64_t big = (int64_t)((p->N + 127) / 128) * ((p->M + 127) / 128);
    if (big <= 64) return launch_skinny<4, false, true>(p, steps, whole, stream);
    if (big <= 512) return launch_tiles<4, 4, 3, 2>(p, steps, whole, stream);
    return launch_tiles<4, 8, 3, 2>(p, steps, whole, stream);
}

}  // extern "C"
