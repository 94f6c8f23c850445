// mxfp4.hip — 4-bit microscaled floating point (OCP MX v1.0, MXFP4): quantise, read back, and the product of two such matrices.
//
// A block of 32 consecutive values of a row is 2^e * q, q in e2m1: e = max(floor(log2 amax) - 2, -127), so amax * 2^-e lies in [4, 8)
// and is the only place where the largest code, 6, saturates.  The scaled matrix instructions take 32 values of a row in a lane -- 16 bytes of codes
// and that block's scale byte -- which is the memory layout itself, no shuffle: 16x16x128 (lane l: row l % 16, values 32 (l / 16) on)
// for few rows, 32x32x64 (row l % 32, values 32 (l / 32) on) for tiles.  Products are exact, sums f32.
#include <type_traits>

#include "apart.h"
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

// Four neighbouring lanes hold a block, eight values each: a wave reads 1 KB (16-bit) in a row and writes 256 bytes of codes.  HBM bound: 16384 x 8192
// bf16 to codes 59 us, 5.7 TB/s, and back 60 us, 5.6 TB/s (f32 109 us, 5.6 TB/s; back 155 us, 3.9 TB/s: 32 bytes a lane to store).
// Rows that do not begin at whole 16 bytes are read and written as single values: 16384 x 8191 133 us, back 185 us.
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

// the same over 32 x 32 rows and 64 values: lane l holds row l % 32, values 32 (l / 32) .. + 31
typedef __attribute__((ext_vector_type(16))) float f32x16;
template <int J>
__device__ __forceinline__ f32x16 mfma_fp4_32(uint4 a, uint4 b, f32x16 c, uint32_t sa, uint32_t sb) {
    const i32x8 va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, J, (int)sa, J, (int)sb);
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
// A workgroup computes 32 weight rows x 16 activation rows over rounds of 64 steps of 128 values: each of its sixteen waves takes four
// consecutive steps of a round straight from memory, 256 bytes of every weight row and 16 bytes of its scales, all in flight at once (steps dealt
// out in turn instead would send all waves to the same memory channels where a row is a power of two long: 8192 x 8192 against one row 11.3 us
// that way).  The waves' sums are added through LDS in wave order.  Raw rows are quantised by the workgroup together, under the weights' loads, into LDS.
// 8192 x 8192 against one row of codes 9.3 us (3.8 TB/s of weights), a raw row 9.7 us, sixteen 10.7 and 14.1 us (every workgroup quantises the rows
// for itself).
constexpr int SKW = 16, SKU = 4, ROUND = SKW * SKU;                       // steps of a round
constexpr int XPITCH = ROUND * 64 + 16, SPITCH = ROUND * 4 + 16;          // bytes of a row's codes and scales in LDS, off the banks' period

// the scales of four steps of a row, a byte each for this lane's block (kb): from s on, the row ends at `steps`
__device__ __forceinline__ uint32_t four_scales(const uint8_t *all, int64_t row, int64_t rows, int s, int steps, int kb) {
    const uint32_t pick = (uint32_t)kb * 0x0101u + 0x0400u;
    uint4 v = make_uint4(0, 0, 0, 0);
    int over = 0;
    if (steps >= 4) {                                // 16 bytes; moved back where they would end behind the matrix
        const int64_t at = (row * steps + s) * 4, last = rows * steps * 4 - 16;
        over = at > last ? (int)(at - last) : 0;
        __builtin_memcpy(&v, all + at - over, 16);
    } else {
        const uint32_t *w = (const uint32_t *)all + row * steps + s;
        v.x = w[0];
        if (s + 1 < steps) v.y = w[1];
        if (s + 2 < steps) v.z = w[2];
    }
    const uint32_t lo = __builtin_amdgcn_perm(v.y, v.x, pick), hi = __builtin_amdgcn_perm(v.w, v.z, pick);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u) >> ((over * 2) & 31);
}

// RAW 0: codes, 1: 16-bit rows, 2: f32 rows
template <int RAW, bool VEC>
__global__ __launch_bounds__(64 * SKW) void skinny_kernel(onedc_mxfp4_params p, int steps, int whole) {
    extern __shared__ __attribute__((aligned(16))) char smem[];              // raw rows' codes, then their scales; the sums over them
    typedef float Red[2][16][20];
    Red *const red = (Red *)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, kb = lane >> 4;
    const int nt = (p.N + 31) / 32;
    const int n0 = (int)(blockIdx.x % nt) * 32;
    const int64_t m0 = (int64_t)(blockIdx.x / nt) * 16, m = m0 + r < p.M ? m0 + r : p.M - 1;
    const int rows = (int)(p.M - m0 < 16 ? p.M - m0 : 16);
    const int na = min(n0 + r, p.N - 1), nc = min(n0 + 16 + r, p.N - 1);
    const uint4 *wa = (const uint4 *)p.wc + (int64_t)na * steps * 4 + kb, *wb = (const uint4 *)p.wc + (int64_t)nc * steps * 4 + kb;
    char *const xscale = smem + 16 * XPITCH;
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int first = 0; first < steps; first += ROUND) {
        const int s = first + wave * SKU;
        uint4 a[SKU], c[SKU], x[SKU];
        uint32_t xa = 0, xc = 0, sx = 0;
        if (s < steps) {
#pragma unroll
            for (int u = 0; u < SKU; ++u) {
                const int su = min(s + u, steps - 1);
                a[u] = wa[su * 4], c[u] = wb[su * 4];
                if (!RAW) x[u] = ((const uint4 *)p.xc)[(m * steps + su) * 4 + kb];
            }
            xa = four_scales((const uint8_t *)p.ws, na, p.N, s, steps, kb);
            xc = four_scales((const uint8_t *)p.ws, nc, p.N, s, steps, kb);
            if (!RAW) sx = four_scales((const uint8_t *)p.xs, m, p.M, s, steps, kb);
        }
        if (RAW) {
            // a row a pass: 1024 threads, eight values each, four neighbours a block
            const int k = first * 128 + threadIdx.x * 8;
            if (first) __syncthreads();              // (the last round's codes have been multiplied)
            for (int i = 0; i < rows; i += 4) {
                Eight<RAW == 2, VEC> v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q].load(p.xr, (m0 + i + q) * p.xr_cs + p.xr_co + k, i + q < rows ? p.K - k : 0);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t sc = block_scale(quad_max<0x4e>(quad_max<0xb1>(v[q].amax_bits())));
                    if (i + q >= rows) continue;     // (uniform)
                    *(uint32_t *)(smem + (i + q) * XPITCH + threadIdx.x * 4) = v[q].codes(sc);
                    if ((threadIdx.x & 3) == 0) xscale[(i + q) * SPITCH + (threadIdx.x >> 2)] = (char)sc;
                }
            }
            __syncthreads();
            if (s < steps) {
                const int row = min(r, rows - 1);
#pragma unroll
                for (int u = 0; u < SKU; ++u) x[u] = *(const uint4 *)(smem + row * XPITCH + (wave * SKU + u) * 64 + kb * 16);
                const uint4 v = *(const uint4 *)(xscale + row * SPITCH + wave * SKU * 4);
                const uint32_t pick = (uint32_t)kb * 0x0101u + 0x0400u;
                sx = __builtin_amdgcn_perm(__builtin_amdgcn_perm(v.w, v.z, pick), __builtin_amdgcn_perm(v.y, v.x, pick), 0x05040100u);
            }
        }
        if (s >= steps) continue;                    // (wave-uniform, like the next)
        acc[0] = mfma_fp4<0>(a[0], x[0], acc[0], xa, sx), acc[1] = mfma_fp4<0>(c[0], x[0], acc[1], xc, sx);
        if (s + 1 < steps) acc[0] = mfma_fp4<1>(a[1], x[1], acc[0], xa, sx), acc[1] = mfma_fp4<1>(c[1], x[1], acc[1], xc, sx);
        if (s + 2 < steps) acc[0] = mfma_fp4<2>(a[2], x[2], acc[0], xa, sx), acc[1] = mfma_fp4<2>(c[2], x[2], acc[1], xc, sx);
        if (s + 3 < steps) acc[0] = mfma_fp4<3>(a[3], x[3], acc[0], xa, sx), acc[1] = mfma_fp4<3>(c[3], x[3], acc[1], xc, sx);
    }
    if (RAW) __syncthreads();
    // lane: activation row r, weight rows 4 kb + e of each half
    *(f32x4 *)&red[wave][0][r][kb * 4] = acc[0];
    *(f32x4 *)&red[wave][1][r][kb * 4] = acc[1];
    __syncthreads();
    const bool glu = p.epi == ONEDC_EPI_GEGLU;
    const int out = glu ? p.N / 2 : p.N, pieces = glu ? 2 : 4;             // eight outputs each
    // first one sum a thread (512 of them), then the row's pieces
    float total = 0.f;
    const int tr = (threadIdx.x >> 5) & 15, tn = threadIdx.x & 31;
    if (threadIdx.x < 512) {
#pragma unroll
        for (int w = 0; w < SKW; ++w) total += red[w][tn >> 4][tr][tn & 15];
        total = p.alpha * total + bias_of(p, n0 + tn);
    }
    __syncthreads();
    float (*const row32)[36] = (float (*)[36])smem;
    if (threadIdx.x < 512) row32[tr][tn] = total;
    __syncthreads();
    const int t = threadIdx.x, row = t / pieces, c = (t - row * pieces) * 8, n = (glu ? n0 / 2 : n0) + c;
    if (t >= 16 * pieces || m0 + row >= p.M || n >= out) return;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = glu ? row32[row][c + j] * gelu_f(row32[row][16 + c + j]) : activation(p, row32[row][c + j]);
    store8(p, m0 + row, n, out, v, whole && n + 8 <= out);
}

// ---- tiles: the matrix cores and what feeds them bound it ---------------------------------------------------------------------------------
// A workgroup of WN x WM waves computes 32 WN FN weight rows x 32 WM FM activation rows.  A stage is two steps of 128 values of both operands,
// LDS-DMA'd into a ring of NST: rows of 128 bytes whose 16-byte chunks are permuted so that the rows that a fragment read touches
// together lie on different banks.  Scales come eight steps (32 bytes a row) at a time; byte permutes collect a lane's scales into the
// words that the matrix instruction picks from.
// The DMA is written as instructions (it has no destination register): behind the builtin the compiler drains every DMA in flight
// before each LDS read.
// 32x32x64 in place of 16x16x128: 6.4 against 5.2 - 5.9 PFLOP/s from registers on random codes, where power bounds it (9.7 on zeros).
// 16384 x 8192 x 8192, 256 x 256: 544 - 572 us, 3.8 - 4.0 PFLOP/s.  Without the DMA it takes 465, without the LDS reads 524, without both
// 373, without the stores 507, the products alone 337: the feeding and the power limit bound it together; the matrix pipe is busy 0.44 of the
// time, and of the LDS reads' cycles 0.48 are conflicts.  Stages of one step in rings of three and four, 2 x 4 waves, other spacings of the DMA and
// outputs stored from registers (605 us) gained nothing.  4096^3 40 us, 3.4 PFLOP/s; 8655 x 10240 x 1280 gated 103 - 115 us, 2.0 - 2.2 PFLOP/s: ten
// steps a tile, its GELU costs as much as its products.
#define MX_VMCNT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")

typedef __attribute__((ext_vector_type(4))) int i32x4;
// (2 GB at most: a tile's own rows span far less, and offsets from 0xffff0000 on are behind every end)
__device__ __forceinline__ i32x4 raw_rsrc(const void *base, int64_t bytes) {
    const uint64_t a = (uint64_t)base;
    return i32x4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), (int)(bytes < 0x7ffffff0ll ? bytes : 0x7ffffff0ll), 0x00020000};
}
// 16 bytes a lane from base + voff + soff to lds + 16 lane; a lane whose voff lies behind the descriptor's end writes zeros
// (m0 is reserved: nothing else in these kernels reads it.  Five wait states: one for m0, five for a scalar operand that a vector instruction may
// have written just before.  No memory clobber: LDS reads may pass it, the waits and barriers order what has to be.)
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned voff, unsigned soff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff));
}

constexpr int KS = 2, ROW = 64 * KS;               // steps of a stage, bytes of its rows

// WN x WM waves of FN x FM blocks of 32 x 32; KG such teams share the tile, each with a ring of its own and a part of K, and the first adds their
// sums in order
template <int WN, int WM, int FN, int FM, int NST, int OCC, int KG>
__global__ __launch_bounds__(64 * WN * WM * KG, OCC) void tile_kernel(onedc_mxfp4_params p, int steps, int tiles_n, int tiles_m, int whole) {
    constexpr int NW = WN * WM, TN = 32 * WN * FN, TM = 32 * WM * FM, STAGE = (TN + TM) * ROW;
    constexpr int RI = 1024 / ROW;                   // rows of a DMA instruction
    constexpr int IN = TN / RI / NW, IM = TM / RI / NW, NI = IN + IM;
    constexpr int GROUP = (TN + TM) * 32, NSC = ((TN + TM) / 32 + NW - 1) / NW, RING = NST * STAGE;     // scales of eight steps, behind the ring
    constexpr int GS = 8 / KS;                       // stages of a group of scales
    static_assert(TN % (RI * NW) == 0 && TM % (RI * NW) == 0, "whole DMA instructions a wave");
    extern __shared__ __attribute__((aligned(16))) char all_smem[];
    const int lane = threadIdx.x & 63, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, kb = lane >> 5;
    const int team = KG > 1 ? any_wave / NW : 0, wave = any_wave - team * NW;
    char *const smem = all_smem + team * (RING + GROUP);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
    const int wn = wave / WM, wm = wave - wn * WM;
    // tiles that run at the same time on one XCD share operands: eight rows of tiles deep, then along n
    const int logical = xcd_logical_tile(blockIdx.x, tiles_n * tiles_m);
    const int band = 8 * tiles_n, b0 = logical / band, in = logical - b0 * band, deep = min(8, tiles_m - b0 * 8);
    const int tn = in / deep, tm = b0 * 8 + in - tn * deep;
    const int n0 = tn * TN;
    const int64_t m0 = (int64_t)tm * TM;

    // codes: rows past the last read zeros (their byte offset lies behind the descriptor's end), and so does the second half of a last
    // stage that ends with an odd step
    const unsigned row_bytes = (unsigned)steps * 64;
    const i32x4 w_rsrc = raw_rsrc((const char *)p.wc + (int64_t)n0 * row_bytes, (int64_t)(p.N - n0) * row_bytes);
    const i32x4 x_rsrc = raw_rsrc((const char *)p.xc + m0 * row_bytes, (p.M - m0) * (int64_t)row_bytes);
    const int srow = wave * RI + (lane >> 3), schunk = (lane & 7) ^ (srow & 7);
    const unsigned voff = (unsigned)srow * row_bytes + (unsigned)schunk * 16;
    unsigned wv[IN], xv[IM];
#pragma unroll
    for (int q = 0; q < IN; ++q) wv[q] = voff + (unsigned)(q * RI * NW) * row_bytes;
#pragma unroll
    for (int q = 0; q < IM; ++q) xv[q] = voff + (unsigned)(q * RI * NW) * row_bytes;
    // Instruction d of a stage's NI.  A stage behind the last, and the second half of a last one that ends with an odd step, write zeros: so
    // every stage issues the same number, and the products need no branch.
    auto stage_one = [&](int d, int t, int slot) {
        const unsigned dst = lds0 + slot * STAGE + wave * 1024;
        const unsigned behind = t * KS + (schunk >> 2) >= steps ? 0xffff0000u : 0u;
        const unsigned soff = t * KS < steps ? (unsigned)t * ROW : 0u;           // (never past the descriptor's end: it is taken off that)
        if (d < IN) dma16(w_rsrc, wv[d < IN ? d : 0] | behind, soff, dst + d * NW * 1024);
        else dma16(x_rsrc, xv[d < IN ? 0 : d - IN] | behind, soff, dst + TN * ROW + (d - IN) * NW * 1024);
    };
    auto stage = [&](int t, int slot) {
#pragma unroll
        for (int d = 0; d < NI; ++d) stage_one(d, t, slot);
    };

    // scales: four bytes a step and row.  What would end behind the matrix (a last row's last group) moves back by `over` bytes
    const int srb = steps * 4;
    const int64_t sw_all = (int64_t)(p.N - n0) * srb - 16, sx_all = (p.M - m0) * (int64_t)srb - 16;
    const int sw_max = (int)(sw_all < 0x7ffffff0ll ? sw_all : 0x7ffffff0ll), sx_max = (int)(sx_all < 0x7ffffff0ll ? sx_all : 0x7ffffff0ll);
    // (the descriptors begin up to 16 bytes in front of the tile's first row, so that moving back stays inside)
    const int64_t sw_base = (int64_t)n0 * srb, sx_base = m0 * (int64_t)srb;
    const int64_t sw_lo = sw_base < 16 ? sw_base : 16, sx_lo = sx_base < 16 ? sx_base : 16;
    const i32x4 sw_rsrc = raw_rsrc((const char *)p.ws + sw_base - sw_lo, sw_all + 16 + sw_lo);
    const i32x4 sx_rsrc = raw_rsrc((const char *)p.xs + sx_base - sx_lo, sx_all + 16 + sx_lo);
    auto stage_scales = [&](int g) {
#pragma unroll
        for (int q = 0; q < NSC; ++q) {
            const int first = min((q * NW + wave) * 32, TN + TM - 32);          // (a wave without rows of its own repeats the last ones)
            const bool w = first < TN;                                          // wave-uniform
            const int row = (w ? first : first - TN) + (lane >> 1);
            const int off = min(row * srb + g * 32 + (lane & 1) * 16, w ? sw_max : sx_max) + (int)(w ? sw_lo : sx_lo);
            dma16(w ? sw_rsrc : sx_rsrc, (unsigned)off, 0, lds0 + RING + first * 32);
        }
    };
    // sc[i][h][q], byte J: the scale of this lane's values 64 h + 32 kb .. + 31 of step 4 q + J of the group
    uint32_t sc[FN + FM][2][2];
    const uint32_t pick0 = (uint32_t)kb * 0x0101u + 0x0400u, pick1 = pick0 + 0x0202u;
    auto take_scales = [&](int g) {
        const int left = KG > 1 ? max(steps - 8 * g, 0) : steps - 8 * g;          // steps behind the last: scale 2^-127, never a NaN
        const uint32_t real[2] = {left >= 4 ? ~0u : (1u << 8 * left) - 1, left >= 8 ? ~0u : left <= 4 ? 0u : (1u << 8 * (left - 4)) - 1};
#pragma unroll
        for (int i = 0; i < FN + FM; ++i)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = (i < FN ? wn * FN + i : wm * FM + i - FN) * 32 + r;
                const uint4 raw = *(const uint4 *)(smem + RING + (row + (i < FN ? 0 : TN)) * 32 + q * 16);
                const int over = (max(row * srb + g * 32 + q * 16 - (i < FN ? sw_max : sx_max), 0) * 2) & 31;
                sc[i][0][q] = (__builtin_amdgcn_perm(__builtin_amdgcn_perm(raw.w, raw.z, pick0), __builtin_amdgcn_perm(raw.y, raw.x, pick0), 0x05040100u) >> over) & real[q];
                sc[i][1][q] = (__builtin_amdgcn_perm(__builtin_amdgcn_perm(raw.w, raw.z, pick1), __builtin_amdgcn_perm(raw.y, raw.x, pick1), 0x05040100u) >> over) & real[q];
            }
    };

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int swap = r & 7;

    // a team's groups of scales, and where they begin; every team makes the same turns (those behind the last step multiply zeros)
    const int groups = (((steps + 7) >> 3) + KG - 1) / KG, g0 = team * groups, stages = min(g0 * GS + (steps + KS - 1) / KS, (g0 + groups) * GS);
    stage_scales(g0);
    constexpr int AHEAD = NST > 1 ? NST - 1 : 1;     // stages in flight
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) stage(g0 * GS + i, i);
    int slot = 0, fill = NST - 1;
    // I: stage of the group
    auto go = [&](auto ic, int t) {
        constexpr int I = decltype(ic)::value;
        // This stage's codes (and a new group's scales) have landed: what was issued behind them are the next stages and, up to the stage that
        // was issued together with them, the next group's scales (issued at the end of a group's second stage).
        MX_VMCNT((AHEAD - 1) * NI + (I >= 2 && I <= AHEAD + 1 && NST > 1 ? NSC : 0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (I == 0) take_scales(t * KS >> 3);
        const char *a = smem + slot * STAGE + (wn * FN * 32 + r) * ROW, *b = smem + slot * STAGE + (TN + wm * FM * 32 + r) * ROW;
        // The DMA into the slot that every wave left behind at this barrier is spread over the products: issued in one go it would hold
        // the wave until the address unit has taken it all.
        constexpr int MUL = 2 * KS * FN * FM, EVERY = MUL / (NI + 1) > 0 ? MUL / (NI + 1) : 1;
        int done = 0, sent = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 fa[FN], fb[FM];
                const int at = ((4 * k + 2 * h + kb) ^ swap) << 4;
#pragma unroll
                for (int j = 0; j < FM; ++j) fb[j] = *(const uint4 *)(b + j * 32 * ROW + at);
#pragma unroll
                for (int i = 0; i < FN; ++i) fa[i] = *(const uint4 *)(a + i * 32 * ROW + at);
                constexpr int J0 = I * KS;
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int j = 0; j < FM; ++j) {
                        if (k == 0) acc[i][j] = mfma_fp4_32<J0 & 3>(fa[i], fb[j], acc[i][j], sc[i][h][J0 >> 2], sc[FN + j][h][J0 >> 2]);
                        else acc[i][j] = mfma_fp4_32<(J0 + 1) & 3>(fa[i], fb[j], acc[i][j], sc[i][h][((J0 + 1) & 7) >> 2], sc[FN + j][h][((J0 + 1) & 7) >> 2]);
                        if (NST > 1 && ++done % EVERY == 0 && sent < NI) stage_one(sent++, t + AHEAD, fill);
                    }
            }
        if (NST == 1) {                              // one slot: everybody has read it, then it is filled again
            __syncthreads();
            stage(t + 1, 0);
        } else {
#pragma unroll
            for (int d = 0; d < NI; ++d)
                if (d >= sent) stage_one(d, t + AHEAD, fill);
            fill = slot;
            slot = slot + 1 == NST ? 0 : slot + 1;
        }
        if (I == 1) stage_scales((t * KS >> 3) + 1);             // (every wave has taken this group's: a barrier ago)
    };
    for (int g = g0; g < g0 + groups; ++g) {
        const int t = g * GS;
        go(std::integral_constant<int, 0>(), t);
        if (t + 1 < stages) go(std::integral_constant<int, 1>(), t + 1);
        if (t + 2 < stages) go(std::integral_constant<int, 2>(), t + 2);
        if (t + 3 < stages) go(std::integral_constant<int, 3>(), t + 3);
    }
    MX_VMCNT(0);
    __syncthreads();                                 // the rings are free: the waves' own scratch from here
    if constexpr (KG > 1) {
        f32x4 *const sums = (f32x4 *)(all_smem + NW * 32 * (FN * 32 + 4) * 4);          // behind that scratch
        constexpr int PER = FN * FM * 4;
        if (team) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                sums[(((team - 1) * NW + wave) * PER + i) * 64 + lane] = *((const f32x4 *)&acc[0][0] + i);
        }
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int t = 0; t < KG - 1; ++t)
#pragma unroll
            for (int i = 0; i < PER; ++i) *((f32x4 *)&acc[0][0] + i) += sums[((t * NW + wave) * PER + i) * 64 + lane];
    }

    // epilogue: 32 activation rows at a time through LDS, so that a row's outputs leave as whole lines.  Of a block a lane holds activation
    // row r and weight rows 8 q + 4 kb + e (q = 0 .. 3, e = 0 .. 3); a gated layer's block is 16 values and their 16 gates
    constexpr int PITCH = FN * 32 + 4;
    float *const my = (float *)smem + wave * 32 * PITCH;
    const int nw = n0 + wn * FN * 32;
    float bias[FN][16];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = nw + i * 32 + q * 8 + kb * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[i][q * 4 + e] = p.bias ? p.bias[min(n + e, p.N - 1)] : 0.f;
        }
    auto finish = [&](auto ec) {
        constexpr int EPI = decltype(ec)::value;
        constexpr bool GLU = EPI == ONEDC_EPI_GEGLU;
        constexpr int WIDE = GLU ? FN * 16 : FN * 32, PIECES = WIDE / 8;         // outputs of a row, in pieces of eight
        const int out = GLU ? p.N / 2 : p.N, no = GLU ? nw / 2 : nw;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int64_t mt = m0 + (wm * FM + j) * 32;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int q = 0; q < (GLU ? 2 : 4); ++q) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float t = __builtin_fmaf(p.alpha, acc[i][j][q * 4 + e], bias[i][q * 4 + e]);
                        if (GLU) v[e] = t * gelu_f(__builtin_fmaf(p.alpha, acc[i][j][(q * 4 + e + 8) & 15], bias[i][(q * 4 + e + 8) & 15]));
                        else v[e] = EPI == ONEDC_EPI_SILU ? silu_f(t) : EPI == ONEDC_EPI_LEAKY ? leaky(t, p.slope) : t;
                    }
                    *(f32x4 *)(my + r * PITCH + i * (GLU ? 16 : 32) + q * 8 + kb * 4) = v;
                }
#pragma unroll
            for (int t0 = 0; t0 < 32 * PIECES; t0 += 64) {
                const int t = t0 + lane, row = t / PIECES, c = (t - row * PIECES) * 8, n = no + c;
                const f32x4 lo = *(const f32x4 *)(my + row * PITCH + c), hi = *(const f32x4 *)(my + row * PITCH + c + 4);
                const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                if (mt + row < p.M && n < out) store8(p, mt + row, n, out, v, whole && n + 8 <= out);
            }
        }
    };
    switch (p.epi) {
    case ONEDC_EPI_GEGLU: finish(std::integral_constant<int, ONEDC_EPI_GEGLU>()); break;
    case ONEDC_EPI_SILU: finish(std::integral_constant<int, ONEDC_EPI_SILU>()); break;
    case ONEDC_EPI_LEAKY: finish(std::integral_constant<int, ONEDC_EPI_LEAKY>()); break;
    default: finish(std::integral_constant<int, ONEDC_EPI_LINEAR>());
    }
}

// the codes and the scales of a matrix
OnedcMem codes_of(const void *p, int64_t rows, int K) { return onedc_mem(p, rows * ((K + 127) / 128) * 64); }
OnedcMem scales_of(const void *p, int64_t rows, int K) { return onedc_mem(p, rows * ((K + 127) / 128) * 4); }

bool held_ok(const void *codes, const void *scales) { return ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0; }
// whole 16-byte pieces of eight (16-bit) or four (f32) values at every row
bool whole_ok(const void *t, int cs, int co, bool f32) { return ((uintptr_t)t & 15) == 0 && ((cs | co) & (f32 ? 3 : 7)) == 0; }

template <bool F32, bool VEC>
int launch_quantize(const void *x, int x_cs, int x_co, void *codes, void *scales, int64_t rows, int K, void *stream) {
    const int per = (K + 127) / 128 * 16;
    const int64_t wgs = (rows * per + 256 * QN - 1) / (256 * QN);
    if (!onedc_grid_fits(wgs, 256)) return -2;
    hipLaunchKernelGGL((quantize_kernel<F32, VEC>), dim3((unsigned)wgs), dim3(256), 0, as_stream(stream), x,
                       x_cs, x_co, (uint32_t *)codes, (uint8_t *)scales, rows, K, per, OnedcFastDiv(per));
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <bool F32, bool VEC>
int launch_dequantize(const void *codes, const void *scales, void *y, int y_cs, int y_co, int64_t rows, int K, void *stream) {
    const int per = (K + 127) / 128 * 16;
    const int64_t wgs = (rows * per + 256 * QN - 1) / (256 * QN);
    if (!onedc_grid_fits(wgs, 256)) return -2;
    hipLaunchKernelGGL((dequantize_kernel<F32, VEC>), dim3((unsigned)wgs), dim3(256), 0, as_stream(stream),
                       (const uint32_t *)codes, (const uint8_t *)scales, y, y_cs, y_co, rows, K, per, OnedcFastDiv(per));
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <int RAW, bool VEC>
int launch_skinny(const onedc_mxfp4_params *p, int steps, int whole, void *stream) {
    const int64_t wgs = (int64_t)((p->N + 31) / 32) * ((p->M + 15) / 16);
    if (!onedc_grid_fits(wgs, 64 * SKW)) return -2;
    constexpr int sums = SKW * 2 * 16 * 20 * 4, raw = RAW ? 16 * (XPITCH + SPITCH) : 0, lds = sums > raw ? sums : raw;
    static OnedcLdsAttrOnce once;
    once.ensure({{(const void *)skinny_kernel<RAW, VEC>, lds}});
    hipLaunchKernelGGL((skinny_kernel<RAW, VEC>), dim3((unsigned)wgs), dim3(64 * SKW), lds, as_stream(stream), *p, steps, whole);
    ONEDC_LAUNCH_CHECK();
    return 0;
}
template <int WN, int WM, int FN, int FM, int NST, int OCC, int KG>
int launch_tiles(const onedc_mxfp4_params *p, int steps, int whole, void *stream) {
    static_assert(FN == 1 || FN == 2 || FN == 4, "");
    constexpr int TN = 32 * WN * FN, TM = 32 * WM * FM;
    constexpr int ring = KG * (TN + TM) * (NST * ROW + 32), scratch = WN * WM * (32 * (FN * 32 + 4) * 4 + (KG - 1) * FN * FM * 4096);
    constexpr int lds = ring > scratch ? ring : scratch;
    static_assert(lds <= 160 * 1024, "");
    static OnedcLdsAttrOnce once;
    once.ensure({{(const void *)tile_kernel<WN, WM, FN, FM, NST, OCC, KG>, lds}});
    const int64_t tn = (p->N + TN - 1) / TN, tm = (p->M + TM - 1) / TM;
    if (!onedc_grid_fits(tn * tm, 64 * WN * WM * KG)) return -2;
    hipLaunchKernelGGL((tile_kernel<WN, WM, FN, FM, NST, OCC, KG>), dim3((unsigned)(tn * tm)), dim3(64 * WN * WM * KG), lds, as_stream(stream), *p, steps,
                       (int)tn, (int)tm, whole);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" {

int onedc_mxfp4_quantize(const void *x, int x_f32, int x_cs, int x_co, void *codes, void *scales, int64_t rows, int K, void *stream) {
    if (!x || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > ONEDC_MXFP4_MAX_K || x_co < 0 || (int64_t)x_cs - K < x_co || !held_ok(codes, scales) ||
        rows * ((K + 127) / 128) > (1ll << 36))
        return -2;
    if (!rows) return 0;
    const OnedcMem c = codes_of(codes, rows, K), e = scales_of(scales, rows, K), from = onedc_mem_rows(x, rows, x_cs, x_co, K, x_f32 ? 4 : 2);
    if (onedc_mem_shared(c, from) || onedc_mem_shared(e, from) || onedc_mem_shared(c, e)) return ONEDC_SHARED_MEMORY;
    const bool vec = K % 8 == 0 && whole_ok(x, x_cs, x_co, x_f32);
    if (x_f32) return vec ? launch_quantize<true, true>(x, x_cs, x_co, codes, scales, rows, K, stream) : launch_quantize<true, false>(x, x_cs, x_co, codes, scales, rows, K, stream);
    return vec ? launch_quantize<false, true>(x, x_cs, x_co, codes, scales, rows, K, stream) : launch_quantize<false, false>(x, x_cs, x_co, codes, scales, rows, K, stream);
}

int onedc_mxfp4_dequantize(const void *codes, const void *scales, void *y, int y_f32, int y_cs, int y_co, int64_t rows, int K, void *stream) {
    if (!y || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > ONEDC_MXFP4_MAX_K || y_co < 0 || (int64_t)y_cs - K < y_co || !held_ok(codes, scales) ||
        rows * ((K + 127) / 128) > (1ll << 36))
        return -2;
    if (!rows) return 0;
    const OnedcMem to = onedc_mem_rows(y, rows, y_cs, y_co, K, y_f32 ? 4 : 2);
    if (onedc_mem_shared(to, codes_of(codes, rows, K)) || onedc_mem_shared(to, scales_of(scales, rows, K))) return ONEDC_SHARED_MEMORY;
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
        (int64_t)p->y_cs - out < p->y_co || (p->res && (p->r_co < 0 || (int64_t)p->r_cs - out < p->r_co)) || !held_ok(p->wc, p->ws))
        return -2;
    if (p->xc ? !held_ok(p->xc, p->xs) : (p->xr_co < 0 || (int64_t)p->xr_cs - p->K < p->xr_co)) return -2;
    if (!p->xc && p->M > ONEDC_MXFP4_ROWS_RAW) return -4;
    if (!p->M) return 0;
    const OnedcMem y[1] = {onedc_mem_rows(p->y, p->M, p->y_cs, p->y_co, out, p->y_f32 ? 4 : 2)};
    const OnedcMem read[] = {codes_of(p->wc, p->N, p->K), scales_of(p->ws, p->N, p->K), p->xc ? codes_of(p->xc, p->M, p->K) : OnedcMem(),
                             p->xc ? scales_of(p->xs, p->M, p->K) : onedc_mem_rows(p->xr, p->M, p->xr_cs, p->xr_co, p->K, p->xr_f32 ? 4 : 2),
                             onedc_mem(p->bias, (int64_t)p->N * 4)};
    if (onedc_mem_any_shared(y, read)) return ONEDC_SHARED_MEMORY;
    const int steps = (p->K + 127) / 128;
    const int whole = whole_ok(p->y, p->y_cs, p->y_co, p->y_f32) && (!p->res || whole_ok(p->res, p->r_cs, p->r_co, p->y_f32));
    if (!p->xc) {
        const bool vec = p->K % 8 == 0 && whole_ok(p->xr, p->xr_cs, p->xr_co, p->xr_f32);
        if (p->xr_f32) return vec ? launch_skinny<2, true>(p, steps, whole, stream) : launch_skinny<2, false>(p, steps, whole, stream);
        return vec ? launch_skinny<1, true>(p, steps, whole, stream) : launch_skinny<1, false>(p, steps, whole, stream);
    }
    // (the tiles' scale reads need 16 bytes in all)
    if (p->M <= ONEDC_MXFP4_ROWS_RAW || (int64_t)p->N * steps < 4) return launch_skinny<0, true>(p, steps, whole, stream);
    // Tiles, by how many of them there are for 256 CUs.  One card, the shapes in turn (f16, gated ones with a bias and operands that no cache holds):
    //   256 x 256, eight waves, two stages: the fewest bytes into LDS a product.  From 160 tiles on, where it pads no tenth more than 128 x 128
    //     (8192 x 4096 x 5120: 94 us against 109; 16384 x 8192 x 8192: 544 against 626); gated layers, whose epilogue runs under nothing else on
    //     the CU, only from 32 steps on (8192 x 10240 x 4096: 203 us against 207 of 128 x 256; with 30 steps 228 against 231, with 20 175 against
    //     173, with 10 121 against 110, with 5 190 against 173)
    //   64 x 64, two teams of four waves that halve a long K, while there is no second workgroup for a CU: one team waits where the other
    //     multiplies (300 x 520 x 8192: 11.5 us against 14.2, 1024 x 1024 x 8192: 13.0 against 15.6; with 10 steps 9.8 against 5.9, three or four
    //     teams 10.2 and 10.5 in the first case where two took 9.8)
    //   64 x 64, three stages, while they fit the CUs' first four each (2048 x 1280 x 5120: 18 us against 21; 4096 x 1280 x 5120: 29 against 27)
    //   128 x 128: one stage and three workgroups a CU that load and multiply in turn; two stages where there are less than two a CU
    //     (4096 x 1280 x 5120: 27 us against 30; 8192 x 4096 x 5120: 112 against 109)
    //   128 x 256, four waves, one stage, two workgroups a CU: gated layers of very many tiles, the more the longer their K (9216 x 10240 x 3840: 231 us
    //     against 240, 16384 x 10240 x 1280: 191 against 197; 8655 x 10240 x 1280 110 both, 36864 x 5120 x 640 173 against 172; linear
    //     36864 x 640 x 640 28 against 25.5)
    const auto tiles = [&](int64_t t) { return ((p->N + t - 1) / t) * ((p->M + t - 1) / t); };
    const bool gated = p->epi == ONEDC_EPI_GEGLU;
    if (tiles(256) >= 160 && tiles(256) * 40 <= tiles(128) * 11 && (!gated || steps >= 32)) return launch_tiles<4, 2, 2, 4, 2, 2, 1>(p, steps, whole, stream);
    if (tiles(64) <= 256 && steps >= 32) return launch_tiles<2, 2, 1, 1, 3, 2, 2>(p, steps, whole, stream);
    if (tiles(64) <= 1024) return launch_tiles<2, 2, 1, 1, 3, 4, 1>(p, steps, whole, stream);
    if (tiles(128) <= 512) return launch_tiles<2, 2, 2, 2, 2, 2, 1>(p, steps, whole, stream);
    if (gated && tiles(128) > 2048) return launch_tiles<2, 2, 2, 4, 1, 2, 1>(p, steps, whole, stream);
    return launch_tiles<2, 2, 2, 2, 1, 3, 1>(p, steps, whole, stream);
}

}  // extern "C"
