// mxfp4.hip — 4-bit microscaled floating point (OCP MX v1.0, MXFP4): quantise, read back, and the product of two such matrices.
//
// A block of 32 consecutive values of a row is 2^e * q, q in e2m1: e = max(floor(log2 amax) - 2, -127), so amax * 2^-e lies in [4, 8)
// and is the only place where the largest code, 6, saturates.  v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 rows over
// 128 values: lane l holds row l % 16, values 32 (l / 16) .. + 31 (16 bytes of codes) and that block's scale byte -- the memory
// layout itself, no shuffle.  Its products are exact, the sums f32.
#include "elem.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;

// e2m1 code of |a| in units of the block's scale, round half to even
__device__ __forceinline__ uint32_t e2m1(float v) {
    const float a = fabsf(v);
    const float r = a < 2.f ? rintf(a * 2.f) : a < 4.f ? rintf(a) + 2.f : fminf(rintf(a * 0.5f) + 4.f, 7.f);
    return (uint32_t)(int)r | ((__float_as_uint(v) >> 28) & 8u);
}
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t m = code & 7u;
    const float a = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    return code & 8u ? -a : a;
}

// scale byte of a block from the bits of its largest magnitude, and the factor that takes values to code units
__device__ __forceinline__ uint32_t block_scale(uint32_t amax_bits, float *inv) {
    if (amax_bits >= 0x7f800000u) {                  // a NaN or an infinity: the whole block reads back as NaN
        *inv = 0.f;
        return 255u;
    }
    const int ex = (int)(amax_bits >> 23);           // biased exponent; 0 (zero, subnormal) lands on the lowest scale too
    const int s = ex > 2 ? ex - 2 : 0;
    *inv = __uint_as_float((uint32_t)(254 - s) << 23);
    return (uint32_t)s;
}

template <bool F32>
__device__ __forceinline__ float load_x(const void *x, int64_t i) {
    return Elem<F32>::get((const typename Elem<F32>::T *)x + i);
}

// one thread per block of 32; blocks past the row's last value are the padding's
template <bool F32>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, int x_cs, int x_co, uint4 *codes, uint8_t *scales, int64_t rows, int K,
                                                       int nb) {
    const int64_t total = rows * nb;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / nb;
        const int k0 = (int)(i - row * nb) * 32;
        float v[32];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = k0 + j < K ? load_x<F32>(x, row * x_cs + x_co + k0 + j) : 0.f;
            amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
        }
        float inv;
        const uint32_t s = block_scale(amax, &inv);
        uint32_t w[4] = {0, 0, 0, 0};
        if (s != 255u)
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j >> 3] |= e2m1(v[j] * inv) << (4 * (j & 7));
        codes[i] = make_uint4(w[0], w[1], w[2], w[3]);
        scales[i] = (uint8_t)s;
    }
}

template <bool F32>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint4 *codes, const uint8_t *scales, void *y, int y_cs, int y_co, int64_t rows,
                                                         int K, int nb) {
    const int64_t total = rows * nb;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / nb;
        const int k0 = (int)(i - row * nb) * 32;
        const uint4 c = codes[i];
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        const int s = scales[i];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (k0 + j >= K) continue;
            const float q = e2m1_value((w[j >> 3] >> (4 * (j & 7))) & 15u);
            const float v = s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(q, s - 127);
            const int64_t at = row * y_cs + y_co + k0 + j;
            if (F32) ((float *)y)[at] = v;
            else ((a16_t *)y)[at] = f2a(v);
        }
    }
}

__device__ __forceinline__ f32x4 mfma_fp4(uint4 a, uint4 b, f32x4 c, int sa, int sb) {
    const i32x8 va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, 0, sa, 0, sb);
}

__device__ __forceinline__ float activation(const onedc_mxfp4_params &p, float v) {
    return p.epi == ONEDC_EPI_SILU ? silu_f(v) : p.epi == ONEDC_EPI_LEAKY ? leaky(v, p.slope) : v;
}
__device__ __forceinline__ void store_y(const onedc_mxfp4_params &p, int64_t m, int n, float v) {
    if (p.res) v += p.y_f32 ? ((const float *)p.res)[m * p.r_cs + p.r_co + n] : a2f(((const a16_t *)p.res)[m * p.r_cs + p.r_co + n]);
    if (p.y_f32) ((float *)p.y)[m * p.y_cs + p.y_co + n] = v;
    else ((a16_t *)p.y)[m * p.y_cs + p.y_co + n] = f2a(v);
}

// A wave computes 32 weight rows x 16 activation rows, fragments straight from memory.  Raw rows (p.xr) are quantised by the lane that
// multiplies them.
__global__ __launch_bounds__(64) void linear_kernel(onedc_mxfp4_params p, int steps) {
    const int lane = threadIdx.x, r = lane & 15, kb = lane >> 4;
    const int nt = (p.N + 31) / 32;
    const int n0 = (int)(blockIdx.x % nt) * 32;
    const int64_t m0 = (int64_t)(blockIdx.x / nt) * 16;
    const int64_t m = m0 + r < p.M ? m0 + r : p.M - 1;
    const int na = n0 + r < p.N ? n0 + r : p.N - 1, nc = n0 + 16 + r < p.N ? n0 + 16 + r : p.N - 1;
    const uint4 *wa = (const uint4 *)p.wc + (int64_t)na * steps * 4 + kb, *wb = (const uint4 *)p.wc + (int64_t)nc * steps * 4 + kb;
    const uint8_t *sa = (const uint8_t *)p.ws + (int64_t)na * steps * 4 + kb, *sb = (const uint8_t *)p.ws + (int64_t)nc * steps * 4 + kb;
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    for (int s = 0; s < steps; ++s) {
        uint4 x;
        int sx;
        if (p.xc) {
            x = ((const uint4 *)p.xc)[m * steps * 4 + s * 4 + kb];
            sx = ((const uint8_t *)p.xs)[m * steps * 4 + s * 4 + kb];
        } else {
            const int k0 = s * 128 + kb * 32;
            float v[32];
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const int64_t at = m * p.xr_cs + p.xr_co + k0 + j;
                v[j] = k0 + j >= p.K ? 0.f : p.xr_f32 ? load_x<true>(p.xr, at) : load_x<false>(p.xr, at);
                amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
            }
            float inv;
            sx = (int)block_scale(amax, &inv);
            uint32_t w[4] = {0, 0, 0, 0};
            if (sx != 255)
#pragma unroll
                for (int j = 0; j < 32; ++j) w[j >> 3] |= e2m1(v[j] * inv) << (4 * (j & 7));
            x = make_uint4(w[0], w[1], w[2], w[3]);
        }
        acc[0] = mfma_fp4(wa[s * 4], x, acc[0], sa[s * 4], sx);
        acc[1] = mfma_fp4(wb[s * 4], x, acc[1], sb[s * 4], sx);
    }
    if (m0 + r >= p.M) return;                       // lane: activation row r, weight rows 4 kb + e of each half
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int a = n0 + kb * 4 + e, c = a + 16;
        if (p.epi == ONEDC_EPI_GEGLU) {
            if (c >= p.N) continue;
            const float v = p.alpha * acc[0][e] + (p.bias ? p.bias[a] : 0.f), g = p.alpha * acc[1][e] + (p.bias ? p.bias[c] : 0.f);
            store_y(p, m0 + r, n0 / 2 + kb * 4 + e, v * gelu_f(g));
        } else {
            if (a < p.N) store_y(p, m0 + r, a, activation(p, p.alpha * acc[0][e] + (p.bias ? p.bias[a] : 0.f)));
            if (c < p.N) store_y(p, m0 + r, c, activation(p, p.alpha * acc[1][e] + (p.bias ? p.bias[c] : 0.f)));
        }
    }
}

bool held_ok(const void *codes, const void *scales) { return ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0; }

}  // namespace

extern "C" {

int onedc_mxfp4_quantize(const void *x, int x_f32, int x_cs, int x_co, void *codes, void *scales, int64_t rows, int K, void *stream) {
    if (!x || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > (1 << 24) || x_co < 0 || x_cs - K < x_co || !held_ok(codes, scales)) return -2;
    if (!rows) return 0;
    const int nb = (K + 127) / 128 * 4;
    const int64_t blocks = (rows * nb + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (x_f32) hipLaunchKernelGGL(quantize_kernel<true>, grid, dim3(256), 0, as_stream(stream), x, x_cs, x_co, (uint4 *)codes, (uint8_t *)scales, rows, K, nb);
    else hipLaunchKernelGGL(quantize_kernel<false>, grid, dim3(256), 0, as_stream(stream), x, x_cs, x_co, (uint4 *)codes, (uint8_t *)scales, rows, K, nb);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

int onedc_mxfp4_dequantize(const void *codes, const void *scales, void *y, int y_f32, int y_cs, int y_co, int64_t rows, int K, void *stream) {
    if (!y || !codes || !scales) return -1;
    if (rows < 0 || rows > 0x7fffffff || K < 1 || K > (1 << 24) || y_co < 0 || y_cs - K < y_co || !held_ok(codes, scales)) return -2;
    if (!rows) return 0;
    const int nb = (K + 127) / 128 * 4;
    const int64_t blocks = (rows * nb + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (y_f32) hipLaunchKernelGGL(dequantize_kernel<true>, grid, dim3(256), 0, as_stream(stream), (const uint4 *)codes, (const uint8_t *)scales, y, y_cs, y_co, rows, K, nb);
    else hipLaunchKernelGGL(dequantize_kernel<false>, grid, dim3(256), 0, as_stream(stream), (const uint4 *)codes, (const uint8_t *)scales, y, y_cs, y_co, rows, K, nb);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

int onedc_mxfp4_linear(const onedc_mxfp4_params *p, void *stream) {
    if (!p || !p->wc || !p->ws || !p->y || (!p->xr && (!p->xc || !p->xs))) return -1;
    if (p->epi != ONEDC_EPI_LINEAR && p->epi != ONEDC_EPI_LEAKY && p->epi != ONEDC_EPI_SILU && p->epi != ONEDC_EPI_GEGLU) return -3;
    if (p->epi == ONEDC_EPI_GEGLU && p->N % 32) return -3;
    const int out = p->epi == ONEDC_EPI_GEGLU ? p->N / 2 : p->N;
    if (p->M < 0 || p->M > 0x7fffffff || p->N < 1 || p->N > (1 << 24) || p->K < 1 || p->K > (1 << 24) || p->y_co < 0 || p->y_cs - out < p->y_co ||
        (p->res && (p->r_co < 0 || p->r_cs - out < p->r_co)) || !held_ok(p->wc, p->ws))
        return -2;
    if (p->xc ? !held_ok(p->xc, p->xs) : (p->xr_co < 0 || p->xr_cs - p->K < p->xr_co)) return -2;
    if (!p->xc && p->M > ONEDC_MXFP4_ROWS_RAW) return -4;
    if (!p->M) return 0;
    const int64_t tiles = (int64_t)((p->N + 31) / 32) * ((p->M + 15) / 16);
    if (tiles > 0x7fffffff) return -2;
    hipLaunchKernelGGL(linear_kernel, dim3((unsigned)tiles), dim3(64), 0, as_stream(stream), *p,
                       (p->K + 127) / 128);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
