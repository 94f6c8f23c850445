// rotary.hip — rotary positions over several axes: pair i of every head of a token turns by pos[token][axis[i]] * freq[i].
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// The angle is kept in turns: phase = pos * turns[i] in f64, minus its nearest whole number, so that positions of any size lose
// nothing; sine and cosine of the remaining half turn in f32.
#include "elem.h"

namespace {

// cosine and sine of the angle of pair i at token n of picture b
__device__ __forceinline__ float2 phase(const onedc_rotary_params &p, int64_t b, int n, int i) {
    const int64_t at = b * p.pos_bs + (int64_t)n * p.axes + p.axis[i];
    const double pos = p.pos_f32 ? (double)((const float *)p.pos)[at] : (double)((const int32_t *)p.pos)[at];
    const double t = pos * p.turns[i];
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    return make_float2(c, p.inverse ? -s : s);
}

// one thread per (token, head, pair or passed-through dim)
template <bool F32>
__global__ __launch_bounds__(256) void rotary_kernel(onedc_rotary_params p) {
    typedef Elem<F32> E;
    const int heads = p.qh + p.kh, per = p.D - p.pairs;
    const int64_t total = (int64_t)p.B * p.N * heads * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t th = i / per;
        const int j = (int)(i - th * per);
        const int64_t row = th / heads;
        const int h = (int)(th - row * heads);
        const bool isq = h < p.qh;
        const typename E::T *src = isq ? (const typename E::T *)p.q + row * p.q_cs + p.q_co + h * p.D
                                       : (const typename E::T *)p.k + row * p.k_cs + p.k_co + (h - p.qh) * p.D;
        typename E::T *dst = isq ? (typename E::T *)p.qo + row * p.qo_cs + p.qo_co + h * p.D
                                 : (typename E::T *)p.ko + row * p.ko_cs + p.ko_co + (h - p.qh) * p.D;
        if (j >= p.pairs) {
            dst[p.pairs + j] = src[p.pairs + j];
            continue;
        }
        const int64_t b = row / p.N;
        const float2 cs = phase(p, b, (int)(row - b * p.N), j);
        const int ia = p.neighbours ? 2 * j : j, ib = p.neighbours ? 2 * j + 1 : j + p.pairs;
        const float a = E::get(src + ia), v = E::get(src + ib);
        E::put(dst + ia, a * cs.x - v * cs.y);
        E::put(dst + ib, v * cs.x + a * cs.y);
    }
}

}  // namespace

extern "C" int onedc_rotary_axes(const onedc_rotary_params *p, void *stream) {
    if (!p || !p->q || !p->qo || !p->pos || !p->turns || !p->axis || (p->kh > 0 && (!p->k || !p->ko))) return -1;
    if (p->B < 0 || p->N < 0 || p->D < 1 || p->D > 4096 || p->pairs < 0 || 2 * p->pairs > p->D || p->axes < 1 || p->axes > 16 || p->qh < 1 ||
        p->kh < 0 || p->qh > 4096 || p->kh > 4096 || (int64_t)p->B * p->N > 0x7fffffff || p->pos_bs < 0)
        return -2;
    const int cq = p->qh * p->D, ck = p->kh * p->D;
    if (p->q_co < 0 || p->q_cs - cq < p->q_co || p->qo_co < 0 || p->qo_cs - cq < p->qo_co) return -2;
    if (p->kh && (p->k_co < 0 || p->k_cs - ck < p->k_co || p->ko_co < 0 || p->ko_cs - ck < p->ko_co)) return -2;
    const int64_t total = (int64_t)p->B * p->N * (p->qh + p->kh) * (p->D - p->pairs);
    if (!total) return 0;
    const int64_t blocks = (total + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (p->x_f32) hipLaunchKernelGGL(rotary_kernel<true>, grid, dim3(256), 0, as_stream(stream), *p);
    else hipLaunchKernelGGL(rotary_kernel<false>, grid, dim3(256), 0, as_stream(stream), *p);
    ONEDC_LAUNCH_CHECK();
    return 0;
}
