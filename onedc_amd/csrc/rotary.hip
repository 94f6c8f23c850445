// rotary.hip — rotary positions over several axes: pair i of every head of a token turns by pos[token][axis[i]] * freq[i].
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// The angle is kept in turns: phase = pos * turns[i] in f64, minus its nearest whole number, so that positions of any size lose
// nothing; sine and cosine of the remaining half turn in f32.
//
// Bound by HBM: q and k are read and written once, 3 operations an element.  What has to stay off that path are the angles: a
// workgroup computes the sines and cosines of its T tokens once, into LDS, and all heads of those tokens read them from there (neighbouring
// lanes hold neighbouring heads, so most of a wave's LDS reads are one address).  Pieces of 16 bytes where the sizes allow it, two or four of a
// thread in flight.  16-bit heads: 49152 tokens x 32 x 80 in 101 us, 5.0 TB/s (a copy of 1 GB reaches 5.15; with the angles computed at every element
// 328 us), 36864 x 16 x 80 40 - 44 us, or, held by the last-level cache, 31 - 33; pairs of which only four share a piece (16384 x 32 x 72, held too)
// 26 us, single values (32000 x 16 x 42) 26 us, 3.3 TB/s; f32 heads (16384 x 32 x 72) 58 us, 5.2 TB/s; one token 3.0 us in a graph, a launch's own time.
#include <type_traits>

#include "apart.h"
#include "conv_common.h"
#include "elem.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_TABLE = 8192;           // pairs of sine and cosine in LDS: 64 KB, all that a launch has without asking for more

// VEC values at p as f32
template <bool F32, int VEC>
struct Piece {
    typedef typename Elem<F32>::T T;
    typedef __attribute__((ext_vector_type(VEC))) T V;
    V v;
    __device__ __forceinline__ void load(const T *p) { v = *(const V *)p; }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (F32) return v[i];
        else return a2f(v[i]);
    }
    __device__ __forceinline__ void set(int i, float a, float b) {       // values i, i + 1
        if constexpr (F32) {
            v[i] = a;
            v[i + 1] = b;
        } else {
            const uint32_t w = pack_a2(a, b);
            v[i] = (T)(w & 0xffffu);
            v[i + 1] = (T)(w >> 16);
        }
    }
    __device__ __forceinline__ void store(T *p) const { *(V *)p = v; }
};
template <bool F32>
struct Piece<F32, 1> {
    typedef typename Elem<F32>::T T;
    T v;
    __device__ __forceinline__ void load(const T *p) { v = *p; }
    __device__ __forceinline__ float get(int) const { return Elem<F32>::get(&v); }
    __device__ __forceinline__ void set1(float a) { Elem<F32>::put(&v, a); }
    __device__ __forceinline__ void store(T *p) const { *p = v; }
};

// A token's heads are cut into units of VEC values: `turn` units a head that turn (two pieces each with pairs of halves, one with pairs of
// neighbours), then the pieces that pass through.
struct Units {
    int turn, per, T;                     // turning units and all units of a head; tokens of a workgroup
    OnedcFastDiv by_unit, by_head, by_pair;
};

// units of a thread in flight
template <bool F32, int VEC, bool NEIGHBOURS, int FLY>
__global__ __launch_bounds__(NT) void rotary_kernel(onedc_rotary_params p, Units u) {
    typedef typename Elem<F32>::T T;
    extern __shared__ __attribute__((aligned(16))) float table[];         // [T][pairs] cosines, then sines
    const int64_t row0 = (int64_t)blockIdx.x * u.T;
    const int64_t rows = (int64_t)p.B * p.N;
    const int tokens = (int)(rows - row0 < u.T ? rows - row0 : u.T);
    float *const cosines = table, *const sines = table + u.T * p.pairs;

    for (int i = threadIdx.x; i < tokens * p.pairs; i += NT) {
        const int t = u.by_pair.div(i), j = i - t * p.pairs;
        const int64_t row = row0 + t, b = row / p.N;
        const int64_t at = b * p.pos_bs + (row - b * p.N) * p.axes + p.axis[j];
        const double pos = p.pos_f32 ? (double)((const float *)p.pos)[at] : (double)((const int32_t *)p.pos)[at];
        const double turn = pos * p.turns[j];
        float s, c;
        sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
        cosines[i] = c;
        sines[i] = p.inverse ? -s : s;
    }
    __syncthreads();

    const int heads = p.qh + p.kh, total = tokens * heads * u.per;
    constexpr bool TWO = VEC == 1 || !NEIGHBOURS;    // pieces of a turning unit
    for (int i0 = threadIdx.x; i0 < total; i0 += NT * FLY) {
        T *dst[FLY];
        int first[FLY], second[FLY], entry[FLY];     // where its pieces begin in the head, and its pairs in the table (-1: passes through)
        Piece<F32, VEC> a[FLY], b[FLY];
#pragma unroll
        for (int q = 0; q < FLY; ++q) {
            const int i = min(i0 + q * NT, total - 1);       // (behind the last: loaded, not stored)
            const int th = u.by_unit.div(i), unit = i - th * u.per;
            const int t = u.by_head.div(th), h = th - t * heads;
            const int64_t row = row0 + t;
            const bool isq = h < p.qh;
            const T *src = isq ? (const T *)p.q + row * p.q_cs + p.q_co + h * p.D : (const T *)p.k + row * p.k_cs + p.k_co + (h - p.qh) * p.D;
            dst[q] = isq ? (T *)p.qo + row * p.qo_cs + p.qo_co + h * p.D : (T *)p.ko + row * p.ko_cs + p.ko_co + (h - p.qh) * p.D;
            const bool turns = unit < u.turn;
            const int wide = VEC == 1 && NEIGHBOURS ? 2 : VEC, passed = 2 * p.pairs + (unit - u.turn) * VEC;
            first[q] = turns ? unit * wide : passed;
            second[q] = !turns ? passed : NEIGHBOURS ? unit * wide + 1 : unit * VEC + p.pairs;
            entry[q] = turns ? t * p.pairs + unit * (VEC == 1 ? 1 : NEIGHBOURS ? VEC / 2 : VEC) : -1;
            a[q].load(src + first[q]);
            if (TWO) b[q].load(src + second[q]);
        }
#pragma unroll
        for (int q = 0; q < FLY; ++q) {
            if (i0 + q * NT >= total) continue;
            if (entry[q] >= 0) {
                if constexpr (VEC == 1) {                                 // one pair
                    const float c = cosines[entry[q]], s = sines[entry[q]], x = a[q].get(0), y = b[q].get(0);
                    a[q].set1(x * c - y * s), b[q].set1(y * c + x * s);
                } else if constexpr (NEIGHBOURS) {                         // VEC / 2 pairs
                    typedef __attribute__((ext_vector_type(VEC / 2))) float C;
                    const C c = *(const C *)(cosines + entry[q]), s = *(const C *)(sines + entry[q]);
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) {
                        const float x = a[q].get(2 * j), y = a[q].get(2 * j + 1);
                        a[q].set(2 * j, x * c[j] - y * s[j], y * c[j] + x * s[j]);
                    }
                } else {                                                  // VEC pairs
                    typedef __attribute__((ext_vector_type(4))) float C;   // (four at a time: the table is 16-byte aligned)
                    C c[VEC / 4], s[VEC / 4];
#pragma unroll
                    for (int j = 0; j < VEC / 4; ++j) {
                        c[j] = *(const C *)(cosines + entry[q] + 4 * j);
                        s[j] = *(const C *)(sines + entry[q] + 4 * j);
                    }
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) {
                        const float x0 = a[q].get(j), x1 = a[q].get(j + 1), y0 = b[q].get(j), y1 = b[q].get(j + 1);
                        const float c0 = c[j / 4][j % 4], c1 = c[j / 4][j % 4 + 1], s0 = s[j / 4][j % 4], s1 = s[j / 4][j % 4 + 1];
                        a[q].set(j, x0 * c0 - y0 * s0, x1 * c1 - y1 * s1);
                        b[q].set(j, y0 * c0 + x0 * s0, y1 * c1 + x1 * s1);
                    }
                }
                if (TWO) b[q].store(dst[q] + second[q]);
            }
            a[q].store(dst[q] + first[q]);
        }
    }
}

template <bool F32, int VEC>
int launch(const onedc_rotary_params *p, void *stream) {
    Units u;
    u.turn = VEC == 1 ? p->pairs : p->neighbours ? 2 * p->pairs / VEC : p->pairs / VEC;
    u.per = u.turn + (p->D - 2 * p->pairs) / VEC;
    // tokens a workgroup: up to 2048 units (8 a thread), fewer where that leaves under two workgroups a CU
    const int64_t rows = (int64_t)p->B * p->N;
    const int heads = p->qh + p->kh;
    int64_t T = 2048 / ((int64_t)heads * u.per), most = (rows + 511) / 512;
    if (T > most) T = most;
    if (p->pairs && T > MAX_TABLE / p->pairs) T = MAX_TABLE / p->pairs;
    u.T = (int)(T < 1 ? 1 : T);
    u.by_unit = OnedcFastDiv(u.per), u.by_head = OnedcFastDiv(heads), u.by_pair = OnedcFastDiv(p->pairs ? p->pairs : 1);
    if (!onedc_grid_fits((rows + u.T - 1) / u.T, NT)) return -2;
    const dim3 grid((unsigned)((rows + u.T - 1) / u.T));
    const size_t lds = (size_t)u.T * p->pairs * 8;
    // four units of a thread in flight, two for small calls, whose threads have no more (tensors that no cache holds: 36864 x 16 x 80 39.6 us against
    // 41.8, 49152 x 32 x 80 102 against 109; 8000 x 16 x 64 8.3 against 7.9)
    const bool many = rows * heads * p->D * (F32 ? 8 : 4) > (32ll << 20);
    const auto go = [&](auto nb, auto fly) {
        hipLaunchKernelGGL((rotary_kernel<F32, VEC, decltype(nb)::value, decltype(fly)::value>), grid, dim3(NT), lds, as_stream(stream), *p, u);
    };
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    if (p->neighbours) many ? go(std::true_type(), Four()) : go(std::true_type(), Two());
    else many ? go(std::false_type(), Four()) : go(std::false_type(), Two());
    ONEDC_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" int onedc_rotary_axes(const onedc_rotary_params *p, void *stream) {
    if (!p || !p->q || !p->qo || !p->pos || !p->turns || !p->axis || (p->kh > 0 && (!p->k || !p->ko))) return -1;
    if (p->B < 0 || p->N < 0 || p->D < 1 || p->D > 4096 || p->pairs < 0 || 2 * p->pairs > p->D || p->axes < 1 || p->axes > 16 || p->qh < 1 ||
        p->kh < 0 || p->qh > 4096 || p->kh > 4096 || (int64_t)p->B * p->N > 0x7fffffff || p->pos_bs < 0)
        return -2;
    const int64_t cq = p->qh * p->D, ck = p->kh * p->D;
    if (p->q_co < 0 || p->q_cs - cq < p->q_co || p->qo_co < 0 || p->qo_cs - cq < p->qo_co) return -2;
    if (p->kh && (p->k_co < 0 || p->k_cs - ck < p->k_co || p->ko_co < 0 || p->ko_cs - ck < p->ko_co)) return -2;
    if (!p->B || !p->N) return 0;
    const auto rows = [&](const void *t, int64_t cs, int64_t co, int64_t c) { return onedc_mem_rows(t, (int64_t)p->B * p->N, cs, co, c, p->x_f32 ? 4 : 2); };
    const OnedcMem out[] = {rows(p->qo, p->qo_cs, p->qo_co, cq), p->kh ? rows(p->ko, p->ko_cs, p->ko_co, ck) : OnedcMem()};
    const OnedcMem plan[] = {onedc_mem(p->pos, ((p->B - 1) * p->pos_bs + (int64_t)p->N * p->axes) * 4), onedc_mem(p->turns, (int64_t)p->pairs * 8),
                             onedc_mem(p->axis, (int64_t)p->pairs * 4)};
    if (onedc_mem_any_shared(out, plan)) return ONEDC_SHARED_MEMORY;
    // the widest piece that divides a head's parts and every row's beginning: 16 bytes, 8 bytes, or single values
    const int part = p->neighbours ? 2 * p->pairs : p->pairs, size = p->x_f32 ? 4 : 2;
    int bits = part | (p->D - 2 * p->pairs) | p->D | p->q_cs | p->q_co | p->qo_cs | p->qo_co;
    uintptr_t at = (uintptr_t)p->q | (uintptr_t)p->qo;
    if (p->kh) {
        bits |= p->k_cs | p->k_co | p->ko_cs | p->ko_co;
        at |= (uintptr_t)p->k | (uintptr_t)p->ko;
    }
    const auto fits = [&](int vec) { return bits % vec == 0 && at % (unsigned)(vec * size) == 0; };
    if (p->x_f32) return fits(4) ? launch<true, 4>(p, stream) : launch<true, 1>(p, stream);
    return fits(8) ? launch<false, 8>(p, stream) : fits(4) ? launch<false, 4>(p, stream) : launch<false, 1>(p, stream);
}
