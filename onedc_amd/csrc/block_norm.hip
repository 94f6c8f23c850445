// block_norm.hip — norms before and after a transformer sub-block fused with its gate and the residual scale, and the backward pass.
//
//   t = x + alpha * gate * P(f)      xo = round(t)      y = (norm(t) * w + b) * (1 + scale) + shift
//
// norm(v) = (v - m) * r with m = mean (LayerNorm; 0 for RMSNorm) and r = 1 / sqrt(mean((v - m)^2) + eps).
// Backward, with u = dy * (1 + scale) * w and h = norm(t):
//   dt = dxo + r * (u - [mean(u)] - h * mean(u * h))                   ([..]: LayerNorm only)
//   df = the same step through norm(f) on alpha * gate * post_w * dt, or alpha * gate * dt without the post norm
// and every parameter gradient follows from four sums over the rows of a picture: S1 = sum dy, S2 = sum dy * norm(t),
// T1 = sum dt, T2 = sum dt * norm(f) (f itself without the post norm).
#include <iterator>
#include <type_traits>

#include "apart.h"
#include "elem.h"

namespace {

constexpr int NT = 256;

// ---- rows in registers: up to 16384 channels (backward: 8192) --------------------------------------------------------------------------
// Bound by HBM: x and f are read once, xo and y written once (backward: four read, two written).  A row belongs to L neighbouring lanes
// (8 .. 64, or a workgroup of 256, 512 or 1024), which hold it as IT pieces of eight channels each: piece i of lane l begins at channel
// 8 (i L + l).  Statistics are two passes over registers -- mean, then squared deviations -- and log2 L exchanges between lanes.  A
// workgroup takes a run of rows of one picture, so that the vectors per picture (gate, scale, shift) and per channel are combined once:
//   A = alpha gate post_w, Ab = alpha gate post_b (join);  W = w (1 + scale), S = b (1 + scale) + shift (norm behind it)
// into LDS where several rows of a wave share them, into registers where a thread owns its channels.  The next row's loads are in
// flight while a row is computed.
// 16-bit, gated, modulated, norms on both sides: 16 x 9216 x 320 in 81 us (4.7 TB/s of 5.15 that a large copy reaches), 16 x 2304 x 640 33 us (5.7),
// 16 x 576 x 1280 21 us (4.5), 16 x 2304 x 643 36 us (5.3), 16 x 576 x 4096 63 us (4.8); with every gradient backward 131 us (4.3), 71 us (4.0),
// 56 us (2.5: 160 pieces leave 96 of 256 lanes idle, and every sum is a barrier), 84 us (3.4), 113 us (4.0), of which the sums over the rows are 7 to 11.
// Norm alone 36, 21 and 13 us of the first three, join alone 47, 24 and 15.
// Outputs stored past the cache take the first to 62 us and give it all back in whoever reads them.

// sum over the L neighbouring lanes of v's row, the same bits in each of them
template <int O>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), O, 0xf, 0xf, true));
}
typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
__device__ __forceinline__ float lanes_sum(float v, int L) {      // (L is wave-uniform; without branches the exchanges of two sums overlap)
    v = dpp_add<0xb1>(v);                            // lane ^ 1
    v = dpp_add<0x4e>(v);                            // lane ^ 2
    v = dpp_add<0x141>(v);                           // mirrored within 8
    const float w = dpp_add<0x140>(v);               // mirrored within 16
    v = L > 8 ? w : v;
    const u32x2_t a = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    v = L > 16 ? __uint_as_float(a[0]) + __uint_as_float(a[1]) : v;
    const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return L > 32 ? __uint_as_float(b[0]) + __uint_as_float(b[1]) : v;
}
// sum over a wave's groups of L lanes, lane by lane
__device__ __forceinline__ float groups_sum(float v, int L) {
    if (L <= 8) v = dpp_add<0x128>(v);               // rotated by 8 within 16
    if (L <= 16) {
        const u32x2_t a = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (L <= 32) {
        const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
        v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    return v;
}
// ... or over the workgroup; red: two floats a wave, alternated so that one barrier a sum is enough
template <int NTH, bool SHARED>
struct RowSum {
    float *red;
    int L, turn;
    float C, inv_C;
    __device__ __forceinline__ float2 operator()(float v, float w) {
        if constexpr (SHARED) return make_float2(lanes_sum(v, L), lanes_sum(w, L));
        v = lanes_sum(v, 64), w = lanes_sum(w, 64);
        float2 *r = (float2 *)red + turn * (NTH / 64);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = make_float2(v, w);
        __syncthreads();
        float2 s = r[0];
#pragma unroll
        for (int i = 1; i < NTH / 64; ++i) s.x += r[i].x, s.y += r[i].y;
        return s;
    }
    // v / C, rounded once but for a rare last bit.  INF: an infinite v stays infinite (its remainder, inf - inf, is taken as a finite number)
    template <bool INF = false>
    __device__ __forceinline__ float over_C(float v) const {
        const float q = v * inv_C, e = __builtin_fmaf(-q, C, v);
        return __builtin_fmaf(INF ? __builtin_fmaxf(e, -3.4e38f) : e, inv_C, q);
    }
    template <bool INF = false>
    __device__ __forceinline__ float mean(float v) {
        if constexpr (SHARED) return over_C<INF>(lanes_sum(v, L));
        return over_C<INF>((*this)(v, 0.f).x);
    }
    __device__ __forceinline__ float2 means(float v, float w) {
        const float2 s = (*this)(v, w);
        return make_float2(over_C(s.x), over_C(s.y));
    }
};

// Eight channels as they lie in memory (any alignment of the type's own).  A row's ragged last piece is read from the row's last eight
// channels and moved down when it is needed: a load of single values would be waited for on the spot, in every one of a row's operands
// (16 x 2304 x 643: 167 us the backward pass that way).
template <bool F32>
struct Eight {
    uint4 w[F32 ? 2 : 1];
    // left: channels of the row from here on; past: how many of the eight lie behind its end
    __device__ __forceinline__ void load(const void *base, int64_t at, int left, int past) {
        typedef typename Elem<F32>::T T;
        if (left > 0) {
            __builtin_memcpy(w, (const T *)base + at - past, sizeof(w));
        } else {
#pragma unroll
            for (int j = 0; j < (F32 ? 2 : 1); ++j) w[j] = make_uint4(0, 0, 0, 0);
        }
    }
    // `past` channels down, zeros behind
    __device__ __forceinline__ void settle(int past) {
        constexpr int N = F32 ? 8 : 4;               // words
        uint32_t u[N];
        __builtin_memcpy(u, w, sizeof(w));
#pragma unroll
        for (int by = N / 2; by > 0; by >>= 1) {
            const bool on = past & (F32 ? by : 2 * by);
#pragma unroll
            for (int j = 0; j < N; ++j) u[j] = on ? j + by < N ? u[j + by] : 0u : u[j];
        }
        if (!F32) {
            const uint32_t half = (past & 1) * 16;
#pragma unroll
            for (int j = 0; j < N; ++j) u[j] = __builtin_amdgcn_alignbit(j + 1 < N ? u[j + 1] : 0u, u[j], half);
        }
        __builtin_memcpy(w, u, sizeof(w));
    }
    __device__ __forceinline__ float get(int j) const {
        const uint32_t *u = (const uint32_t *)w;
        if constexpr (F32) return __uint_as_float(u[j]);
        else return j & 1 ? a2f_hi(u[j >> 1]) : a2f_lo(u[j >> 1]);
    }
};
template <bool F32, bool TAIL>
__device__ __forceinline__ void put8(void *base, int64_t at, const float (&v)[8], int left) {
    typedef typename Elem<F32>::T T;
    T *p = (T *)base + at;
    if (left >= 8) {
        uint4 w[F32 ? 2 : 1];
        uint32_t *u = (uint32_t *)w;
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = pack_a2(v[2 * j], v[2 * j + 1]);
        }
        __builtin_memcpy(p, w, sizeof(w));
    } else if (TAIL) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) Elem<F32>::put(p + j, v[j]);
    }
}

// A thread's first piece of a row: its lane.  The ragged last piece reads channels of the piece in front of it, and a call may be in place: the
// two belong to one wave, whose loads of a row are issued in front of its stores.
template <bool SHARED, bool TAIL, int NTH>
__device__ __forceinline__ int piece_of(int L, int C) {
    const int lane = threadIdx.x & (L - 1);
    if (SHARED || !TAIL) return lane;
    const int last = (C >> 3) & (NTH - 1), a = (last + 1) & (NTH - 1), b = (last - 1) & (NTH - 1);
    return last & 63 ? lane : lane == a ? b : lane == b ? a : lane;
}

struct Plan {
    int L, run_rows, runs;                // lanes a row; rows of a run, runs of a picture
    int has;                              // which combined vectors there are
};
enum { HAS_A = 1, HAS_AB = 2, HAS_W = 4, HAS_S = 8 };

__device__ __forceinline__ float at(const float *v, int64_t i, float none) { return v ? v[i] : none; }
__device__ __forceinline__ float combined(const onedc_block_norm_params &p, int which, int64_t b, int c) {
    if (which == HAS_A || which == HAS_AB) {
        const float g = p.alpha * at(p.gate, b * p.gate_rs + c, 1.f);
        return which == HAS_A ? g * at(p.post_w, c, 1.f) : g * at(p.post_b, c, 0.f);
    }
    const float s = 1.f + at(p.scale, b * p.scale_rs + c, 0.f);
    return which == HAS_W ? s * at(p.w, c, 1.f) : __builtin_fmaf(s, at(p.b, c, 0.f), at(p.shift, b * p.shift_rs + c, 0.f));
}

// One combined vector of a picture: in LDS (SHARED), or this thread's channels of it in registers
template <int IT, bool SHARED, int WHICH>
struct Vector {
    float v[SHARED ? 1 : IT][8];
    const float *lds;
    int last;
    bool on;
    // lds: where the next vector begins
    __device__ __forceinline__ void make(const onedc_block_norm_params &p, bool on_, int64_t b, int c0, int step, float *&at_lds) {
        on = on_;
        if (!on) return;
        if constexpr (SHARED) {
            last = ((p.C + 7) & ~7) - (WHICH == HAS_A ? 0 : 8);
            for (int c = threadIdx.x; c < ((p.C + 7) & ~7); c += blockDim.x) at_lds[c] = c < p.C ? combined(p, WHICH, b, c) : 0.f;
            if (WHICH == HAS_A && threadIdx.x < 8) at_lds[last + threadIdx.x] = 0.f;
            lds = at_lds;
            at_lds += last + 8;
        } else {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = c0 + i * step + j;
                    const float q = combined(p, WHICH, b, min(c, p.C - 1));
                    v[i][j] = WHICH != HAS_A || c < p.C ? q : 0.f;
                }
        }
    }
    // eight of them from channel c on; a piece behind the row gets the last ones, which multiply zeros and are not stored, but of A zeros: an
    // infinite gate there would make a sum over the row no number
    __device__ __forceinline__ void get(int i, int c, float (&o)[8]) const {
        if constexpr (SHARED) {
            c = min(c, last);
            const f32x4 a = *(const f32x4 *)(lds + c), b = *(const f32x4 *)(lds + c + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = a[j], o[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = v[i][j];
        }
    }
};

// v -> (v - mean) * r in place; values behind C stay 0.  Returns r.
template <bool TAIL, int IT, class Sum>
__device__ __forceinline__ float normalise(float (&v)[IT][8], int c0, int step, int C, int kind, float eps, Sum &sum) {
    if (kind == ONEDC_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
        const float m = sum.mean(s);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const float mi = c0 + i * step < C ? m : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = TAIL && c0 + i * step + j >= C ? 0.f : v[i][j] - mi;
        }
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) q = __builtin_fmaf(v[i][j], v[i][j], q);
    const float r = rsqrtf(sum.template mean<true>(q) + eps);         // (0 where the squares leave f32's range)
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= r;
    return r;
}

// What a call has, known to the compiler for the join between two sub-blocks in full; GENERIC asks the arguments (join and norm with a post_b:
// 16 x 9216 x 320 85 us against 84 without, 16 x 2304 x 640 39 against 35, 16 x 576 x 1280 25 against 23).
enum { GENERIC = 0, JOIN = 1, JOIN_POST = 2 };

// NTH 256: rows of up to 64 lanes (SHARED), or one row a workgroup
template <int NTH, bool SHARED, int IT, bool X32, bool F32, bool TAIL, int OPT>
__global__ __launch_bounds__(NTH, NTH > 256 ? 1 : IT > 2 ? 3 : 4) void block_norm_rows_kernel(onedc_block_norm_params p, Plan pl) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const bool has_f = OPT || p.f, has_y = OPT || p.y, post = OPT ? OPT == JOIN_POST : p.post;
    const int b = blockIdx.x / pl.runs, run = blockIdx.x - b * pl.runs;
    const int L = SHARED ? pl.L : NTH, step = 8 * L, c0 = piece_of<SHARED, TAIL, NTH>(L, p.C) * 8, each = NTH / L;
    float *at_lds = lds + 4 * (NTH / 64);
    Vector<IT, SHARED, HAS_A> A;
    Vector<IT, SHARED, HAS_AB> Ab;
    Vector<IT, SHARED, HAS_W> W;
    Vector<IT, SHARED, HAS_S> S;
    A.make(p, OPT || pl.has & HAS_A, b, c0, step, at_lds);
    Ab.make(p, !OPT && pl.has & HAS_AB, b, c0, step, at_lds);
    W.make(p, OPT || pl.has & HAS_W, b, c0, step, at_lds);
    S.make(p, OPT || pl.has & HAS_S, b, c0, step, at_lds);
    RowSum<NTH, SHARED> sum = {lds, L, 0, (float)p.C, 1.f / (float)p.C};
    const int n1 = min(p.N, (run + 1) * pl.run_rows);
    const int64_t row0 = (int64_t)b * p.N;
    Eight<X32> x[IT];
    Eight<F32> f[IT];
    auto past = [&](int i) { return TAIL ? max(c0 + i * step + 8 - p.C, 0) & 7 : 0; };       // (8 on: a piece behind the row)
    auto settle = [&](auto &piece, int i) {
        if (TAIL) piece.settle(past(i));
    };
    auto load = [&](auto &to, const void *from, int cs, int co, int n) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + i * step;
            to[i].load(from, (row0 + n) * cs + co + c, n < n1 ? p.C - c : 0, past(i));
        }
    };
    int n = run * pl.run_rows + threadIdx.x / L;
    load(x, p.x, p.x_cs, p.x_co, n);
    if (has_f) load(f, p.f, p.f_cs, p.f_co, n);
    __syncthreads();
    int cl = c0;
    // (every thread makes every turn: sums over a workgroup have barriers)
    for (int left_rows = n1 - run * pl.run_rows; left_rows > 0; left_rows -= each, n += each) {
        if (SHARED && IT > 1) asm volatile("" : "+v"(cl));        // (else the compiler keeps all of a thread's LDS vectors in registers, and spills)
        const bool more = left_rows > each;
        float t[IT][8];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            settle(x[i], i);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = x[i].get(j);
        }
        if (more) load(x, p.x, p.x_cs, p.x_co, n + each);
        if (has_f) {
            float v[IT][8];
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                settle(f[i], i);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = f[i].get(j);
            }
            if (more) load(f, p.f, p.f_cs, p.f_co, n + each);
            if (post) normalise<TAIL>(v, c0, step, p.C, p.kind, p.eps, sum);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = c0 + i * step;
                float a[8];
                if (A.on) A.get(i, cl + i * step, a);
#pragma unroll
                for (int j = 0; j < 8; ++j) t[i][j] = __builtin_fmaf(A.on ? a[j] : p.alpha, v[i][j], t[i][j]);
                if (Ab.on) {
                    Ab.get(i, cl + i * step, a);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[i][j] += c + (TAIL ? j : 0) < p.C ? a[j] : 0.f;
                }
                if (c < p.C && n < n1) put8<X32, TAIL>(p.xo, (row0 + n) * p.xo_cs + p.xo_co + c, t[i], p.C - c);
            }
        }
        if (has_y) {
            normalise<TAIL>(t, c0, step, p.C, p.kind, p.eps, sum);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = c0 + i * step;
                float w[8];
                if (W.on) {
                    W.get(i, cl + i * step, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[i][j] *= w[j];
                }
                if (S.on) {
                    S.get(i, cl + i * step, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[i][j] += w[j];
                }
                if (c < p.C && n < n1) put8<F32, TAIL>(p.y, (row0 + n) * p.y_cs + p.y_co + c, t[i], p.C - c);
            }
        }
    }
}

// Backward: dx and df of a row; a thread keeps the four sums of its channels over its run of rows, the lane groups of a workgroup add
// theirs in a fixed order, and part[run of a picture][4][C rounded up to 8] goes to the next kernel.
template <int NTH, bool SHARED, int IT, bool X32, bool F32, bool TAIL, int OPT>
__global__ __launch_bounds__(NTH, NTH > 256 ? 1 : IT > 1 ? 2 : 3) void block_norm_rows_backward_kernel(onedc_block_norm_params p,
                                                                                                       onedc_block_norm_grad g, Plan pl, float *part) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const bool has_f = OPT || p.f, has_dy = OPT || g.dy, has_dxo = OPT || g.dxo, has_dx = OPT || g.dx, has_df = OPT || g.df;
    const bool post = OPT ? OPT == JOIN_POST : p.post;
    const int b = blockIdx.x / pl.runs, run = blockIdx.x - b * pl.runs;
    const int L = SHARED ? pl.L : NTH, step = 8 * L, c0 = piece_of<SHARED, TAIL, NTH>(L, p.C) * 8, each = NTH / L;
    float *at_lds = lds + 4 * (NTH / 64);
    Vector<IT, SHARED, HAS_A> A;
    Vector<IT, SHARED, HAS_W> W;
    A.make(p, OPT || pl.has & HAS_A, b, c0, step, at_lds);
    W.make(p, OPT || pl.has & HAS_W, b, c0, step, at_lds);
    RowSum<NTH, SHARED> sum = {lds, L, 0, (float)p.C, 1.f / (float)p.C};
    const int n1 = min(p.N, (run + 1) * pl.run_rows);
    const int64_t row0 = (int64_t)b * p.N;
    // (raw until they are needed, and replaced by the next row's at once: rows of two pieces a lane fit 256 registers so)
    Eight<X32> rt[IT], rd[IT];
    Eight<F32> rf[IT], ry[IT];
    auto past = [&](int i) { return TAIL ? max(c0 + i * step + 8 - p.C, 0) & 7 : 0; };       // (8 on: a piece behind the row)
    auto settle = [&](auto &piece, int i) {
        if (TAIL) piece.settle(past(i));
    };
    auto load = [&](auto &to, const void *from, int cs, int co, int n) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + i * step;
            to[i].load(from, (row0 + n) * cs + co + c, n < n1 ? p.C - c : 0, past(i));
        }
    };
    float s1[IT][8], s2[IT][8], t1[IT][8], t2[IT][8];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s1[i][j] = s2[i][j] = t1[i][j] = t2[i][j] = 0.f;
    int n = run * pl.run_rows + threadIdx.x / L;
    if (has_dy) {
        load(rt, p.x, p.x_cs, p.x_co, n);
        load(ry, g.dy, g.dy_cs, g.dy_co, n);
    }
    if (has_dxo) load(rd, g.dxo, g.dxo_cs, g.dxo_co, n);
    if (has_f) load(rf, p.f, p.f_cs, p.f_co, n);
    __syncthreads();
    int cl = c0;
    for (int left_rows = n1 - run * pl.run_rows; left_rows > 0; left_rows -= each, n += each) {
        if (SHARED) asm volatile("" : "+v"(cl));
        const bool more = left_rows > each;
        const float eps = n < n1 ? p.eps : 1.f;          // (a lane group without a row has zeros: they must not meet an infinite r in the sums)
        float d[IT][8], f[IT][8];
        if (has_dy) {
            float h[IT][8], u[IT][8];
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                settle(rt[i], i), settle(ry[i], i);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = rt[i].get(j), u[i][j] = ry[i].get(j);
            }
            if (more) {
                load(rt, p.x, p.x_cs, p.x_co, n + each);
                load(ry, g.dy, g.dy_cs, g.dy_co, n + each);
            }
            const float r = normalise<TAIL>(h, c0, step, p.C, p.kind, eps, sum);
            float su = 0.f, sh = 0.f;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                float w[8];
                if (W.on) W.get(i, cl + i * step, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    s1[i][j] += u[i][j];
                    s2[i][j] = __builtin_fmaf(u[i][j], h[i][j], s2[i][j]);
                    if (W.on) u[i][j] *= w[j];
                    su += u[i][j];
                    sh = __builtin_fmaf(u[i][j], h[i][j], sh);
                }
            }
            const float2 m = sum.means(su, sh);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const float mu = p.kind == ONEDC_NORM_LAYER && c0 + i * step < p.C ? m.x : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    d[i][j] = r * (u[i][j] - mu - h[i][j] * m.y);
                    if (TAIL && c0 + i * step + j >= p.C) d[i][j] = 0.f;
                }
            }
        }
        if (has_dxo) {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                settle(rd[i], i);
#pragma unroll
                for (int j = 0; j < 8; ++j) d[i][j] = has_dy ? d[i][j] + rd[i].get(j) : rd[i].get(j);
            }
            if (more) load(rd, g.dxo, g.dxo_cs, g.dxo_co, n + each);
        }
        if (has_dx && n < n1) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if (c0 + i * step < p.C) put8<X32, TAIL>(g.dx, (row0 + n) * g.dx_cs + g.dx_co + c0 + i * step, d[i], p.C - c0 - i * step);
        }
        if (has_f) {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                settle(rf[i], i);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[i][j] = rf[i].get(j);
            }
            if (more) load(rf, p.f, p.f_cs, p.f_co, n + each);
        } else {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
        }
        float r = 1.f;
        if (post) r = normalise<TAIL>(f, c0, step, p.C, p.kind, eps, sum);
        float sv = 0.f, sf = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            float a[8];
            if (A.on) A.get(i, cl + i * step, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t1[i][j] += d[i][j];
                t2[i][j] = __builtin_fmaf(d[i][j], f[i][j], t2[i][j]);
                d[i][j] *= A.on ? a[j] : p.alpha;
                sv += d[i][j];
                sf = __builtin_fmaf(d[i][j], f[i][j], sf);
            }
        }
        if (!has_df) continue;
        if (post) {
            const float2 m = sum.means(sv, sf);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const float mv = p.kind == ONEDC_NORM_LAYER ? m.x : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) d[i][j] = r * (d[i][j] - mv - f[i][j] * m.y);
            }
        }
        if (n < n1) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if (c0 + i * step < p.C) put8<F32, TAIL>(g.df, (row0 + n) * g.df_cs + g.df_co + c0 + i * step, d[i], p.C - c0 - i * step);
        }
    }
    if (!part) return;
    const int C8 = (p.C + 7) & ~7;
    f32x4 *out = (f32x4 *)(part + (int64_t)blockIdx.x * 4 * C8);
    if constexpr (!SHARED) {                         // the thread's channels are nobody else's
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + i * step;
            if (c >= p.C) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float(&v)[8] = q == 0 ? s1[i] : q == 1 ? s2[i] : q == 2 ? t1[i] : t2[i];
                out[(q * C8 + c) / 4] = f32x4{v[0], v[1], v[2], v[3]};
                out[(q * C8 + c) / 4 + 1] = f32x4{v[4], v[5], v[6], v[7]};
            }
        }
    } else {
        // the lane groups of a wave by exchanges, then the waves in turn
        auto add_groups = [&](float (&v)[IT][8]) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = groups_sum(v[i][j], L);
        };
        add_groups(s1), add_groups(s2), add_groups(t1), add_groups(t2);
        float *acc = lds + 4 * (NTH / 64);           // over the vectors
        for (int k = 0; k < NTH / 64; ++k) {
            __syncthreads();
            if ((int)(threadIdx.x >> 6) != k || (int)(threadIdx.x & 63) >= L) continue;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = c0 + i * step;
                if (c >= p.C) continue;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float(&v)[8] = q == 0 ? s1[i] : q == 1 ? s2[i] : q == 2 ? t1[i] : t2[i];
                    f32x4 *to = (f32x4 *)(acc + q * C8 + c);
                    f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
                    if (k) lo += to[0], hi += to[1];
                    to[0] = lo, to[1] = hi;
                }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < C8; c += NTH) out[c] = ((const f32x4 *)acc)[c];
    }
}

// ---- wider rows, and rows of less than a piece: a workgroup passes over its row again for every sum ----------------------------------------
// Bound by the latency of those passes, which come from the caches: 512 x 20000 in 85 us (1.0 TB/s), backward 286 us (256 threads a row instead
// of 1024: 212 and 494); a million rows of four channels 676 us, backward 1.3 ms.
constexpr int NTW = 1024;
int simple_threads(int C) { return C < 8 ? 64 : NTW; }

// sum of v over the workgroup, the same value in every thread
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += red[i];
    return s;
}

// mean (0 for RMSNorm) and reciprocal deviation of the C values v(c)
template <class V>
__device__ __forceinline__ float2 row_norm(V v, int C, int kind, float eps, float *red) {
    float m = 0.f;
    if (kind == ONEDC_NORM_LAYER) {
        float s = 0.f;
        for (int c = threadIdx.x; c < C; c += blockDim.x) s += v(c);
        m = block_sum(s, red) / C;
    }
    float q = 0.f;
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
        const float d = v(c) - m;
        q += d * d;
    }
    return make_float2(m, rsqrtf(block_sum(q, red) / C + eps));
}

template <bool X32, bool F32>
__global__ __launch_bounds__(NTW) void block_norm_kernel(onedc_block_norm_params p) {
    typedef Elem<X32> X;
    typedef Elem<F32> F;
    __shared__ float red[NTW / 64];
    for (int64_t row = blockIdx.x; row < (int64_t)p.B * p.N; row += gridDim.x) {
        const int64_t b = row / p.N;
        const typename X::T *x = (const typename X::T *)p.x + row * p.x_cs + p.x_co;
        const typename F::T *f = p.f ? (const typename F::T *)p.f + row * p.f_cs + p.f_co : nullptr;
        const float *gate = p.gate ? p.gate + b * p.gate_rs : nullptr;
        float2 fn = make_float2(0.f, 1.f);
        if (p.post) fn = row_norm([&](int c) { return F::get(f + c); }, p.C, p.kind, p.eps, red);
        auto joined = [&](int c) {
            float t = X::get(x + c);
            if (f) {
                const float v = (F::get(f + c) - fn.x) * fn.y * at(p.post_w, c, 1.f) + at(p.post_b, c, 0.f);
                t = __builtin_fmaf(p.alpha * at(gate, c, 1.f), v, t);
            }
            return t;
        };
        if (p.y) {
            const float2 tn = row_norm(joined, p.C, p.kind, p.eps, red);
            const float *scale = p.scale ? p.scale + b * p.scale_rs : nullptr, *shift = p.shift ? p.shift + b * p.shift_rs : nullptr;
            typename F::T *y = (typename F::T *)p.y + row * p.y_cs + p.y_co;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                const float v = (joined(c) - tn.x) * tn.y * at(p.w, c, 1.f) + at(p.b, c, 0.f);
                F::put(y + c, __builtin_fmaf(v, 1.f + at(scale, c, 0.f), at(shift, c, 0.f)));
            }
        }
        if (p.xo) {                                      // (behind the norm's passes: xo may be x)
            typename X::T *xo = (typename X::T *)p.xo + row * p.xo_cs + p.xo_co;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) X::put(xo + c, joined(c));
        }
    }
}

// dx and df of a row, and the row's four column terms added to this run's sums: sums[4][C rounded up to 8] in memory, one column
// owned by one thread for the whole run (fixed order)
template <bool X32, bool F32>
__global__ __launch_bounds__(NTW) void block_norm_backward_kernel(onedc_block_norm_params p, onedc_block_norm_grad g, float *part,
                                                                 int runs, int run_rows) {
    typedef Elem<X32> X;
    typedef Elem<F32> F;
    __shared__ float red[NTW / 64];
    const int b = blockIdx.x / runs, run = blockIdx.x - b * runs;
    const int n0 = run * run_rows, n1 = min(p.N, n0 + run_rows);
    const float *gate = p.gate ? p.gate + (int64_t)b * p.gate_rs : nullptr;
    const float *scale = p.scale ? p.scale + (int64_t)b * p.scale_rs : nullptr;
    const int C8 = (p.C + 7) & ~7;
    float *sums = part ? part + (int64_t)blockIdx.x * 4 * C8 : nullptr;
    if (sums)
        for (int c = threadIdx.x; c < 4 * C8; c += blockDim.x) sums[c] = 0.f;      // (a thread's own columns differ from these: barrier below)
    __syncthreads();
    for (int n = n0; n < n1; ++n) {
        const int64_t row = (int64_t)b * p.N + n;
        const typename X::T *t = (const typename X::T *)p.x + row * p.x_cs + p.x_co;
        const typename F::T *f = p.f ? (const typename F::T *)p.f + row * p.f_cs + p.f_co : nullptr;
        const typename F::T *dy = g.dy ? (const typename F::T *)g.dy + row * g.dy_cs + g.dy_co : nullptr;
        const typename X::T *dxo = g.dxo ? (const typename X::T *)g.dxo + row * g.dxo_cs + g.dxo_co : nullptr;
        float2 tn = make_float2(0.f, 0.f), fn = make_float2(0.f, 1.f);
        float mu = 0.f, mh = 0.f;
        auto hat = [&](int c) { return (X::get(t + c) - tn.x) * tn.y; };
        auto u = [&](int c) { return F::get(dy + c) * (1.f + at(scale, c, 0.f)) * at(p.w, c, 1.f); };
        if (dy) {
            tn = row_norm([&](int c) { return X::get(t + c); }, p.C, p.kind, p.eps, red);
            float su = 0.f, sh = 0.f;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                const float v = u(c);
                su += v;
                sh += v * hat(c);
            }
            mu = p.kind == ONEDC_NORM_LAYER ? block_sum(su, red) / p.C : 0.f;
            mh = block_sum(sh, red) / p.C;
        }
        auto dt = [&](int c) {
            float v = dxo ? X::get(dxo + c) : 0.f;
            if (dy) v += tn.y * (u(c) - mu - hat(c) * mh);
            return v;
        };
        auto fhat = [&](int c) { return (F::get(f + c) - fn.x) * fn.y; };
        auto w = [&](int c) { return dt(c) * p.alpha * at(gate, c, 1.f) * at(p.post_w, c, 1.f); };
        float mw = 0.f, mf = 0.f;
        if (p.post) {
            fn = row_norm([&](int c) { return F::get(f + c); }, p.C, p.kind, p.eps, red);
            float sw = 0.f, sf = 0.f;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                const float v = w(c);
                sw += v;
                sf += v * fhat(c);
            }
            mw = p.kind == ONEDC_NORM_LAYER ? block_sum(sw, red) / p.C : 0.f;
            mf = block_sum(sf, red) / p.C;
        }
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
            const float d = dt(c), fh = f ? fhat(c) : 0.f;
            if (sums) {
                const float e = dy ? F::get(dy + c) : 0.f;
                sums[c] += e;
                sums[C8 + c] += dy ? e * hat(c) : 0.f;
                sums[2 * C8 + c] += d;
                sums[3 * C8 + c] += d * fh;
            }
            // (dx may be dxo, df may be dy: this thread's own columns, read above)
            const float wc = w(c);
            if (g.dx) X::put((typename X::T *)g.dx + row * g.dx_cs + g.dx_co + c, d);
            if (g.df) F::put((typename F::T *)g.df + row * g.df_cs + g.df_co + c, p.post ? fn.y * (wc - mw - fh * mf) : wc);
        }
        __syncthreads();
    }
}

// The parameter gradients, in f64 and in a fixed order.  First a picture: 32 channels x 32 shares of its runs a workgroup.  What has a row
// per picture is finished here; the picture's parts of what is summed over the pictures go on, parts[picture][7][C].
enum { P_GATE, P_SCALE, P_SHIFT, P_W, P_B, P_POST_W, P_POST_B, PARTS };
__device__ __forceinline__ void finish(const onedc_block_norm_params &p, const onedc_block_norm_grad &g, int c, const double (&t)[PARTS]) {
    if (g.d_gate && !p.gate_rs) g.d_gate[c] = (float)t[P_GATE];
    if (g.d_scale && !p.scale_rs) g.d_scale[c] = (float)t[P_SCALE];
    if (g.d_shift && !p.shift_rs) g.d_shift[c] = (float)t[P_SHIFT];
    if (g.d_w) g.d_w[c] = (float)t[P_W];
    if (g.d_b) g.d_b[c] = (float)t[P_B];
    if (g.d_post_w) g.d_post_w[c] = (float)t[P_POST_W];
    if (g.d_post_b) g.d_post_b[c] = (float)t[P_POST_B];
}

__global__ __launch_bounds__(NT) void block_norm_picture_kernel(onedc_block_norm_params p, onedc_block_norm_grad g, const float *part, double *parts,
                                                                int runs) {
    __shared__ double red[32][4][32];
    const int columns = (p.C + 31) / 32, C8 = (p.C + 7) & ~7;
    const int64_t b = blockIdx.x / columns;
    const int first = (int)(blockIdx.x - b * columns) * 32, share = threadIdx.x >> 3, at4 = (threadIdx.x & 7) * 4;
    double sum[4][4] = {};
    if (first + at4 < p.C)
#pragma unroll 2
        for (int r = share; r < runs; r += 32)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x4 v = *(const f32x4 *)(part + ((b * runs + r) * 4 + k) * C8 + first + at4);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[k][e] += v[e];
            }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[share][k][at4 + e] = sum[k][e];
    __syncthreads();
    // two threads a sum, sixteen shares each
    const int which = threadIdx.x & 127, half = threadIdx.x >> 7;
    double total = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += red[half * 16 + i][which >> 5][which & 31];
    __syncthreads();
    red[half][which >> 5][which & 31] = total;
    __syncthreads();
    const int c = first + threadIdx.x;
    if (threadIdx.x >= 32 || c >= p.C) return;
    double s[4];                                     // S1, S2, T1, T2
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = red[0][k][threadIdx.x] + red[1][k][threadIdx.x];
    const double w = at(p.w, c, 1.f), bb = at(p.b, c, 0.f), pw = at(p.post_w, c, 1.f), pb = at(p.post_b, c, 0.f);
    const double sc = 1.0 + at(p.scale, b * p.scale_rs + c, 0.f), ga = p.alpha * (double)at(p.gate, b * p.gate_rs + c, 1.f);
    const double t[PARTS] = {p.alpha * (pw * s[3] + pb * s[2]), w * s[1] + bb * s[0], s[0], sc * s[1], sc * s[0], ga * s[3], ga * s[2]};
    if (g.d_gate && p.gate_rs) g.d_gate[b * p.C + c] = (float)t[P_GATE];
    if (g.d_scale && p.scale_rs) g.d_scale[b * p.C + c] = (float)t[P_SCALE];
    if (g.d_shift && p.shift_rs) g.d_shift[b * p.C + c] = (float)t[P_SHIFT];
    if (parts) {
#pragma unroll
        for (int k = 0; k < PARTS; ++k) parts[(b * PARTS + k) * p.C + c] = t[k];
    } else if (p.B == 1) {
        finish(p, g, c, t);
    }
}
// then the pictures: 16 channels x 16 shares of them a workgroup
__global__ __launch_bounds__(NT) void block_norm_all_kernel(onedc_block_norm_params p, onedc_block_norm_grad g, const double *parts) {
    __shared__ double red[16][PARTS][16];
    const int lane = threadIdx.x & 15, share = threadIdx.x >> 4, c = blockIdx.x * 16 + lane;
    double t[PARTS] = {0, 0, 0, 0, 0, 0, 0};
    if (c < p.C)
        for (int64_t b = share; b < p.B; b += 16)
#pragma unroll
            for (int k = 0; k < PARTS; ++k) t[k] += parts[(b * PARTS + k) * p.C + c];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) red[share][k][lane] = t[k];
    __syncthreads();
    if (share || c >= p.C) return;
    for (int i = 1; i < 16; ++i)
#pragma unroll
        for (int k = 0; k < PARTS; ++k) t[k] += red[i][k][lane];
    finish(p, g, c, t);
}

int check_view(const void *p, int cs, int co, int C) { return !p || (cs >= C && co >= 0 && co <= cs - C) ? 0 : -2; }

int check_common(const onedc_block_norm_params *p) {
    if (!p) return -1;
    // (2^30 rows: a run of them, and the workgroup's turn behind it, are counted in 31 bits)
    if (p->B < 0 || p->N < 0 || p->C < 1 || p->C > (1 << 20) || (int64_t)p->B * p->N > (1 << 30)) return -2;
    if (!p->B || !p->N) return 0;                    // no rows: nothing is read or written (the pointers of empty tensors are NULL)
    if (!p->x) return -1;
    if (check_view(p->x, p->x_cs, p->x_co, p->C) || check_view(p->f, p->f_cs, p->f_co, p->C)) return -2;
    if (p->gate_rs < 0 || p->scale_rs < 0 || p->shift_rs < 0) return -2;
    if (p->kind != ONEDC_NORM_LAYER && p->kind != ONEDC_NORM_RMS) return -3;
    if (p->f_f32 && !p->x_f32) return -3;
    if (!p->f && (p->post || p->gate)) return -3;
    if (!p->post && (p->post_w || p->post_b)) return -3;
    return 0;
}

bool wants_sums(const onedc_block_norm_grad *g) {
    return g->d_post_w || g->d_post_b || g->d_gate || g->d_w || g->d_b || g->d_scale || g->d_shift;
}
bool wants_all(const onedc_block_norm_params *p, const onedc_block_norm_grad *g) {
    return g->d_post_w || g->d_post_b || g->d_w || g->d_b || (g->d_gate && !p->gate_rs) || (g->d_scale && !p->scale_rs) || (g->d_shift && !p->shift_rs);
}
// Without a parameter per picture the pictures are one.
onedc_block_norm_params joined_pictures(const onedc_block_norm_params *p) {
    onedc_block_norm_params q = *p;
    if (!p->gate_rs && !p->scale_rs && !p->shift_rs) {
        q.N = p->B * p->N;
        q.B = q.N ? 1 : 0;
    }
    return q;
}

// The vectors that a call reads: per channel, and per picture
constexpr int VECTORS = 7;
void vectors_of(const onedc_block_norm_params *p, OnedcMem (&m)[VECTORS]) {
    const auto each = [&](const float *v, int rs) { return onedc_mem_rows(v, rs ? p->B : 1, rs, 0, p->C, 4); };
    const float *all[] = {p->post_w, p->post_b, p->w, p->b};
    for (int i = 0; i < 4; ++i) m[i] = onedc_mem(all[i], (int64_t)p->C * 4);
    m[4] = each(p->gate, p->gate_rs), m[5] = each(p->scale, p->scale_rs), m[6] = each(p->shift, p->shift_rs);
}
OnedcMem rows_of(const onedc_block_norm_params *p, const void *t, int cs, int co, int f32) {
    return onedc_mem_rows(t, (int64_t)p->B * p->N, cs, co, p->C, f32 ? 4 : 2);
}
// A parameter's gradient lies apart from everything else; dx and df apart from the vectors (from rows of x, f, dy and dxo: the caller's affair, who
// may name some of them again); the workspace apart from all
bool gradients_apart(const onedc_block_norm_params *p, const onedc_block_norm_grad *g, int64_t need) {
    OnedcMem v[VECTORS];
    vectors_of(p, v);
    const int64_t one = (int64_t)p->C * 4, each = one * p->B;
    const OnedcMem d[] = {onedc_mem(g->d_post_w, one), onedc_mem(g->d_post_b, one), onedc_mem(g->d_w, one), onedc_mem(g->d_b, one),
                          onedc_mem(g->d_gate, p->gate_rs ? each : one), onedc_mem(g->d_scale, p->scale_rs ? each : one),
                          onedc_mem(g->d_shift, p->shift_rs ? each : one), onedc_mem(need ? g->ws : nullptr, need)};
    const OnedcMem out[] = {rows_of(p, g->dx, g->dx_cs, g->dx_co, p->x_f32), rows_of(p, g->df, g->df_cs, g->df_co, p->f_f32)};
    const OnedcMem in[] = {rows_of(p, p->x, p->x_cs, p->x_co, p->x_f32), rows_of(p, p->f, p->f_cs, p->f_co, p->f_f32),
                           rows_of(p, g->dy, g->dy_cs, g->dy_co, p->f_f32), rows_of(p, g->dxo, g->dxo_cs, g->dxo_co, p->x_f32)};
    if (onedc_mem_any_shared(d, v) || onedc_mem_any_shared(d, out) || onedc_mem_any_shared(d, in) || onedc_mem_any_shared(out, v)) return false;
    for (const OnedcMem *a = d; a != std::end(d); ++a)
        for (const OnedcMem *b = d; b != a; ++b)
            if (onedc_mem_shared(*a, *b)) return false;
    return true;
}

// How rows lie in lanes, by the row's width alone.  Two pieces a lane, in as few lanes as that takes: 4.4 TB/s at 320 channels and 5.4 at
// 640 against 4.2 / 3.0 with one piece (twice the lanes, half of them idle) and, three pieces, 4.3 / 5.0; five pieces spill.  Three where two
// of 64 lanes end (1280 channels: 4.3 against 3.8 for one row a workgroup), but not with a ragged end, whose code takes their registers.
// Wider rows belong to a workgroup each, one piece a thread (two from 8192 channels on, forward).
struct Shape {
    int threads, it;                      // threads a workgroup; pieces a lane; 0: not a row for registers
    bool shared;                          // several rows a workgroup
};
Shape row_shape(int C, int widest, bool back, int *L) {
    const int pieces = (C + 7) / 8;
    Shape s = {NT, 0, true};
    if (C < 8) return s;                             // (less than a piece: the simple kernel)
    for (*L = 8; *L <= 64; *L *= 2)
        if (pieces <= 2 * *L) {
            s.it = pieces <= *L ? 1 : 2;
            return s;
        }
    *L = 64;
    if (pieces <= 192 && C % 8 == 0 && !back) {
        s.it = 3;
        return s;
    }
    s.shared = false;
    for (s.threads = 256; s.threads <= 1024; s.threads *= 2)
        if (pieces <= s.threads) {
            s.it = 1;
            break;
        }
    if (!s.it && C <= widest) s.threads = 1024, s.it = 2;
    *L = s.threads;
    return s;
}
// a run: whole turns of a workgroup; about `want` runs altogether
void cut_runs(const onedc_block_norm_params &p, int each, int want, Plan *pl) {
    const int turns = (p.N + each - 1) / each;
    want = (want + p.B - 1) / p.B;
    want = want < 1 ? 1 : want > turns ? turns : want;
    pl->run_rows = (turns + want - 1) / want * each;
    pl->runs = (p.N + pl->run_rows - 1) / pl->run_rows;
}
// of the workspace: the pictures' sums, in front of the runs' (whole 16 bytes)
int64_t pictures_bytes(const onedc_block_norm_params &q, const onedc_block_norm_grad *g) {
    return q.B > 1 && wants_all(&q, g) ? (((int64_t)q.B * q.C * PARTS * (int64_t)sizeof(double) + 15) & ~15ll) : 0;
}
constexpr int WIDEST = 16384, WIDEST_BACK = 8192;
constexpr int SIMPLE_RUNS = 512;

// shape and runs of a backward pass; false: the simple kernel (it cuts runs of its own)
bool backward_plan(const onedc_block_norm_params &p, bool sums, Shape *s, Plan *pl) {
    *s = row_shape(p.C, WIDEST_BACK, true, &pl->L);
    if (!s->it) {
        cut_runs(p, 1, p.C < 8 ? 32 * SIMPLE_RUNS : SIMPLE_RUNS, pl);
        return false;
    }
    const int each = s->threads / pl->L;
    int want = s->threads == NT ? 1024 : 512;
    if (sums) {                                      // fewer of them: a run's sums are 16 bytes a channel to write and to read
        const int64_t fours = (int64_t)p.B * p.N / (4 * each);
        want = fours < want / 2 ? (int)fours : want / 2;
        want = want < 256 ? 256 : want;
    }
    cut_runs(p, each, want, pl);
    pl->has = (p.f && (p.gate || p.post_w) ? HAS_A : 0) | (p.w || p.scale ? HAS_W : 0);
    return true;
}

// one instance of a kernel template for every shape, type and end of a row, and what the call has
template <class Call>
void by_shape(const Shape &s, bool x32, bool f32, bool tail, int opt, Call &&call) {
    auto types = [&](auto nth, auto shared, auto it) {
        auto ends = [&](auto x, auto f) {
            auto has = [&](auto end) {
                if (opt == JOIN) call(nth, shared, it, x, f, end, std::integral_constant<int, JOIN>());
                else if (opt == JOIN_POST) call(nth, shared, it, x, f, end, std::integral_constant<int, JOIN_POST>());
                else call(nth, shared, it, x, f, end, std::integral_constant<int, GENERIC>());
            };
            if (tail) has(std::true_type());
            else has(std::false_type());
        };
        if (f32) ends(std::true_type(), std::true_type());
        else if (x32) ends(std::true_type(), std::false_type());
        else ends(std::false_type(), std::false_type());
    };
    typedef std::integral_constant<int, 1> I1;
    typedef std::integral_constant<int, 2> I2;
    typedef std::integral_constant<int, 3> I3;
    if (s.shared) {
        if (s.it == 1) types(std::integral_constant<int, NT>(), std::true_type(), I1());
        else if (s.it == 2) types(std::integral_constant<int, NT>(), std::true_type(), I2());
        else types(std::integral_constant<int, NT>(), std::true_type(), I3());
    } else if (s.threads == 256) {
        types(std::integral_constant<int, 256>(), std::false_type(), I1());
    } else if (s.threads == 512) {
        types(std::integral_constant<int, 512>(), std::false_type(), I1());
    } else if (s.it == 1) {
        types(std::integral_constant<int, 1024>(), std::false_type(), I1());
    } else {
        types(std::integral_constant<int, 1024>(), std::false_type(), I2());
    }
}

}  // namespace

extern "C" {

int onedc_block_norm(const onedc_block_norm_params *p, void *stream) {
    const int rc = check_common(p);
    if (rc) return rc;
    const int64_t rows = (int64_t)p->B * p->N;
    if (!rows) return 0;
    if (!p->y && !p->xo) return -1;
    if (check_view(p->xo, p->xo_cs, p->xo_co, p->C) || check_view(p->y, p->y_cs, p->y_co, p->C)) return -2;
    if (!p->f != !p->xo) return -3;
    if (!p->y && (p->w || p->b || p->scale || p->shift)) return -3;
    OnedcMem vectors[VECTORS];
    vectors_of(p, vectors);
    const OnedcMem out[] = {rows_of(p, p->xo, p->xo_cs, p->xo_co, p->x_f32), rows_of(p, p->y, p->y_cs, p->y_co, p->f_f32)};
    if (onedc_mem_any_shared(out, vectors)) return ONEDC_SHARED_MEMORY;
    const onedc_block_norm_params q = joined_pictures(p);
    Plan pl;
    const Shape shape = row_shape(p->C, WIDEST, false, &pl.L);
    if (shape.it) {
        pl.has = (p->f && (p->gate || p->post_w) ? HAS_A : 0) | (p->f && p->post_b ? HAS_AB : 0) | (p->y && (p->w || p->scale) ? HAS_W : 0) |
                 (p->y && (p->b || p->shift) ? HAS_S : 0);
        cut_runs(q, shape.threads / pl.L, shape.threads > 256 ? 512 : 1024, &pl);
        if (!onedc_grid_fits((int64_t)q.B * pl.runs, shape.threads)) return -2;
        const int opt = !p->f || !p->y || p->post_b ? GENERIC : p->post ? JOIN_POST : JOIN;
        if (opt) pl.has = HAS_A | HAS_W | HAS_S;
        const size_t lds = shape.threads / 64 * 16 + (shape.shared ? (size_t)(__builtin_popcount(pl.has) * ((p->C + 7) & ~7) + 8) * 4 : 0);
        const dim3 grid((unsigned)((int64_t)q.B * pl.runs));
        by_shape(shape, p->x_f32, p->f_f32, p->C & 7, opt, [&](auto nth, auto shared, auto it, auto x32, auto f32, auto tail, auto what) {
            constexpr int NTH = decltype(nth)::value, IT = decltype(it)::value;
            constexpr bool SH = decltype(shared)::value, X = decltype(x32)::value, F = decltype(f32)::value, TL = decltype(tail)::value;
            constexpr int OPT = decltype(what)::value;
            hipLaunchKernelGGL((block_norm_rows_kernel<NTH, SH, IT, X, F, TL, OPT>), grid, dim3(NTH), lds, as_stream(stream), q, pl);
        });
        ONEDC_LAUNCH_CHECK();
        return 0;
    }
    if (p->f_f32)
        hipLaunchKernelGGL((block_norm_kernel<true, true>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(simple_threads(p->C)), 0, as_stream(stream), *p);
    else if (p->x_f32)
        hipLaunchKernelGGL((block_norm_kernel<true, false>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(simple_threads(p->C)), 0, as_stream(stream), *p);
    else
        hipLaunchKernelGGL((block_norm_kernel<false, false>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(simple_threads(p->C)), 0, as_stream(stream), *p);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

int64_t onedc_block_norm_backward_ws_bytes(const onedc_block_norm_params *p, const onedc_block_norm_grad *g) {
    if (check_common(p) || !g || !wants_sums(g) || !p->B || !p->N) return 0;
    const onedc_block_norm_params q = joined_pictures(p);
    Shape s;
    Plan pl;
    backward_plan(q, true, &s, &pl);
    return pictures_bytes(q, g) + (int64_t)q.B * pl.runs * 4 * ((p->C + 7) & ~7) * sizeof(float);
}

int onedc_block_norm_backward(const onedc_block_norm_params *p, const onedc_block_norm_grad *g, void *stream) {
    const int rc = check_common(p);
    if (rc) return rc;
    if (!g) return -1;
    const bool any = p->B && p->N;
    if (any) {
        if (!g->dy && !g->dxo) return -1;
        if (check_view(g->dy, g->dy_cs, g->dy_co, p->C) || check_view(g->dxo, g->dxo_cs, g->dxo_co, p->C) ||
            check_view(g->dx, g->dx_cs, g->dx_co, p->C) || check_view(g->df, g->df_cs, g->df_co, p->C))
            return -2;
        if (!g->dy && (p->w || p->b || p->scale || p->shift)) return -3;
        if ((g->df || g->d_gate || g->d_post_w || g->d_post_b) && !p->f) return -3;
        if ((g->d_gate && !p->gate) || (g->d_post_w && !p->post_w) || (g->d_post_b && !p->post_b) || (g->d_w && !p->w) || (g->d_b && !p->b) ||
            (g->d_scale && !p->scale) || (g->d_shift && !p->shift))
            return -3;
    }
    const bool sums = wants_sums(g);
    const onedc_block_norm_params q = joined_pictures(p);
    Shape shape;
    Plan pl;
    const bool rows = any && backward_plan(q, sums, &shape, &pl);
    if (any && !onedc_grid_fits((int64_t)q.B * pl.runs, rows ? shape.threads : simple_threads(p->C))) return -2;
    if (sums && !onedc_grid_fits((int64_t)(any ? q.B : p->B) * ((p->C + 31) / 32), NT)) return -2;
    const int64_t need = onedc_block_norm_backward_ws_bytes(p, g);
    if (need && (!g->ws || g->ws_bytes < need || (uintptr_t)g->ws & 15)) return -15;
    if (!gradients_apart(p, g, need)) return ONEDC_SHARED_MEMORY;
    if (!any) {
        if (sums) {                                  // no rows: every sum is 0
            onedc_block_norm_params none = *p;
            if (p->B) {
                hipLaunchKernelGGL(block_norm_picture_kernel, dim3((unsigned)((int64_t)p->B * ((p->C + 31) / 32))), dim3(NT), 0, as_stream(stream),
                                   none, *g, (const float *)nullptr, (double *)nullptr, 0);
                ONEDC_LAUNCH_CHECK();
            }
            none.B = 0;
            hipLaunchKernelGGL(block_norm_all_kernel, dim3((p->C + 15) / 16), dim3(NT), 0, as_stream(stream), none, *g, (const double *)nullptr);
            ONEDC_LAUNCH_CHECK();
        }
        return 0;
    }
    double *pictures = sums && pictures_bytes(q, g) ? (double *)g->ws : nullptr;
    float *part = sums ? (float *)((char *)g->ws + pictures_bytes(q, g)) : nullptr;
    const dim3 grid((unsigned)((int64_t)q.B * pl.runs));
    if (rows) {
        const size_t scratch = shape.shared ? (size_t)4 * ((p->C + 7) & ~7) * 4 : 0;          // (the vectors, two at most and A's zeros, then the sums)
        const size_t lds = shape.threads / 64 * 16 + scratch;
        const int opt = !p->f || !g->dy || !g->dxo || !g->dx || !g->df ? GENERIC : p->post ? JOIN_POST : JOIN;
        by_shape(shape, p->x_f32, p->f_f32, p->C & 7, opt, [&](auto nth, auto shared, auto it, auto x32, auto f32, auto tail, auto what) {
            constexpr int NTH = decltype(nth)::value, IT = decltype(it)::value;
            constexpr bool SH = decltype(shared)::value, X = decltype(x32)::value, F = decltype(f32)::value, TL = decltype(tail)::value;
            constexpr int OPT = decltype(what)::value;
            if constexpr (IT == 1 || (SH && IT == 2))
                hipLaunchKernelGGL((block_norm_rows_backward_kernel<NTH, SH, IT, X, F, TL, OPT>), grid, dim3(NTH), lds, as_stream(stream), q, *g, pl, part);
        });
    } else if (p->f_f32) {
        hipLaunchKernelGGL((block_norm_backward_kernel<true, true>), grid, dim3(simple_threads(p->C)), 0, as_stream(stream), q, *g, part, pl.runs, pl.run_rows);
    } else if (p->x_f32) {
        hipLaunchKernelGGL((block_norm_backward_kernel<true, false>), grid, dim3(simple_threads(p->C)), 0, as_stream(stream), q, *g, part, pl.runs, pl.run_rows);
    } else {
        hipLaunchKernelGGL((block_norm_backward_kernel<false, false>), grid, dim3(simple_threads(p->C)), 0, as_stream(stream), q, *g, part, pl.runs, pl.run_rows);
    }
    ONEDC_LAUNCH_CHECK();
    if (sums) {
        hipLaunchKernelGGL(block_norm_picture_kernel, dim3((unsigned)((int64_t)q.B * ((p->C + 31) / 32))), dim3(NT), 0, as_stream(stream), q, *g, part,
                           pictures, pl.runs);
        ONEDC_LAUNCH_CHECK();
        if (pictures) {
            hipLaunchKernelGGL(block_norm_all_kernel, dim3((p->C + 15) / 16), dim3(NT), 0, as_stream(stream), q, *g, (const double *)pictures);
            ONEDC_LAUNCH_CHECK();
        }
    }
    return 0;
}

}  // extern "C"
