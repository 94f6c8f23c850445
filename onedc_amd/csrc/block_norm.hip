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
#include "elem.h"

namespace {

constexpr int NT = 256;

// ---- rows in registers: up to MAX_C channels -------------------------------------------------------------------------------------------
// Bound by HBM: x and f are read once, xo and y written once (backward: four read, two written).  A row belongs to L neighbouring lanes
// (8 .. 64, or the whole workgroup), which hold it as IT pieces of eight channels each: piece i of lane l begins at channel 8 (i L + l).
// Statistics are two passes over registers -- mean, then squared deviations -- and log2 L exchanges between lanes.  A workgroup
// takes a run of rows of one picture, so that the vectors per picture (gate, scale, shift) and per channel are combined once, in LDS:
//   A = alpha gate post_w, Ab = alpha gate post_b (join);  W = w (1 + scale), S = b (1 + scale) + shift (norm behind it)
// and the next rows' loads are in flight while a row is computed.

// sum over the L neighbouring lanes of v's row, the same bits in each of them
template <int O>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), O, 0xf, 0xf, true));
}
__device__ __forceinline__ float lanes_sum(float v, int L) {
    v = dpp_add<0xb1>(v);                            // lane ^ 1
    v = dpp_add<0x4e>(v);                            // lane ^ 2
    v = dpp_add<0x141>(v);                           // mirrored within 8
    if (L > 8) v = dpp_add<0x140>(v);                // mirrored within 16
    if (L > 16) v += __shfl_xor(v, 16);
    if (L > 32) v += __shfl_xor(v, 32);
    return v;
}
// ... or over the workgroup; red: two floats a wave, alternated so that one barrier a sum is enough
struct RowSum {
    float *red;
    int L, turn;
    __device__ __forceinline__ float operator()(float v) {
        if (L <= 64) return lanes_sum(v, L);
        v = lanes_sum(v, 64);
        float *r = red + turn * (NT / 64);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
        return (r[0] + r[1]) + (r[2] + r[3]);
    }
};

// eight channels as they lie in memory (any alignment of the type's own)
template <bool F32>
struct Eight {
    uint4 w[F32 ? 2 : 1];
    // TAIL: the row may end inside the piece
    template <bool TAIL>
    __device__ __forceinline__ void load(const void *base, int64_t at, int left) {
        typedef typename Elem<F32>::T T;
        const T *p = (const T *)base + at;
        if (left >= 8) {
            __builtin_memcpy(w, p, sizeof(w));
        } else if (!TAIL) {
#pragma unroll
            for (int j = 0; j < (F32 ? 2 : 1); ++j) w[j] = make_uint4(0, 0, 0, 0);
        } else {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : (T)0;
            __builtin_memcpy(w, v, sizeof(w));
        }
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

struct Plan {
    int L, run_rows, runs;                // lanes a row; rows of a run, runs of a picture
    int has;                              // 1: A, 2: Ab, 4: W, 8: S are in LDS (in this order, C8 floats each)
};
enum { HAS_A = 1, HAS_AB = 2, HAS_W = 4, HAS_S = 8 };

__device__ __forceinline__ float at(const float *v, int64_t i, float none) { return v ? v[i] : none; }

// the combined vectors of picture b
__device__ __forceinline__ void combine(const onedc_block_norm_params &p, int has, int64_t b, float *lds, int C8) {
    float *A = lds, *Ab = A + (has & HAS_A ? C8 : 0), *W = Ab + (has & HAS_AB ? C8 : 0), *S = W + (has & HAS_W ? C8 : 0);
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        if (has & (HAS_A | HAS_AB)) {
            const float g = p.alpha * at(p.gate, b * p.gate_rs + c, 1.f);
            if (has & HAS_A) A[c] = g * at(p.post_w, c, 1.f);
            if (has & HAS_AB) Ab[c] = g * at(p.post_b, c, 0.f);
        }
        if (has & (HAS_W | HAS_S)) {
            const float s = 1.f + at(p.scale, b * p.scale_rs + c, 0.f);
            if (has & HAS_W) W[c] = s * at(p.w, c, 1.f);
            if (has & HAS_S) S[c] = s * at(p.b, c, 0.f) + at(p.shift, b * p.shift_rs + c, 0.f);
        }
    }
}
__device__ __forceinline__ void take8(const float *v, int c, float (&o)[8]) {
    const f32x4 a = *(const f32x4 *)(v + c), b = *(const f32x4 *)(v + c + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = a[j], o[4 + j] = b[j];
}

// v -> (v - mean) * r in place; values behind C stay 0.  Returns r.
template <bool TAIL, int IT>
__device__ __forceinline__ float normalise(float (&v)[IT][8], int c0, int step, int C, int kind, float eps, RowSum &sum) {
    if (kind == ONEDC_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
        const float m = sum(s) / C;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = c0 + i * step + (TAIL ? j : 0) < C ? v[i][j] - m : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) q = __builtin_fmaf(v[i][j], v[i][j], q);
    const float r = rsqrtf(sum(q) / C + eps);
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= r;
    return r;
}

template <int IT, bool X32, bool F32, bool TAIL>
__global__ __launch_bounds__(NT, IT > 2 ? 3 : 4) void block_norm_rows_kernel(onedc_block_norm_params p, Plan pl) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int C8 = (p.C + 7) & ~7;
    const int b = blockIdx.x / pl.runs, run = blockIdx.x - b * pl.runs;
    combine(p, pl.has, b, lds + 2 * (NT / 64), C8);
    const float *A = lds + 2 * (NT / 64), *Ab = A + (pl.has & HAS_A ? C8 : 0), *W = Ab + (pl.has & HAS_AB ? C8 : 0), *S = W + (pl.has & HAS_W ? C8 : 0);
    RowSum sum = {lds, pl.L, 0};
    const int lane = threadIdx.x & (pl.L - 1), step = 8 * pl.L, c0 = lane * 8, each = NT / pl.L;
    const int n1 = min(p.N, (run + 1) * pl.run_rows);
    const int64_t row0 = (int64_t)b * p.N;
    Eight<X32> x[IT];
    Eight<F32> f[IT];
    auto load = [&](int n) {
        const int64_t row = row0 + n;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + i * step, left = n < n1 ? p.C - c : 0;
            x[i].template load<TAIL>(p.x, row * p.x_cs + p.x_co + c, left);
            if (p.f) f[i].template load<TAIL>(p.f, row * p.f_cs + p.f_co + c, left);
        }
    };
    int n = run * pl.run_rows + threadIdx.x / pl.L;
    load(n);
    __syncthreads();
    int cl = c0;
    // (every thread makes every turn: sums over a workgroup have barriers)
    for (int left_rows = n1 - run * pl.run_rows; left_rows > 0; left_rows -= each, n += each) {
        if (IT > 2) asm volatile("" : "+v"(cl));        // (else the compiler keeps all of a thread's LDS vectors in registers, and spills)
        float t[IT][8];
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = x[i].get(j);
        if (p.f) {
            float v[IT][8];
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = f[i].get(j);
            if (left_rows > each) load(n + each);
            if (p.post) normalise<TAIL>(v, c0, step, p.C, p.kind, p.eps, sum);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = c0 + i * step;
                if (c < p.C) {
                    float a[8], ab[8];
                    if (pl.has & HAS_A) take8(A, cl + i * step, a);
                    if (pl.has & HAS_AB) take8(Ab, cl + i * step, ab);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        t[i][j] = __builtin_fmaf(pl.has & HAS_A ? a[j] : p.alpha, v[i][j], t[i][j]);
                        if (pl.has & HAS_AB) t[i][j] += ab[j];
                        if (TAIL && c + j >= p.C) t[i][j] = 0.f;                       // (LDS behind C is not written)
                    }
                    if (n < n1) put8<X32, TAIL>(p.xo, (row0 + n) * p.xo_cs + p.xo_co + c, t[i], p.C - c);
                }
            }
        } else if (left_rows > each) {
            load(n + each);
        }
        if (p.y) {
            normalise<TAIL>(t, c0, step, p.C, p.kind, p.eps, sum);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = c0 + i * step;
                if (c < p.C && n < n1) {
                    float w[8], s[8];
                    if (pl.has & HAS_W) {
                        take8(W, cl + i * step, w);
#pragma unroll
                        for (int j = 0; j < 8; ++j) t[i][j] *= w[j];
                    }
                    if (pl.has & HAS_S) {
                        take8(S, cl + i * step, s);
#pragma unroll
                        for (int j = 0; j < 8; ++j) t[i][j] += s[j];
                    }
                    put8<F32, TAIL>(p.y, (row0 + n) * p.y_cs + p.y_co + c, t[i], p.C - c);
                }
            }
        }
    }
}

// ---- wider rows: a workgroup passes over its row again for every sum -------------------------------------------------------------------

// sum of v over the workgroup, the same value in every thread
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) s += red[i];
    return s;
}

// mean (0 for RMSNorm) and reciprocal deviation of the C values v(c)
template <class V>
__device__ __forceinline__ float2 row_norm(V v, int C, int kind, float eps, float *red) {
    float m = 0.f;
    if (kind == ONEDC_NORM_LAYER) {
        float s = 0.f;
        for (int c = threadIdx.x; c < C; c += NT) s += v(c);
        m = block_sum(s, red) / C;
    }
    float q = 0.f;
    for (int c = threadIdx.x; c < C; c += NT) {
        const float d = v(c) - m;
        q += d * d;
    }
    return make_float2(m, rsqrtf(block_sum(q, red) / C + eps));
}

template <bool X32, bool F32>
__global__ __launch_bounds__(NT) void block_norm_kernel(onedc_block_norm_params p) {
    typedef Elem<X32> X;
    typedef Elem<F32> F;
    __shared__ float red[NT / 64];
    const int64_t row = blockIdx.x;
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
        for (int c = threadIdx.x; c < p.C; c += NT) {
            const float v = (joined(c) - tn.x) * tn.y * at(p.w, c, 1.f) + at(p.b, c, 0.f);
            F::put(y + c, __builtin_fmaf(v, 1.f + at(scale, c, 0.f), at(shift, c, 0.f)));
        }
    }
    if (p.xo) {                                      // (behind the norm's passes: xo may be x)
        typename X::T *xo = (typename X::T *)p.xo + row * p.xo_cs + p.xo_co;
        for (int c = threadIdx.x; c < p.C; c += NT) X::put(xo + c, joined(c));
    }
}

// dx and df of a row, and the row's four column terms added to this run's sums: sums[4][C] in LDS-free global scratch, one column
// owned by one thread for the whole run (fixed order)
template <bool X32, bool F32>
__global__ __launch_bounds__(NT) void block_norm_backward_kernel(onedc_block_norm_params p, onedc_block_norm_grad g, float *part,
                                                                 int runs, int run_rows) {
    typedef Elem<X32> X;
    typedef Elem<F32> F;
    __shared__ float red[NT / 64];
    const int b = blockIdx.x / runs, run = blockIdx.x - b * runs;
    const int n0 = run * run_rows, n1 = min(p.N, n0 + run_rows);
    const float *gate = p.gate ? p.gate + (int64_t)b * p.gate_rs : nullptr;
    const float *scale = p.scale ? p.scale + (int64_t)b * p.scale_rs : nullptr;
    float *sums = part ? part + (int64_t)blockIdx.x * 4 * p.C : nullptr;
    if (sums)
        for (int c = threadIdx.x; c < 4 * p.C; c += NT) sums[c] = 0.f;      // (a thread's own columns differ from these: barrier below)
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
            for (int c = threadIdx.x; c < p.C; c += NT) {
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
            for (int c = threadIdx.x; c < p.C; c += NT) {
                const float v = w(c);
                sw += v;
                sf += v * fhat(c);
            }
            mw = p.kind == ONEDC_NORM_LAYER ? block_sum(sw, red) / p.C : 0.f;
            mf = block_sum(sf, red) / p.C;
        }
        for (int c = threadIdx.x; c < p.C; c += NT) {
            const float d = dt(c), fh = f ? fhat(c) : 0.f;
            if (sums) {
                const float e = dy ? F::get(dy + c) : 0.f;
                sums[c] += e;
                sums[p.C + c] += dy ? e * hat(c) : 0.f;
                sums[2 * p.C + c] += d;
                sums[3 * p.C + c] += d * fh;
            }
            // (dx may be dxo, df may be dy: this thread's own columns, read above)
            const float wc = w(c);
            if (g.dx) X::put((typename X::T *)g.dx + row * g.dx_cs + g.dx_co + c, d);
            if (g.df) F::put((typename F::T *)g.df + row * g.df_cs + g.df_co + c, p.post ? fn.y * (wc - mw - fh * mf) : wc);
        }
        __syncthreads();
    }
}

// The parameter gradients of one column from the runs' sums
__global__ void block_norm_params_kernel(onedc_block_norm_params p, onedc_block_norm_grad g, const float *part, int runs) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.C) return;
    const double w = at(p.w, c, 1.f), bb = at(p.b, c, 0.f), pw = at(p.post_w, c, 1.f), pb = at(p.post_b, c, 0.f), alpha = p.alpha;
    double dw = 0, db = 0, dpw = 0, dpb = 0, dgate = 0, dscale = 0, dshift = 0;
    for (int b = 0; b < p.B; ++b) {
        double s[4] = {0, 0, 0, 0};
        for (int r = 0; r < runs; ++r)
            for (int k = 0; k < 4; ++k) s[k] += part[(((int64_t)b * runs + r) * 4 + k) * p.C + c];
        const double sc = 1.0 + at(p.scale, (int64_t)b * p.scale_rs + c, 0.f), ga = alpha * at(p.gate, (int64_t)b * p.gate_rs + c, 1.f);
        dw += sc * s[1];
        db += sc * s[0];
        dpw += ga * s[3];
        dpb += ga * s[2];
        const double gt = alpha * (pw * s[3] + pb * s[2]), gs = w * s[1] + bb * s[0];
        if (g.d_gate && p.gate_rs) g.d_gate[(int64_t)b * p.C + c] = (float)gt;
        if (g.d_scale && p.scale_rs) g.d_scale[(int64_t)b * p.C + c] = (float)gs;
        if (g.d_shift && p.shift_rs) g.d_shift[(int64_t)b * p.C + c] = (float)s[0];
        dgate += gt;
        dscale += gs;
        dshift += s[0];
    }
    if (g.d_gate && !p.gate_rs) g.d_gate[c] = (float)dgate;
    if (g.d_scale && !p.scale_rs) g.d_scale[c] = (float)dscale;
    if (g.d_shift && !p.shift_rs) g.d_shift[c] = (float)dshift;
    if (g.d_w) g.d_w[c] = (float)dw;
    if (g.d_b) g.d_b[c] = (float)db;
    if (g.d_post_w) g.d_post_w[c] = (float)dpw;
    if (g.d_post_b) g.d_post_b[c] = (float)dpb;
}

int check_view(const void *p, int cs, int co, int C) { return !p || (cs >= C && co >= 0 && co <= cs - C) ? 0 : -2; }

int check_common(const onedc_block_norm_params *p) {
    if (!p) return -1;
    if (p->B < 0 || p->N < 0 || p->C < 1 || p->C > (1 << 20) || (int64_t)p->B * p->N > 0x7fffffff) return -2;
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

struct Runs {
    int runs, rows;        // runs of `rows` token rows per picture
};
Runs backward_runs(const onedc_block_norm_params *p) {
    const int want = p->B > 0 ? (512 + p->B - 1) / p->B : 1;
    Runs r;
    r.rows = (p->N + want - 1) / want;
    if (r.rows < 1) r.rows = 1;
    r.runs = (p->N + r.rows - 1) / r.rows;
    if (r.runs < 1) r.runs = 1;
    return r;
}

// Rows in registers: as few lanes a row as hold it in IT pieces of eight, so that few of them idle and exchanges stay short.  false: too wide.
bool row_plan(const onedc_block_norm_params *p, int most_it, int64_t most_lds, int has, int arrays, int want_runs, Plan *pl, int *it) {
    const int pieces = (p->C + 7) / 8;
    pl->has = has;
    for (pl->L = 8; pl->L <= NT; pl->L = pl->L == 64 ? NT : 2 * pl->L)
        if (pieces <= most_it * pl->L) break;
    if (pl->L > NT || (int64_t)arrays * ((p->C + 7) & ~7) * 4 + 64 > most_lds) return false;
    *it = (pieces + pl->L - 1) / pl->L;
    // whole turns of the workgroup (NT / L rows each) a run
    const int each = NT / pl->L, turns = (p->N + each - 1) / each;
    int want = (want_runs + p->B - 1) / p->B;
    want = want < 1 ? 1 : want > turns ? turns : want;
    pl->run_rows = (turns + want - 1) / want * each;
    pl->runs = (p->N + pl->run_rows - 1) / pl->run_rows;
    return true;
}

bool wants_sums(const onedc_block_norm_grad *g) {
    return g->d_post_w || g->d_post_b || g->d_gate || g->d_w || g->d_b || g->d_scale || g->d_shift;
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
    int has = 0;
    if (p->f && (p->gate || p->post_w)) has |= HAS_A;
    if (p->f && p->post_b) has |= HAS_AB;
    if (p->y && (p->w || p->scale)) has |= HAS_W;
    if (p->y && (p->b || p->shift)) has |= HAS_S;
    Plan pl;
    int it;
    onedc_block_norm_params q = *p;
    if (!p->gate_rs && !p->scale_rs && !p->shift_rs && rows <= 0x7fffffff) q.B = 1, q.N = (int)rows;     // one picture, as far as this goes
    if (row_plan(&q, 5, 128 << 10, has, __builtin_popcount(has), 1024, &pl, &it)) {
        const size_t lds = 64 + (size_t)__builtin_popcount(has) * ((p->C + 7) & ~7) * 4;
        const dim3 grid((unsigned)((int64_t)q.B * pl.runs));
        const bool tail = p->C & 7;
#define BN_ROWS(IT, X, F, TAIL)                                                                                           \
    do {                                                                                                                  \
        static OnedcLdsAttrOnce once;                                                                                     \
        once.ensure({{(const void *)block_norm_rows_kernel<IT, X, F, TAIL>, 128 << 10}});                                 \
        hipLaunchKernelGGL((block_norm_rows_kernel<IT, X, F, TAIL>), grid, dim3(NT), lds, as_stream(stream), q, pl);      \
    } while (0)
#define BN_ROWS_TAIL(IT, X, F) do { if (tail) BN_ROWS(IT, X, F, true); else BN_ROWS(IT, X, F, false); } while (0)
#define BN_ROWS_IT(X, F) do { if (it <= 2) BN_ROWS_TAIL(2, X, F); else BN_ROWS_TAIL(5, X, F); } while (0)
        if (p->f_f32) BN_ROWS_IT(true, true);
        else if (p->x_f32) BN_ROWS_IT(true, false);
        else BN_ROWS_IT(false, false);
        ONEDC_LAUNCH_CHECK();
        return 0;
    }
    if (p->f_f32)
        hipLaunchKernelGGL((block_norm_kernel<true, true>), dim3((unsigned)rows), dim3(NT), 0, as_stream(stream), *p);
    else if (p->x_f32)
        hipLaunchKernelGGL((block_norm_kernel<true, false>), dim3((unsigned)rows), dim3(NT), 0, as_stream(stream), *p);
    else
        hipLaunchKernelGGL((block_norm_kernel<false, false>), dim3((unsigned)rows), dim3(NT), 0, as_stream(stream), *p);
    ONEDC_LAUNCH_CHECK();
    return 0;
}

int64_t onedc_block_norm_backward_ws_bytes(const onedc_block_norm_params *p, const onedc_block_norm_grad *g) {
    if (check_common(p) || !g || !wants_sums(g)) return 0;
    return (int64_t)p->B * backward_runs(p).runs * 4 * p->C * sizeof(float);
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
    const int64_t need = onedc_block_norm_backward_ws_bytes(p, g);
    if (need && (!g->ws || g->ws_bytes < need)) return -15;
    const Runs r = backward_runs(p);
    float *part = sums ? (float *)g->ws : nullptr;
    if (any) {
        const dim3 grid((unsigned)(p->B * r.runs));
        if (p->f_f32)
            hipLaunchKernelGGL((block_norm_backward_kernel<true, true>), grid, dim3(NT), 0, as_stream(stream), *p, *g, part, r.runs, r.rows);
        else if (p->x_f32)
            hipLaunchKernelGGL((block_norm_backward_kernel<true, false>), grid, dim3(NT), 0, as_stream(stream), *p, *g, part, r.runs, r.rows);
        else
            hipLaunchKernelGGL((block_norm_backward_kernel<false, false>), grid, dim3(NT), 0, as_stream(stream), *p, *g, part, r.runs, r.rows);
        ONEDC_LAUNCH_CHECK();
    }
    if (sums) {
        hipLaunchKernelGGL(block_norm_params_kernel, dim3((p->C + 255) / 256), dim3(256), 0, as_stream(stream), *p, *g, part,
                           p->N > 0 ? r.runs : 0);
        ONEDC_LAUNCH_CHECK();
    }
    return 0;
}

}  // extern "C"
