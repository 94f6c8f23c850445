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

__device__ __forceinline__ float at(const float *v, int64_t i, float none) { return v ? v[i] : none; }

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
