// Short depthwise causal convolution with an optional SiLU: forward, backward, and one token of running sequences.
//   pre[t] = bias + sum_w weight[w] x[t - W + 1 + w]     y = act(pre)
//   dpre = dy act'(pre)     dx[t] = sum_w weight[w] dpre[t + W - 1 - w]     dweight[w] = sum_t dpre[t] x[t - W + 1 + w]     dbias = sum_t dpre[t]
// Bound by HBM: forward x in, y out; backward x and dy in, dx out (pre is formed again from x, cheaper than 4 bytes of it saved per element).
// A thread owns a few neighbouring channels and walks down a run of tokens, so that every row of x is read once, with 16-byte accesses, and the
// window of W - 1 rows stays in registers; only the rows around the ends of a run are read twice (they come from L2).
#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int CONV_BATCH = 4;            // rows requested together

// V elements of a row as floats: V = 8 or 4 neighbours from channel d0 on
template <int DT, int V>
__device__ __forceinline__ void conv_load(const void* base, size_t row, int d0, int D, bool vec, float (&v)[V]) {
    if (vec) {
        if constexpr (V == 8) ld8(base, DT, row + d0, v);
        else {
            const float4 f = ld4(base, DT, row + d0);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = d0 + e < D ? ld1(base, DT, row + d0 + e) : 0.f;
    }
}
template <int DT, int V>
__device__ __forceinline__ void conv_store(void* base, size_t row, int d0, int D, bool vec, const float (&v)[V]) {
    if (vec) {
        if constexpr (V == 8) st8<DT>(base, row + d0, v);
        else st4(base, DT, row + d0, make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (d0 + e < D) st1(base, DT, row + d0 + e, v[e]);
    }
}
template <int V>
__device__ __forceinline__ void conv_params(const float* weight, const float* bias, int W, int w, int d0, int D, float (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = d0 + e >= D ? 0.f : weight ? weight[(size_t)(d0 + e) * W + w] : bias ? bias[d0 + e] : 0.f;
}

// The W - 1 rows in front of token `a` of a sequence that starts at `s`: its own tokens, its state, or zeros
template <int DT, int W, int V>
__device__ __forceinline__ void conv_window(const void* x, long long stride, const void* state, int n, int a, int s, int d0, int D, bool vec, bool svec, float (&win)[W - 1][V]) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        const int at = a - (W - 1) + j;
#pragma unroll
        for (int e = 0; e < V; ++e) win[j][e] = 0.f;
        if (at >= s) conv_load<DT, V>(x, (size_t)at * stride, d0, D, vec, win[j]);
        else if (state) conv_load<DT, V>(state, ((size_t)n * (W - 1) + (at - s + W - 1)) * D, d0, D, svec, win[j]);
    }
}

template <int DT, int W, int V>
__global__ void __launch_bounds__(128) conv_fwd_kernel(const MkdaConvFwd p, const int run, const bool vec, const bool svec) {
    follow_stream();
    const int D = p.D, d0 = (blockIdx.x * 128 + threadIdx.x) * V;
    if (d0 >= D) return;
    float wt[W][V], bias[V];
#pragma unroll
    for (int w = 0; w < W; ++w) conv_params<V>(p.weight, nullptr, W, w, d0, D, wt[w]);
    conv_params<V>(nullptr, p.bias, W, 0, d0, D, bias);
    if (blockIdx.y == 0 && p.S.has_empty && p.last) {      // an empty sequence hands its state through
        for (int n = 0; n < p.S.N; ++n) {
            const Span q = sequence(p.S, n);
            if (q.start != q.end) continue;
            float win[W - 1][V];
            conv_window<DT, W, V>(p.x, p.x_stride, p.state, n, q.start, q.start, d0, D, vec, svec, win);
#pragma unroll
            for (int j = 0; j < W - 1; ++j) conv_store<DT, V>(p.last, ((size_t)n * (W - 1) + j) * D, d0, D, svec, win[j]);
        }
    }
    const int t0 = (int)blockIdx.y * run, t1 = min(t0 + run, p.S.TT);
    if (t0 >= t1) return;
    int n = sequence_of(p.S, t0);
    for (int a = t0; a < t1 && n < p.S.N; ++n) {
        const Span q = sequence(p.S, n);
        const int b = min(t1, q.end);
        if (b <= a) continue;
        float xs[CONV_BATCH + W - 1][V];
        float win[W - 1][V];
        conv_window<DT, W, V>(p.x, p.x_stride, p.state, n, a, q.start, d0, D, vec, svec, win);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) xs[j][e] = win[j][e];
        int t = a;
        for (; t < b; t += CONV_BATCH) {
            const int cnt = min(CONV_BATCH, b - t);
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u)
                if (u < cnt) conv_load<DT, V>(p.x, (size_t)(t + u) * p.x_stride, d0, D, vec, xs[W - 1 + u]);
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u) {
                if (u >= cnt) break;
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float pre = bias[e];
#pragma unroll
                    for (int w = 0; w < W; ++w) pre = fmaf(wt[w][e], xs[u + w][e], pre);
                    y[e] = p.silu ? pre * sigmoidf_(pre) : pre;
                }
                conv_store<DT, V>(p.y, (size_t)(t + u) * D, d0, D, svec, y);
            }
            if (cnt == CONV_BATCH) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) xs[j][e] = xs[CONV_BATCH + j][e];
            } else {
                for (int u = 0; u < cnt; ++u)
#pragma unroll
                    for (int j = 0; j < CONV_BATCH + W - 2; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) xs[j][e] = xs[j + 1][e];
            }
        }
        if (b == q.end && p.last) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = xs[j][e];
                conv_store<DT, V>(p.last, ((size_t)n * (W - 1) + j) * D, d0, D, svec, v);
            }
        }
        a = b;
    }
}

// Backward: a run of tokens [t0, t1) per block row.  Within a sequence the walk goes W - 1 tokens past the run's end (their dpre belongs to the
// run's dx) and starts with a window of zeros: dpre in front of the run only matters for rows of other runs, and in front of the sequence there is
// none.  At its first tokens a sequence's walk emits the gradient of its state.
template <int DT, int W, int V>
__global__ void __launch_bounds__(128) conv_bwd_kernel(const MkdaConvBwd p, const int run, const bool vec, const bool svec) {
    follow_stream();
    const int D = p.D, d0 = (blockIdx.x * 128 + threadIdx.x) * V;
    if (d0 >= D) return;
    float wt[W][V], bias[V], dw[W][V], db[V];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        conv_params<V>(p.weight, nullptr, W, w, d0, D, wt[w]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[w][e] = 0.f;
    }
    conv_params<V>(nullptr, p.bias, W, 0, d0, D, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) db[e] = 0.f;
    if (blockIdx.y == 0 && p.S.has_empty && p.dstate) {
        for (int n = 0; n < p.S.N; ++n) {
            const Span q = sequence(p.S, n);
            if (q.start != q.end) continue;
            for (int j = 0; j < W - 1; ++j) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = 0.f;
                if (p.dlast) conv_load<DT, V>(p.dlast, ((size_t)n * (W - 1) + j) * D, d0, D, svec, v);
                conv_store<DT, V>(p.dstate, ((size_t)n * (W - 1) + j) * D, d0, D, svec, v);
            }
        }
    }
    const int t0 = (int)min((long long)blockIdx.y * run, (long long)p.S.TT), t1 = min(t0 + run, p.S.TT);
    int n = t0 < t1 ? sequence_of(p.S, t0) : p.S.N;
    for (int a = t0; a < t1 && n < p.S.N; ++n) {
        const Span q = sequence(p.S, n);
        const int b = min(t1, q.end);
        if (b <= a) continue;
        float xs[CONV_BATCH + W - 1][V], dp[CONV_BATCH + W - 1][V], win[W - 1][V];
        conv_window<DT, W, V>(p.x, p.x_stride, p.state, n, a, q.start, d0, D, vec, svec, win);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) { xs[j][e] = win[j][e]; dp[j][e] = 0.f; }
        const int stop = b + W - 1;                        // one past the last step
        for (int t = a; t < stop; t += CONV_BATCH) {
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u) {
#pragma unroll
                for (int e = 0; e < V; ++e) xs[W - 1 + u][e] = dp[W - 1 + u][e] = 0.f;
                if (t + u < q.end && t + u < stop) {
                    conv_load<DT, V>(p.x, (size_t)(t + u) * p.x_stride, d0, D, vec, xs[W - 1 + u]);
                    conv_load<DT, V>(p.dy, (size_t)(t + u) * D, d0, D, svec, dp[W - 1 + u]);
                }
            }
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u) {
                const int at = t + u;
                if (at >= stop) break;
                if (p.silu && at < q.end) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float pre = bias[e];
#pragma unroll
                        for (int w = 0; w < W; ++w) pre = fmaf(wt[w][e], xs[u + w][e], pre);
                        const float sg = sigmoidf_(pre);
                        dp[W - 1 + u][e] *= sg * fmaf(pre, 1.f - sg, 1.f);
                    }
                }
                if (at < b) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float g = dp[W - 1 + u][e];
                        db[e] += g;
#pragma unroll
                        for (int w = 0; w < W; ++w) dw[w][e] = fmaf(g, xs[u + w][e], dw[w][e]);
                    }
                }
                const int to = at - (W - 1);               // the row whose gradient is complete now
                if (to < a && (a != q.start || !p.dstate)) continue;
                float g[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    g[e] = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w) g[e] = fmaf(wt[W - 1 - w][e], dp[u + w][e], g[e]);
                }
                if (p.dlast && to >= q.end - (W - 1)) {
                    float v[V];
                    conv_load<DT, V>(p.dlast, ((size_t)n * (W - 1) + (to - q.end + W - 1)) * D, d0, D, svec, v);
#pragma unroll
                    for (int e = 0; e < V; ++e) g[e] += v[e];
                }
                if (to >= a) conv_store<DT, V>(p.dx, (size_t)to * D, d0, D, svec, g);
                else conv_store<DT, V>(p.dstate, ((size_t)n * (W - 1) + (to - q.start + W - 1)) * D, d0, D, svec, g);
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) { xs[j][e] = xs[CONV_BATCH + j][e]; dp[j][e] = dp[CONV_BATCH + j][e]; }
        }
        a = b;
    }
    float* part = p.part + (size_t)blockIdx.y * (W + 1) * D;
#pragma unroll
    for (int w = 0; w <= W; ++w)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (d0 + e < D) part[(size_t)w * D + d0 + e] = w < W ? dw[w < W ? w : 0][e] : db[e];
}

template <int DT, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const MkdaConvStep p, const bool vec, const bool svec) {
    follow_stream();
    const int D = p.D, d0 = (blockIdx.x * 128 + threadIdx.x) * V, n = blockIdx.y;
    if (d0 >= D) return;
    float rows[W][V], wt[W][V], bias[V], y[V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_load<DT, V>(p.state, ((size_t)n * (W - 1) + j) * D, d0, D, svec, rows[j]);
    conv_load<DT, V>(p.x, (size_t)n * p.x_stride, d0, D, vec, rows[W - 1]);
#pragma unroll
    for (int w = 0; w < W; ++w) conv_params<V>(p.weight, nullptr, W, w, d0, D, wt[w]);
    conv_params<V>(nullptr, p.bias, W, 0, d0, D, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float pre = bias[e];
#pragma unroll
        for (int w = 0; w < W; ++w) pre = fmaf(wt[w][e], rows[w][e], pre);
        y[e] = p.silu ? pre * sigmoidf_(pre) : pre;
    }
    conv_store<DT, V>(p.y, (size_t)n * D, d0, D, svec, y);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_store<DT, V>(p.state, ((size_t)n * (W - 1) + j) * D, d0, D, svec, rows[j + 1]);
}

template <typename F>
static bool with_taps(int W, F f) {
    switch (W) {
        case 2: f(std::integral_constant<int, 2>()); return true;
        case 3: f(std::integral_constant<int, 3>()); return true;
        case 4: f(std::integral_constant<int, 4>()); return true;
        default: return false;
    }
}

}  // namespace mkda

using namespace mkda;

extern "C" int mkda_conv_fwd(const MkdaConvFwd* p, void* stream) {
    if (!p || !p->weight || (p->S.TT && (!p->x || !p->y))) return set_error(MKDA_ERR_ARG, "conv_fwd: null argument");
    if (p->W < 2 || p->W > 4 || p->D <= 0 || !good_sequences(p->S)) return set_error(MKDA_ERR_ARG, "conv_fwd: 2 to 4 taps, at least one channel");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "conv_fwd: unsupported dtype");
    if (p->S.N == 0 || (p->S.TT == 0 && !(p->last && p->S.has_empty))) return MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        with_taps(p->W, [&](auto w) {
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value, V = DT == MKDA_F32 ? 4 : 8;
            const int blocks = (p->D + 128 * V - 1) / (128 * V);
            const bool wide = p->D % V == 0, vec = wide && p->x_stride % V == 0 && aligned16(p->x), svec = wide && aligned16(p->y) && aligned16(p->state) && aligned16(p->last);
            // tokens per run: 64 where that leaves eight blocks per SM, fewer in short calls
            long long run = (long long)p->S.TT * blocks / (8ll * sm_count());
            run = run < 8 ? 8 : run > 64 ? 64 : run / 4 * 4;
            if (p->S.TT > run * 65535) run = (p->S.TT + 65534) / 65535;
            const int rows = (int)((p->S.TT + run - 1) / run);
            launch(conv_fwd_kernel<DT, W, V>, dim3(blocks, rows ? rows : 1), 128, 0, (cudaStream_t)stream, *p, (int)run, vec, svec);
        });
    });
    return check_launch("conv_fwd");
}

extern "C" int mkda_conv_bwd(const MkdaConvBwd* p, void* stream) {
    if (!p || !p->weight || !p->part || (p->S.TT && (!p->x || !p->dy || !p->dx))) return set_error(MKDA_ERR_ARG, "conv_bwd: null argument");
    if (p->W < 2 || p->W > 4 || p->D <= 0 || !good_sequences(p->S)) return set_error(MKDA_ERR_ARG, "conv_bwd: 2 to 4 taps, at least one channel");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "conv_bwd: unsupported dtype");
    if (p->part_rows < 1 || p->part_rows > 65535) return set_error(MKDA_ERR_ARG, "conv_bwd: 1 to 65535 rows of partial sums");
    with_dtype(p->dtype, [&](auto dt) {
        with_taps(p->W, [&](auto w) {
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value, V = 4;
            const int blocks = (p->D + 128 * V - 1) / (128 * V), run = (p->S.TT + p->part_rows - 1) / p->part_rows;
            const bool wide = p->D % V == 0, vec = wide && p->x_stride % V == 0 && aligned16(p->x);
            const bool svec = wide && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->state) && aligned16(p->dlast) && aligned16(p->dstate);
            launch(conv_bwd_kernel<DT, W, V>, dim3(blocks, p->part_rows), 128, 0, (cudaStream_t)stream, *p, run, vec, svec);
        });
    });
    return check_launch("conv_bwd");
}

extern "C" int mkda_conv_step(const MkdaConvStep* p, void* stream) {
    if (!p || !p->weight || (p->N && (!p->x || !p->state || !p->y))) return set_error(MKDA_ERR_ARG, "conv_step: null argument");
    if (p->W < 2 || p->W > 4 || p->D <= 0 || p->N < 0 || p->N > 65535) return set_error(MKDA_ERR_ARG, "conv_step: 2 to 4 taps, at least one channel, at most 65535 sequences");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "conv_step: unsupported dtype");
    if (p->N == 0) return MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        with_taps(p->W, [&](auto w) {
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value, V = DT == MKDA_F32 ? 4 : 8;
            const bool wide = p->D % V == 0, vec = wide && p->x_stride % V == 0 && aligned16(p->x), svec = wide && aligned16(p->y) && aligned16(p->state);
            launch(conv_step_kernel<DT, W, V>, dim3((p->D + 128 * V - 1) / (128 * V), p->N), 128, 0, (cudaStream_t)stream, *p, vec, svec);
        });
    });
    return check_launch("conv_step");
}
