// Short depthwise causal convolution with an optional SiLU: forward, backward, and one token of running sequences.
//   pre[t] = bias + sum_w weight[w] x[t - W + 1 + w]     y = act(pre)
//   dpre = dy act'(pre)     dx[t] = sum_w weight[w] dpre[t + W - 1 - w]     dweight[w] = sum_t dpre[t] x[t - W + 1 + w]     dbias = sum_t dpre[t]
// Bound by HBM: forward x in, y out; backward x and dy in, dx out (pre is formed again from x, cheaper than 4 bytes of it saved per element).
// A thread owns a few neighbouring channels and walks down a run of tokens, so that every row of x is read once, with 16-byte accesses, and the
// window of W - 1 rows stays in registers; only the rows around the ends of a run are read twice (they come from L2).
// bf16, four taps: forward 32749 x 8192 176 us (6.1 TB/s), 8192 x 4096 30 us (4.5 TB/s, one wave of blocks and its start-up); backward 8192 x 4096 48 us (4.2 TB/s; half of the issue
// slots, waits for the packed products of 13 warps per SM), of which the check of every token against the ends of its run and sequence was 12.
#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int CONV_BATCH = 4;            // rows requested together, and places of the ring that holds the window (a power of two, at least W)

// The V channels of a thread from d0 on: neighbours, but one in 128 in fp32 rows that do not allow 16-byte accesses, whose single elements are then neighbours in a warp (8192 x 4097 forward
// 61 us; shifted from aligned words, as 16-bit rows are, 114).  `vec`: rows allow 16-byte (8-byte) accesses.
template <int DT, bool vec>
__device__ __forceinline__ constexpr int conv_step() { return DT == MKDA_F32 && !vec ? 128 : 1; }
template <int DT, int V, bool vec>
__device__ __forceinline__ int conv_channel() { return conv_step<DT, vec>() == 1 ? (blockIdx.x * 128 + threadIdx.x) * V : blockIdx.x * 128 * V + threadIdx.x; }
// Their elements in a row, as they lie in memory, those past the last channel zero
template <int DT, int V>
struct alignas(DT == MKDA_F32 ? V * 4 : V * 2) ConvRaw { uint32_t w[DT == MKDA_F32 ? V : V / 2]; };
template <int DT, int V>
__device__ __forceinline__ ConvRaw<DT, V> conv_raw(const void* base, size_t row, int d0, int D, bool vec) {
    ConvRaw<DT, V> r;
    constexpr int WORDS = DT == MKDA_F32 ? V : V / 2, SIZE = DT == MKDA_F32 ? 4 : 2;
    const char* p = static_cast<const char*>(base) + (row + d0) * SIZE;
    if (!vec && DT == MKDA_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) r.w[e] = d0 + 128 * e < D ? *reinterpret_cast<const uint32_t*>(p + 512 * e) : 0u;
    } else if (!vec) {
        const Words<4 * WORDS> v = load_shifted<4 * WORDS>(p, min(V, D - d0) * SIZE);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) r.w[i] = v.w[i];
    } else if constexpr (WORDS == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    }
    return r;
}
template <int DT, int V>
__device__ __forceinline__ ConvRaw<DT, V> conv_zero() {
    ConvRaw<DT, V> r;
#pragma unroll
    for (uint32_t& w : r.w) w = 0u;
    return r;
}
template <int DT, int V>
__device__ __forceinline__ void conv_unpack(const ConvRaw<DT, V>& r, f32x2 (&v)[V / 2]) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
        if constexpr (DT == MKDA_F32) {
            v[e] = pack2(__uint_as_float(r.w[2 * e]), __uint_as_float(r.w[2 * e + 1]));
        } else if constexpr (DT == MKDA_BF16) {
            v[e] = pack2(__uint_as_float(r.w[e] << 16), __uint_as_float(r.w[e] & 0xffff0000u));
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[e]));
            v[e] = pack2(f.x, f.y);
        }
    }
}
template <int DT, int V, int STEP = 128>
__device__ __forceinline__ void conv_store(void* base, size_t row, int d0, int D, bool vec, const f32x2 (&p)[V / 2]) {
    float v[V];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) unpack2(p[e], v[2 * e], v[2 * e + 1]);
    if (vec) {
        if constexpr (V == 8) st8<DT>(base, row + d0, v);
        else st4(base, DT, row + d0, make_float4(v[0], v[1], v[2], v[3]));
    } else if constexpr (DT == MKDA_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (d0 + e * STEP < D) static_cast<float*>(base)[row + d0 + e * STEP] = v[e];
    } else {
        Words<2 * V> w;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) w.w[e] = pack16<DT>(v[2 * e], v[2 * e + 1]);
        store_shifted<2 * V>(static_cast<uint16_t*>(base) + row + d0, min(V, D - d0) * 2, w);
    }
}
// weights [D][W] and biases of the thread's channels; those past the last channel are zero
template <int W, int V>
__device__ __forceinline__ void conv_params(const float* weight, const float* bias, int d0, int D, int step, f32x2 (&wt)[W][V / 2], f32x2 (&b)[V / 2]) {
    float f[V * W], g[V];
    if (step == 1 && d0 + V <= D && aligned16(weight)) {   // V W numbers in a row
#pragma unroll
        for (int i = 0; i < V * W; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(weight + (size_t)d0 * W + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * W; ++i) f[i] = d0 + i / W * step < D ? weight[(size_t)(d0 + i / W * step) * W + i % W] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = bias && d0 + e * step < D ? bias[d0 + e * step] : 0.f;
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
        b[e] = pack2(g[2 * e], g[2 * e + 1]);
#pragma unroll
        for (int w = 0; w < W; ++w) wt[w][e] = pack2(f[2 * e * W + w], f[(2 * e + 1) * W + w]);
    }
}

// Row `at` of a sequence that starts at `s`, at < s included: its own token, of its state, or zeros
template <int DT, int W, int V>
__device__ __forceinline__ ConvRaw<DT, V> conv_row(const void* x, long long stride, const void* state, int n, int at, int s, int d0, int D, bool vec) {
    if (at >= s) return conv_raw<DT, V>(x, (size_t)at * stride, d0, D, vec);
    if (state) return conv_raw<DT, V>(state, ((size_t)n * (W - 1) + (at - s + W - 1)) * D, d0, D, vec);
    return conv_zero<DT, V>();
}
// Rows on their way.  A thread copies its own channels of the next STAGES - 1 batches into shared memory asynchronously and reads them back itself, so that no
// barrier is needed and more bytes are in flight than its registers could hold (two batches in registers: 212 us for 32749 x 8192 bf16).  Rows that
// start anywhere, which the asynchronous copy cannot shift, pass through registers, a batch at a time.
template <int DT, int V, int STAGES>
struct ConvFeed {
    static constexpr int BYTES = sizeof(ConvRaw<DT, V>), SHARED = STAGES * CONV_BATCH * 128 * BYTES;
    char* buf;                             // [STAGES][CONV_BATCH][128 threads], from this thread's places on
    const char* base;
    size_t pitch;                          // bytes between rows
    int d0, D;
    bool vec;
    const char* next;                      // the first row of the next batch
    __device__ __forceinline__ ConvFeed(char* shared, const void* rows, long long stride, int d0, int D, bool vec)
        : buf(shared + threadIdx.x * BYTES), base(static_cast<const char*>(rows)), pitch((size_t)stride * SIZE), d0(d0), D(D), vec(vec), next(nullptr) {}
    static constexpr int SIZE = DT == MKDA_F32 ? 4 : 2;
    __device__ __forceinline__ char* place(int batch, int u) const { return buf + ((batch % STAGES) * CONV_BATCH + u) * 128 * BYTES; }
    __device__ __forceinline__ void start(int t) { next = base + (size_t)t * pitch + (size_t)d0 * SIZE; }
    __device__ __forceinline__ void copy(char* to, const char* from) const {
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
        if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(at), "l"(from) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(at), "l"(from) : "memory");
    }
    // the next batch, tokens t to t + CONV_BATCH - 1 as far as they lie in front of `end`
    __device__ __forceinline__ void request(int batch, int t, int end) {
        char* to = place(batch, 0);
        if (vec) {
            if (t + CONV_BATCH <= end) {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u) copy(to + u * 128 * BYTES, next + u * pitch);
            } else {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u)
                    if (t + u < end) copy(to + u * 128 * BYTES, next + u * pitch);
            }
            next += CONV_BATCH * pitch;
        } else {
            ConvRaw<DT, V> r[CONV_BATCH];
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u)
                if (t + u < end) r[u] = conv_raw<DT, V>(base, (size_t)(t + u) * (pitch / SIZE), d0, D, false);
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u)
                if (t + u < end) *reinterpret_cast<ConvRaw<DT, V>*>(to + u * 128 * BYTES) = r[u];
        }
    }
    __device__ __forceinline__ ConvRaw<DT, V> take(int batch, int u) const { return *reinterpret_cast<const ConvRaw<DT, V>*>(place(batch, u)); }
};
__device__ __forceinline__ void conv_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int STAGES>
__device__ __forceinline__ void conv_arrived() { asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 2) : "memory"); }

// The ring holds token t at place (t - a) mod CONV_BATCH, `a` the first token of the walk: places are known at compile time in the unrolled batch.
__device__ __forceinline__ constexpr int conv_place(int u) { return (u + 4 * CONV_BATCH) % CONV_BATCH; }

constexpr int CONV_FWD_BLOCKS = 4, CONV_BWD_BLOCKS = 4;      // per SM
template <int DT, int W, int V, bool vec>
__global__ void __launch_bounds__(128, vec ? CONV_FWD_BLOCKS : 3) conv_fwd_kernel(const MkdaConvFwd p, const int run) {
    follow_stream();
    constexpr int P = V / 2;
    constexpr int STAGES = 4;
    __shared__ __align__(16) char shared_rows[ConvFeed<DT, V, STAGES>::SHARED];
    const int D = p.D, d0 = conv_channel<DT, V, vec>(), t0 = (int)min((long long)blockIdx.y * run, (long long)p.S.TT), t1 = min(t0 + run, p.S.TT);
    int n = t0 < t1 ? sequence_of(p.S, t0) : p.S.N;
    if (d0 >= D) return;
    f32x2 wt[W][P], bias[P];
    conv_params<W, V>(p.weight, p.bias, d0, D, conv_step<DT, vec>(), wt, bias);
    ConvFeed<DT, V, STAGES> feed(shared_rows, p.x, p.x_stride, d0, D, vec);
    if (p.S.has_empty && p.last) {                         // an empty sequence hands its state through: the rows of blocks share the sequences
        for (int n = blockIdx.y; n < p.S.N; n += gridDim.y) {
            const Span q = sequence(p.S, n);
            if (q.start != q.end) continue;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                f32x2 v[P];
                conv_unpack<DT, V>(conv_row<DT, W, V>(p.x, p.x_stride, p.state, n, q.start - (W - 1) + j, q.start, d0, D, vec), v);
                conv_store<DT, V>(p.last, ((size_t)n * (W - 1) + j) * D, d0, D, vec, v);
            }
        }
    }
    for (int a = t0; a < t1 && n < p.S.N; ++n) {
        const Span q = sequence(p.S, n);
        const int b = min(t1, q.end);
        if (b <= a) continue;
        f32x2 ring[CONV_BATCH][P];
        feed.start(a);
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) {
            feed.request(k, a + k * CONV_BATCH, b);
            conv_commit();
        }
#pragma unroll
        for (int j = 1; j < W; ++j)
            conv_unpack<DT, V>(conv_row<DT, W, V>(p.x, p.x_stride, p.state, n, a - j, q.start, d0, D, vec), ring[conv_place(-j)]);
        auto token = [&](int t, int k, int u) {
            conv_unpack<DT, V>(feed.take(k, u), ring[u]);
            f32x2 y[P];
#pragma unroll
            for (int e = 0; e < P; ++e) {
                y[e] = bias[e];
#pragma unroll
                for (int w = 0; w < W; ++w) y[e] = fma2(wt[w][e], ring[conv_place(u - (W - 1) + w)][e], y[e]);
                if (p.silu) y[e] = mul2(y[e], sigmoidf2_(y[e]));
            }
            conv_store<DT, V>(p.y, (size_t)(t + u) * D, d0, D, vec, y);
        };
        for (int t = a, k = 0; t < b; t += CONV_BATCH, ++k) {
            conv_arrived<STAGES>();
            feed.request(k + STAGES - 1, t + (STAGES - 1) * CONV_BATCH, b);      // into the places that the batch in front has left
            conv_commit();
            if (t + CONV_BATCH <= b) {                     // without a look at every token
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u) token(t, k, u);
            } else {
#pragma unroll
                for (int u = 0; u < CONV_BATCH - 1; ++u)
                    if (t + u < b) token(t, k, u);
            }
        }
        if (b == q.end && p.last) {                        // rows from memory again: which place of the ring they have is not known at compile time
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                f32x2 v[P];
                conv_unpack<DT, V>(conv_row<DT, W, V>(p.x, p.x_stride, p.state, n, b - (W - 1) + j, q.start, d0, D, vec), v);
                conv_store<DT, V>(p.last, ((size_t)n * (W - 1) + j) * D, d0, D, vec, v);
            }
        }
        a = b;
    }
}

// Backward: a run of tokens [t0, t1) per block row.  Within a sequence the walk goes W - 1 tokens past the run's end (their dpre belongs to the
// run's dx) and starts with a ring of zeros: dpre in front of the run only matters for rows of other runs, and in front of the sequence there is
// none.  At its first tokens a sequence's walk emits the gradient of its state.
template <int DT, int W, int V, bool vec>
__global__ void __launch_bounds__(128, vec ? CONV_BWD_BLOCKS : 3) conv_bwd_kernel(const MkdaConvBwd p, const int run) {
    follow_stream();
    constexpr int P = V / 2;
    constexpr int STAGES = DT == MKDA_F32 ? 3 : 4;
    __shared__ __align__(16) char shared_rows[2][ConvFeed<DT, V, STAGES>::SHARED];
    const int D = p.D, d0 = conv_channel<DT, V, vec>(), t0 = (int)min((long long)blockIdx.y * run, (long long)p.S.TT), t1 = min(t0 + run, p.S.TT);
    int n = t0 < t1 ? sequence_of(p.S, t0) : p.S.N;
    if (d0 >= D) return;
    ConvFeed<DT, V, STAGES> feed_x(shared_rows[0], p.x, p.x_stride, d0, D, vec);
    ConvFeed<DT, V, STAGES> feed_y(shared_rows[1], p.dy, D, d0, D, vec);
    f32x2 wt[W][P], bias[P], dw[W][P], db[P];
    conv_params<W, V>(p.weight, p.bias, d0, D, conv_step<DT, vec>(), wt, bias);
#pragma unroll
    for (int e = 0; e < P; ++e) {
        db[e] = both(0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) dw[w][e] = both(0.f);
    }
    if (p.S.has_empty && p.dstate) {
        for (int n = blockIdx.y; n < p.S.N; n += gridDim.y) {
            const Span q = sequence(p.S, n);
            if (q.start != q.end) continue;
            for (int j = 0; j < W - 1; ++j) {
                const size_t row = ((size_t)n * (W - 1) + j) * D;
                f32x2 v[P];
                conv_unpack<DT, V>(p.dlast ? conv_raw<DT, V>(p.dlast, row, d0, D, vec) : conv_zero<DT, V>(), v);
                conv_store<DT, V>(p.dstate, row, d0, D, vec, v);
            }
        }
    }
    for (int a = t0; a < t1 && n < p.S.N; ++n) {
        const Span q = sequence(p.S, n);
        const int b = min(t1, q.end);
        if (b <= a) continue;
        const int stop = b + W - 1, read = min(stop, q.end);      // one past the last step, and past the last one with a row of its own
        f32x2 xs[CONV_BATCH][P], dp[CONV_BATCH][P];
        feed_x.start(a);
        feed_y.start(a);
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) {
            feed_x.request(k, a + k * CONV_BATCH, read);
            feed_y.request(k, a + k * CONV_BATCH, read);
            conv_commit();
        }
#pragma unroll
        for (int j = 1; j < W; ++j) {
            conv_unpack<DT, V>(conv_row<DT, W, V>(p.x, p.x_stride, p.state, n, a - j, q.start, d0, D, vec), xs[conv_place(-j)]);
#pragma unroll
            for (int e = 0; e < P; ++e) dp[conv_place(-j)][e] = both(0.f);
        }
        // one step; `inner`: the token lies in the run, and the row whose gradient it completes too, away from both ends of the sequence
        auto token = [&](auto inner, int t, int k, int u) {
            constexpr bool INNER = decltype(inner)::value;
            const int at = t + u;
            conv_unpack<DT, V>(INNER || at < read ? feed_x.take(k, u) : conv_zero<DT, V>(), xs[u]);
            conv_unpack<DT, V>(INNER || at < read ? feed_y.take(k, u) : conv_zero<DT, V>(), dp[u]);
            if (p.silu && (INNER || at < read)) {
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    f32x2 pre = bias[e];
#pragma unroll
                    for (int w = 0; w < W; ++w) pre = fma2(wt[w][e], xs[conv_place(u - (W - 1) + w)][e], pre);
                    const f32x2 sg = sigmoidf2_(pre);      // act' = sg (1 + pre (1 - sg))
                    dp[u][e] = mul2(dp[u][e], mul2(sg, fma2(pre, fma2(sg, both(-1.f), both(1.f)), both(1.f))));
                }
            }
            if (INNER || at < b) {
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    db[e] = add2(db[e], dp[u][e]);
#pragma unroll
                    for (int w = 0; w < W; ++w) dw[w][e] = fma2(dp[u][e], xs[conv_place(u - (W - 1) + w)][e], dw[w][e]);
                }
            }
            const int to = at - (W - 1);                   // the row whose gradient is complete now
            if (!INNER && to < a && (a != q.start || !p.dstate)) return;
            f32x2 g[P];
#pragma unroll
            for (int e = 0; e < P; ++e) {
                g[e] = mul2(wt[W - 1][e], dp[conv_place(u - (W - 1))][e]);
#pragma unroll
                for (int w = 1; w < W; ++w) g[e] = fma2(wt[W - 1 - w][e], dp[conv_place(u - (W - 1) + w)][e], g[e]);
            }
            if (!INNER && p.dlast && to >= q.end - (W - 1)) {
                f32x2 v[P];
                conv_unpack<DT, V>(conv_raw<DT, V>(p.dlast, ((size_t)n * (W - 1) + (to - q.end + W - 1)) * D, d0, D, vec), v);
#pragma unroll
                for (int e = 0; e < P; ++e) g[e] = add2(g[e], v[e]);
            }
            if (INNER || to >= a) conv_store<DT, V>(p.dx, (size_t)to * D, d0, D, vec, g);
            else conv_store<DT, V>(p.dstate, ((size_t)n * (W - 1) + (to - q.start + W - 1)) * D, d0, D, vec, g);
        };
        for (int t = a, k = 0; t < stop; t += CONV_BATCH, ++k) {
            conv_arrived<STAGES>();
            feed_x.request(k + STAGES - 1, t + (STAGES - 1) * CONV_BATCH, read);
            feed_y.request(k + STAGES - 1, t + (STAGES - 1) * CONV_BATCH, read);
            conv_commit();
            if (t - (W - 1) >= a && t + CONV_BATCH <= b) {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u) token(std::true_type(), t, k, u);
            } else {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u)
                    if (t + u < stop) token(std::false_type(), t, k, u);
            }
        }
        a = b;
    }
    float* part = p.part + (size_t)blockIdx.y * (W + 1) * D;
#pragma unroll
    for (int w = 0; w < W; ++w) conv_store<MKDA_F32, V, conv_step<DT, vec>()>(part, (size_t)w * D, d0, D, vec, dw[w]);
    conv_store<MKDA_F32, V, conv_step<DT, vec>()>(part, (size_t)W * D, d0, D, vec, db);
}

template <int DT, int W, int V, bool vec>
__global__ void __launch_bounds__(128) conv_step_kernel(const MkdaConvStep p) {
    follow_stream();
    constexpr int P = V / 2;
    const int D = p.D, d0 = conv_channel<DT, V, vec>(), n = blockIdx.y;
    if (d0 >= D) return;
    f32x2 rows[W][P], wt[W][P], y[P];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_unpack<DT, V>(conv_raw<DT, V>(p.state, ((size_t)n * (W - 1) + j) * D, d0, D, vec), rows[j]);
    conv_unpack<DT, V>(conv_raw<DT, V>(p.x, (size_t)n * p.x_stride, d0, D, vec), rows[W - 1]);
    conv_params<W, V>(p.weight, p.bias, d0, D, conv_step<DT, vec>(), wt, y);
#pragma unroll
    for (int e = 0; e < P; ++e) {
#pragma unroll
        for (int w = 0; w < W; ++w) y[e] = fma2(wt[w][e], rows[w][e], y[e]);
        if (p.silu) y[e] = mul2(y[e], sigmoidf2_(y[e]));
    }
    conv_store<DT, V>(p.y, (size_t)n * D, d0, D, vec, y);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_store<DT, V>(p.state, ((size_t)n * (W - 1) + j) * D, d0, D, vec, rows[j + 1]);
}

// Tokens per run, a multiple of the batch: whole waves of blocks, of runs up to 128 tokens (the W - 1 rows in front of a run are read twice), and in short calls
// runs of no less than `least`.
static long long conv_run(long long tokens, int blocks, int per_sm, long long least) {
    const long long resident = (long long)per_sm * sm_count(), work = tokens * blocks, waves = (work + resident * 128 - 1) / (resident * 128);
    long long run = waves ? (work + resident * waves - 1) / (resident * waves) : 1;
    run = (run < least ? least : run) + CONV_BATCH - 1;
    run -= run % CONV_BATCH;
    return (tokens + run - 1) / run > 65535 ? (tokens + 65534) / 65535 : run;
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
    const bool vec4 = p->D % 4 == 0 && p->x_stride % 4 == 0 && aligned16(p->x) && aligned16(p->weight) && aligned16(p->y) && aligned16(p->state) && aligned16(p->last);
    const bool vec8 = vec4 && p->D % 8 == 0 && p->x_stride % 8 == 0;
    with_dtype(p->dtype, [&](auto dt) {
        with_taps(p->W, [&](auto w) {
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value;
            auto run = [&](auto v, auto wide) {
                constexpr int V = decltype(v)::value;
                constexpr bool vec = decltype(wide)::value;
                const int blocks = (p->D + 128 * V - 1) / (128 * V);
                const long long run = conv_run(p->S.TT, blocks, CONV_FWD_BLOCKS, 8);
                const int rows = (int)((p->S.TT + run - 1) / run);
                launch(conv_fwd_kernel<DT, W, V, vec>, dim3(blocks, rows ? rows : 1), 128, 0, (cudaStream_t)stream, *p, (int)run);
            };
            // eight channels of 16 bits a thread, four where rows are only multiples of 8 bytes (8192 x 4096 30 and 31 us)
            using std::integral_constant;
            if constexpr (DT == MKDA_F32) {
                if (vec4) run(integral_constant<int, 4>(), std::true_type());
                else run(integral_constant<int, 4>(), std::false_type());
            } else {
                if (vec8) run(integral_constant<int, 8>(), std::true_type());
                else if (vec4) run(integral_constant<int, 4>(), std::true_type());
                else run(integral_constant<int, 8>(), std::false_type());
            }
        });
    });
    return check_launch("conv_fwd");
}

static long long conv_bwd_run(int TT, int D) { return conv_run(TT, (D + 511) / 512, CONV_BWD_BLOCKS, 16); }
extern "C" int mkda_conv_bwd_part_rows(int TT, int D) {
    const long long run = conv_bwd_run(TT, D);
    return TT > run ? (int)((TT + run - 1) / run) : 1;
}

extern "C" int mkda_conv_bwd(const MkdaConvBwd* p, void* stream) {
    if (!p || !p->weight || !p->part || (p->S.TT && (!p->x || !p->dy || !p->dx))) return set_error(MKDA_ERR_ARG, "conv_bwd: null argument");
    if (p->W < 2 || p->W > 4 || p->D <= 0 || !good_sequences(p->S)) return set_error(MKDA_ERR_ARG, "conv_bwd: 2 to 4 taps, at least one channel");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "conv_bwd: unsupported dtype");
    if (p->part_rows != mkda_conv_bwd_part_rows(p->S.TT, p->D)) return set_error(MKDA_ERR_ARG, "conv_bwd: as many rows of partial sums as mkda_conv_bwd_part_rows says");
    with_dtype(p->dtype, [&](auto dt) {
        with_taps(p->W, [&](auto w) {
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value, V = 4;
            const int blocks = (p->D + 128 * V - 1) / (128 * V), run = (int)conv_bwd_run(p->S.TT, p->D);
            const bool vec = p->D % V == 0 && p->x_stride % V == 0 && aligned16(p->x) && aligned16(p->weight) && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->state) && aligned16(p->dlast) &&
                             aligned16(p->dstate) && aligned16(p->part);
            launch(vec ? conv_bwd_kernel<DT, W, V, true> : conv_bwd_kernel<DT, W, V, false>, dim3(blocks, p->part_rows), 128, 0, (cudaStream_t)stream, *p, run);
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
            constexpr int DT = decltype(dt)::value, W = decltype(w)::value, V = 4;
            const bool vec = p->D % V == 0 && p->x_stride % V == 0 && aligned16(p->x) && aligned16(p->weight) && aligned16(p->y) && aligned16(p->state);
            launch(vec ? conv_step_kernel<DT, W, V, true> : conv_step_kernel<DT, W, V, false>, dim3((p->D + 128 * V - 1) / (128 * V), p->N), 128, 0, (cudaStream_t)stream, *p);
        });
    });
    return check_launch("conv_step");
}
