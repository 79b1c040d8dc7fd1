// Selective scan: a diagonal state of NST numbers per channel,
//   d = softplus(dt + bias)     h_n = exp(d A_n) h_n + d x B_n     y = sum_n C_n h_n + D x     out = y silu(z)
// and its backward pass
//   g_n[t] = dy C_n + exp(d A_n)[t + 1] g_n[t + 1]     e_n = g_n exp(d A_n) h_n[t - 1]
//   dC_n = sum_channels dy h_n     dB_n = sum_channels g_n d x     dA_n = sum_t e_n d     d(d) = x sum_n g_n B_n + sum_n e_n A_n     dx = d sum_n g_n B_n + D dy
//
// Layout.  A thread holds four states of CPT channels; LPC lanes share a channel (4 LPC states, NST padded with states whose B and C are zero).  A block of four
// warps walks a sequence tile by tile: the elementwise part of a tile (loads of eight channels, softplus, gate, stores) is done by all threads with
// one layout, the recurrence with the other, and the tile passes between the two through shared memory.  The rows of the next tile are requested
// before the recurrence of this one and wait in registers.  Sums over the states of a channel are butterflies in which each lane ends with the
// sum of a token of its own.  All in fp32.
#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int SCAN_THREADS = 128, SCAN_WARPS = SCAN_THREADS / 32, CKPT = MKDA_SCAN_CHECKPOINT;

template <int LPC, int CPT, int TILE>
struct ScanShape {
    static constexpr int NP = 4 * LPC;                     // padded states
    static constexpr int CB = SCAN_THREADS / LPC * CPT;    // channels per block
    static constexpr int ROW = CB / 8;                     // pieces of eight channels in a row
    static constexpr int PIECES = (TILE * ROW + SCAN_THREADS - 1) / SCAN_THREADS;      // per thread
    static constexpr int BC = (TILE * NP / 8 + SCAN_THREADS - 1) / SCAN_THREADS;       // pieces of B (and of C) per thread
    static constexpr int YROW = CB + 8;                    // floats of a row of sums: the four tokens of a butterfly lie in different banks
};

// softplus with its relative error small everywhere: log(1 + u) = 2 artanh(u / (2 + u)), u = exp(-|s|) in (0, 1], by the series of artanh
// (argument at most 1/3: seven terms leave 2e-8).  A dt of 1e-3 is a small u; the logarithm of 1 + u would lose its digits.
__device__ __forceinline__ float scan_softplus(float s) {
    const float u = expf_(-fabsf(s)), w = __fdividef(u, 2.f + u), q = w * w;
    float r = fmaf(q, 1.f / 13.f, 1.f / 11.f);
    r = fmaf(q, r, 1.f / 9.f);
    r = fmaf(q, r, 1.f / 7.f);
    r = fmaf(q, r, 1.f / 5.f);
    r = fmaf(q, r, 1.f / 3.f);
    r = fmaf(q, r, 1.f);
    return fmaxf(s, 0.f) + 2.f * w * r;
}

// Sums over the LPC lanes of a channel of four values each: v[0..3] of lane q become one (LPC >= 4: of token q & 3, in v[0]; LPC = 2: of
// tokens q and q + 2, in v[0] and v[1]).
template <int LPC>
__device__ __forceinline__ void lanes_sum4(float (&v)[4], int q) {
    const bool odd = q & 1;
    const float s0 = odd ? v[0] : v[1], s1 = odd ? v[2] : v[3];
    v[0] = (odd ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, s0, 1);
    v[1] = (odd ? v[3] : v[2]) + __shfl_xor_sync(0xffffffffu, s1, 1);
    if constexpr (LPC >= 4) {
        const bool up = q & 2;
        const float s = up ? v[0] : v[1];
        v[0] = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, s, 2);
#pragma unroll
        for (int b = 4; b < LPC; b <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], b);
    }
}
// ... and where they go: sums[token][channel] of the four tokens from `t` on
template <int LPC, int YROW>
__device__ __forceinline__ void put_sums(float* sums, int t, int ch, const float (&v)[4], int q) {
    if constexpr (LPC == 2) {
        sums[(t + q) * YROW + ch] = v[0];
        sums[(t + q + 2) * YROW + ch] = v[1];
    } else if (LPC == 4 || q < 4) {
        sums[(t + (q & 3)) * YROW + ch] = v[0];
    }
}

__device__ __forceinline__ f32x2 lo2(const float4& v) { return pack2(v.x, v.y); }
__device__ __forceinline__ f32x2 hi2(const float4& v) { return pack2(v.z, v.w); }
__device__ __forceinline__ float sum2(f32x2 v) { float a, b; unpack2(v, a, b); return a + b; }

// four states of a channel: NST may be anything up to the padded number
__device__ __forceinline__ float4 ld_states(const float* base, size_t row, int n0, int NST) {
    if ((NST & 3) == 0) return n0 < NST ? *reinterpret_cast<const float4*>(base + row * NST + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = n0 + i < NST ? base[row * NST + n0 + i] : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void st_states(float* base, size_t row, int n0, int NST, const float4& v) {
    if ((NST & 3) == 0) {
        if (n0 < NST) *reinterpret_cast<float4*>(base + row * NST + n0) = v;
        return;
    }
    const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + i < NST) base[row * NST + n0 + i] = w[i];
}

// Channels of a block: `first` of the whole, `count` of them exist (a block never straddles two groups)
struct Channels { int group, first, count; };
__device__ __forceinline__ Channels channels_of(int block, int D, int G, int CB) {
    const int per = D / G, blocks = (per + CB - 1) / CB, g = block / blocks, b = block - g * blocks;
    return Channels{g, g * per + b * CB, min(CB, per - b * CB)};
}

// Forward.  Four warps walk the recurrence and four beside them do the elementwise part, a tile ahead (loads, softplus) and a tile behind (skip, gate, stores); the block's
// barrier joins them once a tile.  A channel's chain is short and there are few warps of it (4096 channels are 512), so what counts is how many cycles a token takes a warp that
// has a scheduler to itself: with the elementwise part in the same warps 168, of which 32 are the exponentials of the special function unit.
constexpr int SCAN_HELPERS = 256;
template <int LPC, int TILE>
struct ScanFwdShared {
    using Sh = ScanShape<LPC, 1, TILE>;
    float2 d[2][TILE][Sh::CB];             // d, d x
    float B[2][TILE][Sh::NP], C[2][TILE][Sh::NP], y[2][TILE][Sh::YROW];
};

template <int DT, int LPC>
__global__ void __launch_bounds__(SCAN_THREADS + SCAN_HELPERS, 1) scan_fwd_kernel(const MkdaScanFwd p, const bool vec, const bool bvec) {
    follow_stream();
    constexpr int TILE = 32;
    using Sh = ScanShape<LPC, 1, TILE>;
    constexpr int NP = Sh::NP, CB = Sh::CB, YROW = Sh::YROW;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    auto& sh = *reinterpret_cast<ScanFwdShared<LPC, TILE>*>(raw_shared);
    const int D = p.D, NST = p.NST;
    const Channels cs = channels_of(blockIdx.x, D, p.G, CB);
    if (threadIdx.x < SCAN_THREADS) {
        const int tid = threadIdx.x, q = tid % LPC, c0 = tid / LPC, n0 = 4 * q;
        const bool there = c0 < cs.count;
        const size_t ch = cs.first + c0;
        const float4 a = there ? ld_states(p.A, ch, n0, NST) : make_float4(0.f, 0.f, 0.f, 0.f);
        const f32x2 A0 = mul2(lo2(a), both(RCP_LN2)), A1 = mul2(hi2(a), both(RCP_LN2));
        for (int slot = blockIdx.y; slot < p.S.N; slot += gridDim.y) {
            const int n = p.S.order ? p.S.order[slot] : slot;
            const Span sq = sequence(p.S, n);
            const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
            const float4 v = p.h0 && there ? ld_states(p.h0, (size_t)n * D + ch, n0, NST) : make_float4(0.f, 0.f, 0.f, 0.f);
            f32x2 h0 = lo2(v), h1 = hi2(v);
            const size_t ck0 = p.ckpt ? (p.S.ckpt_off ? (size_t)p.S.ckpt_off[n] : (size_t)n * ((p.S.T + CKPT - 1) / CKPT)) : 0;
            float* ck = p.ckpt ? p.ckpt + (ck0 * D + ch) * NP + n0 : nullptr;
            __syncthreads();                               // the first tile is there
            for (int k = 0; k < tiles; ++k) {
                const int buf = k & 1, t0 = k * TILE;
                const float2* sd = &sh.d[buf][0][c0];
                const float* sB = &sh.B[buf][0][n0];
                const float* sC = &sh.C[buf][0][n0];
                float* sy = &sh.y[buf][0][0];
                // Four tokens at a time, three groups in flight: what a token reads is requested two groups ahead, its decays are formed one group ahead, between the
                // steps of the chain (the special function unit takes one of them every eight cycles), and the sums of a group are finished in the next one.
                struct Token { float2 d; float4 B, C; };
                auto fetch = [&](int t) {
                    Token x;
                    x.d = sd[t * CB];
                    x.B = *reinterpret_cast<const float4*>(sB + t * NP);
                    x.C = *reinterpret_cast<const float4*>(sC + t * NP);
                    return x;
                };
                Token now[4], next[4];
                f32x2 e[4][2], en[4][2];
                float ys[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) now[u] = fetch(u);
#pragma unroll
                for (int u = 0; u < 4; ++u) next[u] = fetch(4 + u);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    e[u][0] = ex2f2_(mul2(A0, both(now[u].d.x)));
                    e[u][1] = ex2f2_(mul2(A1, both(now[u].d.x)));
                }
#pragma unroll
                for (int t4 = 0; t4 < TILE; t4 += 4) {
                    if (t4 % CKPT == 0 && ck && there && t0 + t4 < len) {
                        float4 w;
                        unpack2(h0, w.x, w.y);
                        unpack2(h1, w.z, w.w);
                        *reinterpret_cast<float4*>(ck + (size_t)((t0 + t4) / CKPT) * D * NP) = w;
                    }
                    float yn[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (t4 + 4 < TILE) {
                            en[u][0] = ex2f2_(mul2(A0, both(next[u].d.x)));
                            en[u][1] = ex2f2_(mul2(A1, both(next[u].d.x)));
                        }
                        const f32x2 dx = both(now[u].d.y);
                        h0 = fma2(e[u][0], h0, mul2(dx, lo2(now[u].B)));
                        h1 = fma2(e[u][1], h1, mul2(dx, hi2(now[u].B)));
                        yn[u] = sum2(fma2(h1, hi2(now[u].C), mul2(h0, lo2(now[u].C))));
                        now[u] = next[u];
                        if (t4 + 8 < TILE) next[u] = fetch(t4 + 8 + u);
                        e[u][0] = en[u][0];
                        e[u][1] = en[u][1];
                    }
                    if (t4) {
                        lanes_sum4<LPC>(ys, q);
                        put_sums<LPC, YROW>(sy, t4 - 4, c0, ys, q);
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) ys[u] = yn[u];
                }
                lanes_sum4<LPC>(ys, q);
                put_sums<LPC, YROW>(sy, TILE - 4, c0, ys, q);
                __syncthreads();
            }
            if (p.ht && there) {
                float4 w;
                unpack2(h0, w.x, w.y);
                unpack2(h1, w.z, w.w);
                st_states(p.ht, (size_t)n * D + ch, n0, NST, w);
            }
            __syncthreads();                               // the last tile has been stored
        }
        return;
    }

    // the elementwise part: four channels of a token in a piece, the same channels in all pieces of a thread; half of the threads bring B, half C
    constexpr int HELPERS = SCAN_HELPERS, ROW = CB / 4, STEP = HELPERS / ROW, PIECES = (TILE * ROW + HELPERS - 1) / HELPERS;
    constexpr int BROW = NP / 4, BSTEP = HELPERS / 2 / BROW, BC = (TILE * BROW * 2 + HELPERS - 1) / HELPERS;
    const int tid = threadIdx.x - SCAN_THREADS, ec = tid % ROW * 4, et = tid / ROW, valid = cs.count - ec;
    const int half = tid / (HELPERS / 2), bn = tid % BROW * 4, bt = tid % (HELPERS / 2) / BROW, bvalid = NST - bn;
    const void* const bc = half ? p.C : p.B;
    const long long bc_stride = half ? p.C_stride : p.B_stride;
    float bias[4], skip[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias[e] = p.dt_bias && ec + e < cs.count ? p.dt_bias[cs.first + ec + e] : 0.f;
        skip[e] = p.skip && ec + e < cs.count ? p.skip[cs.first + ec + e] : 0.f;
    }
    for (int slot = blockIdx.y; slot < p.S.N; slot += gridDim.y) {
        const Span sq = sequence(p.S, p.S.order ? p.S.order[slot] : slot);
        const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
        Raw4<DT> rx[PIECES], rd[PIECES], rz[PIECES], rb[BC];                             // of the tile that is formed next
        Raw4<DT> x1[PIECES], z1[PIECES], x2[PIECES], z2[PIECES];                         // of the tiles one and two behind it
        auto request = [&](int k) {
            const int t0 = k * TILE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int t = t0 + et + i * STEP;
                const int ok = et + i * STEP < TILE && t < len ? valid : 0;
                const size_t tok = (size_t)(sq.start + t);
                rx[i] = load4<DT>(p.x, tok * p.x_stride + cs.first + ec, ok, vec);
                rd[i] = load4<DT>(p.dt, tok * p.dt_stride + cs.first + ec, ok, vec);
                if (p.z) rz[i] = load4<DT>(p.z, tok * p.z_stride + cs.first + ec, ok, vec);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int t = t0 + bt + i * BSTEP;
                const int ok = bt + i * BSTEP < TILE && t < len ? bvalid : 0;
                rb[i] = load4<DT>(bc, (size_t)(sq.start + t) * bc_stride + cs.group * NST + bn, ok, bvec);
            }
        };
        request(0);
        for (int k = -1; k <= tiles; ++k) {                // forms tile k + 1, stores tile k - 1
            if (k + 1 < tiles) {
                const int buf = (k + 1) & 1, t0 = (k + 1) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (t >= TILE) continue;
                    const bool there = t0 + t < len;       // d = 0 behind the last token: the state stays as it is
                    float x[4], d[4];
                    unpack4<DT>(rx[i], x);
                    unpack4<DT>(rd[i], d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        d[e] += bias[e];
                        if (p.softplus) d[e] = scan_softplus(d[e]);
                        d[e] = there ? d[e] : 0.f;
                        x[e] = there ? d[e] * x[e] : 0.f;
                    }
                    // two pairs at a time, in an order that keeps the eight threads of a store apart
                    const float4 w0 = make_float4(d[0], x[0], d[1], x[1]), w1 = make_float4(d[2], x[2], d[3], x[3]);
                    const int r = (tid >> 2) & 1;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 * r]) = r ? w1 : w0;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 - 2 * r]) = r ? w0 : w1;
                }
#pragma unroll
                for (int i = 0; i < BC; ++i) {
                    const int t = bt + i * BSTEP;
                    if (t >= TILE) continue;
                    float v[4];
                    unpack4<DT>(rb[i], v);
                    *reinterpret_cast<float4*>(half ? &sh.C[buf][t][bn] : &sh.B[buf][t][bn]) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
            if (k >= 1) {
                const int buf = (k - 1) & 1, t0 = (k - 1) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (t >= TILE || t0 + t >= len) continue;
                    const float4 s = *reinterpret_cast<const float4*>(&sh.y[buf][t][ec]);
                    float y[4] = {s.x, s.y, s.z, s.w}, x[4], z[4];
                    unpack4<DT>(x2[i], x);
                    if (p.z) unpack4<DT>(z2[i], z);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (p.skip) y[e] = fmaf(skip[e], x[e], y[e]);
                        if (p.z) y[e] *= z[e] * sigmoidf_(z[e]);
                    }
                    store4<DT>(p.y, (size_t)(sq.start + t0 + t) * D + cs.first + ec, min(valid, 4), vec, y);
                }
            }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) { x2[i] = x1[i]; z2[i] = z1[i]; x1[i] = rx[i]; z1[i] = rz[i]; }
            if (k + 2 < tiles) request(k + 2);
            __syncthreads();
        }
    }
}

// Backward: tiles of one checkpoint, from the last to the first.  Each is run forward from its checkpoint (a_n h_n[t - 1], from which h_n follows with one
// operation, goes to shared memory), then backward.  dB and dC are summed over the channels of a thread, then over the lanes of a warp by a
// butterfly that leaves each lane one of the sums, over the warps through shared memory, and over the blocks of channels by mkda_sum_rows: in a fixed order.
template <int LPC, int CPT>
struct ScanBwdShared {
    using Sh = ScanShape<LPC, CPT, CKPT>;
    float4 p[CKPT][CPT][SCAN_THREADS];                     // a h[t - 1]
    float2 d[CKPT][Sh::CB];                                // d, d x
    float dy[CKPT][Sh::CB];
    float B[CKPT][Sh::NP], C[CKPT][Sh::NP];
    float y[CKPT][Sh::YROW], gB[CKPT][Sh::YROW], eA[CKPT][Sh::YROW];
    float red[SCAN_WARPS][CKPT][2 * Sh::NP];               // dB and dC of each warp
    float bias[Sh::CB], skip[Sh::CB];
};

template <int DT, int LPC, int CPT>
__global__ void __launch_bounds__(SCAN_THREADS) scan_bwd_kernel(const MkdaScanBwd a, const bool vec, const bool bvec) {
    follow_stream();
    constexpr int TILE = CKPT;
    using Sh = ScanShape<LPC, CPT, TILE>;
    constexpr int NP = Sh::NP, CB = Sh::CB, ROW = Sh::ROW, PIECES = Sh::PIECES, BC = Sh::BC, YROW = Sh::YROW;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    ScanBwdShared<LPC, CPT>& sh = *reinterpret_cast<ScanBwdShared<LPC, CPT>*>(raw_shared);
    const MkdaScanFwd& p = a.f;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.D, NST = p.NST;
    const Channels cs = channels_of(blockIdx.x, D, p.G, CB);
    for (int c = tid; c < CB; c += SCAN_THREADS) {
        sh.bias[c] = p.dt_bias && c < cs.count ? p.dt_bias[cs.first + c] : 0.f;
        sh.skip[c] = p.skip && c < cs.count ? p.skip[cs.first + c] : 0.f;
    }
    const int q = tid % LPC, c0 = tid / LPC * CPT, n0 = 4 * q;
    f32x2 A[CPT][2], dA[CPT][2];
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const float4 v = c0 + c < cs.count ? ld_states(p.A, cs.first + c0 + c, n0, NST) : make_float4(0.f, 0.f, 0.f, 0.f);
        A[c][0] = mul2(lo2(v), both(RCP_LN2));
        A[c][1] = mul2(hi2(v), both(RCP_LN2));
        dA[c][0] = dA[c][1] = both(0.f);
    }
    const int ec = tid % ROW * 8, et = tid / ROW, valid = cs.count - ec;
    constexpr int STEP = SCAN_THREADS / ROW;
    const int bn = tid % (NP / 8) * 8, bt = tid / (NP / 8), bvalid = NST - bn;
    constexpr int BSTEP = SCAN_THREADS / (NP / 8);
    float acc_skip[8], acc_bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc_skip[e] = acc_bias[e] = 0.f;
    __syncthreads();

    for (int slot = blockIdx.y; slot < p.S.N; slot += gridDim.y) {
        const int n = p.S.order ? p.S.order[slot] : slot;
        const Span sq = sequence(p.S, n);
        const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
        const size_t ck0 = p.S.ckpt_off ? (size_t)p.S.ckpt_off[n] : (size_t)n * ((p.S.T + CKPT - 1) / CKPT);
        f32x2 G[CPT][2], h[CPT][2];                        // G: a[t + 1] g[t + 1]
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const float4 v = a.dht && c0 + c < cs.count ? ld_states(a.dht, (size_t)n * D + cs.first + c0 + c, n0, NST) : make_float4(0.f, 0.f, 0.f, 0.f);
            G[c][0] = lo2(v);
            G[c][1] = hi2(v);
        }
        Raw8 rx[PIECES], rd[PIECES], rz[PIECES], ry[PIECES], rB[BC], rC[BC];
        float4 rh[CPT];
        auto request = [&](int k) {
            const int t0 = k * TILE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int t = t0 + et + i * STEP;
                const int ok = et + i * STEP < TILE && t < len ? valid : 0;
                const size_t tok = (size_t)(sq.start + t);
                rx[i] = load8<DT>(p.x, tok * p.x_stride + cs.first + ec, ok, vec);
                rd[i] = load8<DT>(p.dt, tok * p.dt_stride + cs.first + ec, ok, vec);
                if (p.z) rz[i] = load8<DT>(p.z, tok * p.z_stride + cs.first + ec, ok, vec);
                ry[i] = load8<DT>(a.dy, tok * D + cs.first + ec, ok, vec);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int t = t0 + bt + i * BSTEP;
                const int ok = bt + i * BSTEP < TILE && t < len ? bvalid : 0;
                const size_t tok = (size_t)(sq.start + t);
                rB[i] = load8<DT>(p.B, tok * p.B_stride + cs.group * NST + bn, ok, bvec);
                rC[i] = load8<DT>(p.C, tok * p.C_stride + cs.group * NST + bn, ok, bvec);
            }
#pragma unroll
            for (int c = 0; c < CPT; ++c)
                rh[c] = c0 + c < cs.count ? *reinterpret_cast<const float4*>(p.ckpt + ((ck0 + k) * D + cs.first + c0 + c) * NP + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        if (tiles) request(tiles - 1);
        for (int k = tiles - 1; k >= 0; --k) {
            const int t0 = k * TILE;
            float x[PIECES][8], z[PIECES][8], up[PIECES][8], s[PIECES][8];      // s: dt with its bias
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                unpack8<DT>(rx[i], x[i]);
                unpack8<DT>(rd[i], s[i]);
                if (p.z) unpack8<DT>(rz[i], z[i]);
                unpack8<DT>(ry[i], up[i]);
                const int t = et + i * STEP;
                if (t >= TILE) continue;
                const bool there = t0 + t < len;
                float dy[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    s[i][e] += sh.bias[ec + e];
                    const float d = there ? p.softplus ? scan_softplus(s[i][e]) : s[i][e] : 0.f;
                    sh.d[t][ec + e] = make_float2(d, there ? d * x[i][e] : 0.f);
                    dy[e] = p.z ? up[i][e] * z[i][e] * sigmoidf_(z[i][e]) : up[i][e];
                }
                st8<MKDA_F32>(&sh.dy[t][ec], 0, dy);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int t = bt + i * BSTEP;
                if (t >= TILE) continue;
                float b[8], c[8];
                unpack8<DT>(rB[i], b);
                unpack8<DT>(rC[i], c);
                st8<MKDA_F32>(&sh.B[t][bn], 0, b);
                st8<MKDA_F32>(&sh.C[t][bn], 0, c);
            }
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                h[c][0] = lo2(rh[c]);
                h[c][1] = hi2(rh[c]);
            }
            __syncthreads();
            if (k > 0) request(k - 1);
#pragma unroll 1
            for (int t4 = 0; t4 < TILE; t4 += 4) {
                float ys[CPT][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int t = t4 + u;
                    const float4 B = *reinterpret_cast<const float4*>(&sh.B[t][n0]), C = *reinterpret_cast<const float4*>(&sh.C[t][n0]);
#pragma unroll
                    for (int c = 0; c < CPT; ++c) {
                        const float2 d = sh.d[t][c0 + c];
                        const f32x2 dd = both(d.x), dx = both(d.y);
                        const f32x2 p0 = mul2(ex2f2_(mul2(A[c][0], dd)), h[c][0]), p1 = mul2(ex2f2_(mul2(A[c][1], dd)), h[c][1]);
                        float4 v;
                        unpack2(p0, v.x, v.y);
                        unpack2(p1, v.z, v.w);
                        sh.p[t][c][tid] = v;
                        h[c][0] = fma2(dx, lo2(B), p0);
                        h[c][1] = fma2(dx, hi2(B), p1);
                        ys[c][u] = p.z ? sum2(fma2(h[c][1], hi2(C), mul2(h[c][0], lo2(C)))) : 0.f;
                    }
                }
                if (p.z) {
#pragma unroll
                    for (int c = 0; c < CPT; ++c) {
                        lanes_sum4<LPC>(ys[c], q);
                        put_sums<LPC, YROW>(&sh.y[0][0], t4, c0 + c, ys[c], q);
                    }
                }
            }
#pragma unroll 1
            for (int t4 = TILE - 4; t4 >= 0; t4 -= 4) {
                float gBs[CPT][4], eAs[CPT][4];
#pragma unroll
                for (int u = 3; u >= 0; --u) {
                    const int t = t4 + u;
                    const float4 B = *reinterpret_cast<const float4*>(&sh.B[t][n0]), C = *reinterpret_cast<const float4*>(&sh.C[t][n0]);
                    f32x2 dB0 = both(0.f), dB1 = dB0, dC0 = dB0, dC1 = dB0;
#pragma unroll
                    for (int c = 0; c < CPT; ++c) {
                        const float2 d = sh.d[t][c0 + c];
                        const f32x2 dd = both(d.x), dx = both(d.y), dy = both(sh.dy[t][c0 + c]);
                        const float4 v = sh.p[t][c][tid];
                        const f32x2 p0 = lo2(v), p1 = hi2(v);
                        dC0 = fma2(dy, fma2(dx, lo2(B), p0), dC0);
                        dC1 = fma2(dy, fma2(dx, hi2(B), p1), dC1);
                        const f32x2 g0 = fma2(dy, lo2(C), G[c][0]), g1 = fma2(dy, hi2(C), G[c][1]);
                        dB0 = fma2(dx, g0, dB0);
                        dB1 = fma2(dx, g1, dB1);
                        gBs[c][u] = sum2(fma2(g1, hi2(B), mul2(g0, lo2(B))));
                        const f32x2 e0 = mul2(g0, p0), e1 = mul2(g1, p1);
                        eAs[c][u] = sum2(fma2(e1, A[c][1], mul2(e0, A[c][0])));
                        dA[c][0] = fma2(e0, dd, dA[c][0]);
                        dA[c][1] = fma2(e1, dd, dA[c][1]);
                        G[c][0] = mul2(ex2f2_(mul2(A[c][0], dd)), g0);
                        G[c][1] = mul2(ex2f2_(mul2(A[c][1], dd)), g1);
                    }
                    // over the lanes of other channels: eight sums over 32 / LPC lanes, halved as long as there are lanes to share them
                    float v[8];
                    unpack2(dB0, v[0], v[1]);
                    unpack2(dB1, v[2], v[3]);
                    unpack2(dC0, v[4], v[5]);
                    unpack2(dC1, v[6], v[7]);
                    const int cl = lane / LPC;
                    int first = 0;                         // of the sums that this lane ends with
#pragma unroll
                    for (int b = 0, w = 4; (LPC << b) < 32; ++b, w >>= 1) {
                        if (w >= 1) {
                            const bool up_ = cl >> b & 1;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (i >= w) break;
                                const float give = up_ ? v[i] : v[i + w], keep = up_ ? v[i + w] : v[i];
                                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, LPC << b);
                            }
                            first += up_ ? w : 0;
                        } else {
                            v[0] += __shfl_xor_sync(0xffffffffu, v[0], LPC << b);
                        }
                    }
                    constexpr int KEEP = LPC >= 4 ? LPC / 4 : 1;      // sums per lane: 1, 1, 2 or 4
                    if (LPC > 2 || cl < 8) {
#pragma unroll
                        for (int i = 0; i < KEEP; ++i) sh.red[warp][t][(first + i >= 4 ? NP : 0) + n0 + ((first + i) & 3)] = v[i];
                    }
                }
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    lanes_sum4<LPC>(gBs[c], q);
                    put_sums<LPC, YROW>(&sh.gB[0][0], t4, c0 + c, gBs[c], q);
                    lanes_sum4<LPC>(eAs[c], q);
                    put_sums<LPC, YROW>(&sh.eA[0][0], t4, c0 + c, eAs[c], q);
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int t = et + i * STEP;
                if (t >= TILE || t0 + t >= len) continue;
                float y[8], gB[8], eA[8], ox[8], od[8], oz[8];
                if (p.z) ld8(&sh.y[t][ec], MKDA_F32, 0, y);
                ld8(&sh.gB[t][ec], MKDA_F32, 0, gB);
                ld8(&sh.eA[t][ec], MKDA_F32, 0, eA);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float dy = up[i][e];
                    if (p.z) {
                        const float sg = sigmoidf_(z[i][e]), act = z[i][e] * sg;
                        oz[e] = dy * fmaf(sh.skip[ec + e], x[i][e], y[e]) * sg * fmaf(z[i][e], 1.f - sg, 1.f);
                        dy *= act;
                    }
                    ox[e] = fmaf(sh.skip[ec + e], dy, sh.d[t][ec + e].x * gB[e]);
                    od[e] = fmaf(x[i][e], gB[e], eA[e] * LN2);
                    if (p.softplus) od[e] *= sigmoidf_(s[i][e]);
                    acc_skip[e] = fmaf(dy, x[i][e], acc_skip[e]);
                    acc_bias[e] += od[e];
                }
                const size_t at = (size_t)(sq.start + t0 + t) * D + cs.first + ec;
                const int ok = min(valid, 8);
                store8<DT>(a.dx, at, ok, vec, ox);
                store8<DT>(a.ddt, at, ok, vec, od);
                if (p.z) store8<DT>(a.dz, at, ok, vec, oz);
            }
            for (int i = tid; i < TILE * NP * 2; i += SCAN_THREADS) {
                const int t = i / (2 * NP), o = i % (2 * NP);
                if (t0 + t >= len) break;
                const float v = (sh.red[0][t][o] + sh.red[1][t][o]) + (sh.red[2][t][o] + sh.red[3][t][o]);
                const size_t at = ((size_t)blockIdx.x * p.S.TT + sq.start + t0 + t) * NP;
                if (o < NP) a.part_B[at + o] = v;
                else a.part_C[at + o - NP] = v;
            }
            __syncthreads();                               // the shared tile may be written again
        }
        if (a.dh0) {
#pragma unroll
            for (int c = 0; c < CPT; ++c)
                if (c0 + c < cs.count) {
                    float4 v;
                    unpack2(G[c][0], v.x, v.y);
                    unpack2(G[c][1], v.z, v.w);
                    st_states(a.dh0, (size_t)n * D + cs.first + c0 + c, n0, NST, v);
                }
        }
    }
#pragma unroll
    for (int c = 0; c < CPT; ++c)
        if (c0 + c < cs.count) {
            float4 v;
            unpack2(dA[c][0], v.x, v.y);
            unpack2(dA[c][1], v.z, v.w);
            *reinterpret_cast<float4*>(a.part_A + ((size_t)blockIdx.y * D + cs.first + c0 + c) * NP + n0) = v;
        }
    // the threads that share eight channels, in order
    float* all = reinterpret_cast<float*>(&sh.p[0][0][0]);      // [2][threads][8]
    __syncthreads();
    st8<MKDA_F32>(all, tid * 8, acc_skip);
    st8<MKDA_F32>(all, (SCAN_THREADS + tid) * 8, acc_bias);
    __syncthreads();
    for (int c = tid; c < cs.count; c += SCAN_THREADS) {
        float s0 = 0.f, s1 = 0.f;
        for (int i = c / 8; i < SCAN_THREADS; i += ROW) {
            s0 += all[i * 8 + c % 8];
            s1 += all[(SCAN_THREADS + i) * 8 + c % 8];
        }
        if (a.part_skip) a.part_skip[(size_t)blockIdx.y * D + cs.first + c] = s0;
        if (a.part_bias) a.part_bias[(size_t)blockIdx.y * D + cs.first + c] = s1;
    }
}

// One token of each sequence.  Bound by HBM: the states are read and written.  A thread has four states of a channel, as above.
template <int DT, int LPC>
__global__ void __launch_bounds__(128) scan_step_kernel(const MkdaScanStep p) {
    follow_stream();
    const int q = threadIdx.x % LPC, c = blockIdx.x * (128 / LPC) + threadIdx.x / LPC, n = blockIdx.y, n0 = 4 * q, D = p.D, NST = p.NST;
    const bool there = c < D;
    float y = 0.f;
    if (there) {
        const size_t row = (size_t)n * D + c;
        const float4 h = ld_states(p.state, row, n0, NST), A = ld_states(p.A, c, n0, NST);
        const float x = ld1(p.x, DT, (size_t)n * p.x_stride + c);
        float d = ld1(p.dt, DT, (size_t)n * p.dt_stride + c) + (p.dt_bias ? p.dt_bias[c] : 0.f);
        if (p.softplus) d = scan_softplus(d);
        const float hs[4] = {h.x, h.y, h.z, h.w}, As[4] = {A.x, A.y, A.z, A.w};
        float o[4];
        const int g = c / (D / p.G);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ok = n0 + i < NST;
            const float B = ok ? ld1(p.B, DT, (size_t)n * p.B_stride + g * NST + n0 + i) : 0.f, C = ok ? ld1(p.C, DT, (size_t)n * p.C_stride + g * NST + n0 + i) : 0.f;
            o[i] = fmaf(ex2f_(As[i] * RCP_LN2 * d), hs[i], d * x * B);
            y = fmaf(C, o[i], y);
        }
        st_states(p.state, row, n0, NST, make_float4(o[0], o[1], o[2], o[3]));
        if (q == 0 && p.skip) y = fmaf(p.skip[c], x, y);
    }
#pragma unroll
    for (int b = 1; b < LPC; b <<= 1) y += __shfl_xor_sync(0xffffffffu, y, b);
    if (there && q == 0) {
        if (p.z) {
            const float z = ld1(p.z, DT, (size_t)n * p.z_stride + c);
            y *= z * sigmoidf_(z);
        }
        st1(p.y, DT, (size_t)n * D + c, y);
    }
}

// lanes per channel for NST states
template <typename F>
static void with_lanes(int NST, F f) {
    if (NST <= 8) f(std::integral_constant<int, 2>());
    else if (NST <= 16) f(std::integral_constant<int, 4>());
    else if (NST <= 32) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}
static int bad_scan(int D, int NST, int G, int dtype) {
    if (D <= 0 || G <= 0 || D % G) return set_error(MKDA_ERR_ARG, "scan: the channels must be a multiple of the groups");
    if (NST < 1 || NST > MKDA_SCAN_MAX_STATES) return set_error(MKDA_ERR_ARG, "scan: 1 to 64 states per channel");
    if (dtype < MKDA_F32 || dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "scan: unsupported dtype");
    return MKDA_OK;
}
// rows of channels, and of B and C, that can be read `w` elements at a time
static bool wide_rows(const MkdaScanFwd& f, int w) {
    return f.D / f.G % w == 0 && f.x_stride % w == 0 && f.dt_stride % w == 0 && (!f.z || f.z_stride % w == 0) && aligned16(f.x) && aligned16(f.dt) && aligned16(f.z);
}
static bool wide_states(const MkdaScanFwd& f, int w) { return f.NST % w == 0 && f.B_stride % w == 0 && f.C_stride % w == 0 && aligned16(f.B) && aligned16(f.C); }
static int blocks_of_channels(int D, int G, int CB) { return G * ((D / G + CB - 1) / CB); }

}  // namespace mkda

using namespace mkda;

extern "C" int mkda_scan_padded_states(int NST) { return NST <= 8 ? 8 : NST <= 16 ? 16 : NST <= 32 ? 32 : 64; }

extern "C" int mkda_scan_fwd(const MkdaScanFwd* p, void* stream) {
    if (!p || !p->A || (p->S.TT && (!p->x || !p->dt || !p->B || !p->C || !p->y))) return set_error(MKDA_ERR_ARG, "scan_fwd: null argument");
    if (int e = bad_scan(p->D, p->NST, p->G, p->dtype)) return e;
    if (!good_sequences(p->S) || (p->ckpt && p->S.cu && !p->S.ckpt_off)) return set_error(MKDA_ERR_ARG, "scan_fwd: bad sequences");
    if (!aligned16(p->A) || !aligned16(p->h0) || !aligned16(p->ht) || !aligned16(p->ckpt)) return set_error(MKDA_ERR_ARG, "scan_fwd: A and states must be 16-byte aligned");
    if (p->S.N == 0) return MKDA_OK;
    int rc = MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        with_lanes(p->NST, [&](auto l) {
            constexpr int DT = decltype(dt)::value, LPC = decltype(l)::value, smem = (int)sizeof(ScanFwdShared<LPC, 32>);
            const bool vec = wide_rows(*p, 4) && aligned16(p->y);
            const int blocks = blocks_of_channels(p->D, p->G, ScanShape<LPC, 1, 32>::CB);
            auto* kern = scan_fwd_kernel<DT, LPC>;
            rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "scan_fwd");
            if (rc == MKDA_OK)
                launch(kern, dim3(blocks, p->S.N < 65535 ? p->S.N : 65535), SCAN_THREADS + SCAN_HELPERS, smem, (cudaStream_t)stream, *p, vec, wide_states(*p, 4));
        });
    });
    if (rc != MKDA_OK) return rc;
    return check_launch("scan_fwd");
}

template <int LPC>
static constexpr int bwd_cpt() { return LPC <= 4 ? 2 : 2; }

extern "C" int mkda_scan_bwd_channel_blocks(int D, int G, int NST, int N) {
    (void)N;
    int r = 0;
    if (D > 0 && G > 0 && NST > 0 && NST <= MKDA_SCAN_MAX_STATES)
        with_lanes(NST, [&](auto l) { r = blocks_of_channels(D, G, ScanShape<decltype(l)::value, bwd_cpt<decltype(l)::value>(), CKPT>::CB); });
    return r;
}

extern "C" int mkda_scan_bwd(const MkdaScanBwd* p, void* stream) {
    if (!p || !p->f.A || !p->part_A ||
        (p->f.S.TT && (!p->f.x || !p->f.dt || !p->f.B || !p->f.C || !p->f.ckpt || !p->dy || !p->dx || !p->ddt || (p->f.z && !p->dz) || !p->part_B || !p->part_C)))
        return set_error(MKDA_ERR_ARG, "scan_bwd: null argument");
    if (int e = bad_scan(p->f.D, p->f.NST, p->f.G, p->f.dtype)) return e;
    if (!good_sequences(p->f.S) || (p->f.S.cu && !p->f.S.ckpt_off)) return set_error(MKDA_ERR_ARG, "scan_bwd: bad sequences");
    if (!aligned16(p->f.A) || !aligned16(p->f.ckpt) || !aligned16(p->dht) || !aligned16(p->dh0) || !aligned16(p->part_A))
        return set_error(MKDA_ERR_ARG, "scan_bwd: A, states and partial sums must be 16-byte aligned");
    if (p->slots < 1 || p->slots > 65535 || p->channel_blocks != mkda_scan_bwd_channel_blocks(p->f.D, p->f.G, p->f.NST, p->f.S.N))
        return set_error(MKDA_ERR_ARG, "scan_bwd: 1 to 65535 slots, and as many blocks of channels as mkda_scan_bwd_channel_blocks says");
    int rc = MKDA_OK;
    with_dtype(p->f.dtype, [&](auto dt) {
        with_lanes(p->f.NST, [&](auto l) {
            constexpr int DT = decltype(dt)::value, LPC = decltype(l)::value, CPT = bwd_cpt<LPC>();
            const MkdaScanFwd& f = p->f;
            const bool vec = wide_rows(f, 8) && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->ddt) && aligned16(p->dz);
            auto* kern = scan_bwd_kernel<DT, LPC, CPT>;
            constexpr int smem = (int)sizeof(ScanBwdShared<LPC, CPT>);
            rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "scan_bwd");
            if (rc == MKDA_OK) launch(kern, dim3(p->channel_blocks, p->slots), SCAN_THREADS, smem, (cudaStream_t)stream, *p, vec, wide_states(f, 8));
        });
    });
    return rc != MKDA_OK ? rc : check_launch("scan_bwd");
}

extern "C" int mkda_scan_step(const MkdaScanStep* p, void* stream) {
    if (!p || !p->A || (p->N && (!p->x || !p->dt || !p->B || !p->C || !p->state || !p->y))) return set_error(MKDA_ERR_ARG, "scan_step: null argument");
    if (int e = bad_scan(p->D, p->NST, p->G, p->dtype)) return e;
    if (p->N < 0 || p->N > 65535) return set_error(MKDA_ERR_ARG, "scan_step: at most 65535 sequences");
    if (!aligned16(p->A) || !aligned16(p->state)) return set_error(MKDA_ERR_ARG, "scan_step: A and the states must be 16-byte aligned");
    if (p->N == 0) return MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        with_lanes(p->NST, [&](auto l) {
            constexpr int DT = decltype(dt)::value, LPC = decltype(l)::value;
            launch(scan_step_kernel<DT, LPC>, dim3((p->D + 128 / LPC - 1) / (128 / LPC), p->N), 128, 0, (cudaStream_t)stream, *p);
        });
    });
    return check_launch("scan_step");
}
