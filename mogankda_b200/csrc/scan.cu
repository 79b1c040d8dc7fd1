// Selective scan: a diagonal state of NST numbers per channel,
//   d = softplus(dt + bias)     h_n = exp(d A_n) h_n + d x B_n     y = sum_n C_n h_n + D x     out = y silu(z)
// and its backward pass
//   g_n[t] = dy C_n + exp(d A_n)[t + 1] g_n[t + 1]     e_n = g_n exp(d A_n) h_n[t - 1]
//   dC_n = sum_channels dy h_n     dB_n = sum_channels g_n d x     dA_n = sum_t e_n d     d(d) = x sum_n g_n B_n + sum_n e_n A_n     dx = d sum_n g_n B_n + D dy
//
// Layout.  A thread holds four states of a channel; LPC lanes share a channel (4 LPC states, NST padded with states whose B and C are zero), 128 / LPC channels are a block.
// Four warps of a block walk the recurrence, others do the elementwise part (loads of four channels, softplus, gate, stores), tile by tile, with a layout of their own; tiles pass
// between the two through shared memory.  Sums over the states of a channel are butterflies in which each lane ends with the sum of a token of its own.  All in fp32: a decay
// is off by 2^-24 or so of itself, a state by the accumulated rounding of its memory.
// What bounds it: 16 exponentials per token and channel (16 states) are 118 us of the special function units for 8192 x 4096, HBM 41 us; the walk reads d, d x, B and C of every
// token from shared memory, 10 of its cycles a token and warp, which is 70 to 75 % of what an SM's shared memory gives.  bf16, 16 states, with gate: forward 8192 x 4096
// 280 us, 4 x 2048 x 4096 285 us; backward 2 x 2048 x 4096 406 us.
#include <cfloat>
#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int SCAN_THREADS = 128, SCAN_WARPS = SCAN_THREADS / 32, CKPT = MKDA_SCAN_CHECKPOINT;

template <int LPC>
struct ScanShape {
    static constexpr int NP = 4 * LPC;                     // padded states
    static constexpr int CB = SCAN_THREADS / LPC;          // channels per block
    static constexpr int YROW = CB + 8;                    // floats of a row of sums: the four tokens of a butterfly lie in different banks
};

// softplus with its relative error small everywhere: log(1 + u) = 2 artanh(u / (2 + u)), u = exp(-|s|) in (0, 1], by the series of artanh
// (argument at most 1/3: six terms leave 1.4e-7).  A dt of 1e-3 is a small u; the logarithm of 1 + u would lose its digits.
__device__ __forceinline__ f32x2 scan_softplus2(f32x2 s) {
    float a, b, c, d;
    unpack2(s, a, b);
    const f32x2 u = ex2f2_(pack2(-fabsf(a) * RCP_LN2, -fabsf(b) * RCP_LN2));
    unpack2(add2(u, both(2.f)), c, d);
    const f32x2 w = mul2(u, pack2(rcpf_(c), rcpf_(d))), q = mul2(w, w);
    f32x2 r = fma2(q, both(1.f / 11.f), both(1.f / 9.f));
    r = fma2(q, r, both(1.f / 7.f));
    r = fma2(q, r, both(1.f / 5.f));
    r = fma2(q, r, both(1.f / 3.f));
    r = fma2(q, r, both(1.f));
    return fma2(mul2(w, both(2.f)), r, pack2(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}
__device__ __forceinline__ float scan_softplus(float s) {
    float a, b;
    unpack2(scan_softplus2(both(s)), a, b);
    return a;
}

// exp(d A) for two states, A scaled by log2 e.  2^x of the special function unit is low in the mean: by 0.5e-8 to 1e-8 of itself for x in (-2^-8, 0), 2e-8 to 3e-8 down to -1, 5e-8
// below (measured over 2^18 arguments per octave).  A chain adds that up over its memory: states that keep a thousand tokens were off by 1e-6 to 3e-6 for it, twice what their
// roundings make.  So the argument is raised by 2.2e-8, in the product's own rounding.  An argument up to 8e-8 still gives 1 exactly: d = 0 leaves the state as it is.
__device__ __forceinline__ f32x2 scan_decay(f32x2 A, float d) { return ex2f2_(fma2(A, both(d), both(2.2e-8f))); }

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
__device__ __forceinline__ bool finite2(f32x2 v) { float a, b; unpack2(v, a, b); return fabsf(a) <= FLT_MAX && fabsf(b) <= FLT_MAX; }
__device__ __forceinline__ float sum2(f32x2 v) { float a, b; unpack2(v, a, b); return a + b; }

// four states of a channel: NST may be anything up to the padded number
__device__ __forceinline__ float4 ld_states(const float* base, size_t row, int n0, int NST) {
    if ((NST & 3) == 0) return n0 < NST ? *reinterpret_cast<const float4*>(base + row * NST + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = n0 + i < NST ? base[row * NST + n0 + i] : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}
// rates A, times log2 e, and no infinity: A * 0 has to be 0 where no time passes (the tokens behind a sequence's last one), also where A is infinite or its product with log2 e
// is.  The largest number leaves as little of a state as infinity does, for any d above 1e-36.
// NaN stays NaN.
__device__ __forceinline__ float4 rates(const float4& f) {
    float v[4] = {f.x * RCP_LN2, f.y * RCP_LN2, f.z * RCP_LN2, f.w * RCP_LN2};
#pragma unroll
    for (float& a : v) asm("{.reg .f32 t; max.NaN.f32 t, %0, %1; min.NaN.f32 %0, t, %2;}" : "+f"(a) : "f"(-FLT_MAX), "f"(FLT_MAX));
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

// all bits of those of the states n and n + 1 that are among the NST
__device__ __forceinline__ f32x2 real_states(int n, int NST) { return (n < NST ? 0xffffffffull : 0ull) | (n + 1 < NST ? 0xffffffffull << 32 : 0ull); }

// Channels of a block: `first` of the whole, `count` of them exist (a block never straddles two groups).  A launch has `blocks` blocks of each group, from the from-th on.
struct Channels { int group, first, count; };
__device__ __forceinline__ Channels channels_of(int block, int D, int G, int CB, int from, int blocks) {
    const int per = D / G, g = block / blocks, b = from + block - g * blocks;
    return Channels{g, g * per + b * CB, min(CB, per - b * CB)};
}

// A sequence, or the k-th part of one where sequences are cut: slots go over the sequences first.  `there`: a part that the sequence has.
struct Part { int n, k, start, end; bool there, last; };
__device__ __forceinline__ Part part_of(const MkdaSeqs& s, int slot) {
    const int k = slot / s.N, i = slot - k * s.N, n = s.order ? s.order[i] : i;
    const Span q = sequence(s, n);
    if (!s.seg) return Part{n, 0, q.start, q.end, true, true};
    const long long a = q.start + (long long)k * s.seg;
    const int end = (int)min(a + s.seg, (long long)q.end);
    return Part{n, k, (int)min(a, (long long)q.end), end, k == 0 || a < q.end, a + s.seg >= q.end};
}
__device__ __forceinline__ int parts(const MkdaSeqs& s) { return s.seg ? s.N * s.segs : s.N; }

// Forward.  Four warps walk the recurrence and four beside them do the elementwise part, a tile ahead (loads, softplus) and a tile behind (skip, gate, stores); the block's
// barrier joins them once a tile.  There are few warps on the chain (4096 channels are 512), so what counts is how many cycles a token takes a warp that
// has a scheduler to itself: 168 with the elementwise part in the same warps, 65 now, of which 32 are the exponentials of the special function unit.
constexpr int SCAN_HELPERS = 256, SCAN_LONG = 256;
// The backward kernel: threads beside those on the chain, blocks per SM, and the registers of the two roles out of those of the launch
constexpr int SCAN_BWD_HELPERS = 128, SCAN_BWD_THREADS = SCAN_THREADS + SCAN_BWD_HELPERS, SCAN_BWD_BLOCKS = 2, SCAN_BWD_WALK_REGS = 152, SCAN_BWD_HELP_REGS = 104, SCAN_BWD_LAUNCH_REGS = 128;
static_assert(SCAN_THREADS * SCAN_BWD_WALK_REGS + SCAN_BWD_HELPERS * SCAN_BWD_HELP_REGS <= SCAN_BWD_THREADS * SCAN_BWD_LAUNCH_REGS &&
              SCAN_BWD_THREADS * SCAN_BWD_LAUNCH_REGS * SCAN_BWD_BLOCKS <= 65536, "register split");
template <int LPC, int TILE>
struct ScanFwdShared {
    using Sh = ScanShape<LPC>;
    static constexpr int AHEAD = 8;        // rows behind the last one that are read and not used
    float2 d[2][TILE + AHEAD][Sh::CB];     // d, d x
    float B[2][TILE + AHEAD][Sh::NP], C[2][TILE + AHEAD][Sh::NP], y[2][TILE][Sh::YROW];
};
// four states of a channel
struct Four { f32x2 v[2]; };
__device__ __forceinline__ Four four(const float4& f) { return Four{{lo2(f), hi2(f)}}; }
__device__ __forceinline__ float4 flat(const Four& s) {
    float4 f;
    unpack2(s.v[0], f.x, f.y);
    unpack2(s.v[1], f.z, f.w);
    return f;
}

// `old` behind a part that makes `own` of nothing, in general `both`: nothing stays nothing, and infinity infinite, which no token's decay by itself ends
__device__ __forceinline__ float carried(float old, float both, float own) { return old == 0.f ? own : fabsf(old) > FLT_MAX ? old + own : both; }
// What enters a part: the state (or its gradient) that enters the sequence, carried over the parts in front (behind).  A (scaled by log2 e): of this lane.  A part's decay
// goes in by two halves, since the whole may leave the range where decay times state does not.
__device__ __forceinline__ void carry(Four& s, const Four& A, const MkdaSeqs& S, int n, int from, int to, int step, const float* seg_h, const float* seg_d, int D, size_t ch, int NP, int n0) {
    for (int j = from; j != to; j += step) {
        const size_t i = ((size_t)j * S.N + n) * D + ch;
        const Four h = four(*reinterpret_cast<const float4*>(seg_h + i * NP + n0));
        const f32x2 d = both(0.5f * seg_d[i]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const f32x2 half = ex2f2_(mul2(A.v[e], d)), first = mul2(half, s.v[e]);
            float a, b, a1, b1;
            unpack2(s.v[e], a, b);
            unpack2(fma2(half, first, h.v[e]), a1, b1);
            float ha, hb;
            unpack2(h.v[e], ha, hb);
            s.v[e] = pack2(carried(a, a1, ha), carried(b, b1, hb));
        }
    }
}

// (8192 x 4096: 280 us.  Two states a lane and twice the warps on the chain 10 % more; B and C in 16 bits side by side, or d and d x doubled for packed products, 20 %.)
// FILL: there are states that fill up a channel's lanes.  Their B and C are zero, but 0 times an infinite d or x is not: a tile after which they are not zero is walked once more
// (clearing them after every token of every tile lengthens the chain: 12 states, 8192 x 4096, 314 us for 272).
template <int DT, int LPC, int TILE, bool FILL>
__global__ void __launch_bounds__(SCAN_THREADS + SCAN_HELPERS, 1) scan_fwd_kernel(const MkdaScanFwd p, const bool vec, const bool bvec) {
    follow_stream();
    using Sh = ScanShape<LPC>;
    constexpr int NP = Sh::NP, CB = Sh::CB, YROW = Sh::YROW;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    auto& sh = *reinterpret_cast<ScanFwdShared<LPC, TILE>*>(raw_shared);
    const int D = p.D, NST = p.NST;
    const Channels cs = channels_of(blockIdx.x, D, p.G, CB, 0, (D / p.G + CB - 1) / CB);
    if (threadIdx.x < SCAN_THREADS) {
        const int tid = threadIdx.x, q = tid % LPC, c0 = tid / LPC, n0 = 4 * q;
        const bool there = c0 < cs.count;
        const size_t ch = cs.first + c0;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const Four A = four(rates(there ? ld_states(p.A, ch, n0, NST) : zero));
        const f32x2 real[2] = {real_states(n0, NST), real_states(n0 + 2, NST)};
        for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
            const Part sq = part_of(p.S, slot);
            if (!sq.there) continue;
            const int n = sq.n, len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
            Four h = four(p.h0 && there ? ld_states(p.h0, (size_t)n * D + ch, n0, NST) : zero);
            if (there) carry(h, A, p.S, n, 0, sq.k, 1, p.seg_h, p.seg_d, D, ch, NP, n0);
            if constexpr (FILL) { h.v[0] &= real[0]; h.v[1] &= real[1]; }
            const size_t ck0 = p.ckpt ? (p.S.ckpt_off ? (size_t)p.S.ckpt_off[n] : (size_t)n * ((p.S.T + CKPT - 1) / CKPT)) : 0;
            float* ck = p.ckpt ? p.ckpt + ((ck0 + (size_t)sq.k * (p.S.seg / CKPT)) * D + ch) * NP + n0 : nullptr;
            __syncthreads();                               // the first tile is there
            for (int k = 0; k < tiles; ++k) {
                const int buf = k & 1, t0 = k * TILE;
                const float2* sd = &sh.d[buf][0][c0];
                const float* sB = &sh.B[buf][0][n0];
                const float* sC = &sh.C[buf][0][n0];
                float* sy = &sh.y[buf][0][0];
                const Four entered = h;
                // Four tokens at a time, three groups in flight: what a token reads is requested two groups ahead, its decays are formed one group ahead, between the
                // steps of the chain (the special function unit takes one of them every eight cycles), and the sums of a group are finished in the next one.
                struct Token { float2 d; Four B, C; };
                auto fetch = [&](int t) {
                    Token x;
                    x.d = sd[t * CB];
                    x.B = four(*reinterpret_cast<const float4*>(sB + t * NP));
                    x.C = four(*reinterpret_cast<const float4*>(sC + t * NP));
                    return x;
                };
                Token now[4], next[4];
                Four e[4];
                float ys[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) now[u] = fetch(u);
#pragma unroll
                for (int u = 0; u < 4; ++u) next[u] = fetch(4 + u);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) e[u].v[i] = scan_decay(A.v[i], now[u].d.x);
#pragma unroll                                             // by 2, 4 or 8 groups 413, 341 and 315 us
                for (int t4 = 0; t4 < TILE; t4 += 4) {
                    if (t4 % CKPT == 0 && ck && there && t0 + t4 < len) *reinterpret_cast<float4*>(ck + (size_t)((t0 + t4) / CKPT) * D * NP) = flat(h);
                    float yn[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const f32x2 dx = both(now[u].d.y);
                        f32x2 y;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x2 d = e[u].v[i];
                            e[u].v[i] = scan_decay(A.v[i], next[u].d.x);
                            h.v[i] = fma2(d, h.v[i], mul2(dx, now[u].B.v[i]));
                            y = i ? fma2(h.v[i], now[u].C.v[i], y) : mul2(h.v[i], now[u].C.v[i]);
                        }
                        yn[u] = sum2(y);
                        now[u] = next[u];
                        next[u] = fetch(t4 + 8 + u);
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
                if constexpr (FILL) {
                    if (__any_sync(0xffffffffu, ((h.v[0] & ~real[0]) | (h.v[1] & ~real[1])) != 0)) {      // once more, the whole warp, clearing them after every token
                        h = entered;
#pragma unroll 1
                        for (int t4 = 0; t4 < TILE; t4 += 4) {
                            if (t4 % CKPT == 0 && ck && there && t0 + t4 < len) *reinterpret_cast<float4*>(ck + (size_t)((t0 + t4) / CKPT) * D * NP) = flat(h);
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const Token x = fetch(t4 + u);
                                f32x2 y;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    h.v[i] = fma2(scan_decay(A.v[i], x.d.x), h.v[i], mul2(both(x.d.y), x.B.v[i])) & real[i];
                                    y = i ? fma2(h.v[i], x.C.v[i], y) : mul2(h.v[i], x.C.v[i]);
                                }
                                ys[u] = sum2(y);
                            }
                            lanes_sum4<LPC>(ys, q);
                            put_sums<LPC, YROW>(sy, t4, c0, ys, q);
                        }
                    }
                }
                __syncthreads();
            }
            if (p.ht && there && sq.last) st_states(p.ht, (size_t)n * D + ch, n0, NST, flat(h));
            __syncthreads();                               // the last tile has been stored
        }
        return;
    }

    // the elementwise part: four channels of a token in a piece, the same channels in all pieces of a thread; half of the threads bring B, half C
    constexpr int HELPERS = SCAN_HELPERS, ROW = CB / 4, STEP = HELPERS / ROW, PIECES = (TILE * ROW + HELPERS - 1) / HELPERS;
    constexpr int BROW = NP / 4, BSTEP = HELPERS / 2 / BROW, BC = (TILE * BROW * 2 + HELPERS - 1) / HELPERS;
    const int tid = threadIdx.x - SCAN_THREADS, ec = tid % ROW * 4, et = tid / ROW, valid = cs.count - ec;
    const int half = tid / (HELPERS / 2), bn = tid % BROW * 4, bt = tid % (HELPERS / 2) / BROW, bvalid = NST - bn;
    constexpr int SIZE = DT == MKDA_F32 ? 4 : 2;
    const size_t x_pitch = (size_t)p.x_stride * SIZE, d_pitch = (size_t)p.dt_stride * SIZE, z_pitch = (size_t)p.z_stride * SIZE, y_pitch = (size_t)D * SIZE,
                 b_pitch = (size_t)(half ? p.C_stride : p.B_stride) * SIZE;
    float fb[4], fs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        fb[e] = p.dt_bias && ec + e < cs.count ? p.dt_bias[cs.first + ec + e] : 0.f;
        fs[e] = p.skip && ec + e < cs.count ? p.skip[cs.first + ec + e] : 0.f;
    }
    const f32x2 bias[2] = {pack2(fb[0], fb[1]), pack2(fb[2], fb[3])}, skip[2] = {pack2(fs[0], fs[1]), pack2(fs[2], fs[3])};
    const bool whole = STEP * PIECES == TILE && BSTEP * BC == TILE;      // every piece of every thread lies in the tile
    for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
        const Part sq = part_of(p.S, slot);
        if (!sq.there) continue;
        const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
        struct Rows { Raw4<DT> x[PIECES], d[PIECES], z[PIECES], b[BC]; };
        Rows even, odd;                                    // rows on their way, of every other tile: requested two steps before they are used
        Raw4<DT> x1[PIECES], z1[PIECES], x2[PIECES], z2[PIECES];      // of the two tiles behind the one that is formed
        // where this thread's first piece of the next tile to be requested, and to be stored, lies
        const size_t row = (size_t)sq.start + et, col = (size_t)(cs.first + ec) * SIZE;
        const char *px = static_cast<const char*>(p.x) + row * x_pitch + col, *pd = static_cast<const char*>(p.dt) + row * d_pitch + col,
                   *pz = static_cast<const char*>(p.z) + row * z_pitch + col,
                   *pb = static_cast<const char*>(half ? p.C : p.B) + ((size_t)sq.start + bt) * b_pitch + (size_t)(cs.group * NST + bn) * SIZE;
        char* py = static_cast<char*>(p.y) + row * y_pitch + col;
        auto request = [&](Rows& r, int k) {
            const int left = len - k * TILE;               // tokens from the tile's first on
            const bool inside = whole && left >= TILE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int t = et + i * STEP, ok = inside || (t < TILE && t < left) ? valid : 0;
                r.x[i] = load4<DT>(px + i * STEP * x_pitch, 0, ok, vec);
                r.d[i] = load4<DT>(pd + i * STEP * d_pitch, 0, ok, vec);
                if (p.z) r.z[i] = load4<DT>(pz + i * STEP * z_pitch, 0, ok, vec);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int t = bt + i * BSTEP;
                r.b[i] = load4<DT>(pb + i * BSTEP * b_pitch, 0, inside || (t < TILE && t < left) ? bvalid : 0, bvec);
            }
            px += TILE * x_pitch; pd += TILE * d_pitch; pz += TILE * z_pitch; pb += TILE * b_pitch;
        };
        auto step = [&](Rows& r, int k) {                  // forms tile k + 1, stores tile k - 1
            if (k + 1 < tiles) {
                const int buf = (k + 1) & 1, left = len - (k + 1) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (!whole && t >= TILE) continue;
                    f32x2 x[2], d[2];
                    unpack4_2<DT>(r.x[i], x);
                    unpack4_2<DT>(r.d[i], d);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        d[e] = add2(d[e], bias[e]);
                        if (p.softplus) d[e] = scan_softplus2(d[e]);
                        x[e] = mul2(d[e], x[e]);
                    }
                    float4 w0, w1;
                    unpack2(d[0], w0.x, w0.z);
                    unpack2(x[0], w0.y, w0.w);
                    unpack2(d[1], w1.x, w1.z);
                    unpack2(x[1], w1.y, w1.w);
                    if (left < TILE && t >= left) w0 = w1 = make_float4(0.f, 0.f, 0.f, 0.f);      // d = 0 behind the last token: the state stays as it is
                    // two pairs at a time, in an order that keeps the eight threads of a store apart
                    const int o = (tid >> 2) & 1;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 * o]) = o ? w1 : w0;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 - 2 * o]) = o ? w0 : w1;
                }
#pragma unroll
                for (int i = 0; i < BC; ++i) {
                    const int t = bt + i * BSTEP;
                    if (!whole && t >= TILE) continue;
                    float v[4];
                    unpack4<DT>(r.b[i], v);
                    *reinterpret_cast<float4*>(half ? &sh.C[buf][t][bn] : &sh.B[buf][t][bn]) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
            if (k >= 1) {
                const int buf = (k - 1) & 1, left = len - (k - 1) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if ((!whole && t >= TILE) || t >= left) continue;
                    const float4 f = *reinterpret_cast<const float4*>(&sh.y[buf][t][ec]);
                    f32x2 y[2] = {lo2(f), hi2(f)}, x[2], z[2];
                    unpack4_2<DT>(x2[i], x);
                    if (p.z) unpack4_2<DT>(z2[i], z);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (p.skip) y[e] = fma2(skip[e], x[e], y[e]);
                        if (p.z) y[e] = mul2(y[e], mul2(z[e], sigmoidf2_(z[e])));
                    }
                    float v[4];
                    unpack2(y[0], v[0], v[1]);
                    unpack2(y[1], v[2], v[3]);
                    store4<DT>(py + i * STEP * y_pitch, 0, min(valid, 4), vec, v);
                }
                py += TILE * y_pitch;
            }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) { x2[i] = x1[i]; z2[i] = z1[i]; x1[i] = r.x[i]; z1[i] = r.z[i]; }
            if (k + 3 < tiles) request(r, k + 3);
            __syncthreads();
        };
        request(even, 0);
        if (tiles > 1) request(odd, 1);
        for (int k = -1; k <= tiles; k += 2) {
            step(even, k);
            if (k + 1 <= tiles) step(odd, k + 1);
        }
    }
}

// Where there are fewer blocks than SMs and the sequences are long, these are cut into parts that run side by side.  This kernel finds what each part makes of nothing,
//   forward   h over the part from h = 0 (all parts but a sequence's last)     REV   g in front of the part from g = 0 behind it (all but the first)
// and the sum of its d, from which the part's decay follows; the main kernels carry the state over the parts in front of theirs.  It is the forward kernel without
// results per token; REV walks from the last token to the first.
template <int DT, int LPC, int TILE>
struct ScanPreShared {
    using Sh = ScanShape<LPC>;
    static constexpr int AHEAD = 8;
    float2 d[2][TILE + AHEAD][Sh::CB];     // d, and d x or the gradient of y
    float B[2][TILE + AHEAD][Sh::NP];      // B or C
};
template <int DT, int LPC, int TILE, bool REV>
__global__ void __launch_bounds__(SCAN_THREADS + SCAN_HELPERS, 1) scan_pre_kernel(const MkdaScanFwd p, const void* up, float* out_h, float* out_d, const int from, const int blocks, const bool vec, const bool bvec) {
    follow_stream();
    using Sh = ScanShape<LPC>;
    constexpr int NP = Sh::NP, CB = Sh::CB;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    auto& sh = *reinterpret_cast<ScanPreShared<DT, LPC, TILE>*>(raw_shared);
    const int D = p.D, NST = p.NST;
    const Channels cs = channels_of(blockIdx.x, D, p.G, CB, from, blocks);
    auto wanted = [](const Part& q) { return q.there && (REV ? q.k > 0 : !q.last); };
    if (threadIdx.x < SCAN_THREADS) {
        const int tid = threadIdx.x, q = tid % LPC, c0 = tid / LPC, n0 = 4 * q;
        const bool there = c0 < cs.count;
        const size_t ch = cs.first + c0;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const Four A = four(rates(there ? ld_states(p.A, ch, n0, NST) : zero));
        for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
            const Part sq = part_of(p.S, slot);
            if (!wanted(sq)) continue;
            const int tiles = (sq.end - sq.start + TILE - 1) / TILE;
            Four h = four(zero);
            float sum = 0.f;
            __syncthreads();                               // the first tile is there
            for (int k = 0; k < tiles; ++k) {
                const float2* sd = &sh.d[k & 1][0][c0];
                const float* sB = &sh.B[k & 1][0][n0];
                struct Token { float2 d; Four B; };
                auto fetch = [&](int t) { return Token{sd[t * CB], four(*reinterpret_cast<const float4*>(sB + t * NP))}; };
                Token now[4], next[4];
                Four e[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) now[u] = fetch(u);
#pragma unroll
                for (int u = 0; u < 4; ++u) next[u] = fetch(4 + u);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) e[u].v[i] = scan_decay(A.v[i], now[u].d.x);
#pragma unroll
                for (int t4 = 0; t4 < TILE; t4 += 4) {
                    float part[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        part[u] = now[u].d.x;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x2 a = e[u].v[i], v = both(now[u].d.y);
                            e[u].v[i] = scan_decay(A.v[i], next[u].d.x);
                            h.v[i] = REV ? mul2(a, fma2(v, now[u].B.v[i], h.v[i])) : fma2(a, h.v[i], mul2(v, now[u].B.v[i]));
                        }
                        now[u] = next[u];
                        next[u] = fetch(t4 + 8 + u);
                    }
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                }
                __syncthreads();
            }
            if (there) {
                const size_t i = ((size_t)sq.k * p.S.N + sq.n) * D + ch;
                *reinterpret_cast<float4*>(out_h + i * NP + n0) = flat(h);
                if (q == 0) out_d[i] = sum;
            }
        }
        return;
    }
    constexpr int HELPERS = SCAN_HELPERS, ROW = CB / 4, STEP = HELPERS / ROW, PIECES = (TILE * ROW + HELPERS - 1) / HELPERS;
    constexpr int BROW = NP / 4, BSTEP = HELPERS / BROW, BC = (TILE * BROW + HELPERS - 1) / HELPERS;
    const int tid = threadIdx.x - SCAN_THREADS, ec = tid % ROW * 4, et = tid / ROW, valid = cs.count - ec;
    const int bn = tid % BROW * 4, bt = tid / BROW, bvalid = NST - bn;
    float fb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) fb[e] = p.dt_bias && ec + e < cs.count ? p.dt_bias[cs.first + ec + e] : 0.f;
    const f32x2 bias[2] = {pack2(fb[0], fb[1]), pack2(fb[2], fb[3])};
    for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
        const Part sq = part_of(p.S, slot);
        if (!wanted(sq)) continue;
        const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
        struct Rows { Raw4<DT> d[PIECES], x[PIECES], z[PIECES], b[BC]; };      // x: x or the gradient of the output
        Rows even, odd;
        auto request = [&](Rows& r, int k) {               // row i of tile k is token TILE k + i, REV: from the end
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int row = et + i * STEP, t = k * TILE + row, ok = row < TILE && t < len ? valid : 0;
                const size_t tok = (size_t)(REV ? sq.end - 1 - t : sq.start + t), col = cs.first + ec;
                r.d[i] = load4<DT>(p.dt, tok * p.dt_stride + col, ok, vec);
                r.x[i] = REV ? load4<DT>(up, tok * D + col, ok, vec) : load4<DT>(p.x, tok * p.x_stride + col, ok, vec);
                if (REV && p.z) r.z[i] = load4<DT>(p.z, tok * p.z_stride + col, ok, vec);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int row = bt + i * BSTEP, t = k * TILE + row, ok = row < TILE && t < len ? bvalid : 0;
                const size_t tok = (size_t)(REV ? sq.end - 1 - t : sq.start + t), col = cs.group * NST + bn;
                r.b[i] = REV ? load4<DT>(p.C, tok * p.C_stride + col, ok, bvec) : load4<DT>(p.B, tok * p.B_stride + col, ok, bvec);
            }
        };
        auto step = [&](Rows& r, int k) {                  // forms tile k + 1
            if (k + 1 < tiles) {
                const int buf = (k + 1) & 1, left = len - (k + 1) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (t >= TILE) continue;
                    f32x2 d[2], x[2];
                    unpack4_2<DT>(r.d[i], d);
                    unpack4_2<DT>(r.x[i], x);
                    if (REV && p.z) {
                        f32x2 z[2];
                        unpack4_2<DT>(r.z[i], z);
#pragma unroll
                        for (int e = 0; e < 2; ++e) x[e] = mul2(x[e], mul2(z[e], sigmoidf2_(z[e])));
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        d[e] = add2(d[e], bias[e]);
                        if (p.softplus) d[e] = scan_softplus2(d[e]);
                        if (!REV) x[e] = mul2(d[e], x[e]);
                    }
                    float4 w0, w1;
                    unpack2(d[0], w0.x, w0.z);
                    unpack2(x[0], w0.y, w0.w);
                    unpack2(d[1], w1.x, w1.z);
                    unpack2(x[1], w1.y, w1.w);
                    if (t >= left) w0 = w1 = make_float4(0.f, 0.f, 0.f, 0.f);
                    const int o = (tid >> 2) & 1;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 * o]) = o ? w1 : w0;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 - 2 * o]) = o ? w0 : w1;
                }
#pragma unroll
                for (int i = 0; i < BC; ++i) {
                    const int t = bt + i * BSTEP;
                    if (t >= TILE) continue;
                    float v[4];
                    unpack4<DT>(r.b[i], v);
                    *reinterpret_cast<float4*>(&sh.B[buf][t][bn]) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
            if (k + 3 < tiles) request(r, k + 3);
            __syncthreads();
        };
        request(even, 0);
        if (tiles > 1) request(odd, 1);
        for (int k = -1; k < tiles; k += 2) {
            step(even, k);
            if (k + 1 < tiles) step(odd, k + 1);
        }
    }
}

// Backward: tiles of one checkpoint, from the last to the first, with the same two roles.  A tile is run forward from its checkpoint, then backward:
// a_n h_n[t - 1], from which h_n follows with one operation, stays in the registers of the lane in between (the decays beside it, not formed twice, left the rest too few:
// 1.5 % more).  dB and dC are summed over the lanes of a warp by a butterfly
// that leaves each lane one of the sums, over the warps through shared memory, and over the blocks of channels by mkda_sum_rows: in a fixed order.  bf16 with 16 states fits the
// registers; fp32 with 8 states keeps 456 bytes a thread in local memory (and one block per SM, for its shared memory), with 64 states 192, and scan_pre_kernel with tiles of 64 76.  Two blocks per SM: the
// chain and the butterflies are latency, and two channels per thread, which halve the butterflies but take the registers of the second block, were slower (525 us).
template <int DT, int LPC>
struct ScanBwdShared {
    static constexpr int PIECES = (CKPT * SCAN_THREADS / LPC / 4 + SCAN_BWD_HELPERS - 1) / SCAN_BWD_HELPERS;
    Raw4<DT> kept[4][4][PIECES][SCAN_BWD_HELPERS];         // x, dt, z and dy of the last tiles, each thread's own: registers are what the second block needs
    using Sh = ScanShape<LPC>;
    float2 d[2][CKPT][Sh::CB];                             // d, d x
    float dy[2][CKPT][Sh::CB];
    float B[2][CKPT][Sh::NP], C[2][CKPT][Sh::NP];
    float y[2][CKPT][Sh::YROW], gB[2][CKPT][Sh::YROW], eA[2][CKPT][Sh::YROW];
    float red[2][SCAN_WARPS][CKPT][2 * Sh::NP];            // dB and dC of each warp
};

template <int DT, int LPC>
__global__ void __launch_bounds__(SCAN_BWD_THREADS, SCAN_BWD_BLOCKS) scan_bwd_kernel(const MkdaScanBwd a, const bool vec, const bool bvec) {
    follow_stream();
    constexpr int TILE = CKPT;
    using Sh = ScanShape<LPC>;
    constexpr int NP = Sh::NP, CB = Sh::CB, YROW = Sh::YROW;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    auto& sh = *reinterpret_cast<ScanBwdShared<DT, LPC>*>(raw_shared);
    const MkdaScanFwd& p = a.f;
    const int D = p.D, NST = p.NST;
    const Channels cs = channels_of(blockIdx.x, D, p.G, CB, a.first_block, a.blocks);
    if (threadIdx.x < SCAN_THREADS) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(SCAN_BWD_WALK_REGS));
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, q = tid % LPC, c0 = tid / LPC, n0 = 4 * q, cl = lane / LPC;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const bool z = p.z, there = c0 < cs.count;
        const size_t ch = cs.first + c0;
        const Four A = four(rates(there ? ld_states(p.A, ch, n0, NST) : zero));
        Four dA = four(zero);
        for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
            const Part sq = part_of(p.S, slot);
            if (!sq.there) continue;
            const int n = sq.n, len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
            const size_t ck0 = (p.S.ckpt_off ? (size_t)p.S.ckpt_off[n] : (size_t)n * ((p.S.T + CKPT - 1) / CKPT)) + (size_t)sq.k * (p.S.seg / CKPT);
            auto checkpoint = [&](int k) { return there ? *reinterpret_cast<const float4*>(p.ckpt + ((ck0 + k) * D + ch) * NP + n0) : zero; };
            Four G = four(a.dht && there ? ld_states(a.dht, (size_t)n * D + ch, n0, NST) : zero);      // a[t + 1] g[t + 1]
            if (there && p.S.seg) {
                const Span all = sequence(p.S, n);
                carry(G, A, p.S, n, max((all.end - all.start + p.S.seg - 1) / p.S.seg - 1, 0), sq.k, -1, a.seg_g, a.seg_d, D, ch, NP, n0);
            }
            float4 rh = tiles ? checkpoint(tiles - 1) : zero;
            __syncthreads();                               // the first tile is there
            for (int j = 0; j < tiles; ++j) {
                const int buf = j & 1;
                const float2* sd = &sh.d[buf][0][c0];
                const float* sdy = &sh.dy[buf][0][c0];
                const float* sB = &sh.B[buf][0][n0];
                const float* sC = &sh.C[buf][0][n0];
                constexpr int SUMS = TILE / 4 * (LPC == 2 ? 2 : 1);      // sums over states that a lane ends with
                Four h = four(rh), P[TILE], dAt = four(zero);
                float ysum[SUMS];                          // they wait in registers: a store in between would keep reads behind it
#pragma unroll
                for (int t4 = 0; t4 < TILE; t4 += 4) {
                    float ys[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float2 d = sd[(t4 + u) * CB];
                        const Four B = four(*reinterpret_cast<const float4*>(sB + (t4 + u) * NP)), C = four(*reinterpret_cast<const float4*>(sC + (t4 + u) * NP));
                        f32x2 y;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x2 v = mul2(scan_decay(A.v[i], d.x), h.v[i]);
                            P[t4 + u].v[i] = v;
                            h.v[i] = fma2(both(d.y), B.v[i], v);
                            y = i ? fma2(h.v[i], C.v[i], y) : mul2(h.v[i], C.v[i]);
                        }
                        ys[u] = sum2(y);
                    }
                    if (z) {
                        lanes_sum4<LPC>(ys, q);
                        ysum[t4 / 4] = ys[0];
                        if constexpr (LPC == 2) ysum[TILE / 4 + t4 / 4] = ys[1];
                    }
                }
                if (tiles - 2 - j >= 0) rh = checkpoint(tiles - 2 - j);
                asm volatile("" ::: "memory");             // what the first pass has read is read again: kept for sixteen tokens it would not fit into the registers
                constexpr int KEEP = LPC >= 4 ? LPC / 4 : 1;      // sums of dB and dC per lane: 1, 1, 2 or 4
                float gsum[SUMS], esum[SUMS], red[TILE][KEEP];
                int first = 0;                             // of the sums of dB and dC that this lane ends with
#pragma unroll
                for (int t4 = TILE - 4; t4 >= 0; t4 -= 4) {
                    __syncwarp();                          // reads of the next tokens stay behind it, or their number takes the registers
                    float gBs[4], eAs[4];
#pragma unroll
                    for (int u = 3; u >= 0; --u) {
                        const int t = t4 + u;
                        const float2 d = sd[t * CB];
                        const float dy = sdy[t * CB];
                        const Four B = four(*reinterpret_cast<const float4*>(sB + t * NP)), C = four(*reinterpret_cast<const float4*>(sC + t * NP));
                        f32x2 v[4], gb, ea;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x2 g = fma2(both(dy), C.v[i], G.v[i]), e = mul2(g, P[t].v[i]);
                            v[i] = mul2(both(d.y), g);
                            v[i + 2] = mul2(both(dy), fma2(both(d.y), B.v[i], P[t].v[i]));
                            gb = i ? fma2(g, B.v[i], gb) : mul2(g, B.v[i]);
                            ea = i ? fma2(e, A.v[i], ea) : mul2(e, A.v[i]);
                            dAt.v[i] = fma2(e, both(d.x), dAt.v[i]);
                            G.v[i] = mul2(scan_decay(A.v[i], d.x), g);
                        }
                        gBs[u] = sum2(gb);
                        eAs[u] = sum2(ea);
                        // over the lanes of other channels: eight sums over 32 / LPC lanes, halved as long as there are lanes to share them
                        float w[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) unpack2(v[i], w[2 * i], w[2 * i + 1]);
                        int at = 0;
#pragma unroll
                        for (int b = 0, k = 4; (LPC << b) < 32; ++b, k >>= 1) {
                            if (k >= 1) {
                                const bool up = cl >> b & 1;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    if (i >= k) break;
                                    const float give = up ? w[i] : w[i + k], keep = up ? w[i + k] : w[i];
                                    w[i] = keep + __shfl_xor_sync(0xffffffffu, give, LPC << b);
                                }
                                at += up ? k : 0;
                            } else {
                                w[0] += __shfl_xor_sync(0xffffffffu, w[0], LPC << b);
                            }
                        }
                        first = at;
#pragma unroll
                        for (int i = 0; i < KEEP; ++i) red[t][i] = w[i];
                    }
                    lanes_sum4<LPC>(gBs, q);
                    lanes_sum4<LPC>(eAs, q);
                    gsum[t4 / 4] = gBs[0];
                    esum[t4 / 4] = eAs[0];
                    if constexpr (LPC == 2) {
                        gsum[TILE / 4 + t4 / 4] = gBs[1];
                        esum[TILE / 4 + t4 / 4] = eAs[1];
                    }
                }
                auto put = [&](float* to, const float (&v)[SUMS]) {
#pragma unroll
                    for (int i = 0; i < TILE / 4; ++i) {
                        if constexpr (LPC == 2) {
                            to[(4 * i + q) * YROW + c0] = v[i];
                            to[(4 * i + q + 2) * YROW + c0] = v[TILE / 4 + i];
                        } else if (LPC == 4 || q < 4) {
                            to[(4 * i + (q & 3)) * YROW + c0] = v[i];
                        }
                    }
                };
                if (z) put(&sh.y[buf][0][0], ysum);
                put(&sh.gB[buf][0][0], gsum);
                put(&sh.eA[buf][0][0], esum);
                if (LPC > 2 || cl < 8) {
#pragma unroll
                    for (int t = 0; t < TILE; ++t)
#pragma unroll
                        for (int i = 0; i < KEEP; ++i) sh.red[buf][warp][t][(first + i >= 4 ? NP : 0) + n0 + ((first + i) & 3)] = red[t][i];
                }
                if (j == 0 && len % TILE) {                // the same for all lanes
                    if (!(finite2(dAt.v[0]) && finite2(dAt.v[1]))) {
                        // The tokens that fill up the last tile add e * 0, which an infinite state behind the last token makes NaN and the definition does not have.  Formed anew without
                        // them, each token's state from the checkpoint: seldom enough, and the loop above stays as it is (with P set to zero there 2 x 2048 x 4096 took 409 us for 401).
                        Four g1 = four(a.dht && there ? ld_states(a.dht, (size_t)n * D + ch, n0, NST) : zero);
                        dAt = four(zero);
#pragma unroll 1
                        for (int t = len % TILE - 1; t >= 0; --t) {
                            Four hs = four(checkpoint(tiles - 1)), v;
                            float2 d;
#pragma unroll 1
                            for (int s = 0; s <= t; ++s) {
                                d = sd[s * CB];
                                const Four B = four(*reinterpret_cast<const float4*>(sB + s * NP));
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    v.v[i] = mul2(scan_decay(A.v[i], d.x), hs.v[i]);
                                    hs.v[i] = fma2(both(d.y), B.v[i], v.v[i]);
                                }
                            }
                            const Four C = four(*reinterpret_cast<const float4*>(sC + t * NP));
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const f32x2 g = fma2(both(sdy[t * CB]), C.v[i], g1.v[i]);
                                dAt.v[i] = fma2(mul2(g, v.v[i]), both(d.x), dAt.v[i]);
                                g1.v[i] = mul2(scan_decay(A.v[i], d.x), g);
                            }
                        }
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) dA.v[i] = add2(dA.v[i], dAt.v[i]);      // tile by tile: the sum over thousands of tokens loses less
                __syncthreads();
            }
            if (a.dh0 && there && sq.k == 0) st_states(a.dh0, (size_t)n * D + ch, n0, NST, flat(G));
            __syncthreads();                               // the last tile has been stored
        }
        if (there) *reinterpret_cast<float4*>(a.part_A + ((size_t)blockIdx.y * D + ch) * NP + n0) = flat(dA);
        __syncthreads();
        __syncthreads();                                   // the elementwise part's sums over tokens
        return;
    }

    // the elementwise part, laid out as in the forward kernel
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(SCAN_BWD_HELP_REGS));
    constexpr int HELPERS = SCAN_BWD_HELPERS, ROW = CB / 4, STEP = HELPERS / ROW, PIECES = (TILE * ROW + HELPERS - 1) / HELPERS;
    constexpr int BROW = NP / 4, BSTEP = HELPERS / 2 / BROW, BC = (TILE * BROW * 2 + HELPERS - 1) / HELPERS;
    const int tid = threadIdx.x - SCAN_THREADS, ec = tid % ROW * 4, et = tid / ROW, valid = cs.count - ec;
    const int half = tid / (HELPERS / 2), bn = tid % BROW * 4, bt = tid % (HELPERS / 2) / BROW, bvalid = NST - bn;
    constexpr int SIZE = DT == MKDA_F32 ? 4 : 2;
    const size_t x_pitch = (size_t)p.x_stride * SIZE, d_pitch = (size_t)p.dt_stride * SIZE, z_pitch = (size_t)p.z_stride * SIZE, y_pitch = (size_t)D * SIZE,
                 b_pitch = (size_t)(half ? p.C_stride : p.B_stride) * SIZE;
    float fb[4], fs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        fb[e] = p.dt_bias && ec + e < cs.count ? p.dt_bias[cs.first + ec + e] : 0.f;
        fs[e] = p.skip && ec + e < cs.count ? p.skip[cs.first + ec + e] : 0.f;
    }
    const f32x2 bias[2] = {pack2(fb[0], fb[1]), pack2(fb[2], fb[3])}, skip[2] = {pack2(fs[0], fs[1]), pack2(fs[2], fs[3])};
    const f32x2 skips = p.skip ? ~0ull : 0ull;             // without D there is no term of it, also beside values that are infinite (0 times infinity is no 0)
    f32x2 acc_skip[2] = {both(0.f), both(0.f)}, acc_bias[2] = {both(0.f), both(0.f)};
    for (int slot = blockIdx.y; slot < parts(p.S); slot += gridDim.y) {
        const Part sq = part_of(p.S, slot);
        if (!sq.there) continue;
        const int len = sq.end - sq.start, tiles = (len + TILE - 1) / TILE;
        struct Rows { Raw4<DT> x[PIECES], d[PIECES], z[PIECES], y[PIECES], b[BC]; };
        Rows even, odd;                                    // rows on their way, of every other tile: requested two steps before they are used
        const size_t col = (size_t)(cs.first + ec) * SIZE;
        auto request = [&](Rows& r, int j) {               // the j-th tile from the end
            const int t0 = (tiles - 1 - j) * TILE, left = len - t0;
            const size_t row = (size_t)(sq.start + t0 + et), brow = (size_t)(sq.start + t0 + bt);
            const char *px = static_cast<const char*>(p.x) + row * x_pitch + col, *pd = static_cast<const char*>(p.dt) + row * d_pitch + col,
                       *pz = static_cast<const char*>(p.z) + row * z_pitch + col, *py = static_cast<const char*>(a.dy) + row * y_pitch + col,
                       *pb = static_cast<const char*>(half ? p.C : p.B) + brow * b_pitch + (size_t)(cs.group * NST + bn) * SIZE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int t = et + i * STEP, ok = t < TILE && t < left ? valid : 0;
                r.x[i] = load4<DT>(px + i * STEP * x_pitch, 0, ok, vec);
                r.d[i] = load4<DT>(pd + i * STEP * d_pitch, 0, ok, vec);
                if (p.z) r.z[i] = load4<DT>(pz + i * STEP * z_pitch, 0, ok, vec);
                r.y[i] = load4<DT>(py + i * STEP * y_pitch, 0, ok, vec);
            }
#pragma unroll
            for (int i = 0; i < BC; ++i) {
                const int t = bt + i * BSTEP;
                r.b[i] = load4<DT>(pb + i * BSTEP * b_pitch, 0, t < TILE && t < left ? bvalid : 0, bvec);
            }
        };
        auto step = [&](Rows& r, int j) {                  // forms tile j + 1, stores tile j - 1, both from the end
            if (j + 1 < tiles) {
                const int buf = (j + 1) & 1, left = len - (tiles - 2 - j) * TILE;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (t >= TILE) continue;
                    auto& kept = sh.kept[(j + 1) & 3];
                    kept[0][i][tid] = r.x[i];
                    kept[1][i][tid] = r.d[i];
                    if (p.z) kept[2][i][tid] = r.z[i];
                    kept[3][i][tid] = r.y[i];
                    f32x2 x[2], d[2], dy[2];
                    unpack4_2<DT>(r.x[i], x);
                    unpack4_2<DT>(r.d[i], d);
                    unpack4_2<DT>(r.y[i], dy);
                    if (p.z) {
                        f32x2 z[2];
                        unpack4_2<DT>(r.z[i], z);
#pragma unroll
                        for (int e = 0; e < 2; ++e) dy[e] = mul2(dy[e], mul2(z[e], sigmoidf2_(z[e])));
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        d[e] = add2(d[e], bias[e]);
                        if (p.softplus) d[e] = scan_softplus2(d[e]);
                        x[e] = mul2(d[e], x[e]);
                    }
                    float4 w0, w1, g;
                    unpack2(d[0], w0.x, w0.z);
                    unpack2(x[0], w0.y, w0.w);
                    unpack2(d[1], w1.x, w1.z);
                    unpack2(x[1], w1.y, w1.w);
                    unpack2(dy[0], g.x, g.y);
                    unpack2(dy[1], g.z, g.w);
                    if (t >= left) w0 = w1 = g = make_float4(0.f, 0.f, 0.f, 0.f);      // nothing behind the last token: states and their gradients stay as they are
                    const int o = (tid >> 2) & 1;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 * o]) = o ? w1 : w0;
                    *reinterpret_cast<float4*>(&sh.d[buf][t][ec + 2 - 2 * o]) = o ? w0 : w1;
                    *reinterpret_cast<float4*>(&sh.dy[buf][t][ec]) = g;
                }
#pragma unroll
                for (int i = 0; i < BC; ++i) {
                    const int t = bt + i * BSTEP;
                    if (t >= TILE) continue;
                    float v[4];
                    unpack4<DT>(r.b[i], v);
                    *reinterpret_cast<float4*>(half ? &sh.C[buf][t][bn] : &sh.B[buf][t][bn]) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
            if (j >= 1) {
                const int buf = (j - 1) & 1, t0 = (tiles - j) * TILE, left = len - t0;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int t = et + i * STEP;
                    if (t >= TILE || t >= left) continue;
                    const float4 fg = *reinterpret_cast<const float4*>(&sh.gB[buf][t][ec]), fe = *reinterpret_cast<const float4*>(&sh.eA[buf][t][ec]);
                    f32x2 x[2], s[2], dy[2], ox[2], od[2], oz[2];
                    const f32x2 gB[2] = {lo2(fg), hi2(fg)}, eA[2] = {lo2(fe), hi2(fe)};
                    auto& kept = sh.kept[(j - 1) & 3];
                    unpack4_2<DT>(kept[0][i][tid], x);
                    unpack4_2<DT>(kept[1][i][tid], s);
                    unpack4_2<DT>(kept[3][i][tid], dy);
                    if (p.z) {
                        f32x2 z[2];
                        const float4 fy = *reinterpret_cast<const float4*>(&sh.y[buf][t][ec]);
                        const f32x2 y[2] = {lo2(fy), hi2(fy)};
                        unpack4_2<DT>(kept[2][i][tid], z);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {      // silu' = sg (1 + z (1 - sg))
                            const f32x2 sg = sigmoidf2_(z[e]);
                            oz[e] = mul2(mul2(dy[e], fma2(skip[e], x[e] & skips, y[e])), mul2(sg, fma2(z[e], fma2(sg, both(-1.f), both(1.f)), both(1.f))));
                            dy[e] = mul2(dy[e], mul2(z[e], sg));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[e] = add2(s[e], bias[e]);
                        const f32x2 d = p.softplus ? scan_softplus2(s[e]) : s[e];
                        ox[e] = fma2(skip[e], dy[e] & skips, mul2(d, gB[e]));
                        od[e] = fma2(x[e], gB[e], mul2(eA[e], both(LN2)));
                        if (p.softplus) od[e] = mul2(od[e], sigmoidf2_(s[e]));
                        acc_skip[e] = fma2(dy[e], x[e], acc_skip[e]);
                        acc_bias[e] = add2(acc_bias[e], od[e]);
                    }
                    const size_t at = (size_t)(sq.start + t0 + t) * D + cs.first + ec;
                    const int ok = min(valid, 4);
                    float v[4];
                    auto store = [&](void* to, const f32x2 (&o)[2]) {
                        unpack2(o[0], v[0], v[1]);
                        unpack2(o[1], v[2], v[3]);
                        store4<DT>(to, at, ok, vec, v);
                    };
                    store(a.dx, ox);
                    store(a.ddt, od);
                    if (p.z) store(a.dz, oz);
                }
                for (int i = tid; i < TILE * NP / 2; i += HELPERS) {      // four sums at a time: of dB the first half of a row, of dC the second
                    const int t = i / (NP / 2), o = i % (NP / 2) * 4;
                    if (t >= left) break;
                    float4 v = *reinterpret_cast<const float4*>(&sh.red[buf][0][t][o]);
#pragma unroll
                    for (int w = 1; w < SCAN_WARPS; ++w) {
                        const float4 u = *reinterpret_cast<const float4*>(&sh.red[buf][w][t][o]);
                        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
                    }
                    float* to = (o < NP ? a.part_B : a.part_C) + ((size_t)blockIdx.x * p.S.TT + sq.start + t0 + t) * NP + o % NP;
                    *reinterpret_cast<float4*>(to) = v;
                }
            }
            if (j + 3 < tiles) request(r, j + 3);
            __syncthreads();
        };
        if (tiles > 0) request(even, 0);
        if (tiles > 1) request(odd, 1);
        for (int j = -1; j <= tiles; j += 2) {
            step(even, j);
            if (j + 1 <= tiles) step(odd, j + 1);
        }
    }
    // the threads that share four channels, in order
    float* all = reinterpret_cast<float*>(raw_shared);     // [2][HELPERS][4]: no tile is left
    static_assert(sizeof(ScanBwdShared<DT, LPC>) >= 2 * HELPERS * 16, "sums of all threads");
    float v[4];
    __syncthreads();
    unpack2(acc_skip[0], v[0], v[1]);
    unpack2(acc_skip[1], v[2], v[3]);
    *reinterpret_cast<float4*>(all + tid * 4) = make_float4(v[0], v[1], v[2], v[3]);
    unpack2(acc_bias[0], v[0], v[1]);
    unpack2(acc_bias[1], v[2], v[3]);
    *reinterpret_cast<float4*>(all + (HELPERS + tid) * 4) = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    for (int c = tid; c < cs.count; c += HELPERS) {
        float s0 = 0.f, s1 = 0.f;
        for (int i = c / 4; i < HELPERS; i += ROW) {
            s0 += all[i * 4 + c % 4];
            s1 += all[(HELPERS + i) * 4 + c % 4];
        }
        if (a.part_skip) a.part_skip[(size_t)blockIdx.y * D + cs.first + c] = s0;
        if (a.part_bias) a.part_bias[(size_t)blockIdx.y * D + cs.first + c] = s1;
    }
}

// One token of each sequence.  Bound by HBM: the states are read and written.  A thread has four states of a channel, as above, of ROWS = 4 or 1 sequences, whose states
// are requested together and share A.  With four the lanes of a channel share the rest: a lane reads x, dt and z of one of the sequences (two lanes: of two) and ends with its sum.
template <int DT, int LPC, int ROWS, bool FILL>
__global__ void __launch_bounds__(128) scan_step_kernel(const MkdaScanStep p, const bool bvec) {
    follow_stream();
    constexpr int MINE = ROWS == 1 ? 1 : LPC == 2 ? 2 : 1;      // sequences whose elementwise part this lane has: q & 3, or q and q + 2
    const int q = threadIdx.x % LPC, c = blockIdx.x * (128 / LPC) + threadIdx.x / LPC, first = blockIdx.y * ROWS, n0 = 4 * q, D = p.D, NST = p.NST;
    const bool there = c < D;
    const int rows = there ? min(ROWS, p.N - first) : 0, g = there && p.G > 1 ? c / (D / p.G) : 0, mine = ROWS == 1 ? 0 : q & 3;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 h[ROWS];
    Raw4<DT> rB[ROWS], rC[ROWS];
    const size_t row = (size_t)first * D + c, at = (size_t)g * NST + n0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        h[r] = r < rows ? ld_states(p.state, row + (size_t)r * D, n0, NST) : zero;
        rB[r] = load4<DT>(p.B, (size_t)(first + r) * p.B_stride + at, r < rows ? NST - n0 : 0, bvec);
        rC[r] = load4<DT>(p.C, (size_t)(first + r) * p.C_stride + at, r < rows ? NST - n0 : 0, bvec);
    }
    float x[MINE], d[MINE], z[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const bool ok = mine + 2 * i < rows;
        const size_t n = (size_t)(first + mine + 2 * i);
        x[i] = ok ? ld1(p.x, DT, n * p.x_stride + c) : 0.f;
        d[i] = ok ? ld1(p.dt, DT, n * p.dt_stride + c) : 0.f;
        z[i] = ok && p.z ? ld1(p.z, DT, n * p.z_stride + c) : 0.f;
    }
    Four A = four(there ? ld_states(p.A, c, n0, NST) : zero);
    const f32x2 real[2] = {real_states(n0, NST), real_states(n0 + 2, NST)};      // states that fill up the lanes stay zero beside infinite values
    const float bias = there && p.dt_bias ? p.dt_bias[c] : 0.f, skip = there && p.skip ? p.skip[c] : 0.f;
    // not held to the fp32 range as rates() does, which took 0.16 of 2.2 us: every token here is one of a sequence
#pragma unroll
    for (int i = 0; i < 2; ++i) A.v[i] = mul2(A.v[i], both(RCP_LN2));
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        d[i] += bias;
        if (p.softplus) d[i] = scan_softplus(d[i]);
    }
    float y[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        f32x2 B[2], C[2], s;
        unpack4_2<DT>(rB[r], B);
        unpack4_2<DT>(rC[r], C);
        float dr = d[0], dx = d[0] * x[0];
        if constexpr (ROWS > 1) {
            const int i = LPC == 2 ? r / 2 : 0;
            dr = __shfl_sync(0xffffffffu, d[i < MINE ? i : 0], LPC == 2 ? r & 1 : r, LPC);
            dx = __shfl_sync(0xffffffffu, d[i < MINE ? i : 0] * x[i < MINE ? i : 0], LPC == 2 ? r & 1 : r, LPC);
        }
        Four o = four(h[r]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o.v[i] = fma2(scan_decay(A.v[i], dr), o.v[i], mul2(both(dx), B[i]));
            if constexpr (FILL) o.v[i] &= real[i];
            s = i ? fma2(C[i], o.v[i], s) : mul2(C[i], o.v[i]);
        }
        if (r < rows) st_states(p.state, row + (size_t)r * D, n0, NST, flat(o));
        y[r] = sum2(s);
    }
    if constexpr (ROWS > 1) {
        lanes_sum4<LPC>(y, q);
    } else {
#pragma unroll
        for (int b = 1; b < LPC; b <<= 1) y[0] += __shfl_xor_sync(0xffffffffu, y[0], b);
    }
    if (q > (ROWS == 1 ? 0 : 3)) return;
#pragma unroll
    for (int i = 0; i < MINE; ++i)
        if (mine + 2 * i < rows) {
            float v = p.skip ? fmaf(skip, x[i], y[i]) : y[i];      // 0 times infinity is no 0
            if (p.z) v *= z[i] * sigmoidf_(z[i]);
            st1(p.y, DT, row + (size_t)(mine + 2 * i) * D, v);
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
static bool good_parts(const MkdaSeqs& s) { return s.seg == 0 || (s.seg > 0 && s.seg % 64 == 0 && s.segs >= 1 && (long long)s.N * s.segs <= 0x7fffffff); }
static int rows_of_blocks(const MkdaSeqs& s) {
    const long long n = s.seg ? (long long)s.N * s.segs : s.N;
    return (int)(n < 65535 ? n : 65535);
}
template <int DT, int LPC, bool REV>
static int launch_scan_pre(const MkdaScanFwd& p, const void* up, float* out_h, float* out_d, int from, int blocks, bool vec, cudaStream_t stream) {
    constexpr int TILE = LPC == 2 ? 32 : 64, smem = (int)sizeof(ScanPreShared<DT, LPC, TILE>);
    auto* kern = scan_pre_kernel<DT, LPC, TILE, REV>;
    if (int e = ensure_smem(reinterpret_cast<const void*>(kern), smem, "scan: parts")) return e;
    launch(kern, dim3(p.G * blocks, rows_of_blocks(p.S)), SCAN_THREADS + SCAN_HELPERS, smem, stream, p, up, out_h, out_d, from, blocks, vec, wide_states(p, 4));
    return check_launch("scan: parts");
}

}  // namespace mkda

using namespace mkda;

extern "C" int mkda_scan_padded_states(int NST) { return NST <= 8 ? 8 : NST <= 16 ? 16 : NST <= 32 ? 32 : 64; }

extern "C" int mkda_scan_fwd(const MkdaScanFwd* p, void* stream) {
    if (!p || !p->A || (p->S.TT && (!p->x || !p->dt || !p->B || !p->C || !p->y))) return set_error(MKDA_ERR_ARG, "scan_fwd: null argument");
    if (int e = bad_scan(p->D, p->NST, p->G, p->dtype)) return e;
    if (!good_sequences(p->S) || (p->ckpt && p->S.cu && !p->S.ckpt_off)) return set_error(MKDA_ERR_ARG, "scan_fwd: bad sequences");
    if (!good_parts(p->S) || (p->S.seg && (!p->seg_h || !p->seg_d || !aligned16(p->seg_h)))) return set_error(MKDA_ERR_ARG, "scan_fwd: parts of a multiple of 64 tokens, with their workspace");
    if (!aligned16(p->A) || !aligned16(p->h0) || !aligned16(p->ht) || !aligned16(p->ckpt)) return set_error(MKDA_ERR_ARG, "scan_fwd: A and states must be 16-byte aligned");
    if (p->S.N == 0) return MKDA_OK;
    int rc = MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        with_lanes(p->NST, [&](auto l) {
            constexpr int DT = decltype(dt)::value, LPC = decltype(l)::value;
            const bool vec = wide_rows(*p, 4) && aligned16(p->y);
            const int blocks = blocks_of_channels(p->D, p->G, ScanShape<LPC>::CB);
            if (p->S.seg) rc = launch_scan_pre<DT, LPC, false>(*p, nullptr, p->seg_h, p->seg_d, 0, blocks / p->G, vec, (cudaStream_t)stream);
            if (rc != MKDA_OK) return;
            auto run = [&](auto tile) {
                constexpr int TILE = decltype(tile)::value, smem = (int)sizeof(ScanFwdShared<LPC, TILE>);
                auto* kern = p->NST == 4 * LPC ? scan_fwd_kernel<DT, LPC, TILE, false> : scan_fwd_kernel<DT, LPC, TILE, true>;
                rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "scan_fwd");
                if (rc == MKDA_OK)
                    launch(kern, dim3(blocks, rows_of_blocks(p->S)), SCAN_THREADS + SCAN_HELPERS, smem, (cudaStream_t)stream, *p, vec, wide_states(*p, 4));
            };
            // 64 tokens a tile from 256 tokens per sequence on; with two lanes per channel the rows of 64 would not fit into the registers
            if (LPC == 2 || (p->S.seg ? p->S.seg < SCAN_LONG : (long long)p->S.TT < SCAN_LONG * (long long)p->S.N)) run(std::integral_constant<int, 32>());
            else run(std::integral_constant<int, LPC == 2 ? 32 : 64>());
        });
    });
    if (rc != MKDA_OK) return rc;
    return check_launch("scan_fwd");
}

extern "C" int mkda_scan_bwd_channel_blocks(int D, int G, int NST) {
    int r = 0;
    if (D > 0 && G > 0 && NST > 0 && NST <= MKDA_SCAN_MAX_STATES)
        with_lanes(NST, [&](auto l) { r = blocks_of_channels(D, G, ScanShape<decltype(l)::value>::CB); });
    return r;
}

extern "C" int mkda_scan_bwd(const MkdaScanBwd* p, void* stream) {
    if (!p || !p->f.A || !p->part_A ||
        (p->f.S.TT && (!p->f.x || !p->f.dt || !p->f.B || !p->f.C || !p->f.ckpt || !p->dy || !p->dx || !p->ddt || (p->f.z && !p->dz) || !p->part_B || !p->part_C)))
        return set_error(MKDA_ERR_ARG, "scan_bwd: null argument");
    if (int e = bad_scan(p->f.D, p->f.NST, p->f.G, p->f.dtype)) return e;
    if (!good_sequences(p->f.S) || (p->f.S.cu && !p->f.S.ckpt_off)) return set_error(MKDA_ERR_ARG, "scan_bwd: bad sequences");
    if (!good_parts(p->f.S) || (p->f.S.seg && (!p->seg_g || !p->seg_d || !aligned16(p->seg_g)))) return set_error(MKDA_ERR_ARG, "scan_bwd: parts of a multiple of 64 tokens, with their workspace");
    if (!aligned16(p->f.A) || !aligned16(p->f.ckpt) || !aligned16(p->dht) || !aligned16(p->dh0) || !aligned16(p->part_A) || !aligned16(p->part_B) || !aligned16(p->part_C))
        return set_error(MKDA_ERR_ARG, "scan_bwd: A, states and partial sums must be 16-byte aligned");
    if (p->slots < 1 || p->slots > 65535 || p->channel_blocks != mkda_scan_bwd_channel_blocks(p->f.D, p->f.G, p->f.NST))
        return set_error(MKDA_ERR_ARG, "scan_bwd: 1 to 65535 slots, and as many blocks of channels as mkda_scan_bwd_channel_blocks says");
    const int per_group = p->channel_blocks / p->f.G;
    if (p->first_block < 0 || p->blocks < 0 || p->blocks > per_group || p->first_block > per_group - (p->blocks ? p->blocks : per_group))
        return set_error(MKDA_ERR_ARG, "scan_bwd: blocks of channels that the groups do not have");
    MkdaScanBwd q = *p;
    if (!q.blocks) q.blocks = per_group;
    int rc = MKDA_OK;
    with_dtype(p->f.dtype, [&](auto dt) {
        with_lanes(p->f.NST, [&](auto l) {
            constexpr int DT = decltype(dt)::value, LPC = decltype(l)::value;
            const MkdaScanFwd& f = p->f;
            const bool vec = wide_rows(f, 4) && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->ddt) && aligned16(p->dz);
            constexpr int smem = (int)sizeof(ScanBwdShared<DT, LPC>);
            if (f.S.seg) rc = launch_scan_pre<DT, LPC, true>(f, p->dy, p->seg_g, p->seg_d, q.first_block, q.blocks, vec, (cudaStream_t)stream);
            if (rc != MKDA_OK) return;
            auto* kern = scan_bwd_kernel<DT, LPC>;
            static const int regs = kernel_registers(reinterpret_cast<const void*>(kern));
            if (regs != SCAN_BWD_LAUNCH_REGS) { rc = set_error(MKDA_ERR_LAUNCH, "scan_bwd: built with other registers than its roles share"); return; }
            rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "scan_bwd");
            if (rc == MKDA_OK) launch(kern, dim3(f.G * q.blocks, p->slots), SCAN_BWD_THREADS, smem, (cudaStream_t)stream, q, vec, wide_states(f, 4));
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
            const bool bvec = p->NST % 4 == 0 && p->B_stride % 4 == 0 && p->C_stride % 4 == 0 && aligned16(p->B) && aligned16(p->C);
            const int blocks = (p->D + 128 / LPC - 1) / (128 / LPC);
            // four sequences a thread where that leaves eight blocks per SM
            const bool fill = p->NST != 4 * LPC;
            if ((long long)blocks * p->N >= 32ll * sm_count())
                launch(fill ? scan_step_kernel<DT, LPC, 4, true> : scan_step_kernel<DT, LPC, 4, false>, dim3(blocks, (p->N + 3) / 4), 128, 0, (cudaStream_t)stream, *p, bvec);
            else
                launch(fill ? scan_step_kernel<DT, LPC, 1, true> : scan_step_kernel<DT, LPC, 1, false>, dim3(blocks, p->N), 128, 0, (cudaStream_t)stream, *p, bvec);
        });
    });
    return check_launch("scan_step");
}
