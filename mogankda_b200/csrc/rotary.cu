// Rotary positions of several axes: pair f of a head is turned by the angle positions[axis(f)][token] * inv_freq[f],
//   (a, b) -> (a cos - b sin, a sin + b cos),
// and back by the opposite angle in the backward pass.  The angle of a far position has more whole turns than 32 bits leave room for: it is formed in 64 bits, in turns, and
// reduced to half a turn to either side before its sine and cosine are taken in 32 bits (error of the angle below 2 pi 2^-26).  A block forms the sines and cosines of its tokens
// once, in shared memory, for all heads of q and k.
// Bound by HBM: each channel is read and written once.
#include <algorithm>
#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int ROTARY_THREADS = 256, ROTARY_BATCH = 4;

__device__ __forceinline__ float2 turn(const MkdaRotary& p, long long token, int f) {
    const int axis = (p.axis_of[f >> 2] >> (8 * (f & 3))) & 255;
    const size_t at = (size_t)axis * p.tokens + token;
    const double pos = p.positions_64 ? (double)static_cast<const long long*>(p.positions)[at] : (double)static_cast<const int*>(p.positions)[at];
    double t = pos * (double)p.inv_freq[f] * 0.15915494309189535;      // 1 / (2 pi)
    t -= rint(t);
    float s, c;
    sincospif(2.f * (float)t, &s, &c);
    return make_float2(c, p.inverse ? -s : s);
}

// P neighbouring elements, in one access (two for eight of fp32)
template <int DT, int P>
struct Piece {
    using T = typename std::conditional<DT == MKDA_F32, uint32_t, uint16_t>::type;
    struct alignas(P * sizeof(T) < 16 ? P * sizeof(T) : 16) Raw { T v[P]; };
    static __device__ __forceinline__ void load(const void* base, size_t idx, Raw& r) { r = *reinterpret_cast<const Raw*>(static_cast<const T*>(base) + idx); }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[P]) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
            if constexpr (DT == MKDA_F32) v[e] = __uint_as_float(r.v[e]);
            else if constexpr (DT == MKDA_BF16) v[e] = __uint_as_float((uint32_t)r.v[e] << 16);
            else v[e] = __half2float(__ushort_as_half(r.v[e]));
        }
    }
    static __device__ __forceinline__ void store(void* base, size_t idx, const float (&v)[P]) {
        Raw r;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            if constexpr (DT == MKDA_F32) r.v[e] = __float_as_uint(v[e]);
            else if constexpr (DT == MKDA_BF16) r.v[e] = __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
            else r.v[e] = __half_as_ushort(__float2half_rn(v[e]));
        }
        *reinterpret_cast<Raw*>(static_cast<T*>(base) + idx) = r;
    }
};
template <int DT>
struct Piece<DT, 8> {
    using T = typename Piece<DT, 4>::T;
    using Raw = Raw8;
    static __device__ __forceinline__ void load(const void* base, size_t idx, Raw& r) { ldraw8<DT>(base, idx, r); }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) { unpack8<DT>(r, v); }
    static __device__ __forceinline__ void store(void* base, size_t idx, const float (&v)[8]) { st8<DT>(base, idx, v); }
};

// Pairs in pieces of P, as many as sizes, strides and addresses allow in one access.  A thread has the same piece of every head that it takes, and goes on from head to head without a
// division (one for the token and one for the head of each piece took as long as the bytes: 32749 tokens x 40 heads 195 us).
template <int DT, int P, bool NEIGHBOURS>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const MkdaRotary p, const int per_block) {
    follow_stream();
    extern __shared__ __align__(16) float2 turns[];        // [per_block][freqs]
    using Q = Piece<DT, P>;
    const int F = p.freqs, D = p.dim, heads = p.heads_q + p.heads_k;
    const long long first = (long long)blockIdx.x * per_block;
    const int n = (int)min((long long)per_block, p.tokens - first);
    for (int e = threadIdx.x; e < n * F; e += ROTARY_THREADS) turns[e] = turn(p, first + e / F, e % F);
    __syncthreads();
    const int pairs = F / P, units = pairs + (D - 2 * F) / P;      // pieces of a head: of pairs, then of channels that stay
    const int at_once = max(1, ROTARY_THREADS / units);            // heads that the block takes together
    for (int unit = threadIdx.x % min(units, ROTARY_THREADS); unit < units; unit += ROTARY_THREADS) {
        int tok = 0, h = threadIdx.x / min(units, ROTARY_THREADS);
        if (h >= at_once) break;                                   // threads that are left over
        const bool turned = unit < pairs;
        const int a = turned ? (NEIGHBOURS ? 2 : 1) * P * unit : 2 * F + P * (unit - pairs), b = a + (NEIGHBOURS ? P : F);
        auto settle = [&] {
            while (h >= heads) { h -= heads; ++tok; }
        };
        settle();
        while (tok < n) {
            typename Q::Raw ra[ROTARY_BATCH], rb[ROTARY_BATCH];
            int toks[ROTARY_BATCH];
            void* to[ROTARY_BATCH];
#pragma unroll
            for (int i = 0; i < ROTARY_BATCH; ++i) {
                toks[i] = tok;
                if (tok >= n) continue;
                const bool of_k = h >= p.heads_q;
                const int hh = of_k ? h - p.heads_q : h;
                const void* from = of_k ? p.k : p.q;
                const size_t at = (size_t)(first + tok) * (of_k ? p.k_stride : p.q_stride) + (size_t)hh * D;
                to[i] = static_cast<typename Q::T*>(of_k ? p.k_out : p.q_out) + ((size_t)(first + tok) * (of_k ? p.heads_k : p.heads_q) + hh) * D;
                Q::load(from, at + a, ra[i]);
                if (turned) Q::load(from, at + b, rb[i]);
                h += at_once;
                settle();
            }
#pragma unroll
            for (int i = 0; i < ROTARY_BATCH; ++i) {
                if (toks[i] >= n) continue;
                float x[P], y[P];
                Q::unpack(ra[i], x);
                if (turned) {
                    Q::unpack(rb[i], y);
                    const float2* cs = turns + (size_t)toks[i] * F + P * unit;
                    float2 t[P];
                    if constexpr (P == 1) {
                        t[0] = *cs;
                    } else {
#pragma unroll
                        for (int e = 0; e < P; e += 2) {
                            const float4 two = *reinterpret_cast<const float4*>(cs + e);
                            t[e] = make_float2(two.x, two.y);
                            t[e + 1] = make_float2(two.z, two.w);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < P; ++e) {          // of neighbours, pair e is elements 2 e and 2 e + 1 of x and y one behind the other
                        float& u = !NEIGHBOURS ? x[e] : 2 * e < P ? x[2 * e < P ? 2 * e : 0] : y[2 * e >= P ? 2 * e - P : 0];
                        float& v = !NEIGHBOURS ? y[e] : 2 * e + 1 < P ? x[2 * e + 1 < P ? 2 * e + 1 : 0] : y[2 * e + 1 >= P ? 2 * e + 1 - P : 0];
                        const float w = u;
                        u = w * t[e].x - v * t[e].y;
                        v = w * t[e].y + v * t[e].x;
                    }
                    Q::store(to[i], b, y);
                }
                Q::store(to[i], a, x);
            }
        }
    }
}

}  // namespace mkda

using namespace mkda;

extern "C" int mkda_rotary(const MkdaRotary* p, void* stream) {
    if (!p) return set_error(MKDA_ERR_ARG, "rotary: null argument");
    if (p->tokens < 0 || p->heads_q < 0 || p->heads_k < 0 || p->heads_q > 65536 || p->heads_k > 65536) return set_error(MKDA_ERR_ARG, "rotary: at most 65536 heads");
    if (p->dim < 1 || p->dim > MKDA_ROTARY_MAX_DIM || p->freqs < 0 || 2 * p->freqs > p->dim) return set_error(MKDA_ERR_ARG, "rotary: heads of 1 to 512 channels, half as many frequencies at most");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "rotary: unsupported dtype");
    if (p->axes < 1 || p->axes > 255) return set_error(MKDA_ERR_ARG, "rotary: 1 to 255 axes");
    for (int f = 0; f < p->freqs; ++f)
        if (((p->axis_of[f >> 2] >> (8 * (f & 3))) & 255) >= p->axes) return set_error(MKDA_ERR_ARG, "rotary: a frequency of an axis that there is not");
    if (p->tokens == 0 || p->heads_q + p->heads_k == 0) return MKDA_OK;
    if ((p->heads_q && (!p->q || !p->q_out)) || (p->heads_k && (!p->k || !p->k_out)) || (p->freqs && (!p->positions || !p->inv_freq))) return set_error(MKDA_ERR_ARG, "rotary: null argument");
    const int size = p->dtype == MKDA_F32 ? 4 : 2;
    int piece = 8;
    auto fits = [&](const void* at) { return reinterpret_cast<uintptr_t>(at) % std::min(16, piece * size) == 0; };
    while (piece > 1 && (p->dim % piece || p->freqs % piece || (p->heads_q && p->q_stride % piece) || (p->heads_k && p->k_stride % piece) || !fits(p->q) || !fits(p->k) || !fits(p->q_out) || !fits(p->k_out))) piece /= 2;
    const int units = (p->heads_q + p->heads_k) * (p->dim - p->freqs) / piece;      // a token's
    // tokens of a block: work for a few batches of its threads, at most 32 KB of sines and cosines, and as many blocks as fill whole waves of the places on the GPU
    int per = std::max(1, 4 * ROTARY_BATCH * ROTARY_THREADS / std::max(units, 1));
    per = std::min(per, std::max(1, 4096 / std::max(p->freqs, 1)));
    with_dtype(p->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto* kern = piece == 8 ? p->interleaved ? rotary_kernel<DT, 8, true> : rotary_kernel<DT, 8, false> : piece == 4 ? p->interleaved ? rotary_kernel<DT, 4, true> : rotary_kernel<DT, 4, false>
                   : piece == 2 ? p->interleaved ? rotary_kernel<DT, 2, true> : rotary_kernel<DT, 2, false> : p->interleaved ? rotary_kernel<DT, 1, true> : rotary_kernel<DT, 1, false>;
        const long long places = (long long)sm_count() * std::min(resident(reinterpret_cast<const void*>(kern), ROTARY_THREADS), 200 * 1024 / std::max(1, per * p->freqs * 8)), waves = (p->tokens + per * places - 1) / (per * places);
        per = (int)((p->tokens + waves * places - 1) / (waves * places));
        launch(kern, dim3((unsigned)(((long long)p->tokens + per - 1) / per)), ROTARY_THREADS, (size_t)per * p->freqs * sizeof(float2), (cudaStream_t)stream, *p, per);
    });
    return check_launch("rotary");
}
