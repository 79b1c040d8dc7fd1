// Rotary positions of several axes: pair f of a head is turned by the angle positions[axis(f)][token] * inv_freq[f],
//   (a, b) -> (a cos - b sin, a sin + b cos),
// and back by the opposite angle in the backward pass.  The angle of a far position has more whole turns than 32 bits leave room for: it is formed in 64 bits, in turns, and
// reduced to half a turn to either side before its sine and cosine are taken in 32 bits (error of the angle below 2 pi 2^-26).  A block forms the sines and cosines of its tokens
// once, in shared memory, for all heads of q and k.
// Bound by HBM: each channel is read and written once.
#include <algorithm>

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

// VEC: pairs in pieces of eight, 16-byte accesses; else pair by pair.  A thread has the same piece of every head that it takes, and goes on from head to head without a division
// (one for the token and one for the head of each piece took as long as the bytes: 32749 tokens x 40 heads 195 us).
template <int DT, bool VEC, bool NEIGHBOURS>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const MkdaRotary p, const int per_block) {
    follow_stream();
    extern __shared__ __align__(16) float2 turns[];        // [per_block][freqs]
    const int F = p.freqs, D = p.dim, heads = p.heads_q + p.heads_k;
    const long long first = (long long)blockIdx.x * per_block;
    const int n = (int)min((long long)per_block, p.tokens - first);
    for (int e = threadIdx.x; e < n * F; e += ROTARY_THREADS) turns[e] = turn(p, first + e / F, e % F);
    __syncthreads();
    constexpr int P = VEC ? 8 : 1;
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
            Raw8 ra[ROTARY_BATCH], rb[ROTARY_BATCH];
            float fa[ROTARY_BATCH], fb[ROTARY_BATCH];
            int toks[ROTARY_BATCH];
            char* to[ROTARY_BATCH];
            constexpr int SIZE = DT == MKDA_F32 ? 4 : 2;
#pragma unroll
            for (int i = 0; i < ROTARY_BATCH; ++i) {
                toks[i] = tok;
                if (tok >= n) continue;
                const bool of_k = h >= p.heads_q;
                const int hh = of_k ? h - p.heads_q : h;
                const void* from = of_k ? p.k : p.q;
                const size_t at = (size_t)(first + tok) * (of_k ? p.k_stride : p.q_stride) + (size_t)hh * D;
                to[i] = static_cast<char*>(of_k ? p.k_out : p.q_out) + ((size_t)(first + tok) * (of_k ? p.heads_k : p.heads_q) + hh) * D * SIZE;
                if constexpr (VEC) {
                    ldraw8<DT>(from, at + a, ra[i]);
                    if (turned) ldraw8<DT>(from, at + b, rb[i]);
                } else {
                    fa[i] = ld1(from, DT, at + a);
                    if (turned) fb[i] = ld1(from, DT, at + b);
                }
                h += at_once;
                settle();
            }
#pragma unroll
            for (int i = 0; i < ROTARY_BATCH; ++i) {
                if (toks[i] >= n) continue;
                const float2* cs = turns + (size_t)toks[i] * F + P * unit;
                if constexpr (VEC) {
                    float x[8], y[8];
                    unpack8<DT>(ra[i], x);
                    if (turned) {
                        unpack8<DT>(rb[i], y);
                        float4 t[4];                           // two pairs' cosine and sine each
#pragma unroll
                        for (int e = 0; e < 4; ++e) t[e] = *reinterpret_cast<const float4*>(cs + 2 * e);
                        auto one = [](float& u, float& v, float c, float s) {
                            const float w = u;
                            u = w * c - v * s;
                            v = w * s + v * c;
                        };
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (NEIGHBOURS) {
                                float (&z)[8] = e < 2 ? x : y;
                                one(z[4 * (e & 1)], z[4 * (e & 1) + 1], t[e].x, t[e].y);
                                one(z[4 * (e & 1) + 2], z[4 * (e & 1) + 3], t[e].z, t[e].w);
                            } else {
                                one(x[2 * e], y[2 * e], t[e].x, t[e].y);
                                one(x[2 * e + 1], y[2 * e + 1], t[e].z, t[e].w);
                            }
                        }
                        st8<DT>(to[i], b, y);
                    }
                    st8<DT>(to[i], a, x);
                } else {
                    if (turned) {
                        st1(to[i], DT, a, fa[i] * cs->x - fb[i] * cs->y);
                        st1(to[i], DT, b, fa[i] * cs->y + fb[i] * cs->x);
                    } else {
                        st1(to[i], DT, a, fa[i]);
                    }
                }
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
    const bool vec = p->dim % 8 == 0 && p->freqs % 8 == 0 && (!p->heads_q || p->q_stride % 8 == 0) && (!p->heads_k || p->k_stride % 8 == 0) && aligned16(p->q) && aligned16(p->k) &&
                     aligned16(p->q_out) && aligned16(p->k_out);
    const int units = (p->heads_q + p->heads_k) * (p->dim - p->freqs) / (vec ? 8 : 1);      // a token's
    // tokens of a block: work for a few batches of its threads, at most 32 KB of sines and cosines, and a block for each place on the GPU as long as there are tokens
    int per = std::max(1, 4 * ROTARY_BATCH * ROTARY_THREADS / std::max(units, 1));
    per = std::min(per, std::max(1, 4096 / std::max(p->freqs, 1)));
    per = (int)std::min<long long>(per, std::max<long long>(1, p->tokens / (4 * sm_count())));
    const long long blocks = ((long long)p->tokens + per - 1) / per;
    with_dtype(p->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto* kern = vec ? p->interleaved ? rotary_kernel<DT, true, true> : rotary_kernel<DT, true, false> : p->interleaved ? rotary_kernel<DT, false, true> : rotary_kernel<DT, false, false>;
        launch(kern, dim3((unsigned)blocks), ROTARY_THREADS, (size_t)per * p->freqs * sizeof(float2), (cudaStream_t)stream, *p, per);
    });
    return check_launch("rotary");
}
