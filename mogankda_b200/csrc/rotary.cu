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

// VEC: pairs in pieces of eight, 16-byte accesses; else pair by pair.
template <int DT, bool VEC>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const MkdaRotary p, const int per_block) {
    follow_stream();
    extern __shared__ __align__(16) float2 turns[];        // [per_block][freqs]
    const int F = p.freqs, D = p.dim, heads = p.heads_q + p.heads_k;
    const long long first = (long long)blockIdx.x * per_block;
    const int n = (int)min((long long)per_block, p.tokens - first);
    for (int e = threadIdx.x; e < n * F; e += ROTARY_THREADS) turns[e] = turn(p, first + e / F, e % F);
    __syncthreads();
    constexpr int P = VEC ? 8 : 1;
    const int pairs = F / P, rest = (D - 2 * F) / P, units = pairs + rest, per_token = heads * units, all = n * per_token;
    for (int base = threadIdx.x; base < all; base += ROTARY_BATCH * ROTARY_THREADS) {
        Raw8 ra[ROTARY_BATCH], rb[ROTARY_BATCH];
        float fa[ROTARY_BATCH], fb[ROTARY_BATCH];
        int tok[ROTARY_BATCH], unit[ROTARY_BATCH];
        size_t to[ROTARY_BATCH];
        bool of_k[ROTARY_BATCH];
#pragma unroll
        for (int i = 0; i < ROTARY_BATCH; ++i) {
            const int u = base + i * ROTARY_THREADS;
            tok[i] = -1;
            if (u >= all) continue;
            tok[i] = u / per_token;
            const int in = u - tok[i] * per_token, h = in / units;
            unit[i] = in - h * units;
            of_k[i] = h >= p.heads_q;
            const int hh = of_k[i] ? h - p.heads_q : h;
            const void* from = of_k[i] ? p.k : p.q;
            const size_t at = (size_t)(first + tok[i]) * (of_k[i] ? p.k_stride : p.q_stride) + (size_t)hh * D;
            to[i] = ((size_t)(first + tok[i]) * (of_k[i] ? p.heads_k : p.heads_q) + hh) * D;
            const bool turned = unit[i] < pairs;
            const int a = turned ? (p.interleaved ? 2 : 1) * P * unit[i] : 2 * F + P * (unit[i] - pairs), b = a + (p.interleaved ? P : F);
            if constexpr (VEC) {
                ldraw8<DT>(from, at + a, ra[i]);
                if (turned) ldraw8<DT>(from, at + b, rb[i]);
            } else {
                fa[i] = ld1(from, DT, at + a);
                if (turned) fb[i] = ld1(from, DT, at + b);
            }
        }
#pragma unroll
        for (int i = 0; i < ROTARY_BATCH; ++i) {
            if (tok[i] < 0) continue;
            void* out = of_k[i] ? p.k_out : p.q_out;
            const bool turned = unit[i] < pairs;
            const int a = turned ? (p.interleaved ? 2 : 1) * P * unit[i] : 2 * F + P * (unit[i] - pairs), b = a + (p.interleaved ? P : F);
            const float2* cs = turns + (size_t)tok[i] * F + P * unit[i];
            if constexpr (VEC) {
                float x[8], y[8];
                unpack8<DT>(ra[i], x);
                if (turned) {
                    unpack8<DT>(rb[i], y);
                    if (p.interleaved) {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float2 t0 = cs[e / 2], t1 = cs[4 + e / 2];
                            const float u = x[e], v = x[e + 1], r = y[e], s = y[e + 1];
                            x[e] = u * t0.x - v * t0.y; x[e + 1] = u * t0.y + v * t0.x;
                            y[e] = r * t1.x - s * t1.y; y[e + 1] = r * t1.y + s * t1.x;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float2 t = cs[e];
                            const float u = x[e], v = y[e];
                            x[e] = u * t.x - v * t.y; y[e] = u * t.y + v * t.x;
                        }
                    }
                    st8<DT>(out, to[i] + b, y);
                }
                st8<DT>(out, to[i] + a, x);
            } else {
                if (turned) {
                    st1(out, DT, to[i] + a, fa[i] * cs->x - fb[i] * cs->y);
                    st1(out, DT, to[i] + b, fa[i] * cs->y + fb[i] * cs->x);
                } else {
                    st1(out, DT, to[i] + a, fa[i]);
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
        launch(vec ? rotary_kernel<DT, true> : rotary_kernel<DT, false>, dim3((unsigned)blocks), ROTARY_THREADS, (size_t)per * p->freqs * sizeof(float2), (cudaStream_t)stream, *p, per);
    });
    return check_launch("rotary");
}
