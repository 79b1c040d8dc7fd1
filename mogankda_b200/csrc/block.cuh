// Shared device code of the operators around the layer (conv.cu, scan.cu, norm.cu): pieces of eight channels that may be ragged or unaligned, and
// the boundaries of sequences.
#pragma once
#include "../../include/mkda_block.h"
#include "common.cuh"
#include "host.h"

namespace mkda {

// Eight consecutive elements from `idx` on, of which the first `valid` exist (the others are zero); `vec`: idx, the address and the row
// allow 16-byte accesses, and valid is 8 or at most 0.
template <int DT>
__device__ __forceinline__ Raw8 load8(const void* base, size_t idx, int valid, bool vec) {
    Raw8 r;
    r.a = make_uint4(0, 0, 0, 0);
    r.b = make_uint4(0, 0, 0, 0);
    if (valid <= 0) return r;
    if (vec) {
        ldraw8<DT>(base, idx, r);
    } else if (DT == MKDA_F32) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = e < valid ? __float_as_uint(static_cast<const float*>(base)[idx + e]) : 0u;
        r.a = make_uint4(w[0], w[1], w[2], w[3]);
        r.b = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = e < valid ? static_cast<const uint16_t*>(base)[idx + e] : 0u;
        r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void store8(void* base, size_t idx, int valid, bool vec, const float (&v)[8]) {
    if (valid <= 0) return;
    if (vec) {
        st8<DT>(base, idx, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) st1(base, DT, idx + e, v[e]);
    }
}

// The same for four elements, 8-byte (fp32: 16-byte) accesses
template <int DT>
struct alignas(DT == MKDA_F32 ? 16 : 8) Raw4 { uint32_t w[DT == MKDA_F32 ? 4 : 2]; };
template <int DT>
__device__ __forceinline__ Raw4<DT> load4(const void* base, size_t idx, int valid, bool vec) {
    Raw4<DT> r;
#pragma unroll
    for (uint32_t& w : r.w) w = 0u;
    if (valid <= 0) return r;
    if (vec) {
        if constexpr (DT == MKDA_F32) {
            const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const float*>(base) + idx);
            r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + idx);
            r.w[0] = v.x; r.w[1] = v.y;
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = e >= valid ? 0u : DT == MKDA_F32 ? static_cast<const uint32_t*>(base)[idx + e] : static_cast<const uint16_t*>(base)[idx + e];
        if constexpr (DT == MKDA_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[e] = w[e];
        } else {
            r.w[0] = w[0] | w[1] << 16;
            r.w[1] = w[2] | w[3] << 16;
        }
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void unpack4(const Raw4<DT>& r, float (&v)[4]) {
    if constexpr (DT == MKDA_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(r.w[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if constexpr (DT == MKDA_BF16) {
                v[2 * e] = __uint_as_float(r.w[e] << 16);
                v[2 * e + 1] = __uint_as_float(r.w[e] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[e]));
                v[2 * e] = f.x; v[2 * e + 1] = f.y;
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ void unpack4_2(const Raw4<DT>& r, f32x2 (&v)[2]) {
    float f[4];
    unpack4<DT>(r, f);
    v[0] = pack2(f[0], f[1]);
    v[1] = pack2(f[2], f[3]);
}
template <int DT>
__device__ __forceinline__ void store4(void* base, size_t idx, int valid, bool vec, const float (&v)[4]) {
    if (valid <= 0) return;
    if (vec) {
        st4(base, DT, idx, make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < valid) st1(base, DT, idx + e, v[e]);
    }
}

struct Span { int start, end; };
__device__ __forceinline__ Span sequence(const MkdaSeqs& s, int n) {
    if (!s.cu) return Span{n * s.T, (n + 1) * s.T};
    return Span{s.cu[n], s.cu[n + 1]};
}
// The sequence that holds token t; N if none does (t behind the last one).  Called by whole warps: 32 boundaries are looked at together, one round trip to memory for up to 32
// sequences where halving takes five.
__device__ __forceinline__ int sequence_of(const MkdaSeqs& s, int t) {
    if (!s.cu) return t / s.T;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = s.N;                                  // the first n in [lo, hi] with cu[n + 1] > t, hi standing for itself
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;      // the last of the lane's candidates
        const unsigned above = __ballot_sync(0xffffffffu, at < hi && s.cu[at + 1] > t);
        const int first = above ? __ffs(above) - 1 : 32;   // every candidate of the lanes in front is too small
        const int full = (hi - lo) / step;                 // lanes whose last candidate was looked at
        if (first < 32) {
            hi = lo + (first + 1) * step - 1;
            lo = lo + first * step;
            if (step == 1) return hi;
        } else {
            lo += full * step;
            if (step == 1) return hi;
        }
    }
    return lo;
}

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Calls f with the dtype as a compile-time constant; false for another one.
template <typename F>
inline bool with_dtype(int dtype, F f) {
    switch (dtype) {
        case MKDA_F32: f(std::integral_constant<int, MKDA_F32>()); return true;
        case MKDA_BF16: f(std::integral_constant<int, MKDA_BF16>()); return true;
        case MKDA_F16: f(std::integral_constant<int, MKDA_F16>()); return true;
        default: return false;
    }
}
inline bool good_sequences(const MkdaSeqs& s) { return s.N >= 0 && s.T >= 0 && s.TT >= 0 && (s.cu || (long long)s.N * s.T == s.TT); }

}  // namespace mkda
