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

struct Span { int start, end; };
__device__ __forceinline__ Span sequence(const MkdaSeqs& s, int n) {
    if (!s.cu) return Span{n * s.T, (n + 1) * s.T};
    return Span{s.cu[n], s.cu[n + 1]};
}
// The sequence that holds token t; N if none does (t behind the last one).
__device__ __forceinline__ int sequence_of(const MkdaSeqs& s, int t) {
    if (!s.cu) return t / s.T;
    int lo = 0, hi = s.N;                                  // the first n with cu[n + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
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
