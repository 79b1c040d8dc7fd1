// Shared device code of the operators around the layer (conv.cu, scan.cu, norm.cu): pieces of eight channels that may be ragged or unaligned, and
// the boundaries of sequences.
#pragma once
#include "../../include/mkda_block.h"
#include "common.cuh"
#include "host.h"

namespace mkda {

// BYTES = 8 or 16 bytes from any address that is a multiple of two on, of which the first `bytes` are wanted (the others read as zero).  Rows of odd widths start anywhere: the one or two aligned
// words of that size that hold a wanted byte are read whole, as neighbouring lanes read theirs, and shifted into place (an aligned word never leaves the allocation that one
// of its bytes lies in).  Element by element a convolution of 8192 x 4097 in bf16 took six times as long as one of 4096 channels.
template <int BYTES>
struct alignas(BYTES) Words { uint32_t w[BYTES / 4]; };
template <int BYTES>
__device__ __forceinline__ Words<BYTES> load_shifted(const void* from, int bytes) {
    constexpr int N = BYTES / 4;
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    const int off = (int)(at & (BYTES - 1));
    const Words<BYTES>* p = reinterpret_cast<const Words<BYTES>*>(at - off);
    uint32_t q[2 * N + 1];
#pragma unroll
    for (uint32_t& v : q) v = 0u;
    if constexpr (BYTES == 16) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        q[0] = a.x; q[1] = a.y; q[2] = a.z; q[3] = a.w;
        if (off + bytes > BYTES) {
            const uint4 b = *reinterpret_cast<const uint4*>(p + 1);
            q[4] = b.x; q[5] = b.y; q[6] = b.z; q[7] = b.w;
        }
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        q[0] = a.x; q[1] = a.y;
        if (off + bytes > BYTES) {
            const uint2 b = *reinterpret_cast<const uint2*>(p + 1);
            q[2] = b.x; q[3] = b.y;
        }
    }
    // by whole words, then by half of one
    if (BYTES == 16 && (off & 8)) {
#pragma unroll
        for (int i = 0; i < 2 * N - 2; ++i) q[i] = q[i + 2];
    }
    if (off & 4) {
#pragma unroll
        for (int i = 0; i < N + 1; ++i) q[i] = q[i + 1];
    }
    Words<BYTES> r;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        r.w[i] = off & 2 ? __funnelshift_r(q[i], q[i + 1], 16) : q[i];
        const int left = bytes - 4 * i;
        if (left < 4) r.w[i] = left < 2 ? 0u : r.w[i] & 0xffffu;
    }
    return r;
}
// The reverse: the first `bytes` bytes of `v`, in the widest stores that the address allows.
template <int BYTES>
__device__ __forceinline__ void store_shifted(void* to, int bytes, const Words<BYTES>& v) {
    constexpr int N = BYTES / 4;
    char* const p = static_cast<char*>(to);
    const uintptr_t at = reinterpret_cast<uintptr_t>(to);
    if (at & 2) {                                          // half a word, whole ones across the borders of v's, half a word
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)v.w[0];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t next = i + 1 < N ? v.w[i + 1 < N ? i + 1 : 0] : 0u;
            if (bytes >= 4 * i + 6) *reinterpret_cast<uint32_t*>(p + 4 * i + 2) = __funnelshift_r(v.w[i], next, 16);
            else if (bytes >= 4 * i + 4) *reinterpret_cast<uint16_t*>(p + 4 * i + 2) = (uint16_t)(v.w[i] >> 16);
        }
    } else if ((at & 7) == 0 && bytes == BYTES) {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(p + 4 * i) = make_uint2(v.w[i], v.w[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (bytes >= 4 * i + 4) *reinterpret_cast<uint32_t*>(p + 4 * i) = v.w[i];
            else if (bytes >= 4 * i + 2) *reinterpret_cast<uint16_t*>(p + 4 * i) = (uint16_t)v.w[i];
        }
    }
}

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
    } else {
        constexpr int SIZE = DT == MKDA_F32 ? 4 : 2;
        const char* p = static_cast<const char*>(base) + idx * SIZE;
        const int bytes = min(valid, 8) * SIZE;
        const Words<16> a = load_shifted<16>(p, min(bytes, 16));
        r.a = make_uint4(a.w[0], a.w[1], a.w[2], a.w[3]);
        if (DT == MKDA_F32 && bytes > 16) {
            const Words<16> b = load_shifted<16>(p + 16, bytes - 16);
            r.b = make_uint4(b.w[0], b.w[1], b.w[2], b.w[3]);
        }
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void store8(void* base, size_t idx, int valid, bool vec, const float (&v)[8]) {
    if (valid <= 0) return;
    if (vec) {
        st8<DT>(base, idx, v);
    } else if constexpr (DT == MKDA_F32) {
        char* p = static_cast<char*>(base) + idx * 4;
        const int bytes = min(valid, 8) * 4;
        store_shifted<16>(p, min(bytes, 16), Words<16>{{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}});
        if (bytes > 16) store_shifted<16>(p + 16, bytes - 16, Words<16>{{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])}});
    } else {
        store_shifted<16>(static_cast<char*>(base) + idx * 2, min(valid, 8) * 2, Words<16>{{pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3]), pack16<DT>(v[4], v[5]), pack16<DT>(v[6], v[7])}});
    }
}

// The same for four elements, 8-byte (fp32: 16-byte) accesses; else element by element (shifting took registers from the scan kernels' other path: backward 400 -> 450 us)
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
// tokens are counted in 32 bits, a run or a tile past the last one included
inline bool good_sequences(const MkdaSeqs& s) { return s.N >= 0 && s.T >= 0 && s.TT >= 0 && s.TT <= MKDA_SEQS_MAX_TOKENS && (s.cu || (long long)s.N * s.T == s.TT); }

}  // namespace mkda
