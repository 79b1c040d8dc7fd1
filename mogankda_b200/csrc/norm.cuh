// What the norms of whole rows share (norm.cu, layer_norm.cu): reductions over the threads of a row, and how many threads and pieces of eight channels a row takes.
#pragma once
#include <type_traits>

#include "block.cuh"

namespace mkda {

// |v| kept, NaN passed on (fmaxf drops it, and a row of NaN would get the scale of a row of zeros)
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Sums (or maxima) of N = 1 or 2 values over the TPR threads of a row (neighbouring lanes where they are fewer than 32), the same in all of them; `part` is shared memory that two calls
// later may be used again
template <int TPR, int N, bool MAX>
__device__ __forceinline__ void row_reduce(float (&v)[N], float (*part)[N]) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float w = __shfl_xor_sync(0xffffffffu, v[k], o);
            v[k] = MAX ? max_nan(v[k], w) : v[k] + w;
        }
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) part[threadIdx.x >> 5][k] = v[k];
        __syncthreads();
        const float4* all = reinterpret_cast<const float4*>(part);      // four values at a time: of four warps, or of two
        auto join = [](float a, float b) { return MAX ? max_nan(a, b) : a + b; };
        float4 t = all[0];
#pragma unroll
        for (int i = 1; i < TPR / 32 * N / 4; ++i) {
            const float4 u = all[i];
            t.x = join(t.x, u.x); t.y = join(t.y, u.y); t.z = join(t.z, u.z); t.w = join(t.w, u.w);
        }
        if constexpr (N == 1) {
            v[0] = join(join(t.x, t.y), join(t.z, t.w));
        } else {
            v[0] = join(t.x, t.z);
            v[1] = join(t.y, t.w);
        }
    }
}
__device__ __forceinline__ void load_any8(const void* base, int dtype, size_t idx, int valid, bool vec, float (&v)[8]) {
    if (valid <= 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    } else if (vec) {
        ld8(base, dtype, idx, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < valid ? ld1(base, dtype, idx + e) : 0.f;
    }
}
template <int DT>
__device__ __forceinline__ float as_held(float v) {
    return DT == MKDA_F32 ? v : DT == MKDA_BF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}

// Threads of a row and pieces of eight channels per thread
template <typename F>
static bool with_width_bwd(int H, F f) {
    using std::integral_constant;
    if (H <= 256) f(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (H <= 1024) f(integral_constant<int, 128>(), integral_constant<int, 1>());
    else if (H <= 2048) f(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (H <= 4096) f(integral_constant<int, 512>(), integral_constant<int, 1>());
    else if (H <= 8192) f(integral_constant<int, 1024>(), integral_constant<int, 1>());
    else if (H <= 16384) f(integral_constant<int, 1024>(), integral_constant<int, 2>());
    else if (H <= MKDA_NORM_MAX_WIDTH) f(integral_constant<int, 1024>(), integral_constant<int, 4>());
    else return false;
    return true;
}
template <typename F>
static bool with_width(int H, F f) {
    using std::integral_constant;
    if (H <= 256) f(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (H <= 512) f(integral_constant<int, 32>(), integral_constant<int, 2>());
    else if (H <= 1024) f(integral_constant<int, 128>(), integral_constant<int, 1>());
    else if (H <= 2048) f(integral_constant<int, 128>(), integral_constant<int, 2>());
    else if (H <= 4096) f(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (H <= 8192) f(integral_constant<int, 512>(), integral_constant<int, 2>());
    else if (H <= 16384) f(integral_constant<int, 1024>(), integral_constant<int, 2>());
    else if (H <= MKDA_NORM_MAX_WIDTH) f(integral_constant<int, 1024>(), integral_constant<int, 4>());
    else return false;
    return true;
}
// Blocks that walk the rows: as many as are resident
template <int TPR, int THREADS>
static int norm_blocks(int rows) {
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    const long long most = (long long)sm_count() * (THREADS / (TPR < 128 ? 128 : TPR) > 0 ? THREADS / (TPR < 128 ? 128 : TPR) : 1), want = ((long long)rows + RPB - 1) / RPB;
    return (int)(want < most ? want : most);
}
static bool good_dtype(int d) { return d >= MKDA_F32 && d <= MKDA_F16; }

}  // namespace mkda
