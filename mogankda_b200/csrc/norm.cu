// RMS norm of whole rows with the residual's addition in front of it, its backward pass, and the second stage of the sums that the backward passes of
// conv.cu, scan.cu and this file leave.
//   s = x + residual (as the residual's type holds it)     r = 1 / sqrt(mean s^2 + eps)     y = s r weight     8 bits: y / scale, scale = max |y| / 448
//   dn = dy weight     ds = r (dn - s r^2 mean(dn s)) + dsum     dweight = sum_rows dy s r
// Bound by HBM: a row stays in the registers of the threads that share it (a warp up to 1024 channels, then blocks of 128, 512 or 1024 threads),
// in pieces of eight channels, so that everything is read once.
#include <cuda_fp8.h>

#include <type_traits>

#include "block.cuh"

namespace mkda {

// |v| kept, NaN passed on (fmaxf drops it, and a row of NaN would get the scale of a row of zeros)
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Sum (or maximum) over the TPR threads of a row, the same in all of them; `part` is shared memory of this use alone
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < TPR / 32; ++i) v = MAX ? max_nan(v, part[i]) : v + part[i];
    }
    return v;
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
__device__ __forceinline__ void store_any8(void* base, int dtype, size_t idx, int valid, bool vec, const float (&v)[8]) {
    if (dtype == MKDA_F32) store8<MKDA_F32>(base, idx, valid, vec, v);
    else if (dtype == MKDA_BF16) store8<MKDA_BF16>(base, idx, valid, vec, v);
    else store8<MKDA_F16>(base, idx, valid, vec, v);
}
__device__ __forceinline__ float as_held(float v, int dtype) {
    return dtype == MKDA_F32 ? v : dtype == MKDA_BF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}

template <int DT, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_fwd_kernel(const MkdaNormFwd p, const bool vec, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    __shared__ float part[2][TPR / 32];
    const int tid = threadIdx.x % TPR, row = blockIdx.x * RPB + threadIdx.x / TPR, H = p.width;
    if (row >= p.rows) return;                             // whole warps, and blocks of one row never
    float s[NV][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) load_any8(p.x, DT, (size_t)row * p.x_stride + (tid + i * TPR) * 8, H - (tid + i * TPR) * 8, vec, s[i]);
    if (p.residual) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float r[8];
            load_any8(p.residual, p.res_dtype, (size_t)row * p.res_stride + c, H - c, vec, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i][e] = as_held(s[i][e] + r[e], p.res_dtype);
            store_any8(p.sum, p.res_dtype, (size_t)row * H + c, min(H - c, 8), vec, s[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(s[i][e], s[i][e], sum);
    const float r = rsqrtf(row_reduce<TPR, false>(sum, part[0]) / (float)H + p.eps);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * TPR) * 8;
        float w[8];
        if (p.weight) load_any8(p.weight, p.weight_dtype, c, H - c, wvec, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[i][e] *= r;
            if (p.weight) s[i][e] *= w[e];
        }
        if (!p.out_e4m3) store_any8(p.y, DT, (size_t)row * H + c, min(H - c, 8), vec, s[i]);
    }
    if (!p.out_e4m3) return;
    if (!p.group) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(s[i][e]));
        top = row_reduce<TPR, true>(top, part[1]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * TPR) * 8;
        float t = top;
        if (p.group) {                                     // 128 channels are sixteen threads
            t = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) t = max_nan(t, fabsf(s[i][e]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, o));
        }
        const float scale = max_nan(t, 0x1p-126f * 448.f) / 448.f, inv = 1.f / scale;
        if (c >= H) continue;
        if (p.group ? c % 128 == 0 : c == 0) p.scale[p.group ? (size_t)row * (H / 128) + c / 128 : row] = scale;
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = __nv_cvt_float_to_fp8(s[i][e] * inv, __NV_SATFINITE, __NV_E4M3);
        uint8_t* out = static_cast<uint8_t*>(p.y) + (size_t)row * H + c;
        if (vec) {
            *reinterpret_cast<uint2*>(out) = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < H) out[e] = (uint8_t)b[e];
        }
    }
}

template <int DT, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_bwd_kernel(const MkdaNormBwd p, const bool vec, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    __shared__ float part[2][2][TPR / 32];
    const int tid = threadIdx.x % TPR, first = blockIdx.x * RPB + threadIdx.x / TPR, H = p.width;
    float dw[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
    int turn = 0;
    for (int row = first; row < p.rows; row += gridDim.x * RPB, turn ^= 1) {
        float s[NV][8], g[NV][8], ss = 0.f, sg = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            load_any8(p.s, p.s_dtype, (size_t)row * p.s_stride + c, H - c, vec, s[i]);
            load_any8(p.dy, DT, (size_t)row * H + c, H - c, vec, g[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float w[8];
            if (p.weight) load_any8(p.weight, p.weight_dtype, c, H - c, wvec, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = fmaf(s[i][e], s[i][e], ss);
                sg = fmaf(p.weight ? g[i][e] * w[e] : g[i][e], s[i][e], sg);
            }
        }
        ss = row_reduce<TPR, false>(ss, part[turn][0]);
        sg = row_reduce<TPR, false>(sg, part[turn][1]);
        const float r = rsqrtf(ss / (float)H + p.eps), k = r * r * (sg / (float)H);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float w[8], o[8];
            if (p.weight) load_any8(p.weight, p.weight_dtype, c, H - c, wvec, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[i][e] = fmaf(g[i][e], s[i][e] * r, dw[i][e]);
                o[e] = r * fmaf(-s[i][e], k, p.weight ? g[i][e] * w[e] : g[i][e]);
            }
            if (p.dsum) {
                float u[8];
                load_any8(p.dsum, p.res_dtype, (size_t)row * H + c, H - c, vec, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += u[e];
            }
            store_any8(p.dx, DT, (size_t)row * H + c, min(H - c, 8), vec, o);
            if (p.dres) store_any8(p.dres, p.res_dtype, (size_t)row * H + c, min(H - c, 8), vec, o);
        }
    }
    if (p.part) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            store8<MKDA_F32>(p.part, (size_t)first * H + c, min(H - c, 8), (H & 3) == 0, dw[i]);
        }
    }
}

// A block adds the rows of 128 columns: 32 threads of four columns each, eight rows at a time, then the eight in order.
__global__ void __launch_bounds__(256) sum_rows_kernel(const MkdaSumRows p) {
    follow_stream();
    __shared__ float4 part[8][32];
    long long blk = blockIdx.x;
    int j = 0;
    for (; j < 5; ++j) {
        const long long n = p.job[j].out ? (p.job[j].cols + 127) / 128 * p.job[j].groups : 0;
        if (blk < n) break;
        blk -= n;
    }
    if (j == 5) return;
    const MkdaSumJob q = p.job[j];
    const long long per = (q.cols + 127) / 128, g = blk / per, c = (blk - g * per) * 128 + 4 * (threadIdx.x & 31);
    const int l = threadIdx.x >> 5;
    const float* in = q.in + (size_t)g * q.rows * q.pitch + c;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (((q.cols | q.pitch) & 3) == 0 && (reinterpret_cast<uintptr_t>(q.in) & 15) == 0) {
        if (c < q.cols) {
#pragma unroll 4
            for (int r = l; r < q.rows; r += 8) {
                const float4 v = *reinterpret_cast<const float4*>(in + (size_t)r * q.pitch);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        }
    } else {
        for (int r = l; r < q.rows; r += 8) {
            const float* v = in + (size_t)r * q.pitch;
            if (c < q.cols) s.x += v[0];
            if (c + 1 < q.cols) s.y += v[1];
            if (c + 2 < q.cols) s.z += v[2];
            if (c + 3 < q.cols) s.w += v[3];
        }
    }
    part[l][threadIdx.x & 31] = s;
    __syncthreads();
    if (l) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        const float4 v = part[i][threadIdx.x];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const long long at = c + e, outer = at / q.inner, inner = at - outer * q.inner;
        if (at < q.cols && inner < q.valid) st1(q.out, q.out_dtype, (size_t)(g * q.out_group + outer * q.out_outer + inner * q.out_inner), o[e]);
    }
}

// Threads of a row and pieces of eight channels per thread
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
static bool good_dtype(int d) { return d >= MKDA_F32 && d <= MKDA_F16; }

}  // namespace mkda

using namespace mkda;

extern "C" int mkda_norm_fwd(const MkdaNormFwd* p, void* stream) {
    if (!p || (p->rows && (!p->x || !p->y || (p->residual && !p->sum) || (p->out_e4m3 && !p->scale)))) return set_error(MKDA_ERR_ARG, "norm_fwd: null argument");
    if (p->rows < 0 || p->width < 1 || p->width > MKDA_NORM_MAX_WIDTH) return set_error(MKDA_ERR_ARG, "norm_fwd: rows of 1 to 32768 channels");
    if (!good_dtype(p->dtype) || (p->residual && !good_dtype(p->res_dtype)) || (p->weight && !good_dtype(p->weight_dtype))) return set_error(MKDA_ERR_ARG, "norm_fwd: unsupported dtype");
    if (p->group != 0 && (p->group != 128 || p->width % 128)) return set_error(MKDA_ERR_ARG, "norm_fwd: one scale per row, or per 128 channels of rows of a multiple of 128");
    if (p->rows == 0) return MKDA_OK;
    const bool vec = p->width % 8 == 0 && p->x_stride % 8 == 0 && (!p->residual || p->res_stride % 8 == 0) && aligned16(p->x) && aligned16(p->residual) && aligned16(p->sum) && aligned16(p->y);
    const bool wvec = p->width % 8 == 0 && aligned16(p->weight);
    with_dtype(p->dtype, [&](auto dt) {
        with_width(p->width, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value, RPB = TPR < 128 ? 128 / TPR : 1;
            launch(norm_fwd_kernel<DT, TPR, NV>, (p->rows + RPB - 1) / RPB, TPR < 128 ? 128 : TPR, 0, (cudaStream_t)stream, *p, vec, wvec);
        });
    });
    return check_launch("norm_fwd");
}

extern "C" int mkda_norm_bwd_part_rows(int rows, int width) {
    int r = 0;
    with_width(width, [&](auto t, auto) {
        constexpr int TPR = decltype(t)::value, RPB = TPR < 128 ? 128 / TPR : 1;
        const int most = sm_count() * (2048 / (TPR < 128 ? 128 : TPR)) / 2, want = (rows + RPB - 1) / RPB;
        r = (want < most ? want : most) * RPB;
    });
    return r;
}

extern "C" int mkda_norm_bwd(const MkdaNormBwd* p, void* stream) {
    if (!p || (p->rows && (!p->s || !p->dy || !p->dx))) return set_error(MKDA_ERR_ARG, "norm_bwd: null argument");
    if (p->rows < 0 || p->width < 1 || p->width > MKDA_NORM_MAX_WIDTH) return set_error(MKDA_ERR_ARG, "norm_bwd: rows of 1 to 32768 channels");
    if (!good_dtype(p->dtype) || !good_dtype(p->s_dtype) || ((p->dsum || p->dres) && !good_dtype(p->res_dtype)) || (p->weight && !good_dtype(p->weight_dtype)))
        return set_error(MKDA_ERR_ARG, "norm_bwd: unsupported dtype");
    if (p->rows == 0) return MKDA_OK;
    if (p->part && (p->part_rows != mkda_norm_bwd_part_rows(p->rows, p->width) || !aligned16(p->part)))
        return set_error(MKDA_ERR_ARG, "norm_bwd: as many rows of partial sums as mkda_norm_bwd_part_rows says, 16-byte aligned");
    const bool vec = p->width % 8 == 0 && p->s_stride % 8 == 0 && aligned16(p->s) && aligned16(p->dy) && aligned16(p->dsum) && aligned16(p->dx) && aligned16(p->dres);
    const bool wvec = p->width % 8 == 0 && aligned16(p->weight);
    with_dtype(p->dtype, [&](auto dt) {
        with_width(p->width, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value, RPB = TPR < 128 ? 128 / TPR : 1;
            launch(norm_bwd_kernel<DT, TPR, NV>, mkda_norm_bwd_part_rows(p->rows, p->width) / RPB, TPR < 128 ? 128 : TPR, 0, (cudaStream_t)stream, *p, vec, wvec);
        });
    });
    return check_launch("norm_bwd");
}

extern "C" int mkda_sum_rows(const MkdaSumRows* p, void* stream) {
    if (!p) return set_error(MKDA_ERR_ARG, "sum_rows: null argument");
    long long blocks = 0;
    for (const MkdaSumJob& q : p->job) {
        if (!q.out) continue;
        if ((!q.in && q.rows > 0) || q.rows < 0 || q.groups < 0 || q.cols < 0 || q.pitch < q.cols || q.inner < 1 || !good_dtype(q.out_dtype)) return set_error(MKDA_ERR_ARG, "sum_rows: bad argument");
        blocks += (q.cols + 127) / 128 * q.groups;
    }
    if (blocks > 0x7fffffffll) return set_error(MKDA_ERR_ARG, "sum_rows: too many columns");
    if (blocks == 0) return MKDA_OK;
    launch(sum_rows_kernel, (unsigned)blocks, 256, 0, (cudaStream_t)stream, *p);
    return check_launch("sum_rows");
}

extern "C" int mkda_block_struct_sizes(int* out, int n) {
#define MKDA_SIZE(S) (int)sizeof(S),
    const int sizes[] = {MKDA_BLOCK_STRUCTS(MKDA_SIZE)};
    const int cnt = (int)(sizeof(sizes) / sizeof(sizes[0]));
    for (int i = 0; i < n && i < cnt; ++i) out[i] = sizes[i];
    return cnt;
}
