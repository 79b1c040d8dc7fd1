// RMS norm of whole rows with the residual's addition in front of it, its backward pass, and the second stage of the sums that the backward passes of
// conv.cu, scan.cu and this file leave.
//   s = x + residual (as the residual's type holds it)     r = 1 / sqrt(mean s^2 + eps)     y = s r weight     8 bits: y / scale, scale = max |y| / 448
//   dn = dy weight     ds = r (dn - s r^2 mean(dn s)) + dsum     dweight = sum_rows dy s r
// Bound by HBM: a row stays in the registers of the threads that share it (a warp for narrow rows, up to 1024 threads for wide ones),
// in pieces of eight channels, so that everything is read once.  8192 x 4096 bf16 with a residual: forward 46 us (5.8 TB/s), backward 50 us (5.4 TB/s) and 5 us for the sum of the
// weight's gradient; 65536 x 2048 with an output in e4m3 169 us (5.6 TB/s).
#include <algorithm>
#include <cuda_fp8.h>

#include <type_traits>

#include "block.cuh"

namespace mkda {

constexpr int NORM_FWD_THREADS = 1024, NORM_BWD_THREADS = 1024;      // per SM

// |v| kept, NaN passed on (fmaxf drops it, and a row of NaN would get the scale of a row of zeros)
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Sums (or maxima) of N = 1 or 2 values over the TPR threads of a row, the same in all of them; `part` is shared memory that two calls later may be used again
template <int TPR, int N, bool MAX>
__device__ __forceinline__ void row_reduce(float (&v)[N], float (*part)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
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

// Blocks walk the rows; the pieces of the next row are requested before this one's sums are formed, so that loads are in flight across the barrier.  RDT: the type of
// the residual, -1 without one.
template <int DT, int RDT, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, 1) norm_fwd_kernel(const MkdaNormFwd p, const bool vec, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1, RT = RDT < 0 ? DT : RDT;
    constexpr bool AHEAD = TPR <= 512, KEEP = AHEAD && NV <= 2;      // a thread of 1024 has registers neither for the next row nor for the weights
    __shared__ __align__(16) float part[2][TPR / 32][1], tops[2][TPR / 32][1];
    const int tid = threadIdx.x % TPR, H = p.width;
    const long long stride = (long long)gridDim.x * RPB;
    const float over = 1.f / (float)H;
    float w[KEEP ? NV : 1][8];
    auto weights = [&](int c, float (&v)[8]) {
        if (p.weight) {
            load_any8(p.weight, p.weight_dtype, c, H - c, wvec, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 1.f;
        }
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) weights((tid + i * TPR) * 8, w[i]);
    }
    Raw8 rx[NV], rr[NV];
    auto request = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8, ok = row < p.rows ? H - c : 0;
            rx[i] = load8<DT>(p.x, (size_t)row * p.x_stride + c, ok, vec);
            if constexpr (RDT >= 0) rr[i] = load8<RT>(p.residual, (size_t)row * p.res_stride + c, ok, vec);
        }
    };
    long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    if (AHEAD) request(row);
    for (int turn = 0; row < p.rows; row += stride, turn ^= 1) {      // rows of a block end together, or a row is a warp
        if (!AHEAD) request(row);
        float s[NV][8], sum[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            unpack8<DT>(rx[i], s[i]);
            if constexpr (RDT >= 0) {
                float r[8];
                unpack8<RT>(rr[i], r);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i][e] = as_held<RT>(s[i][e] + r[e]);
                store8<RT>(p.sum, (size_t)row * H + c, min(H - c, 8), vec, s[i]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[0] = fmaf(s[i][e], s[i][e], sum[0]);
        }
        if (AHEAD) request(row + stride);
        row_reduce<TPR, 1, false>(sum, part[turn]);
        const float r = rsqrtf(fmaf(sum[0], over, p.eps));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float v[8];
            if constexpr (!KEEP) weights(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i][e] = s[i][e] * r * (KEEP ? w[KEEP ? i : 0][e] : v[e]);
            if (!p.out_e4m3) store8<DT>(p.y, (size_t)row * H + c, min(H - c, 8), vec, s[i]);
        }
        if (!p.out_e4m3) continue;
        float top[1] = {0.f};
        if (!p.group) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top[0] = max_nan(top[0], fabsf(s[i][e]));
            row_reduce<TPR, 1, true>(top, tops[turn]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float t = top[0];
            if (p.group) {                                 // 128 channels are sixteen threads
                t = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) t = max_nan(t, fabsf(s[i][e]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, o));
            }
            const float scale = max_nan(t, 0x1p-126f * 448.f) / 448.f, inv = 1.f / scale;
            if (c >= H) continue;
            if (p.group ? c % 128 == 0 : c == 0) p.scale[p.group ? (size_t)row * (H / 128) + c / 128 : row] = scale;
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = __nv_cvt_float2_to_fp8x2(make_float2(s[i][2 * e] * inv, s[i][2 * e + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            uint8_t* out = static_cast<uint8_t*>(p.y) + (size_t)row * H + c;
            if (vec) {
                *reinterpret_cast<uint2*>(out) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < H) out[e] = (uint8_t)(b[e / 2] >> (e & 1) * 8);
            }
        }
    }
}

// RT: the type of what was normalised and of the stream beside it.  Pieces stay as they lie in memory and are widened when they are used, and the weights are in
// shared memory: registers are what keeps more blocks from being resident (64 for 1024 threads per SM; 128 with sixteen channels a thread 90 us where this takes 50).  64 do hold
// one piece a thread, up to 8192 channels (with an fp32 stream 44 to 80 bytes go to local memory); wider rows have two or four, of which 0.2 or 1 to 1.4 KB a thread do.
template <int DT, int RT, int TPR, int NV, bool vec>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR == 32 ? 5 : TPR == 128 ? 8 : 1024 / TPR) norm_bwd_kernel(const MkdaNormBwd p, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    constexpr bool AHEAD = NV == 1;
    __shared__ __align__(16) float part[2][TPR / 32][2];
    extern __shared__ __align__(16) float norm_w[];        // [TPR * NV * 8]
    const int tid = threadIdx.x % TPR, first = blockIdx.x * RPB + threadIdx.x / TPR, H = p.width;
    const long long stride = (long long)gridDim.x * RPB;
    const float over = 1.f / (float)H;
    for (int c = threadIdx.x * 8; c < TPR * NV * 8; c += blockDim.x * 8) {
        float w[8];
        if (p.weight) {
            load_any8(p.weight, p.weight_dtype, c, H - c, wvec, w);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 1.f;
        }
        st8<MKDA_F32>(norm_w, c, w);
    }
    __syncthreads();
    float dw[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
    Raw8 rs[NV], rg[NV], ru[NV];
    auto request = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8, ok = row < p.rows ? H - c : 0;
            rs[i] = load8<RT>(p.s, (size_t)row * p.s_stride + c, ok, vec);
            rg[i] = load8<DT>(p.dy, (size_t)row * H + c, ok, vec);
            if (p.dsum) ru[i] = load8<RT>(p.dsum, (size_t)row * H + c, ok, vec);
        }
    };
    if (AHEAD) request(first);
    int turn = 0;
    for (long long row = first; row < p.rows; row += stride, turn ^= 1) {
        if (!AHEAD) request(row);
        Raw8 qs[NV], qg[NV], qu[NV];
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float s[8], g[8], w[8];
            qs[i] = rs[i]; qg[i] = rg[i]; qu[i] = ru[i];
            unpack8<RT>(qs[i], s);
            unpack8<DT>(qg[i], g);
            ld8(norm_w, MKDA_F32, (tid + i * TPR) * 8, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sums[0] = fmaf(s[e], s[e], sums[0]);
                sums[1] = fmaf(g[e] * w[e], s[e], sums[1]);
            }
        }
        if (AHEAD) request(row + stride);
        row_reduce<TPR, 2, false>(sums, part[turn]);
        const float r = rsqrtf(fmaf(sums[0], over, p.eps)), k = -r * r * (sums[1] * over);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float s[8], g[8], w[8], o[8], u[8];
            unpack8<RT>(qs[i], s);
            unpack8<DT>(qg[i], g);
            ld8(norm_w, MKDA_F32, c, w);
            if (p.dsum) unpack8<RT>(qu[i], u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[i][e] = fmaf(g[e], s[e] * r, dw[i][e]);
                o[e] = r * fmaf(s[e], k, g[e] * w[e]);
                if (p.dsum) o[e] += u[e];
            }
            store8<DT>(p.dx, (size_t)row * H + c, min(H - c, 8), vec, o);
            if (p.dres) store8<RT>(p.dres, (size_t)row * H + c, min(H - c, 8), vec, o);
        }
    }
    if (!p.part) return;
    if constexpr (RPB > 1) {                               // the warps of a block, in order: a row of partial sums per block
        float* all = norm_w + TPR * NV * 8;                // [RPB][TPR * NV * 8]
#pragma unroll
        for (int i = 0; i < NV; ++i) st8<MKDA_F32>(all, (threadIdx.x / TPR) * TPR * NV * 8 + (tid + i * TPR) * 8, dw[i]);
        __syncthreads();
        if (threadIdx.x >= TPR) return;
        for (int w = 1; w < RPB; ++w)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[8];
                ld8(all, MKDA_F32, w * TPR * NV * 8 + (tid + i * TPR) * 8, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) dw[i][e] += v[e];
            }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * TPR) * 8;
        store8<MKDA_F32>(p.part, (size_t)blockIdx.x * H + c, min(H - c, 8), (H & 7) == 0, dw[i]);
    }
}

// A block adds the rows of 1024 / LANES columns: four columns a thread, LANES rows at a time, then the LANES in order.  Many rows of few columns by 32 lanes, few rows of many
// columns by four (128 rows of 2 x 65536 columns 22 us by 32 lanes, 17 by four).
template <int LANES>
__global__ void __launch_bounds__(256) sum_rows_kernel(const MkdaSumRows p) {
    follow_stream();
    constexpr int QUADS = 256 / LANES, COLS = 4 * QUADS;
    __shared__ float4 part[LANES][QUADS];
    long long blk = blockIdx.x;
    int j = 0;
    for (; j < 5; ++j) {
        const long long n = p.job[j].out ? (p.job[j].cols + COLS - 1) / COLS * p.job[j].groups : 0;
        if (blk < n) break;
        blk -= n;
    }
    if (j == 5) return;
    const MkdaSumJob& q = p.job[j];
    const long long per = (q.cols + COLS - 1) / COLS, g = blk / per, first = (blk - g * per) * COLS;
    const int l = threadIdx.x / QUADS, k = threadIdx.x % QUADS;
    const long long c = first + 4 * k;
    const float* in = q.in + (size_t)g * q.rows * q.pitch + c;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (((q.cols | q.pitch) & 3) == 0 && (reinterpret_cast<uintptr_t>(q.in) & 15) == 0) {
        if (c < q.cols) {
#pragma unroll 8
            for (int r = l; r < q.rows; r += LANES) {
                const float4 v = *reinterpret_cast<const float4*>(in + (size_t)r * q.pitch);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        }
    } else {
#pragma unroll 4
        for (int r = l; r < q.rows; r += LANES) {
            const float* v = in + (size_t)r * q.pitch;
            if (c < q.cols) s.x += v[0];
            if (c + 1 < q.cols) s.y += v[1];
            if (c + 2 < q.cols) s.z += v[2];
            if (c + 3 < q.cols) s.w += v[3];
        }
    }
    part[l][k] = s;
    __syncthreads();
    if (threadIdx.x >= COLS) return;
    const float* all = reinterpret_cast<const float*>(part) + threadIdx.x;      // one column per thread
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < LANES; ++i) o += all[COLS * i];
    const long long at = first + threadIdx.x, outer = at / q.inner, inner = at - outer * q.inner;
    if (at < q.cols && inner < q.valid) st1(q.out, q.out_dtype, (size_t)(g * q.out_group + outer * q.out_outer + inner * q.out_inner), o);
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

using namespace mkda;

extern "C" int mkda_norm_fwd(const MkdaNormFwd* p, void* stream) {
    if (!p || (p->rows && (!p->x || !p->y || (p->residual && !p->sum) || (p->out_e4m3 && !p->scale)))) return set_error(MKDA_ERR_ARG, "norm_fwd: null argument");
    if (p->rows < 0 || p->width < 1 || p->width > MKDA_NORM_MAX_WIDTH) return set_error(MKDA_ERR_ARG, "norm_fwd: rows of 1 to 32768 channels");
    if (!good_dtype(p->dtype) || (p->residual && p->res_dtype != p->dtype && p->res_dtype != MKDA_F32) || (p->weight && !good_dtype(p->weight_dtype))) return set_error(MKDA_ERR_ARG, "norm_fwd: unsupported dtype");
    if (p->group != 0 && (p->group != 128 || p->width % 128)) return set_error(MKDA_ERR_ARG, "norm_fwd: one scale per row, or per 128 channels of rows of a multiple of 128");
    if (p->rows == 0) return MKDA_OK;
    const bool vec = p->width % 8 == 0 && p->x_stride % 8 == 0 && (!p->residual || p->res_stride % 8 == 0) && aligned16(p->x) && aligned16(p->residual) && aligned16(p->sum) && aligned16(p->y);
    const bool wvec = p->width % 8 == 0 && aligned16(p->weight);
    with_dtype(p->dtype, [&](auto dt) {
        with_width(p->width, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value;
            auto* kern = !p->residual ? norm_fwd_kernel<DT, -1, TPR, NV> : p->res_dtype == DT ? norm_fwd_kernel<DT, DT, TPR, NV> : norm_fwd_kernel<DT, MKDA_F32, TPR, NV>;
            launch(kern, norm_blocks<TPR, NORM_FWD_THREADS>(p->rows), TPR < 128 ? 128 : TPR, 0, (cudaStream_t)stream, *p, vec, wvec);
        });
    });
    return check_launch("norm_fwd");
}

extern "C" int mkda_norm_bwd_part_rows(int rows, int width) {
    int r = 0;
    with_width_bwd(width, [&](auto t, auto) {
        r = norm_blocks<decltype(t)::value, NORM_BWD_THREADS>(rows);
    });
    return r;
}

extern "C" int mkda_norm_bwd(const MkdaNormBwd* p, void* stream) {
    if (!p || (p->rows && (!p->s || !p->dy || !p->dx))) return set_error(MKDA_ERR_ARG, "norm_bwd: null argument");
    if (p->rows < 0 || p->width < 1 || p->width > MKDA_NORM_MAX_WIDTH) return set_error(MKDA_ERR_ARG, "norm_bwd: rows of 1 to 32768 channels");
    if (!good_dtype(p->dtype) || (p->s_dtype != p->dtype && p->s_dtype != MKDA_F32) || (p->weight && !good_dtype(p->weight_dtype)))
        return set_error(MKDA_ERR_ARG, "norm_bwd: unsupported dtype");
    if (p->rows == 0) return MKDA_OK;
    if (p->part && (p->part_rows != mkda_norm_bwd_part_rows(p->rows, p->width) || !aligned16(p->part)))
        return set_error(MKDA_ERR_ARG, "norm_bwd: as many rows of partial sums as mkda_norm_bwd_part_rows says, 16-byte aligned");
    int rc = MKDA_OK;
    const bool vec = p->width % 8 == 0 && p->s_stride % 8 == 0 && aligned16(p->s) && aligned16(p->dy) && aligned16(p->dsum) && aligned16(p->dx) && aligned16(p->dres);
    const bool wvec = p->width % 8 == 0 && aligned16(p->weight);
    with_dtype(p->dtype, [&](auto dt) {
        with_width_bwd(p->width, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value;
            auto* kern = p->s_dtype == DT ? vec ? norm_bwd_kernel<DT, DT, TPR, NV, true> : norm_bwd_kernel<DT, DT, TPR, NV, false>
                                          : vec ? norm_bwd_kernel<DT, MKDA_F32, TPR, NV, true> : norm_bwd_kernel<DT, MKDA_F32, TPR, NV, false>;
            constexpr int smem = TPR * NV * 8 * 4 * (TPR < 128 ? 1 + 128 / TPR : 1);
            if (smem > 40000) rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "norm_bwd");
            if (rc == MKDA_OK) launch(kern, norm_blocks<TPR, NORM_BWD_THREADS>(p->rows), TPR < 128 ? 128 : TPR, smem, (cudaStream_t)stream, *p, wvec);
        });
    });
    if (rc != MKDA_OK) return rc;
    return check_launch("norm_bwd");
}

extern "C" int mkda_sum_rows(const MkdaSumRows* p, void* stream) {
    if (!p) return set_error(MKDA_ERR_ARG, "sum_rows: null argument");
    long long blocks = 0, wide = 0;
    int most = 0;
    for (const MkdaSumJob& q : p->job) {
        if (!q.out) continue;
        if ((!q.in && q.rows > 0) || q.rows < 0 || q.groups < 0 || q.cols < 0 || q.pitch < q.cols || q.inner < 1 || !good_dtype(q.out_dtype)) return set_error(MKDA_ERR_ARG, "sum_rows: bad argument");
        blocks += (q.cols + 31) / 32 * q.groups;
        wide += (q.cols + 255) / 256 * q.groups;
        most = std::max(most, q.rows);
    }
    if (blocks > 0x7fffffffll) return set_error(MKDA_ERR_ARG, "sum_rows: too many columns");
    if (blocks == 0) return MKDA_OK;
    // four lanes where that leaves two blocks per SM and no job has a long way down its rows
    if (wide >= 2 * sm_count() && most <= 512) launch(sum_rows_kernel<4>, (unsigned)wide, 256, 0, (cudaStream_t)stream, *p);
    else launch(sum_rows_kernel<32>, (unsigned)blocks, 256, 0, (cudaStream_t)stream, *p);
    return check_launch("sum_rows");
}

extern "C" int mkda_block_struct_sizes(int* out, int n) {
#define MKDA_SIZE(S) (int)sizeof(S),
    const int sizes[] = {MKDA_BLOCK_STRUCTS(MKDA_SIZE)};
    const int cnt = (int)(sizeof(sizes) / sizeof(sizes[0]));
    for (int i = 0; i < n && i < cnt; ++i) out[i] = sizes[i];
    return cnt;
}
