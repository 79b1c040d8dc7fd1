// Layer norm of rows, or of each of `groups` equal parts of them (the heads of a token), with the residual's addition in front of it, and its backward pass.
//   s = x + residual (as the residual's type holds it)     m = mean s     r = 1 / sqrt(mean (s - m)^2 + eps)     h = (s - m) r     y = h weight + bias
//   dn = dy weight     ds = r (dn - mean dn - h mean(dn h)) + dsum     dweight = sum_rows dy h     dbias = sum_rows dy
// Bound by HBM: a part stays in the registers of the threads that share it, as in norm.cu, and the next one is on its way.  The variance is that of the differences to the
// mean, a second sum over what is in registers: in one pass it would lose what mean^2 is larger than it.  m and r are kept for the backward pass (8 bytes a part), which then
// has one pair of sums to form.
#include <algorithm>
#include <mutex>

#include "norm.cuh"

namespace mkda {

constexpr int LN_BWD_THREADS = 768;                        // per SM

template <int DT, int RDT, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, 1) layer_norm_fwd_kernel(const MkdaLayerNormFwd p, const bool vec, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1, RT = RDT < 0 ? DT : RDT;
    constexpr bool AHEAD = TPR <= 512, KEEP = AHEAD && NV <= 2;      // a thread of 1024 has registers neither for the next row nor for the weights
    __shared__ __align__(16) float part[2][TPR < 32 ? 1 : TPR / 32][1], part2[2][TPR < 32 ? 1 : TPR / 32][1];
    const int tid = threadIdx.x % TPR, W = p.width / p.groups, g0 = blockIdx.y * W;
    const long long stride = (long long)gridDim.x * RPB;
    const float over = 1.f / (float)W;
    float w[KEEP ? NV : 1][8], b[KEEP ? NV : 1][8];
    auto params = [&](int c, float (&v)[8], float (&u)[8]) {
        if (p.weight) {
            load_any8(p.weight, p.weight_dtype, g0 + c, W - c, wvec, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 1.f;
        }
        if (p.bias) {
            load_any8(p.bias, p.bias_dtype, g0 + c, W - c, wvec, u);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = 0.f;
        }
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) params((tid + i * TPR) * 8, w[i], b[i]);
    }
    Raw8 rx[NV], rr[NV];
    auto request = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8, ok = row < p.rows ? W - c : 0;
            rx[i] = load8<DT>(p.x, (size_t)row * p.x_stride + g0 + c, ok, vec);
            if constexpr (RDT >= 0) rr[i] = load8<RT>(p.residual, (size_t)row * p.res_stride + g0 + c, ok, vec);
        }
    };
    // A block's rows go together: where parts share a warp, those behind the last row are zeros that nobody stores, and take part in the sums' exchanges
    const long long mine = threadIdx.x / TPR;
    long long base = (long long)blockIdx.x * RPB, row = base + mine;
    if (AHEAD) request(row);
    for (int turn = 0; base < p.rows; base += stride, row = base + mine, turn ^= 1) {
        const bool real = row < p.rows;
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
                store8<RT>(p.sum, (size_t)row * p.width + g0 + c, real ? min(W - c, 8) : 0, vec, s[i]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[0] += s[i][e];           // zeros behind the part's end
        }
        if (AHEAD) request(row + stride);
        row_reduce<TPR, 1, false>(sum, part[turn]);
        const float m = sum[0] * over;
        float sq[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = W - (tid + i * TPR) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[i][e] -= m;
                if (e < left) sq[0] = fmaf(s[i][e], s[i][e], sq[0]);
            }
        }
        row_reduce<TPR, 1, false>(sq, part2[turn]);
        const float r = rsqrtf(fmaf(sq[0], over, p.eps));
        if (p.stats && tid == 0 && real) *reinterpret_cast<float2*>(p.stats + 2 * ((size_t)row * p.groups + blockIdx.y)) = make_float2(m, r);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            float v[8], u[8];
            if constexpr (!KEEP) params(c, v, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i][e] = fmaf(s[i][e] * r, KEEP ? w[KEEP ? i : 0][e] : v[e], KEEP ? b[KEEP ? i : 0][e] : u[e]);
            store8<DT>(p.y, (size_t)row * p.width + g0 + c, real ? min(W - c, 8) : 0, vec, s[i]);
        }
    }
}

// RT: the type of what was normalised and of the stream beside it.  As in norm.cu pieces stay as they lie in memory until they are used, and the weights are in shared memory.
template <int DT, int RT, int TPR, int NV, bool vec>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR <= 128 ? 6 : TPR == 1024 ? 1 : 768 / TPR) layer_norm_bwd_kernel(const MkdaLayerNormBwd p, const bool wvec) {
    follow_stream();
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    constexpr bool AHEAD = NV == 1;
    __shared__ __align__(16) float part[2][TPR < 32 ? 1 : TPR / 32][2];
    extern __shared__ __align__(16) float norm_w[];        // [TPR * NV * 8]
    const int tid = threadIdx.x % TPR, W = p.width / p.groups, g0 = blockIdx.y * W;
    const long long mine = threadIdx.x / TPR, stride = (long long)gridDim.x * RPB;
    const float over = 1.f / (float)W;
    for (int c = threadIdx.x * 8; c < TPR * NV * 8; c += blockDim.x * 8) {
        float w[8];
        if (p.weight) {
            load_any8(p.weight, p.weight_dtype, g0 + c, W - c, wvec, w);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 1.f;
        }
        st8<MKDA_F32>(norm_w, c, w);
    }
    __syncthreads();
    float dw[NV][8], db[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = db[i][e] = 0.f;
    Raw8 rs[NV], rg[NV], ru[NV];
    float2 rm = make_float2(0.f, 0.f);
    auto request = [&](long long row) {
        rm = row < p.rows ? *reinterpret_cast<const float2*>(p.stats + 2 * ((size_t)row * p.groups + blockIdx.y)) : make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8, ok = row < p.rows ? W - c : 0;
            rs[i] = load8<RT>(p.s, (size_t)row * p.s_stride + g0 + c, ok, vec);
            rg[i] = load8<DT>(p.dy, (size_t)row * p.width + g0 + c, ok, vec);
            if (p.dsum) ru[i] = load8<RT>(p.dsum, (size_t)row * p.width + g0 + c, ok, vec);
        }
    };
    long long base = (long long)blockIdx.x * RPB, row = base + mine;      // a block's rows go together, as in the forward kernel
    if (AHEAD) request(row);
    for (int turn = 0; base < p.rows; base += stride, row = base + mine, turn ^= 1) {
        const bool real = row < p.rows;
        if (!AHEAD) request(row);
        Raw8 qs[NV], qg[NV], qu[NV];
        const float m = rm.x, r = rm.y;
        float sums[2] = {0.f, 0.f};                        // of dn and of dn h; zeros of dy behind the part's end
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float s[8], g[8], w[8];
            qs[i] = rs[i]; qg[i] = rg[i]; qu[i] = ru[i];
            unpack8<RT>(qs[i], s);
            unpack8<DT>(qg[i], g);
            ld8(norm_w, MKDA_F32, (tid + i * TPR) * 8, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sums[0] = fmaf(g[e], w[e], sums[0]);
                sums[1] = fmaf(g[e] * w[e], (s[e] - m) * r, sums[1]);
            }
        }
        if (AHEAD) request(row + stride);
        row_reduce<TPR, 2, false>(sums, part[turn]);
        const float m1 = sums[0] * over, m2 = sums[1] * over;
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
                const float h = (s[e] - m) * r;
                dw[i][e] = fmaf(g[e], h, dw[i][e]);
                db[i][e] += g[e];
                o[e] = r * (fmaf(g[e], w[e], -m1) - h * m2);
                if (p.dsum) o[e] += u[e];
            }
            const int keep = real ? min(W - c, 8) : 0;
            store8<DT>(p.dx, (size_t)row * p.width + g0 + c, keep, vec, o);
            if (p.dres) store8<RT>(p.dres, (size_t)row * p.width + g0 + c, keep, vec, o);
        }
    }
    if (!p.part) return;
    float* to = p.part + (size_t)blockIdx.x * 2 * p.width + g0;
    const bool pvec = (p.width & 3) == 0 && (W & 7) == 0;  // rows of sums start on 16 bytes
    auto leave = [&](float (&d)[NV][8], float* out) {
        if constexpr (RPB > 1) {                           // the warps of a block, in order: a row of partial sums per block
            float* all = norm_w + TPR * NV * 8;            // [RPB][TPR * NV * 8]
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) st8<MKDA_F32>(all, (threadIdx.x / TPR) * TPR * NV * 8 + (tid + i * TPR) * 8, d[i]);
            __syncthreads();
            if (threadIdx.x < TPR)
                for (int w = 1; w < RPB; ++w)
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        float v[8];
                        ld8(all, MKDA_F32, w * TPR * NV * 8 + (tid + i * TPR) * 8, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e) d[i][e] += v[e];
                    }
        }
        if (threadIdx.x < TPR)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (tid + i * TPR) * 8;
                store8<MKDA_F32>(out, c, min(W - c, 8), pvec, d[i]);
            }
    };
    leave(dw, to);
    leave(db, to + p.width);
}

// Threads of a part: narrow ones share a warp (heads of 128 channels by whole warps, half of them idle: 262112 of 128 channels: forward 49 us, backward 83, where this takes 28 and 66)
template <bool BWD, typename F>
static bool with_part_width(int W, F f) {
    using std::integral_constant;
    if (W <= 64) f(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (W <= 128) f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else return BWD ? with_width_bwd(W, f) : with_width(W, f);
    return true;
}
// Blocks of a group that walk the rows, of `most` that are resident over all groups
template <int TPR>
static int group_blocks(int rows, int groups, int most) {
    constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
    return std::max(1, std::min((int)(((long long)rows + RPB - 1) / RPB), (most + groups - 1) / groups));
}
template <int TPR>
static int bwd_blocks(int rows, int groups) { return group_blocks<TPR>(rows, groups, sm_count() * (TPR == 1024 ? 1 : LN_BWD_THREADS / (TPR < 128 ? 128 : TPR))); }

int resident(const void* func, int threads) {
    struct Known { const void* func; int blocks; };
    static Known known[256];
    static int count = 0;
    static std::mutex mutex;
    std::lock_guard<std::mutex> lock(mutex);
    for (int i = 0; i < count; ++i)
        if (known[i].func == func) return known[i].blocks;
    int blocks = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, func, threads, 0) != cudaSuccess) (void)cudaGetLastError();
    if (blocks < 1) blocks = 1;
    if (count < 256) known[count++] = Known{func, blocks};
    return blocks;
}

}  // namespace mkda

using namespace mkda;

static const char* bad_shape(int rows, int width, int groups) {
    if (rows < 0 || width < 1 || groups < 1 || groups > 65535 || width % groups) return "layer_norm: rows of equal parts, at most 65535";
    if (width / groups > MKDA_NORM_MAX_WIDTH) return "layer_norm: parts of 1 to 32768 channels";
    return nullptr;
}

extern "C" int mkda_layer_norm_fwd(const MkdaLayerNormFwd* p, void* stream) {
    if (!p || (p->rows && (!p->x || !p->y || (p->residual && !p->sum)))) return set_error(MKDA_ERR_ARG, "layer_norm_fwd: null argument");
    if (const char* bad = bad_shape(p->rows, p->width, p->groups)) return set_error(MKDA_ERR_ARG, bad);
    if (!good_dtype(p->dtype) || (p->residual && p->res_dtype != p->dtype && p->res_dtype != MKDA_F32) || (p->weight && !good_dtype(p->weight_dtype)) || (p->bias && !good_dtype(p->bias_dtype)))
        return set_error(MKDA_ERR_ARG, "layer_norm_fwd: unsupported dtype");
    if (reinterpret_cast<uintptr_t>(p->stats) & 7) return set_error(MKDA_ERR_ARG, "layer_norm_fwd: stats must be 8-byte aligned");
    if (p->rows == 0) return MKDA_OK;
    const int W = p->width / p->groups;
    const bool vec = W % 8 == 0 && p->x_stride % 8 == 0 && (!p->residual || p->res_stride % 8 == 0) && aligned16(p->x) && aligned16(p->residual) && aligned16(p->sum) && aligned16(p->y);
    const bool wvec = W % 8 == 0 && aligned16(p->weight) && aligned16(p->bias);
    with_dtype(p->dtype, [&](auto dt) {
        with_part_width<false>(W, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value, THREADS = TPR < 128 ? 128 : TPR;
            auto* kern = !p->residual ? layer_norm_fwd_kernel<DT, -1, TPR, NV> : p->res_dtype == DT ? layer_norm_fwd_kernel<DT, DT, TPR, NV> : layer_norm_fwd_kernel<DT, MKDA_F32, TPR, NV>;
            launch(kern, dim3(group_blocks<TPR>(p->rows, p->groups, sm_count() * resident(reinterpret_cast<const void*>(kern), THREADS)), p->groups), THREADS, 0, (cudaStream_t)stream, *p, vec, wvec);
        });
    });
    return check_launch("layer_norm_fwd");
}

extern "C" int mkda_layer_norm_bwd_part_rows(int rows, int width, int groups) {
    int r = 0;
    if (bad_shape(rows, width, groups)) return 0;
    with_part_width<true>(width / groups, [&](auto t, auto) { r = bwd_blocks<decltype(t)::value>(rows, groups); });
    return r;
}

extern "C" int mkda_layer_norm_bwd(const MkdaLayerNormBwd* p, void* stream) {
    if (!p || (p->rows && (!p->s || !p->dy || !p->dx || !p->stats))) return set_error(MKDA_ERR_ARG, "layer_norm_bwd: null argument");
    if (const char* bad = bad_shape(p->rows, p->width, p->groups)) return set_error(MKDA_ERR_ARG, bad);
    if (!good_dtype(p->dtype) || (p->s_dtype != p->dtype && p->s_dtype != MKDA_F32) || (p->weight && !good_dtype(p->weight_dtype)))
        return set_error(MKDA_ERR_ARG, "layer_norm_bwd: unsupported dtype");
    if (reinterpret_cast<uintptr_t>(p->stats) & 7) return set_error(MKDA_ERR_ARG, "layer_norm_bwd: stats must be 8-byte aligned");
    if (p->part && (p->part_rows != mkda_layer_norm_bwd_part_rows(p->rows, p->width, p->groups) || !aligned16(p->part)))
        return set_error(MKDA_ERR_ARG, "layer_norm_bwd: as many rows of partial sums as mkda_layer_norm_bwd_part_rows says, 16-byte aligned");
    if (p->rows == 0) return MKDA_OK;
    const int W = p->width / p->groups;
    int rc = MKDA_OK;
    const bool vec = W % 8 == 0 && p->s_stride % 8 == 0 && aligned16(p->s) && aligned16(p->dy) && aligned16(p->dsum) && aligned16(p->dx) && aligned16(p->dres);
    const bool wvec = W % 8 == 0 && aligned16(p->weight);
    with_dtype(p->dtype, [&](auto dt) {
        with_part_width<true>(W, [&](auto t, auto n) {
            constexpr int DT = decltype(dt)::value, TPR = decltype(t)::value, NV = decltype(n)::value;
            auto* kern = p->s_dtype == DT ? vec ? layer_norm_bwd_kernel<DT, DT, TPR, NV, true> : layer_norm_bwd_kernel<DT, DT, TPR, NV, false>
                                          : vec ? layer_norm_bwd_kernel<DT, MKDA_F32, TPR, NV, true> : layer_norm_bwd_kernel<DT, MKDA_F32, TPR, NV, false>;
            constexpr int smem = TPR * NV * 8 * 4 * (TPR < 128 ? 1 + 128 / TPR : 1);
            if (smem > 40000) rc = ensure_smem(reinterpret_cast<const void*>(kern), smem, "layer_norm_bwd");
            if (rc == MKDA_OK) launch(kern, dim3(bwd_blocks<TPR>(p->rows, p->groups), p->groups), TPR < 128 ? 128 : TPR, smem, (cudaStream_t)stream, *p, wvec);
        });
    });
    if (rc != MKDA_OK) return rc;
    return check_launch("layer_norm_bwd");
}
