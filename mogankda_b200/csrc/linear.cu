// Linear attention with a decay for each head (linear.cuh): the kernel for any type and size of heads, the states of cut sequences, sums over the v-heads of a group, and the
// single-token form.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "linear.cuh"

namespace mkda {

// ---- any type, 1 to 128 channels: fp32 throughout ------------------------------------------------------------------------------------------------
// A block carries one part of a sequence and v-head, 64 tokens at a time: their rows and the state in shared memory, every product by fused multiply-adds on tiles of registers.  Bound by
// the tiles' way out of shared memory, four cycles for a warp's 16 bytes each, whoever shares them: with four rows and four columns a thread twice what its 49 thousand multiply-adds per
// token at 128 channels take (the older tensor instructions, as compensated TF32, are no faster).  ROWS x COLS: what the channels of b and of c are padded to for the threads' tiles.  64 x 64
// by 256 threads, two blocks to an SM: 4 x 1000 tokens x 8 heads forward 90 us, by 512 threads of two rows 99, 296 x 512 tokens 196 and 229 (201 since decays of states have two parts).  128 channels by 512, in us 279 for 148 x 512
// tokens; 256 threads with eight rows each have too few warps to cover the waits (319).
namespace ls {
constexpr int C = 64, PP = C + 4;
__host__ __device__ constexpr int threads(int rows, int cols) { return rows + cols == 128 ? 256 : 512; }
__host__ __device__ constexpr int pitch(int n) { return (n + 3) / 4 * 4 + 4; }
inline int smem(int M, int V) { return 4 * (2 * C * pitch(M) + C * pitch(V) + C * PP + ((M + 3) / 4 * 4) * pitch(V) + PP); }

// rows [0, len) of `n` channels from global memory, the rest of the C rows and of the pitch zero
template <int DT, int THREADS>
__device__ __forceinline__ void load_rows(float* to, int pit, const void* from, size_t at, long long stride, int n, int len, bool vec) {
    const int quads = pit / 4, step = THREADS / quads;     // rows at once
    const int r0 = threadIdx.x / quads, c = 4 * (threadIdx.x - r0 * quads);
    if (r0 >= step) return;
#pragma unroll 4
    for (int r = r0; r < C; r += step) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < len && c < n) {
            const size_t i = at + (size_t)r * stride + c;
            if (vec) {
                v = ld4(from, DT, i);
            } else {
                v.x = ld1(from, DT, i);
                if (c + 1 < n) v.y = ld1(from, DT, i + 1);
                if (c + 2 < n) v.z = ld1(from, DT, i + 2);
                if (c + 3 < n) v.w = ld1(from, DT, i + 3);
            }
        }
        *reinterpret_cast<float4*>(to + r * pit + c) = v;
    }
}
__device__ __forceinline__ void fma4(float (&d)[4], float a, const float4& b) {
    d[0] = fmaf(a, b.x, d[0]); d[1] = fmaf(a, b.y, d[1]); d[2] = fmaf(a, b.z, d[2]); d[3] = fmaf(a, b.w, d[3]);
}
// d[R][4] += rows x[R] (`xp` floats apart) times the columns y: terms [from, to), multiples of four
template <int R>
__device__ __forceinline__ void product(float (&d)[R][4], const float* x, int xp, const float* y, int yp, int from, int to) {
#pragma unroll 2
    for (int t = from; t < to; t += 4) {
        float4 q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = *reinterpret_cast<const float4*>(y + (t + e) * yp);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float4 f = *reinterpret_cast<const float4*>(x + r * xp + t);
            fma4(d[r], f.x, q[0]); fma4(d[r], f.y, q[1]); fma4(d[r], f.z, q[2]); fma4(d[r], f.w, q[3]);
        }
    }
}
}  // namespace ls

template <int DT, int ROWS, int COLS>
__global__ void __launch_bounds__(ls::threads(ROWS, COLS), ROWS + COLS == 128 ? 2 : 1) linear_simt_kernel(const __grid_constant__ LinearCall call, const bool vec) {
    using namespace ls;
    constexpr int THREADS = threads(ROWS, COLS);
    follow_stream();
    extern __shared__ __align__(16) float smem_f[];
    const LinearKind& k = call.kind[blockIdx.z];
    const int h = blockIdx.x % call.HV, part = blockIdx.x / call.HV, n = call.S.order && !call.S.seg ? call.S.order[blockIdx.y] : blockIdx.y;
    const LinearPart w = linear_part(call.S, n, part, k.back);
    if (w.nothing || (k.states && w.leaves_last)) return;      // what the last part leaves is the main kernel's to find
    const int M = k.M, V = k.V, pm = pitch(M), pv = pitch(V), M4 = (M + 3) / 4 * 4;
    float* sa = smem_f;
    float* sb = sa + C * pm;
    float* sc = sb + C * pm;
    float* sp = sc + C * pv;
    float* st = sp + C * PP;                               // [M4][pv]
    float* pw = st + M4 * pv;                              // lam^0 .. lam^64; what lam^64 and lam to the sequence's last tokens lack
    const int tid = threadIdx.x;
    const float gamma = call.log_decay[h];
    if (tid <= C) pw[tid] = decay_power(gamma, tid);
    else if (tid <= C + 2) pw[tid] = decay_parts(gamma, tid == C + 1 ? C : w.len % C).lo;
    const size_t size = (size_t)M * V;
    const float* in = k.states ? nullptr : call.S.seg ? k.parts + ((size_t)(n * call.S.segs + part) * call.HV + h) * size : k.first ? k.first + ((size_t)n * call.HV + h) * size : nullptr;
    for (int e = tid; e < M4 * pv; e += THREADS) {
        const int m = e / pv, v = e - m * pv;
        st[e] = in && m < M && v < V ? in[k.transposed ? (size_t)v * M + m : (size_t)m * V + v] : 0.f;
    }
    constexpr int ACROSS = COLS / 4, GROUPS = THREADS / ACROSS, OUT = C / GROUPS, STATE = ROWS / GROUPS;      // threads of a row, of a column, and rows of each
    const int v = 4 * (tid % ACROSS), group = tid / ACROSS;
    const int chunks = (w.len + C - 1) / C;
    for (int t = 0; t < chunks; ++t) {
        const int c0 = (k.back ? chunks - 1 - t : t) * C, len = min(C, w.len - c0);
        const size_t tok = w.start + c0;
        __syncthreads();
        if (!k.states) load_rows<DT, THREADS>(sa, pm, k.a, tok * k.a_stride + (size_t)(h / k.a_per) * M, k.a_stride, M, len, vec);
        load_rows<DT, THREADS>(sb, pm, k.b, tok * k.b_stride + (size_t)(h / k.b_per) * M, k.b_stride, M, len, vec);
        load_rows<DT, THREADS>(sc, pv, k.c, tok * k.c_stride + (size_t)(h / k.c_per) * V, k.c_stride, V, len, vec);
        __syncthreads();
        if (!k.states) {
            {                                              // pairs: rows i + STEP u, columns j = tid % 16 + 16 jj
                constexpr int STEP = THREADS / 16, PAIRS = C / STEP;
                const int i = tid >> 4;
                float d[PAIRS][4] = {};
#pragma unroll 2
                for (int m = 0; m < M4; m += 4) {
                    float4 x[PAIRS];
#pragma unroll
                    for (int u = 0; u < PAIRS; ++u) x[u] = *reinterpret_cast<const float4*>(sa + (i + STEP * u) * pm + m);
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const float4 y = *reinterpret_cast<const float4*>(sb + ((tid & 15) + 16 * jj) * pm + m);
#pragma unroll
                        for (int u = 0; u < PAIRS; ++u) d[u][jj] = fmaf(x[u].x, y.x, fmaf(x[u].y, y.y, fmaf(x[u].z, y.z, fmaf(x[u].w, y.w, d[u][jj]))));
                    }
                }
#pragma unroll
                for (int u = 0; u < PAIRS; ++u)
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const int row = i + STEP * u, j = (tid & 15) + 16 * jj, away = k.back ? j - row : row - j;
                        sp[row * PP + j] = away >= 0 && j < len ? d[u][jj] * pw[away] * k.pair_scale : 0.f;
                    }
            }
            __syncthreads();
            if (v < V) {
                float o[OUT][4] = {}, s[OUT][4] = {};
                const int i0 = OUT * group;
                // pairs of these rows: forwards up to the last one, backwards from the first one on
                product<OUT>(o, sp + i0 * PP, PP, sc + v, pv, k.back ? i0 & ~3 : 0, k.back ? C : (i0 + OUT + 3) & ~3);
                float odd = 0.f;
#pragma unroll
                for (int r = 0; r < OUT; ++r) odd += (o[r][0] + o[r][1]) + (o[r][2] + o[r][3]);
                if (!(fabsf(odd) <= FLT_MAX)) {            // 0 times what is not finite is not 0: once more, over the pairs that count
#pragma unroll
                    for (int r = 0; r < OUT; ++r) {
                        o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;
#pragma unroll 1
                        for (int j = k.back ? i0 + r : 0; j < (k.back ? len : min(len, i0 + r + 1)); ++j) fma4(o[r], sp[(i0 + r) * PP + j], *reinterpret_cast<const float4*>(sc + j * pv + v));
                    }
                }
                product<OUT>(s, sa + i0 * pm, pm, st + v, pv, 0, M4);
#pragma unroll
                for (int r = 0; r < OUT; ++r) {
                    const int i = i0 + r;
                    if (i >= len) continue;
                    const float f = pw[k.back ? len - 1 - i : i + 1] * k.state_scale;
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = fmaf(f, s[r][e], o[r][e]);
                    const size_t at = ((tok + i) * call.HV + h) * V + v;
                    if (V % 4 == 0) {
                        st4(k.out, k.out_dtype, at, make_float4(x[0], x[1], x[2], x[3]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (v + e < V) st1(k.out, k.out_dtype, at + e, x[e]);
                    }
                }
            }
            __syncthreads();
        }
        const int m0 = STATE * group;
        if (m0 < M && v < V) {                             // the state
            float acc[STATE][4] = {};
#pragma unroll 4
            for (int j = 0; j < len; ++j) {
                const float f = pw[k.back ? j + 1 : len - 1 - j] * k.in_scale;
                float4 y = *reinterpret_cast<const float4*>(sc + j * pv + v);
                y.x *= f; y.y *= f; y.z *= f; y.w *= f;
                const float* x = sb + j * pm + m0;
#pragma unroll
                for (int r = 0; r < STATE; r += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(x + r);
                    fma4(acc[r], q.x, y);
                    fma4(acc[r + 1], q.y, y);
                    fma4(acc[r + 2], q.z, y);
                    fma4(acc[r + 3], q.w, y);
                }
            }
            const Decay f = {pw[len], pw[len == C ? C + 1 : C + 2]};
#pragma unroll
            for (int r = 0; r < STATE; ++r) {
                if (m0 + r >= M) break;
                float4* s = reinterpret_cast<float4*>(st + (m0 + r) * pv + v);
                float4 x = *s;
                x.x = decayed(f, x.x, acc[r][0]); x.y = decayed(f, x.y, acc[r][1]); x.z = decayed(f, x.z, acc[r][2]); x.w = decayed(f, x.w, acc[r][3]);
                *s = x;
            }
        }
    }
    float* out = k.states ? k.parts + ((size_t)(n * call.S.segs + part + (k.back ? -1 : 1)) * call.HV + h) * size : k.last && w.leaves_last ? k.last + ((size_t)n * call.HV + h) * size : nullptr;
    if (!out) return;
    __syncthreads();
    for (size_t e = tid; e < size; e += THREADS) {
        const int slow = (int)(e / (k.transposed ? M : V)), fast = (int)(e - (size_t)slow * (k.transposed ? M : V));
        out[e] = k.transposed ? st[fast * pv + slow] : st[slow * pv + fast];
    }
}

// ---- cut sequences -------------------------------------------------------------------------------------------------------------------------------
// A part finds what it makes of nothing and leaves it where the next part's entering state belongs; this adds what comes through from further away:
//   parts[p] = (what part p - 1 makes of nothing) + lam^(tokens of part p - 1) parts[p - 1], parts[0] the sequence's initial state; backwards likewise.
__global__ void __launch_bounds__(256) linear_parts_kernel(const __grid_constant__ LinearCall call) {
    follow_stream();
    const LinearKind& k = call.kind[blockIdx.z];
    const int h = blockIdx.x % call.HV, n = blockIdx.y;
    const size_t size = (size_t)k.M * k.V, e = (size_t)(blockIdx.x / call.HV) * 256 + threadIdx.x, pitch = (size_t)call.HV * size;
    const Span w = sequence(call.S, n);
    const int len = w.end - w.start, seg = call.S.seg, parts = part_count(len, seg);
    if (e >= size) return;
    float* at = k.parts + ((size_t)n * call.S.segs * call.HV + h) * size + e;
    float s = k.first ? k.first[((size_t)n * call.HV + h) * size + e] : 0.f;
    const Decay whole = decay_parts(call.log_decay[h], seg), rest = decay_parts(call.log_decay[h], len - (parts - 1) * seg);
    // in the order of the walk; eight parts are requested before the first is written, or each would wait for memory by itself
    const int step = k.back ? -1 : 1;
    float* to = at + (k.back ? (parts - 1) * pitch : 0);
    *to = s;
    for (int p = 1; p < parts; p += 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p + i < parts ? to[(ptrdiff_t)(i + 1) * step * (ptrdiff_t)pitch] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (p + i >= parts) break;
            to += (ptrdiff_t)step * (ptrdiff_t)pitch;
            *to = s = decayed(k.back && p + i == 1 ? rest : whole, s, x[i]);
        }
    }
}

// ---- shared heads --------------------------------------------------------------------------------------------------------------------------------
// out[t][g] = sum over the `per` v-heads of group g, in order, for the tokens from the first sequence's first one (`first`, or 0 without it) on: nobody has written those in front of it
__global__ void __launch_bounds__(256) linear_group_kernel(const float* part, void* out, int dtype, const int* first, int heads, long long rows, int per, int K) {
    follow_stream();
    const bool vec = K % 4 == 0;
    const int step = vec ? 4 : 1;
    const long long all = rows * (K / step);
    for (long long e = (first ? (long long)*first * heads * (K / step) : 0) + (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
        const long long row = e / (K / step);
        const int c = (int)(e - row * (K / step)) * step;
        const float* p = part + (size_t)row * per * K + c;
        if (vec) {
            float4 s = *reinterpret_cast<const float4*>(p);
            for (int r = 1; r < per; ++r) {
                const float4 x = *reinterpret_cast<const float4*>(p + (size_t)r * K);
                s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
            }
            st4(out, dtype, (size_t)row * K + c, s);
        } else {
            float s = p[0];
            for (int r = 1; r < per; ++r) s += p[(size_t)r * K];
            st1(out, dtype, (size_t)row * K + c, s);
        }
    }
}

// ---- single tokens -------------------------------------------------------------------------------------------------------------------------------
// A block per v-head and sequence: S <- lam S + k v^T where it lies, o = scale S^T q.  Eight warps share the rows of the state, a lane has four columns of each of them; all of
// a thread's rows are requested before the first is used.  Bound by HBM: the state is read and written.
// lam has two parts: rounded to 32 bits it is off by up to 2^-25 with one sign at every token, and a memory of a million tokens would be 5 % off.  What the second one adds is less than half
// a step of the state: it goes in beside k v, in front of the last rounding.  An infinite state stays one: a thread that has something that is not finite leaves that part out there.
// 64 sequences x 32 heads of 128 channels 45.3 us, 44.4 with lam in one part (with scalar arithmetic 47.2).
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) linear_step_kernel(const MkdaLinearStep p) {
    follow_stream();
    __shared__ float sq[MKDA_LINEAR_MAX_DIM], sk[MKDA_LINEAR_MAX_DIM], part[8][MKDA_LINEAR_MAX_DIM], decay[2];
    const int h = blockIdx.x, n = blockIdx.y, K = p.K, V = p.V, g = h / (p.HV / p.HK), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, v = 4 * lane;
    float* state = p.state + ((size_t)n * p.HV + h) * K * V;
    const float rate = p.log_decay[h];
    float4 s[16];
    auto row = [&](int i) { return warp + 8 * i; };
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* at = state + (size_t)row(i) * V + v;
        if (row(i) >= K || v >= V) continue;
        if (VEC) {
            s[i] = *reinterpret_cast<const float4*>(at);
        } else {
            s[i].x = at[0];
            if (v + 1 < V) s[i].y = at[1];
            if (v + 2 < V) s[i].z = at[2];
            if (v + 3 < V) s[i].w = at[3];
        }
    }
    if (tid < K) sq[tid] = ld1(p.q, DT, (size_t)n * p.q_stride + (size_t)g * K + tid);
    else if (tid >= 128 && tid - 128 < K) sk[tid - 128] = ld1(p.k, DT, (size_t)n * p.k_stride + (size_t)g * K + tid - 128);
    float x[4] = {0.f, 0.f, 0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (v + e < V) x[e] = ld1(p.v, DT, (size_t)n * p.v_stride + (size_t)h * V + v + e);
    if (tid == 0) {
        const double lam = exp((double)rate);
        decay[0] = (float)lam;
        decay[1] = (float)(lam - (double)decay[0]);
    }
    f32x2 odd = both(0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) odd = fma2(pack2(s[i].z, s[i].w), both(0.f), fma2(pack2(s[i].x, s[i].y), both(0.f), odd));
    float odd0, odd1;
    unpack2(odd, odd0, odd1);
    __syncthreads();
    const float hi = decay[0], lo = decay[1];
    auto update = [&](auto finite) {
        const f32x2 x01 = pack2(x[0], x[1]), x23 = pack2(x[2], x[3]);
        f32x2 o01 = both(0.f), o23 = both(0.f);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (row(i) >= K || v >= V) continue;
            const f32x2 kk = both(sk[row(i)]), qq = both(sq[row(i)]);
            auto next = [&](float a, float b, f32x2 xs) {
                const f32x2 ab = pack2(a, b), small = decltype(finite)::value ? ab : pack2(fabsf(a) <= FLT_MAX ? a : 0.f, fabsf(b) <= FLT_MAX ? b : 0.f);
                return fma2(both(hi), ab, fma2(both(lo), small, mul2(kk, xs)));
            };
            const f32x2 s01 = next(s[i].x, s[i].y, x01), s23 = next(s[i].z, s[i].w, x23);
            o01 = fma2(qq, s01, o01);
            o23 = fma2(qq, s23, o23);
            float4 r;
            unpack2(s01, r.x, r.y);
            unpack2(s23, r.z, r.w);
            float* at = state + (size_t)row(i) * V + v;
            if (VEC) {
                *reinterpret_cast<float4*>(at) = r;
            } else {
                at[0] = r.x;
                if (v + 1 < V) at[1] = r.y;
                if (v + 2 < V) at[2] = r.z;
                if (v + 3 < V) at[3] = r.w;
            }
        }
        unpack2(o01, o[0], o[1]);
        unpack2(o23, o[2], o[3]);
    };
    if (odd0 + odd1 == 0.f) update(std::true_type());
    else update(std::false_type());
    *reinterpret_cast<float4*>(&part[warp][v]) = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (tid < V) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += part[w][tid];
        st1(p.o, DT, ((size_t)n * p.HV + h) * V + tid, p.scale * t);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------------
// The kernels that find the states of cut sequences (`before`) run first.
static int run_linear(const LinearCall& call, const LinearCall& before, cudaStream_t stream) {
    const MkdaSeqs& S = call.S;
    if (S.N == 0) return MKDA_OK;
    const bool tc = linear_tc_takes(call) && linear_tc_takes(before);
    auto run = [&](const LinearCall& c, bool states) {
        if (tc) return launch_linear_tc(c, states, stream);
        int bytes = 0, rc = MKDA_OK, rows = 0, cols = 0;
        bool vec = true;
        for (int i = 0; i < c.kinds; ++i) {
            const LinearKind& k = c.kind[i];
            bytes = std::max(bytes, ls::smem(k.M, k.V));
            rows = std::max(rows, k.M);
            cols = std::max(cols, k.V);
            vec = vec && k.M % 4 == 0 && k.V % 4 == 0 && k.a_stride % 4 == 0 && k.b_stride % 4 == 0 && k.c_stride % 4 == 0 && aligned16(k.a) && aligned16(k.b) && aligned16(k.c);
        }
        with_dtype(c.dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            auto* kern = rows > 64 ? cols > 64 ? linear_simt_kernel<DT, 128, 128> : linear_simt_kernel<DT, 128, 64> : cols > 64 ? linear_simt_kernel<DT, 64, 128> : linear_simt_kernel<DT, 64, 64>;
            rc = ensure_smem(reinterpret_cast<const void*>(kern), 227 * 1024 - 1024, "linear");
            if (rc == MKDA_OK) launch(kern, dim3(c.HV * (S.seg ? S.segs : 1), S.N, c.kinds), ls::threads(rows > 64 ? 128 : 64, cols > 64 ? 128 : 64), bytes, stream, c, vec);
        });
        return rc != MKDA_OK ? rc : check_launch("linear");
    };
    if (S.seg && S.segs > 1) {
        int rc = run(before, true);
        if (rc != MKDA_OK) return rc;
    }
    if (S.seg) {
        size_t size = 0;
        for (int i = 0; i < before.kinds; ++i) size = std::max(size, (size_t)before.kind[i].M * before.kind[i].V);
        launch(linear_parts_kernel, dim3(before.HV * (unsigned)((size + 255) / 256), S.N, before.kinds), 256, 0, stream, before);
        int rc = check_launch("linear parts");
        if (rc != MKDA_OK) return rc;
    }
    return run(call, false);
}

static const char* bad_linear(const MkdaLinearFwd& p) {
    if (!good_sequences(p.S)) return "linear: bad sequences";
    if (p.HK < 1 || p.HV < 1 || p.HV > 65535 || p.HV % p.HK) return "linear: the v-heads, at most 65535, must be a multiple of the q/k-heads";
    if (p.K < 1 || p.K > MKDA_LINEAR_MAX_DIM || p.V < 1 || p.V > MKDA_LINEAR_MAX_DIM) return "linear: heads of 1 to 128 channels";
    if (p.dtype < MKDA_F32 || p.dtype > MKDA_F16) return "linear: unsupported dtype";
    if (p.S.N > 65535) return "linear: at most 65535 sequences";
    if (p.S.seg < 0 || p.S.seg % (p.dtype == MKDA_F32 ? 64 : 128) || (p.S.seg && (p.S.segs < 1 || !p.seg_h))) return "linear: parts of a multiple of 128 tokens (fp32: 64), and a state for each";
    if (p.S.seg && (long long)p.HV * p.S.segs * 64 > 0x7fffffff) return "linear: too many parts";
    if (p.S.seg && !p.S.cu && (long long)p.S.seg * p.S.segs < p.S.T) return "linear: more tokens than the parts have";
    if (!p.log_decay) return "linear: null argument";
    if (any_misaligned(p.h0, p.ht, p.seg_h, p.o)) return "linear: states and outputs must be 16-byte aligned";
    return nullptr;
}

}  // namespace mkda

using namespace mkda;

// q and k of a v-head, v
static LinearKind kind_of(const MkdaLinearFwd& p, const void* a, long long sa, bool a_v, const void* b, long long sb, bool b_v, const void* c, long long sc, bool c_v) {
    const int per = p.HV / p.HK;
    LinearKind k{};
    k.a = a; k.b = b; k.c = c; k.a_stride = sa; k.b_stride = sb; k.c_stride = sc;
    k.a_per = a_v ? 1 : per; k.b_per = b_v ? 1 : per; k.c_per = c_v ? 1 : per;
    k.M = b_v ? p.V : p.K; k.V = c_v ? p.V : p.K;
    k.pair_scale = p.scale; k.in_scale = 1.f; k.state_scale = p.scale;
    k.out_dtype = p.dtype;
    return k;
}
static LinearCall call_of(const MkdaLinearFwd& p) {
    LinearCall c{};
    c.S = p.S; c.HV = p.HV; c.dtype = p.dtype; c.log_decay = p.log_decay;
    return c;
}

extern "C" int mkda_linear_fwd(const MkdaLinearFwd* p, void* stream) {
    if (!p) return set_error(MKDA_ERR_ARG, "linear_fwd: null argument");
    if (const char* bad = bad_linear(*p)) return set_error(MKDA_ERR_ARG, bad);
    if (p->S.TT && (!p->q || !p->k || !p->v || !p->o)) return set_error(MKDA_ERR_ARG, "linear_fwd: null argument");
    LinearCall call = call_of(*p), before = call;
    LinearKind k = kind_of(*p, p->q, p->q_stride, false, p->k, p->k_stride, false, p->v, p->v_stride, true);
    k.out = p->o; k.first = p->h0; k.last = p->ht; k.parts = p->seg_h;
    call.kind[0] = k; call.kinds = 1;
    k.states = 1;
    before.kind[0] = k; before.kinds = 1;
    return run_linear(call, before, (cudaStream_t)stream);
}

extern "C" int mkda_linear_bwd(const MkdaLinearBwd* q, void* stream) {
    if (!q) return set_error(MKDA_ERR_ARG, "linear_bwd: null argument");
    const MkdaLinearFwd& p = q->f;
    if (const char* bad = bad_linear(p)) return set_error(MKDA_ERR_ARG, bad);
    const bool shared = p.HV > p.HK;
    if (p.S.TT && (!p.q || !p.k || !p.v || !q->d_o || !q->dq || !q->dk || !q->dv || (shared && (!q->part_q || !q->part_k)))) return set_error(MKDA_ERR_ARG, "linear_bwd: null argument");
    if ((p.S.seg && !q->seg_g) || any_misaligned(q->d_o, q->dht, q->dq, q->dk, q->dv, q->dh0, q->seg_g, q->part_q, q->part_k))
        return set_error(MKDA_ERR_ARG, "linear_bwd: states, gradients and workspaces must be 16-byte aligned");
    if (q->end < 0 || q->end > p.S.TT) return set_error(MKDA_ERR_ARG, "linear_bwd: the last boundary is behind the tokens");
    const long long so = (long long)p.HV * p.V;
    LinearCall call = call_of(p), before = call;
    LinearKind dq = kind_of(p, q->d_o, so, true, p.v, p.v_stride, true, p.k, p.k_stride, false);
    LinearKind dk = kind_of(p, p.v, p.v_stride, true, q->d_o, so, true, p.q, p.q_stride, false);
    LinearKind dv = kind_of(p, p.k, p.k_stride, false, p.q, p.q_stride, false, q->d_o, so, true);
    dq.transposed = dk.transposed = 1;
    dk.back = dv.back = 1;
    dk.in_scale = dv.in_scale = p.scale;                   // the state's gradient has the scale in it
    dk.state_scale = dv.state_scale = 1.f;
    dq.first = p.h0; dk.first = dv.first = q->dht;
    dv.last = q->dh0;
    dq.parts = p.seg_h; dk.parts = dv.parts = q->seg_g;
    dq.out = shared ? static_cast<void*>(q->part_q) : q->dq; dk.out = shared ? static_cast<void*>(q->part_k) : q->dk; dv.out = q->dv;
    if (shared) dq.out_dtype = dk.out_dtype = MKDA_F32;
    call.kind[0] = dq; call.kind[1] = dk; call.kind[2] = dv; call.kinds = 3;
    LinearKind fs = kind_of(p, nullptr, 0, false, p.k, p.k_stride, false, p.v, p.v_stride, true), bs = dv;
    fs.first = p.h0; fs.parts = p.seg_h;
    fs.states = bs.states = 1;
    before.kind[0] = fs; before.kind[1] = bs; before.kinds = 2;
    int rc = run_linear(call, before, (cudaStream_t)stream);
    if (rc != MKDA_OK || !shared || q->end == 0 || p.S.N == 0) return rc;
    const long long rows = (long long)q->end * p.HK;
    const unsigned blocks = (unsigned)std::min<long long>((rows * p.K + 1023) / 1024, 16ll * sm_count());
    for (int i = 0; i < 2; ++i) {
        launch(linear_group_kernel, dim3(std::max(1u, blocks)), 256, 0, (cudaStream_t)stream, static_cast<const float*>(i ? q->part_k : q->part_q), i ? q->dk : q->dq, p.dtype, p.S.cu, p.HK, rows, p.HV / p.HK, p.K);
        rc = check_launch("linear groups");
        if (rc != MKDA_OK) return rc;
    }
    return MKDA_OK;
}

extern "C" int mkda_linear_step(const MkdaLinearStep* p, void* stream) {
    if (!p || !p->log_decay || (p->N && (!p->q || !p->k || !p->v || !p->state || !p->o))) return set_error(MKDA_ERR_ARG, "linear_step: null argument");
    if (p->N < 0 || p->N > 65535) return set_error(MKDA_ERR_ARG, "linear_step: at most 65535 sequences");
    if (p->HK < 1 || p->HV < 1 || p->HV % p->HK) return set_error(MKDA_ERR_ARG, "linear_step: the v-heads must be a multiple of the q/k-heads");
    if (p->K < 1 || p->K > MKDA_LINEAR_MAX_DIM || p->V < 1 || p->V > MKDA_LINEAR_MAX_DIM) return set_error(MKDA_ERR_ARG, "linear_step: heads of 1 to 128 channels");
    if (p->dtype < MKDA_F32 || p->dtype > MKDA_F16) return set_error(MKDA_ERR_ARG, "linear_step: unsupported dtype");
    if (!aligned16(p->state)) return set_error(MKDA_ERR_ARG, "linear_step: the state must be 16-byte aligned");
    if (p->N == 0) return MKDA_OK;
    with_dtype(p->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        launch(p->V % 4 == 0 ? linear_step_kernel<DT, true> : linear_step_kernel<DT, false>, dim3(p->HV, p->N), 256, 0, (cudaStream_t)stream, *p);
    });
    return check_launch("linear_step");
}
