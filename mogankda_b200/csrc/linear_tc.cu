// Linear attention with a decay for each head (linear.cuh) in bf16 on the Blackwell tensor cores.
//
// A block (one per SM) carries parts of sequences and v-heads one after the other, 128 tokens at a time.  With the rows of a, b and c in shared memory (tiled copies, 128-byte
// swizzle) a stretch is four products with fp32 accumulators in tensor memory:
//   P0 = a b^T                       pairs; the weights lam^|i - j| and the mask are applied to the accumulator, and P leaves as bf16 hi + lo, the left operand of P c
//   O  = a M                         M: the state in front of the stretch as hi + lo in shared memory; lam^(i + 1) is applied to the accumulator's rows
//   O += P c
//   M^T = lam^L M^T + (f c)^T b      f[j] = lam^(L - 1 - j); M^T stays in its accumulator, and f c is split in three parts, so that the state is an fp32 one
// a, b and c are exact in bf16.  Two halves (2^-16) are enough where the result is rounded to bf16, one would show: P and M in one bf16 each are as far off as the result's own rounding.
//
// Roles, joined by mbarriers: a warp that fetches rows into a ring of five tiles, one that issues products, and four warps each for the pairs' weights, for f c, for the state and
// for the output.  Every accumulator row is a lane: token i of P0 and O, channel of c of M^T.
//
// Bound by HBM where there are enough parts: 128 KB per stretch, 3 us of an SM's share; products take 8 x 516 cycles = 2.2 us, and each group of warps less than that.
#include <algorithm>

#include "host.h"
#include "linear.cuh"
#include "umma.cuh"

namespace mkda {
namespace lt {

using umma::mbar_wait;
using umma::signal_tmem;
using umma::wait_mma;

constexpr int C = 128, TILE = 32768, SLOTS = 5, THREADS = 576, WARP_LOAD = 16, WARP_MMA = 17;
constexpr int P = 0, O = 128, S = 256, F = 384;            // tensor-memory columns: pairs, output, state, f c (two buffers of a quarter: 3 x 16 columns each)

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS];
    uint64_t p0_done, p_ready, f_ready[2], f_free[2], s_ready, x_done, in_done, o_scaled, o_done, o_free;
    uint32_t tmem;
    float power[C + 4];                                    // lam^n of the current part's head, one copy per group of warps that reads it
    float power_p[C + 4], power_o[C + 4];
};
constexpr int SMEM = 2 * TILE + SLOTS * TILE + (int)sizeof(Shared);
static_assert(SMEM <= 232448, "shared memory of one block");

struct Maps { CUtensorMap row[4]; };                       // rows of a head, boxes of 64 channels x 128 tokens
struct Plan {
    LinearCall call;
    int map_a[3], map_b[3], map_c[3];                      // per kind
    long long items;
};

struct Item { int kind, h, n, part; };
__device__ __forceinline__ Item item_of(const LinearCall& call, long long w) {
    Item it;
    it.kind = (int)(w % call.kinds);
    w /= call.kinds;
    it.h = (int)(w % call.HV);
    w /= call.HV;
    const int segs = call.S.seg ? call.S.segs : 1;
    it.part = (int)(w % segs);
    const int n = (int)(w / segs);
    it.n = call.S.order ? call.S.order[n] : n;
    return it;
}
// Calls f(kind, item, part) for every item of this block that has something to do, the same ones in every role
template <bool STATES, typename Body>
__device__ __forceinline__ void for_items(const Plan& plan, Body body) {
    for (long long w = blockIdx.x; w < plan.items; w += gridDim.x) {
        const Item it = item_of(plan.call, w);
        const LinearKind& k = plan.call.kind[it.kind];
        const LinearPart part = linear_part(plan.call.S, it.n, it.part, k.back);
        if (part.nothing || (STATES && part.leaves_last)) continue;
        body(k, it, part, (part.len + C - 1) / C);
    }
}
__device__ __forceinline__ int first_of(const LinearKind& k, int chunks, int t) { return (k.back ? chunks - 1 - t : t) * C; }
__device__ __forceinline__ const float* entering(const LinearCall& call, const LinearKind& k, const Item& it, bool states) {
    const size_t size = (size_t)k.M * k.V;
    if (states) return nullptr;
    if (call.S.seg) return k.parts + ((size_t)(it.n * call.S.segs + it.part) * call.HV + it.h) * size;
    return k.first ? k.first + ((size_t)it.n * call.HV + it.h) * size : nullptr;
}
// Powers of lam for one group of 128 threads, between its own barriers
__device__ __forceinline__ void set_powers(float* to, float log_decay, int tid, int barrier) {
    asm volatile("bar.sync %0, 128;" :: "r"(barrier) : "memory");
    to[tid] = decay_power(log_decay, tid);
    if (tid == 0) to[C] = decay_power(log_decay, C);
    asm volatile("bar.sync %0, 128;" :: "r"(barrier) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&f)[32]) {
    uint32_t a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) { a[i] = __float_as_uint(f[i]); b[i] = __float_as_uint(f[16 + i]); }
    umma::tmem_st16(taddr, a);
    umma::tmem_st16(taddr + 16, b);
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, int x, int head, int token, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(umma::smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(umma::smem_u32(bar)) : "memory");
}

// STATES: nothing but what the parts of cut sequences make of a zero state
template <bool STATES>
__global__ void __launch_bounds__(THREADS, 1) linear_tc_kernel(const __grid_constant__ Plan plan, const __grid_constant__ Maps maps) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = smem_raw;                              // no static shared memory: the dynamic block starts on a 1024-byte boundary
    uint8_t* const state_hi = base;                        // M^T [channel of c][channel of b], hi then lo
    uint8_t* const ring = base + 2 * TILE;
    Shared& sh = *reinterpret_cast<Shared*>(ring + SLOTS * TILE);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (umma::smem_u32(base) & 1023) {                     // ... and nothing runs if that ever fails to hold
        follow_stream();
        if (tid == 0) atomicExch(&umma::g_timeout_flag, 1u);
        return;
    }
    if (warp == 0) umma::tmem_alloc(&sh.tmem, 512);
    if (tid == 0) {
        for (int i = 0; i < SLOTS; ++i) { umma::mbar_init(&sh.full[i], 1); umma::mbar_init(&sh.empty[i], 1); }
        for (uint64_t* b : {&sh.p0_done, &sh.f_free[0], &sh.f_free[1], &sh.x_done, &sh.in_done, &sh.o_done}) umma::mbar_init(b, 1);
        for (uint64_t* b : {&sh.p_ready, &sh.f_ready[0], &sh.f_ready[1], &sh.s_ready, &sh.o_scaled, &sh.o_free}) umma::mbar_init(b, 4);
        umma::fence_barrier_init();
    }
    follow_stream();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = sh.tmem;
    const LinearCall& call = plan.call;
    constexpr int PER = STATES ? 2 : 3;                    // tiles of a stretch: (a,) b, c
    auto slot_of = [](uint32_t tile) { return tile % SLOTS; };
    auto parity_of = [](uint32_t tile) { return (tile / SLOTS) & 1u; };

    if (warp == WARP_LOAD) {
        if (umma::elect_one()) {
            uint32_t tile = 0;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                const int idx = it.kind;
                for (int t = 0; t < chunks; ++t) {
                    const int tok = part.start + first_of(k, chunks, t);
                    auto fetch = [&](int map, int head) {
                        const uint32_t s = slot_of(tile);
                        if (tile >= SLOTS) mbar_wait(&sh.empty[s], parity_of(tile) ^ 1u);
                        umma::mbar_expect_tx(&sh.full[s], TILE);
                        load_box(ring + s * TILE, &maps.row[map], 0, head, tok, &sh.full[s]);
                        load_box(ring + s * TILE + TILE / 2, &maps.row[map], 64, head, tok, &sh.full[s]);
                        ++tile;
                    };
                    if (!STATES) fetch(plan.map_a[idx], it.h / k.a_per);
                    fetch(plan.map_b[idx], it.h / k.b_per);
                    fetch(plan.map_c[idx], it.h / k.c_per);
                }
            });
        }
        __syncwarp();
    } else if (warp == WARP_MMA) {
        if (umma::elect_one()) {
            uint32_t n = 0;                                // stretches so far
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart&, int chunks) {
                const int ms = (k.M + 15) / 16, vn = (k.V + 15) / 16 * 16;
                const bool zero = entering(call, k, it, STATES) == nullptr;
                const uint32_t id_p0 = umma::idesc_bf16(128, C), id_in = umma::idesc_bf16(128, vn), id_pc = umma::idesc_bf16(128, vn, 0, 1), id_x = umma::idesc_bf16(128, ms * 16, 0, 1);
                for (int t = 0; t < chunks; ++t, ++n) {
                    const uint32_t ta = n * PER, tb = ta + (STATES ? 0 : 1), tc = tb + 1, par = n & 1;
                    const umma::Opnd a = umma::opnd_k(ring + slot_of(ta) * TILE, nullptr, 128), bk = umma::opnd_k(ring + slot_of(tb) * TILE, nullptr, 128);
                    const umma::Opnd bm = umma::opnd_mn(ring + slot_of(tb) * TILE, nullptr, 128), cm = umma::opnd_mn(ring + slot_of(tc) * TILE, nullptr, 128);
                    const uint64_t ad = umma::opnd_base_desc(a, a.hi);
                    if (!STATES) mbar_wait(&sh.full[slot_of(ta)], parity_of(ta));
                    mbar_wait(&sh.full[slot_of(tb)], parity_of(tb));
                    if (!STATES) {
                        const uint64_t bd = umma::opnd_base_desc(bk, bk.hi);
                        for (int ks = 0; ks < ms; ++ks) umma::mma_bf16(tmem + P, ad + umma::opnd_step16(a, ks), bd + umma::opnd_step16(bk, ks), id_p0, ks != 0);
                        umma::commit(&sh.p0_done);
                        if (n) wait_mma(&sh.o_free, par ^ 1u);
                    }
                    wait_mma(&sh.s_ready, par);
                    const bool from_zero = zero && t == 0;
                    if (!STATES) {
                        if (!from_zero) {
                            const umma::Opnd m = umma::opnd_k(state_hi, state_hi + TILE, 128);
                            const uint64_t mh = umma::opnd_base_desc(m, m.hi), ml = umma::opnd_base_desc(m, m.lo);
                            for (int ks = 0; ks < ms; ++ks) {
                                const uint32_t ao = umma::opnd_step16(a, ks), mo = umma::opnd_step16(m, ks);
                                umma::mma_bf16(tmem + O, ad + ao, ml + mo, id_in, ks != 0);
                                umma::mma_bf16(tmem + O, ad + ao, mh + mo, id_in, 1u);
                            }
                        }
                        umma::commit(&sh.in_done);
                        umma::commit(&sh.empty[slot_of(ta)]);
                    }
                    const uint64_t bmd = umma::opnd_base_desc(bm, bm.hi);
                    uint32_t acc = !from_zero;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {          // 32 tokens: the smallest of the three parts of f c first
                        wait_mma(&sh.f_ready[q & 1], (2 * n + (q >> 1)) & 1);
#pragma unroll
                        for (int part = 2; part >= 0; --part)
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks) {
                                umma::mma_bf16_ta(tmem + S, tmem + F + 64 * (q & 1) + 16 * part + 8 * ks, bmd + umma::opnd_step16(bm, 2 * q + ks), id_x, acc);
                                acc = 1u;
                            }
                        umma::commit(&sh.f_free[q & 1]);
                    }
                    umma::commit(&sh.x_done);
                    umma::commit(&sh.empty[slot_of(tb)]);
                    if (!STATES) {
                        wait_mma(&sh.p_ready, par);
                        wait_mma(&sh.o_scaled, par);
                        mbar_wait(&sh.full[slot_of(tc)], parity_of(tc));
                        const uint64_t cd = umma::opnd_base_desc(cm, cm.hi);
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t at = tmem + P + 32 * (ks >> 1) + 8 * (ks & 1);
                            umma::mma_bf16_ta(tmem + O, at + 16, cd + umma::opnd_step16(cm, ks), id_pc, ks != 0 || !from_zero);
                            umma::mma_bf16_ta(tmem + O, at, cd + umma::opnd_step16(cm, ks), id_pc, 1u);
                        }
                        umma::commit(&sh.o_done);
                    }
                    umma::commit(&sh.empty[slot_of(tc)]);
                }
            });
            if (n) mbar_wait(&sh.empty[slot_of(n * PER - 1)], parity_of(n * PER - 1));      // the last arrival of a product
        }
        __syncwarp();
    } else if (warp < 4) {
        // ---- pairs: row i = this lane's token
        if (!STATES) {
            uint32_t n = 0;
            const int i = tid;
            float* const power = sh.power_p;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                set_powers(power, call.log_decay[it.h], tid, 1);
                for (int t = 0; t < chunks; ++t, ++n) {
                    const int len = min(C, part.len - first_of(k, chunks, t));
                    wait_mma(&sh.p0_done, n & 1);
#pragma unroll 1
                    for (int blk = 0; blk < 4; ++blk) {
                        const uint32_t at = umma::tmem_addr(tmem, warp, P + 32 * blk);
                        uint32_t h[16], l[16];
                        if (k.back ? blk < warp || 32 * blk >= len : blk > warp) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) h[e] = l[e] = 0u;
                        } else {
                            float v[32];
                            umma::tmem_ld32(at, v);
                            const int away = k.back ? 32 * blk - i : i - 32 * blk;      // of column 0
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float x[2];
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    const int d = k.back ? away + e + u : away - e - u;
                                    const bool good = d >= 0 && (!k.back || 32 * blk + e + u < len);
                                    x[u] = good ? v[e + u] * (power[good ? d : 0] * k.pair_scale) : 0.f;
                                }
                                umma::split2(x[0], x[1], h[e / 2], l[e / 2]);
                            }
                        }
                        umma::tmem_st16(at, h);
                        umma::tmem_st16(at + 16, l);
                    }
                    umma::tmem_wait_st();
                    signal_tmem(&sh.p_ready, lane);
                }
            });
        }
    } else if (warp < 8) {
        // ---- f c, transposed: row = this lane's channel of c
        uint32_t n = 0;
        const int ch = tid - 128, k8 = ch >> 3;
        float* const power = sh.power;
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            set_powers(power, call.log_decay[it.h], ch, 2);
            for (int t = 0; t < chunks; ++t, ++n) {
                const int len = min(C, part.len - first_of(k, chunks, t));
                const uint32_t tb = n * PER + (STATES ? 0 : 1), tc = tb + 1;
                uint8_t* const c = ring + slot_of(tc) * TILE;
                mbar_wait(&sh.full[slot_of(tc)], parity_of(tc));
                if (len < C) {                             // rows behind the part's end belong to somebody else: 0 times what is not finite is not 0
                    uint8_t* const b = ring + slot_of(tb) * TILE;
                    mbar_wait(&sh.full[slot_of(tb)], parity_of(tb));
                    for (int e = ch; e < (C - len) * 16; e += 128) {
                        const uint32_t off = umma::tile_chunk_offset(128, len + (e >> 4), e & 15);
                        *reinterpret_cast<uint4*>(b + off) = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(c + off) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("bar.sync 2, 128;" ::: "memory");
                    __syncwarp();
                }
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[3][16];
                    const int j0 = 32 * q, at = k.back ? j0 + 1 : len - 1 - j0;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float x[2], r[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t off = umma::tile_chunk_offset(128, j0 + e + u, k8) + 2 * (ch & 7);
                            const float v = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(c + off) << 16);
                            const int d = k.back ? at + e + u : at - e - u;
                            x[u] = v * (power[max(d, 0)] * k.in_scale);      // behind the part's end v is 0
                        }
                        w[0][e / 2] = umma::pack_bf16x2(x[0], x[1]);
                        r[0] = x[0] - __uint_as_float(w[0][e / 2] << 16);
                        r[1] = x[1] - __uint_as_float(w[0][e / 2] & 0xffff0000u);
                        w[1][e / 2] = umma::pack_bf16x2(r[0], r[1]);
                        r[0] -= __uint_as_float(w[1][e / 2] << 16);
                        r[1] -= __uint_as_float(w[1][e / 2] & 0xffff0000u);
                        w[2][e / 2] = umma::pack_bf16x2(r[0], r[1]);
                    }
                    const uint32_t use = 2 * n + (q >> 1);         // of this buffer
                    if (use) wait_mma(&sh.f_free[q & 1], (use - 1) & 1);
#pragma unroll
                    for (int p = 0; p < 3; ++p) umma::tmem_st16(umma::tmem_addr(tmem, warp, F + 64 * (q & 1) + 16 * p), w[p]);
                    umma::tmem_wait_st();
                    umma::signal(&sh.f_ready[q & 1], lane);
                }
            }
        });
    } else if (warp < 12) {
        // ---- the state: row = this lane's channel of c, columns the channels of b
        uint32_t n = 0;
        const int ch = tid - 256;
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            const float* in = entering(call, k, it, STATES);
            const size_t size = (size_t)k.M * k.V;
            float* out = STATES ? k.parts + ((size_t)(it.n * call.S.segs + it.part + (k.back ? -1 : 1)) * call.HV + it.h) * size
                                : k.last && part.leaves_last ? k.last + ((size_t)it.n * call.HV + it.h) * size : nullptr;
            const float gamma = call.log_decay[it.h], whole = decay_power(gamma, C), rest = decay_power(gamma, part.len % C);
            auto at = [&](int m) { return k.transposed ? (size_t)ch * k.M + m : (size_t)m * k.V + ch; };
            auto from_memory = [&](int m0, float (&v)[32]) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = in && ch < k.V && m0 + e < k.M ? in[at(m0 + e)] : 0.f;
            };
            for (int t = 0; t < chunks; ++t, ++n) {
                const bool from_zero = t == 0 && !in;
                if (t) wait_mma(&sh.x_done, (n - 1) & 1);
                if (!from_zero) {
                    const bool short_one = part.len - first_of(k, chunks, t) < C;
                    const float f = short_one ? rest : whole;
#pragma unroll 1
                    for (int m0 = 0; m0 < k.M; m0 += 32) {
                        float v[32];
                        if (t) umma::tmem_ld32(umma::tmem_addr(tmem, warp, S + m0), v);
                        else from_memory(m0, v);
                        if (!STATES) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                const float x[8] = {v[e], v[e + 1], v[e + 2], v[e + 3], v[e + 4], v[e + 5], v[e + 6], v[e + 7]};
                                umma::store_split8(state_hi, state_hi + TILE, 128, ch, (m0 + e) >> 3, x);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= f;
                        __syncwarp();
                        tmem_st32(umma::tmem_addr(tmem, warp, S + m0), v);
                    }
                    umma::tmem_wait_st();
                }
                umma::signal(&sh.s_ready, lane);
            }
            if (chunks) wait_mma(&sh.x_done, (n - 1) & 1);
            if (!out) return;
#pragma unroll 1
            for (int m0 = 0; m0 < k.M; m0 += 32) {
                float v[32];
                __syncwarp();
                if (chunks) umma::tmem_ld32(umma::tmem_addr(tmem, warp, S + m0), v);
                else from_memory(m0, v);
                if (ch < k.V)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (m0 + e < k.M) out[at(m0 + e)] = v[e];
            }
        });
    } else if (warp < 16) {
        // ---- the output: row i = this lane's token
        if (!STATES) {
            uint32_t n = 0;
            const int i = tid - 384;
            float* const power = sh.power_o;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                set_powers(power, call.log_decay[it.h], i, 3);
                const bool zero = entering(call, k, it, STATES) == nullptr;
                for (int t = 0; t < chunks; ++t, ++n) {
                    const int c0 = first_of(k, chunks, t), len = min(C, part.len - c0);
                    wait_mma(&sh.in_done, n & 1);
                    if (!zero || t) {
                        const float f = power[k.back ? max(len - 1 - i, 0) : i + 1] * k.state_scale;
#pragma unroll 1
                        for (int m0 = 0; m0 < k.V; m0 += 32) {
                            float v[32];
                            umma::tmem_ld32(umma::tmem_addr(tmem, warp, O + m0), v);
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] *= f;
                            tmem_st32(umma::tmem_addr(tmem, warp, O + m0), v);
                        }
                        umma::tmem_wait_st();
                    }
                    signal_tmem(&sh.o_scaled, lane);
                    wait_mma(&sh.o_done, n & 1);
                    const size_t row = ((size_t)(part.start + c0 + i) * call.HV + it.h) * k.V;
#pragma unroll 1
                    for (int m0 = 0; m0 < k.V; m0 += 32) {
                        float v[32];
                        __syncwarp();
                        umma::tmem_ld32(umma::tmem_addr(tmem, warp, O + m0), v);
                        if (m0 + 32 >= k.V) signal_tmem(&sh.o_free, lane);
                        if (i >= len) continue;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (m0 + e >= k.V) break;
                            const float x[8] = {v[e], v[e + 1], v[e + 2], v[e + 3], v[e + 4], v[e + 5], v[e + 6], v[e + 7]};
                            if (k.out_dtype == MKDA_F32) st8<MKDA_F32>(k.out, row + m0 + e, x);
                            else st8<MKDA_BF16>(k.out, row + m0 + e, x);
                        }
                    }
                }
            });
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (warp == 0) umma::tmem_dealloc(tmem, 512);
}

}  // namespace lt

bool linear_tc_takes(const LinearCall& call) {
    if (call.dtype != MKDA_BF16 || call.S.TT < 1) return false;
    for (int i = 0; i < call.kinds; ++i) {
        const LinearKind& k = call.kind[i];
        if (k.M % 8 || k.V % 8 || (k.a && (k.a_stride % 8 || !aligned16(k.a))) || k.b_stride % 8 || k.c_stride % 8 || !aligned16(k.b) || !aligned16(k.c)) return false;
    }
    return true;
}

int launch_linear_tc(const LinearCall& call, bool states, cudaStream_t stream) {
    lt::Plan plan{};
    lt::Maps maps{};
    plan.call = call;
    struct Known { const void* base; long long stride; int heads, dim; } known[4];
    int count = 0, rc = MKDA_OK;
    auto map = [&](const void* base, long long stride, int per, int dim) {
        const int heads = call.HV / per;
        for (int i = 0; i < count; ++i)
            if (known[i].base == base && known[i].stride == stride && known[i].heads == heads && known[i].dim == dim) return i;
        if (rc == MKDA_OK) rc = make_heads_map(&maps.row[count], base, call.S.TT, heads, dim, stride, "linear");
        known[count] = {base, stride, heads, dim};
        return count++;
    };
    for (int i = 0; i < call.kinds; ++i) {
        const LinearKind& k = call.kind[i];
        plan.map_a[i] = k.a ? map(k.a, k.a_stride, k.a_per, k.M) : 0;
        plan.map_b[i] = map(k.b, k.b_stride, k.b_per, k.M);
        plan.map_c[i] = map(k.c, k.c_stride, k.c_per, k.V);
    }
    if (rc != MKDA_OK) return rc;
    plan.items = (long long)call.S.N * (call.S.seg ? call.S.segs : 1) * call.HV * call.kinds;
    auto* kern = states ? lt::linear_tc_kernel<true> : lt::linear_tc_kernel<false>;
    rc = ensure_smem(reinterpret_cast<const void*>(kern), lt::SMEM, "linear");
    if (rc != MKDA_OK) return rc;
    launch(kern, dim3((unsigned)std::min<long long>(plan.items, sm_count())), lt::THREADS, lt::SMEM, stream, plan, maps);
    return check_launch("linear");
}
int linear_tc_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, umma::g_timeout_flag, sizeof(unsigned int)) == cudaSuccess ? 0 : -1; }
int linear_tc_status_clear() {
    const unsigned int zero = 0;
    return cudaMemcpyToSymbol(umma::g_timeout_flag, &zero, sizeof(zero)) == cudaSuccess ? 0 : -1;
}

}  // namespace mkda
