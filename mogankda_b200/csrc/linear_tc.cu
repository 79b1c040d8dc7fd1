// Linear attention with a decay for each head (linear.cuh) in bf16 on the Blackwell tensor cores.
//
// A block (one per SM) carries parts of sequences and v-heads one after the other, 128 tokens at a time.  With the rows of a, b and c in shared memory (tiled copies, 128-byte
// swizzle) a stretch is four products with fp32 accumulators in tensor memory:
//   P0 = a b^T                       pairs; the weights lam^|i - j| and the mask are applied to the accumulator, and P leaves as bf16 hi + lo, the left operand of P c
//   O  = a M                         M: the state in front of the stretch as hi + lo in shared memory; lam^(i + 1) is applied to the accumulator's rows
//   O += P c
//   X = (f c)^T b                    what goes into the state, f[j] = lam^(L - 1 - j); f c is split in three parts, so that the state, fp32 in registers, is exact to 32 bits
// a, b and c are exact in bf16.  Two halves (2^-16) are enough where the result is rounded to bf16, one would show: P and M in one bf16 each are as far off as the result's own rounding.
//
// Roles, joined by mbarriers: a warp that fetches rows into a ring of five tiles, one that issues products, and four warps each for the pairs' weights, for f c, for the state and
// for the output.  Every accumulator row is a lane: token i of P0 and O, channel of c of X and of the state M^T.
//
// Bound by HBM where there are enough parts: 128 KB per stretch, 3 us of an SM's share; products take 8 x 516 cycles = 2.2 us, and each group of warps less than that.
#include <algorithm>
#include <type_traits>

#include "host.h"
#include "linear.cuh"
#include "umma.cuh"

namespace mkda {
namespace lt {

using umma::mbar_wait;
using umma::signal_tmem;
using umma::wait_mma;

constexpr int C = 128, TILE = 32768, SLOTS = 5, THREADS = 1024;
constexpr int WARP_PAIRS = 0, WARP_FACTORS = 8, WARP_STATE = 16, WARP_OUT = 20, WARP_LOAD = 28, WARP_MMA = 29;
constexpr int P = 0, O = 128, X = 256, F = 384;            // tensor-memory columns: pairs, output, what goes into the state, f c (two buffers of a quarter: 3 x 16 columns each)
// Registers: a thread of the state has 128 values of it.
constexpr int LAUNCH_REGS = 64, WORK_REGS = 48, STATE_REGS = 160, ISSUE_REGS = 40;
static_assert(6 * WORK_REGS + STATE_REGS + ISSUE_REGS <= 8 * LAUNCH_REGS, "registers of the launch");

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS];
    uint64_t p0_done, p_ready, f_ready[2], f_free[2], s_ready, x_done, in_done, o_scaled, o_done, o_free;
    uint32_t tmem;
    // of the current part's head, a copy for each group of warps that reads it: scale lam^n and lam^(31 - e) (backwards lam^e); f; lam^n times the scale
    __align__(16) float pair[C], column[32], factor[C], row[C + 4];
};
constexpr int SMEM = 2 * TILE + SLOTS * TILE + (int)sizeof(Shared);
static_assert(SMEM <= 232448, "shared memory of one block");

struct Maps { CUtensorMap row[4]; };                       // rows of a head, boxes of 64 channels x 128 tokens
struct Plan {
    LinearCall call;
    int map_a[3], map_b[3], map_c[3];                      // per kind
    int wide[3];                                           // bf16 rows of the output leave in pieces of 32 bytes
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
__device__ __forceinline__ void group_sync(int barrier) { asm volatile("bar.sync %0, 256;" :: "r"(barrier) : "memory"); }
// A pair of values as bf16 pairs: hi, and what is left of them, two rounded parts in all
__device__ __forceinline__ uint32_t take_bf16(f32x2& v) {          // hi; v becomes the rest, exactly
    float a, b;
    unpack2(v, a, b);
    const uint32_t h = umma::pack_bf16x2(a, b);
    v = fma2(pack2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)), both(-1.f), v);
    return h;
}
__device__ __forceinline__ uint32_t as_bf16(f32x2 v) {
    float a, b;
    unpack2(v, a, b);
    return umma::pack_bf16x2(a, b);
}
// Four 8 x 8 blocks of 16-bit values, transposed: lane t gets elements (2 (t % 4), t / 4) and (2 (t % 4) + 1, t / 4) of each; lane t gives the address of row t % 8 of block t / 8
__device__ __forceinline__ void load_transposed(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 lanes x 16 columns: lane t of the warp gives column 4 i + t % 4 of rows t / 4 (v[2 i]) and 8 + t / 4 (v[2 i + 1])
__device__ __forceinline__ void tmem_st_16x16(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
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
        for (uint64_t* b : {&sh.p_ready, &sh.f_ready[0], &sh.f_ready[1], &sh.o_scaled, &sh.o_free}) umma::mbar_init(b, 8);
        umma::mbar_init(&sh.s_ready, 4);
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

    if (warp >= WARP_LOAD) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(ISSUE_REGS));
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
                // FULL: 128 channels in all heads, every loop unrolled; the address of a tile passes through an empty statement, or descriptors are kept over the loop and spilled
                auto stretch = [&](auto full, int ms, int vn, bool from_zero) {
                    constexpr bool FULL = decltype(full)::value;
                    const uint32_t ta = n * PER, tb = ta + (STATES ? 0 : 1), tc = tb + 1, par = n & 1;
                    const uint32_t id_p0 = umma::idesc_bf16(128, C), id_in = umma::idesc_bf16(128, FULL ? C : vn), id_pc = umma::idesc_bf16(128, FULL ? C : vn, 0, 1),
                                   id_x = umma::idesc_bf16(128, FULL ? C : ms * 16, 0, 1);
                    auto k_major = [&](uint32_t addr) {
                        asm volatile("" : "+r"(addr));
                        return umma::make_desc(addr);
                    };
                    auto mn_major = [&](uint32_t addr) {
                        asm volatile("" : "+r"(addr));
                        return umma::make_desc(addr, TILE / 2 / 16);
                    };
                    auto k_step = [](int ks) { return (uint64_t)((ks >> 2) * (TILE / 2 / 16) + (ks & 3) * 2); };
                    auto mn_step = [](int ks) { return (uint64_t)(ks * 128); };
                    const uint32_t ring_at = umma::smem_u32(ring), state_at = umma::smem_u32(state_hi);
                    if (!STATES) mbar_wait(&sh.full[slot_of(ta)], parity_of(ta));
                    mbar_wait(&sh.full[slot_of(tb)], parity_of(tb));
                    if (!STATES) {
                        const uint64_t ad = k_major(ring_at + slot_of(ta) * TILE), bd = k_major(ring_at + slot_of(tb) * TILE);
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            if (FULL || ks < ms) umma::mma_bf16(tmem + P, ad + k_step(ks), bd + k_step(ks), id_p0, ks != 0);
                        umma::commit(&sh.p0_done);
                    }
                    wait_mma(&sh.s_ready, par);
                    const uint64_t bm = mn_major(ring_at + slot_of(tb) * TILE);
                    auto into_state = [&](int q) {         // 32 tokens: the smallest of the three parts of f c first
                        wait_mma(&sh.f_ready[q & 1], (2 * n + (q >> 1)) & 1);
#pragma unroll
                        for (int part = 2; part >= 0; --part)
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks)
                                umma::mma_bf16_ta(tmem + X, tmem + F + 64 * (q & 1) + 16 * part + 8 * ks, bm + mn_step(2 * q + ks), id_x, q + ks != 0 || part != 2);
                        umma::commit(&sh.f_free[q & 1]);
                    };
                    // The first half of X lies in front of the product with the state, which waits for the last stretch's output to be read; the second half's parts of f c are made beside it
                    into_state(0);
                    into_state(1);
                    if (!STATES) {
                        if (n) wait_mma(&sh.o_free, par ^ 1u);
                        if (!from_zero) {
                            const uint64_t ad = k_major(ring_at + slot_of(ta) * TILE), mh = k_major(state_at), ml = k_major(state_at + TILE);
#pragma unroll
                            for (int ks = 0; ks < 8; ++ks)
                                if (FULL || ks < ms) {
                                    umma::mma_bf16_fill(tmem + O, ad + k_step(ks), ml + k_step(ks), id_in, ks != 0);
                                    umma::mma_bf16_lastuse(tmem + O, ad + k_step(ks), mh + k_step(ks), id_in, 1u);
                                }
                        }
                        umma::commit(&sh.in_done);
                        umma::commit(&sh.empty[slot_of(ta)]);
                    }
                    into_state(2);
                    into_state(3);
                    umma::commit(&sh.x_done);
                    umma::commit(&sh.empty[slot_of(tb)]);
                    if (!STATES) {
                        wait_mma(&sh.p_ready, par);
                        wait_mma(&sh.o_scaled, par);
                        mbar_wait(&sh.full[slot_of(tc)], parity_of(tc));
                        const uint64_t cd = mn_major(ring_at + slot_of(tc) * TILE);
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t at = tmem + P + 16 * ks;
                            umma::mma_bf16_ta(tmem + O, at + 8, cd + mn_step(ks), id_pc, ks != 0 || !from_zero);
                            umma::mma_bf16_ta(tmem + O, at, cd + mn_step(ks), id_pc, 1u);
                        }
                        umma::commit(&sh.o_done);
                    }
                    umma::commit(&sh.empty[slot_of(tc)]);
                };
                for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart&, int chunks) {
                    const int ms = (k.M + 15) / 16, vn = (k.V + 15) / 16 * 16;
                    const bool zero = entering(call, k, it, STATES) == nullptr;
                    if (ms == 8 && vn == C) {
                        for (int t = 0; t < chunks; ++t, ++n) stretch(std::true_type(), ms, vn, zero && t == 0);
                    } else {
                        for (int t = 0; t < chunks; ++t, ++n) stretch(std::false_type(), ms, vn, zero && t == 0);
                    }
                });
                if (n) mbar_wait(&sh.empty[slot_of(n * PER - 1)], parity_of(n * PER - 1));      // the last arrival of a product
            }
            __syncwarp();
        }
    } else if (warp < WARP_FACTORS) {
        // ---- pairs: row i = this lane's token, half of the columns.  Off the diagonal the weight is a factor of the row times one of the column, neither above 1
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(WORK_REGS));
        if (!STATES) {
            uint32_t n = 0;
            const int w = warp & 3, half = warp >> 2, i = 32 * w + lane;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                const float gamma = call.log_decay[it.h];
                group_sync(1);
                if (half == 0) sh.pair[i] = decay_power(gamma, i) * k.pair_scale;
                else if (i < 32) sh.column[i] = decay_power(gamma, k.back ? i : 31 - i);
                group_sync(1);
                for (int t = 0; t < chunks; ++t, ++n) {
                    const int len = min(C, part.len - first_of(k, chunks, t));
                    wait_mma(&sh.p0_done, n & 1);
#pragma unroll 1
                    for (int j0 = 64 * half; j0 < 64 * half + 64; j0 += 16) {      // 16 columns leave as 8 of hi and 8 of lo in their place
                        const uint32_t at = umma::tmem_addr(tmem, w, P + j0);
                        const int blk = j0 >> 5;
                        if (k.back ? blk < w || j0 >= len : blk > w) {
                            const uint32_t none[16] = {};
                            umma::tmem_st16(at, none);
                            continue;
                        }
                        float v[16];
                        umma::tmem_ld16(at, v);
                        if (blk == w) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const int d = k.back ? j0 + e - i : i - j0 - e;
                                v[e] = d >= 0 ? v[e] * sh.pair[max(d, 0)] : 0.f;
                            }
                        } else {
                            const f32x2 r = both(sh.pair[k.back ? 32 * blk - i : i - 32 * blk - 31]);
                            const float* column = sh.column + (j0 & 16);
#pragma unroll
                            for (int e = 0; e < 16; e += 4) {
                                const float4 c = *reinterpret_cast<const float4*>(column + e);
                                unpack2(mul2(pack2(v[e], v[e + 1]), mul2(r, pack2(c.x, c.y))), v[e], v[e + 1]);
                                unpack2(mul2(pack2(v[e + 2], v[e + 3]), mul2(r, pack2(c.z, c.w))), v[e + 2], v[e + 3]);
                            }
                        }
                        if (k.back && j0 + 16 > len) {     // columns behind the part's end
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (j0 + e >= len) v[e] = 0.f;
                        }
                        uint32_t h[8], l[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            f32x2 x = pack2(v[2 * e], v[2 * e + 1]);
                            h[e] = take_bf16(x);
                            l[e] = as_bf16(x);
                        }
                        umma::tmem_st8(at, h);
                        umma::tmem_st8(at + 8, l);
                    }
                    umma::tmem_wait_st();
                    signal_tmem(&sh.p_ready, lane);
                }
            });
        }
    } else if (warp < WARP_STATE) {
        // ---- f c, transposed: row = channel of c, 16 of them a warp.  Blocks of 8 tokens x 8 channels come transposed out of shared memory, in the layout that 16 rows of tensor
        // memory take
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(WORK_REGS));
        uint32_t n = 0;
        const int me = tid - 32 * WARP_FACTORS, w = warp & 3, half = (warp - WARP_FACTORS) >> 2;
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            const float gamma = call.log_decay[it.h];
            int factors_of = -1;                           // tokens that the table is for
            for (int t = 0; t < chunks; ++t, ++n) {
                const int len = min(C, part.len - first_of(k, chunks, t));
                const uint32_t tb = n * PER + (STATES ? 0 : 1), tc = tb + 1;
                uint8_t* const c = ring + slot_of(tc) * TILE;
                if (len != factors_of) {
                    group_sync(2);
                    if (me < C) sh.factor[me] = me < len ? decay_power(gamma, k.back ? me + 1 : len - 1 - me) * k.in_scale : 0.f;
                    factors_of = len;
                    group_sync(2);
                }
                mbar_wait(&sh.full[slot_of(tc)], parity_of(tc));
                if (len < C) {                             // rows behind the part's end belong to somebody else: 0 times what is not finite is not 0
                    uint8_t* const b = ring + slot_of(tb) * TILE;
                    mbar_wait(&sh.full[slot_of(tb)], parity_of(tb));
                    for (int e = me; e < (C - len) * 16; e += 256) {
                        const uint32_t off = umma::tile_chunk_offset(128, len + (e >> 4), e & 15);
                        *reinterpret_cast<uint4*>(b + off) = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(c + off) = make_uint4(0, 0, 0, 0);
                    }
                    umma::fence_async_smem();
                    group_sync(2);
                    __syncwarp();
                }
                const uint32_t rows = umma::smem_u32(c);
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    const uint32_t use = 2 * n + (q >> 1);         // of this buffer
                    uint32_t part_[3][8];
#pragma unroll
                    for (int g2 = 0; g2 < 2; ++g2) {       // 16 tokens: blocks (tokens 0..7, channels 0..7), (0..7, 8..15), (8..15, 0..7), (8..15, 8..15)
                        uint32_t r[4];
                        const int j = 32 * q + 16 * g2 + ((lane >> 4) << 3) + (lane & 7), k8 = (32 * w + 16 * half) / 8 + ((lane >> 3) & 1);
                        load_transposed(rows + umma::tile_chunk_offset(128, j, k8), r);
#pragma unroll
                        for (int m = 0; m < 4; ++m) {      // of this lane's two tokens in each 8
                            const f32x2 f = *reinterpret_cast<const f32x2*>(sh.factor + 32 * q + 16 * g2 + 8 * (m >> 1) + 2 * (lane & 3));
                            f32x2 x = mul2(pack2(__uint_as_float(r[m] << 16), __uint_as_float(r[m] & 0xffff0000u)), f);
                            const int to = 2 * (2 * g2 + (m >> 1)) + (m & 1);
                            part_[0][to] = take_bf16(x);
                            part_[1][to] = take_bf16(x);
                            part_[2][to] = as_bf16(x);
                        }
                    }
                    if (use) wait_mma(&sh.f_free[q & 1], (use - 1) & 1);
#pragma unroll
                    for (int p = 0; p < 3; ++p) tmem_st_16x16(umma::tmem_addr(tmem, w, F + 64 * (q & 1) + 16 * p) + ((uint32_t)(16 * half) << 16), part_[p]);
                    umma::tmem_wait_st();
                    signal_tmem(&sh.f_ready[q & 1], lane);
                }
            }
        });
    } else if (warp < WARP_OUT) {
        // ---- the state: row = this lane's channel of c, columns the channels of b, in registers.  What a stretch adds comes from an accumulator of its own: the tensor cores cut off what
        // does not fit into 32 bits, and over a long sequence's products that is an error of one sign (2.5e-6 of the state behind 32 k tokens, this way 0.4e-6).
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(STATE_REGS));
        uint32_t n = 0;
        const int ch = tid - 32 * WARP_STATE;
        f32x2 s[64];
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            const float* in = entering(call, k, it, STATES);
            const size_t size = (size_t)k.M * k.V;
            float* out = STATES ? k.parts + ((size_t)(it.n * call.S.segs + it.part + (k.back ? -1 : 1)) * call.HV + it.h) * size
                                : k.last && part.leaves_last ? k.last + ((size_t)it.n * call.HV + it.h) * size : nullptr;
            const float gamma = call.log_decay[it.h], whole = decay_power(gamma, C), rest = decay_power(gamma, part.len % C);
            const size_t first = k.transposed ? (size_t)ch * k.M : ch, step = k.transposed ? 1 : k.V;
#pragma unroll
            for (int m = 0; m < 128; m += 2) {
                float v[2] = {0.f, 0.f};
                if (in && ch < k.V) {
                    if (m < k.M) v[0] = in[first + m * step];
                    if (m + 1 < k.M) v[1] = in[first + (m + 1) * step];
                }
                s[m / 2] = pack2(v[0], v[1]);
            }
            __syncwarp();
            for (int t = 0; t <= chunks; ++t) {
                f32x2 f = both(1.f);
                if (t) {
                    const bool short_one = part.len - first_of(k, chunks, t - 1) < C;
                    f = both(short_one ? rest : whole);
                    wait_mma(&sh.x_done, (n - 1) & 1);
                }
                const bool store = !STATES && t < chunks && (t || in);
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    if (16 * g >= k.M) break;
                    if (t) {
                        float x[16];
                        umma::tmem_ld16(umma::tmem_addr(tmem, warp, X + 16 * g), x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[8 * g + e] = fma2(s[8 * g + e], f, pack2(x[2 * e], x[2 * e + 1]));
                    }
                    if (store) {
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            uint32_t h[4], l[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                f32x2 x = s[8 * g + e + j];
                                h[j] = take_bf16(x);
                                l[j] = as_bf16(x);
                            }
                            uint8_t* const to = state_hi + umma::tile_chunk_offset(128, ch, 2 * g + e / 4);
                            *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                            *reinterpret_cast<uint4*>(to + TILE) = make_uint4(l[0], l[1], l[2], l[3]);
                        }
                    }
                }
                if (t == chunks) break;
                umma::signal(&sh.s_ready, lane);
                ++n;
            }
            if (!out || ch >= k.V) return;
#pragma unroll
            for (int m = 0; m < 128; m += 2) {
                float a, b;
                unpack2(s[m / 2], a, b);
                if (m < k.M) out[first + m * step] = a;
                if (m + 1 < k.M) out[first + (m + 1) * step] = b;
            }
        });
    } else {
        // ---- the output: row i = this lane's token, half of the channels
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(WORK_REGS));
        if (!STATES) {
            uint32_t n = 0;
            const int w = warp & 3, half = (warp - WARP_OUT) >> 2, i = 32 * w + lane, m_first = 64 * half;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                const float gamma = call.log_decay[it.h];
                group_sync(3);
                if (half == 0) sh.row[i] = decay_power(gamma, i) * k.state_scale;
                else if (i == 0) sh.row[C] = decay_power(gamma, C) * k.state_scale;
                group_sync(3);
                const bool zero = entering(call, k, it, STATES) == nullptr, wide = plan.wide[it.kind], fp32 = k.out_dtype == MKDA_F32;
                const int m_end = min(k.V, m_first + 64);
                for (int t = 0; t < chunks; ++t, ++n) {
                    const int c0 = first_of(k, chunks, t), len = min(C, part.len - c0);
                    wait_mma(&sh.in_done, n & 1);
                    if (!zero || t) {
                        const f32x2 f = both(sh.row[k.back ? max(len - 1 - i, 0) : i + 1]);
#pragma unroll 1
                        for (int m0 = m_first; m0 < m_end; m0 += 16) {
                            const uint32_t at = umma::tmem_addr(tmem, w, O + m0);
                            float v[16];
                            umma::tmem_ld16(at, v);
#pragma unroll
                            for (int g = 0; g < 16; g += 8) {
                                f32x2 x[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) x[e] = mul2(pack2(v[g + 2 * e], v[g + 2 * e + 1]), f);
                                umma::tmem_st8(at + g, x);
                            }
                        }
                        umma::tmem_wait_st();
                    }
                    signal_tmem(&sh.o_scaled, lane);
                    wait_mma(&sh.o_done, n & 1);
                    const size_t row = ((size_t)(part.start + c0 + i) * call.HV + it.h) * k.V;
#pragma unroll 1
                    for (int m0 = m_first; m0 < m_first + 64; m0 += 16) {
                        float v[16];
                        __syncwarp();
                        if (m0 < m_end) umma::tmem_ld16(umma::tmem_addr(tmem, w, O + m0), v);
                        if (m0 == m_first + 48) signal_tmem(&sh.o_free, lane);
                        if (i >= len || m0 >= m_end) continue;
                        if (fp32) {
                            float* to = static_cast<float*>(k.out) + row + m0;
#pragma unroll
                            for (int e = 0; e < 16; e += 4)
                                if (m0 + e < m_end) *reinterpret_cast<float4*>(to + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                        } else {
                            uint16_t* to = static_cast<uint16_t*>(k.out) + row + m0;
                            uint32_t u[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) u[e] = umma::pack_bf16x2(v[2 * e], v[2 * e + 1]);
                            if (wide) {
                                st32b(to, u);
                            } else {
                                *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
                                if (m0 + 8 < m_end) *reinterpret_cast<uint4*>(to + 8) = make_uint4(u[4], u[5], u[6], u[7]);
                            }
                        }
                    }
                    __syncwarp();
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
        plan.wide[i] = k.V % 16 == 0 && !any_misaligned32(k.out);
    }
    if (rc != MKDA_OK) return rc;
    plan.items = (long long)call.S.N * (call.S.seg ? call.S.segs : 1) * call.HV * call.kinds;
    auto* kern = states ? lt::linear_tc_kernel<true> : lt::linear_tc_kernel<false>;
    rc = ensure_smem(reinterpret_cast<const void*>(kern), lt::SMEM, "linear");
    if (rc != MKDA_OK) return rc;
    static const int regs = std::min(kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<true>)), kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<false>)));
    if (regs < lt::LAUNCH_REGS) return set_error(MKDA_ERR_LAUNCH, "linear: built with fewer registers than its warps redistribute");
    launch(kern, dim3((unsigned)std::min<long long>(plan.items, sm_count())), lt::THREADS, lt::SMEM, stream, plan, maps);
    return check_launch("linear");
}
int linear_tc_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, umma::g_timeout_flag, sizeof(unsigned int)) == cudaSuccess ? 0 : -1; }
int linear_tc_status_clear() {
    const unsigned int zero = 0;
    return cudaMemcpyToSymbol(umma::g_timeout_flag, &zero, sizeof(zero)) == cudaSuccess ? 0 : -1;
}

}  // namespace mkda
