// Linear attention with a decay for each head (linear.cuh) in bf16 and fp16 on the Blackwell tensor cores.
//
// A block (one per SM) carries parts of sequences and v-heads one after the other, 128 tokens at a time.  With the rows of a, b and c in shared memory (tiled copies, 128-byte
// swizzle) a stretch is four products with fp32 accumulators in tensor memory:
//   P0 = a b^T                       pairs; the weights lam^|i - j| and the mask are applied to the accumulator, and P leaves as hi + lo in 16 bits, the left operand of P c
//   O  = a M                         M: the state in front of the stretch as hi + lo in shared memory; lam^(i + 1) is applied to the accumulator's rows
//   O += P c
//   X = (f c)^T b                    what goes into the state, f[j] = lam^(L - 1 - j); f c is split in three parts, so that the state, fp32 in registers, is exact to 32 bits; in two
//                                  where no state leaves, and in fp16
// a, b and c are exact as they are.  Two halves (2^-16) are enough where the result is rounded to bf16, one would show: P and M in one bf16 each are as far off as the result's own rounding.
//
// Roles, joined by mbarriers: a warp that fetches rows into a ring of five tiles, one that issues products, and eight warps each for the pairs' weights and the output, for f c and for
// the state.  Every accumulator row is a lane: token i of P0 and O, channel of c of X and of the state M^T.
//
// Bound by the hand-overs between the products and, in runs that last, by 1000 W: a stretch takes 3.3 us where few SMs are busy, 4.2 (7 k cycles) where all are.  HBM alone would
// take 2.9 (128 KB), the products 7 or 8 x 516 cycles, the warps' arithmetic less.  16384 tokens x 148 heads 587 us, 0.64 of HBM; fp16 4 x 2048 x 16 heads with the backward pass 271 us, where
// the fp32 units (linear.cu) take 2890.
#include <algorithm>
#include <cfloat>

#include "host.h"
#include "linear.cuh"
#include "umma.cuh"

namespace mkda {
namespace lt {

using umma::signal_tmem;

constexpr int C = 128, TILE = 32768, SLOTS = 5, THREADS = 896;
constexpr int WARP_FACTORS = 8, WARP_STATE = 16, WARP_LOAD = 24, WARP_MMA = 25, WARP_STORE = 26;
constexpr int P = 0, O = 128, X = 256, F = 384;            // tensor-memory columns: pairs, output, what goes into the state, f c (two buffers of a quarter: 3 x 16 columns each)
// Registers: a thread of the state has 64 values of it.
constexpr int LAUNCH_REGS = 72, FACTOR_REGS = 48, STATE_REGS = 104, ISSUE_REGS = 56;
static_assert(2 * (LAUNCH_REGS + FACTOR_REGS + STATE_REGS) + ISSUE_REGS <= 7 * LAUNCH_REGS, "registers of the launch");

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS];
    uint64_t p0_done, p_ready, f_ready[2], f_free[2], s_ready, x_done, in_done, o_scaled, o_done, o_free, o_staged[2], e_ready[2];
    // of even and odd stretches: which 16 channels of c have values that are not finite (by the warp that made f c of them), and (edge) the first of them in each channel in the order of the walk
    uint8_t bad[2][8];
    // of the current part's head, a copy for each group of warps that reads it: f, weights of the pairs by j - i + 128 (0 where a pair does not count), lam^n times the scale
    float factor[C], pair[2 * C], row[C + 1];
    uint32_t tmem;
    // fp16: powers of two that the state and the channels of f c are scaled by, of even and odd stretches, and the largest exponents that warps find for the state and for the rows of the
    // pairs (of half of the columns each)
    float s_scale[2];
    uint8_t f_scale[2][C], s_top[8], p_top[2][C];
    uint8_t edge[2][C];
};
constexpr int SMEM = 2 * TILE + SLOTS * TILE + (int)sizeof(Shared);
static_assert(SMEM <= 232448, "shared memory of one block");

struct Maps { CUtensorMap row[4], out[3]; };               // rows of a head, boxes of 64 channels x 128 tokens; out per kind
struct Plan {
    LinearCall call;
    int map_a[3], map_b[3], map_c[3];                      // per kind
    uint32_t items;
};

// Waits for the phase of `bar` with the given parity, at most `tries` times a microsecond; on expiry the status word is set, and the waits behind it are short.  umma::mbar_wait is longer
// by a reading of the clock and a loop: the roles' code together is about as large as the instruction cache, and each runs through its own once a stretch.
__device__ __forceinline__ void mbar_wait(uint64_t* bar, uint32_t parity, uint32_t& tries) {
    for (uint32_t left = tries;; --left) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(umma::smem_u32(bar)), "r"(parity), "r"(1000u) : "memory");
        if (ok) break;
        if (left == 0) {
            atomicExch(&umma::g_timeout_flag, 1u);
            tries = 32;
            break;
        }
    }
}
__device__ __forceinline__ void wait_mma(uint64_t* bar, uint32_t parity, uint32_t& tries) {
    mbar_wait(bar, parity, tries);
    umma::fence_after_sync();
}

struct Item { int kind, h, n, part; };
__device__ __forceinline__ Item item_of(const LinearCall& call, uint32_t w) {
    Item it;
    const uint32_t kinds = call.kinds, heads = call.HV, segs = call.S.seg ? call.S.segs : 1;
    it.kind = (int)(w % kinds);
    w /= kinds;
    it.h = (int)(w % heads);
    w /= heads;
    it.part = (int)(w % segs);
    const int n = (int)(w / segs);
    it.n = call.S.order ? call.S.order[n] : n;
    return it;
}
// Calls body(kind, item, part, stretches) for every item of this block that has something to do, the same ones in every role.  The longest sequences come first; every other round of
// the blocks runs the other way, so that who got the longest of one gets the shortest of the next (11 documents of 204 to 1712 tokens x 48: 28 stretches for the busiest block, 24 so).
template <bool STATES, typename Body>
__device__ __forceinline__ void for_items(const Plan& plan, Body body) {
#pragma unroll 1
    for (uint32_t round = 0; round * gridDim.x < plan.items; ++round) {      // items + blocks stay below 2^32
        const uint32_t w = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (w >= plan.items) continue;
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
// A pair of values in 16 bits, and back
template <bool HALF>
__device__ __forceinline__ uint32_t as_part(f32x2 v) {
    float a, b;
    unpack2(v, a, b);
    return HALF ? pack16<MKDA_F16>(a, b) : umma::pack_bf16x2(a, b);
}
template <bool HALF>
__device__ __forceinline__ f32x2 of_part(uint32_t h) {
    if constexpr (HALF) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        return pack2(f.x, f.y);
    } else {
        return pack2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
    }
}
// hi; v becomes the rest, exactly
template <bool HALF>
__device__ __forceinline__ uint32_t take_part(f32x2& v) {
    const uint32_t h = as_part<HALF>(v);
    v = fma2(of_part<HALF>(h), both(-1.f), v);
    return h;
}
// The power of two that brings a value of this exponent to [2^(to - 1), 2^to)
__device__ __forceinline__ int exponent_of(float v) { return (int)(__float_as_uint(v) >> 23) & 255; }
__device__ __forceinline__ float scale_of(int exponent, int to) { return __uint_as_float((uint32_t)min(max(to - 1 + 254 - exponent, 4), 250) << 23); }
// ... `top`; 1 for 0
__device__ __forceinline__ float scale_to(float top, int to) { return top == 0.f ? 1.f : scale_of(exponent_of(top), to); }
__device__ __forceinline__ float warp_top(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ int top_of(const uint8_t (&tops)[8]) {
    int v = tops[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = max(v, (int)tops[i]);
    return v;
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

__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int head, int token, const void* src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
                 :: "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(umma::smem_u32(src)) : "memory");
}
// z stays 0 as long as the pairs of 16-bit values are finite
template <bool HALF>
__device__ __forceinline__ void note_not_finite(uint32_t& z, uint32_t v) {
    if constexpr (HALF) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(z) : "r"(v), "r"(0u));
    else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(z) : "r"(v), "r"(0u));
}
// Whether a state of 32 bits leaves: f c then has three parts, else two, as the state that only meets bf16 rows needs no more
template <bool STATES>
__device__ __forceinline__ bool exact_state(const LinearKind& k) { return STATES || k.last; }

// STATES: nothing but what the parts of cut sequences make of a zero state
// HALF: fp16 rows.  Their products are exact as those of bf16 are, but pair weights, f c and states leave fp16's range where bf16 has fp32's: each is scaled by a power of two that
// keeps it below 2^15, and its two parts are off by 2^-22 of the value or 2^-39 of the largest that shares the power of two.  That is, for pairs, of one row, found from its accumulator:
// from the stretch's largest q and k, one large token took the bits of all others, also of those in front of it.  For f c it is one channel, which is one of the state and of the results,
// for the state its largest value.
template <bool STATES, bool HALF>
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
    if (tid < 2) *reinterpret_cast<unsigned long long*>(sh.bad[tid]) = 0;
    if (tid == 0) {
        for (int i = 0; i < SLOTS; ++i) { umma::mbar_init(&sh.full[i], 1); umma::mbar_init(&sh.empty[i], 1); }
        for (uint64_t* b : {&sh.p0_done, &sh.f_free[0], &sh.f_free[1], &sh.x_done, &sh.in_done, &sh.o_done}) umma::mbar_init(b, 1);
        for (uint64_t* b : {&sh.p_ready, &sh.f_ready[0], &sh.f_ready[1], &sh.s_ready, &sh.o_scaled, &sh.o_free, &sh.o_staged[0], &sh.o_staged[1], &sh.e_ready[0], &sh.e_ready[1]}) umma::mbar_init(b, 8);
        umma::fence_barrier_init();
    }
    follow_stream();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = sh.tmem;
    uint32_t tries = 1u << 17;
    const LinearCall& call = plan.call;
    constexpr int PER = STATES ? 2 : 3;                    // tiles of a stretch: (a,) b, c
    auto slot_of = [](uint32_t tile) { return tile % SLOTS; };
    auto parity_of = [](uint32_t tile) { return (tile / SLOTS) & 1u; };
    // where rows of the output lie before they leave, in blocks of 128 bytes of each row: bf16 in the place of b, fp32 from channel 64 on in that of c
    auto staging = [&](uint32_t n, bool fp32, int channel) {
        return fp32 ? ring + slot_of(n * PER + 1 + (channel >> 6)) * TILE + ((channel >> 5) & 1) * (TILE / 2) : ring + slot_of(n * PER + 1) * TILE + (channel >> 6) * (TILE / 2);
    };

    if (warp >= WARP_LOAD) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(ISSUE_REGS));
        if (warp == WARP_LOAD) {
            if (umma::elect_one()) {
                uint32_t tile = 0;
                for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                    const int idx = it.kind;
#pragma unroll 1
                    for (int t = 0; t < chunks; ++t) {
                        const int tok = part.start + first_of(k, chunks, t);
                        auto fetch = [&](int map, int head) {
                            const uint32_t s = slot_of(tile);
                            if (tile >= SLOTS) mbar_wait(&sh.empty[s], parity_of(tile) ^ 1u, tries);
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
                // Short loops: a product takes 65 cycles and an iteration less, while unrolled code of this and the other roles pushes each other out of the instruction caches
                const uint64_t k_desc = umma::make_desc(0), mn_desc = umma::make_desc(0, TILE / 2 / 16);
                const uint32_t ring_at = umma::smem_u32(ring) >> 4, state_at = umma::smem_u32(state_hi) >> 4;
                auto tile_at = [&](uint32_t tile) { return ring_at + slot_of(tile) * (TILE / 16); };
                auto k_step = [](int ks) { return (uint32_t)((ks >> 2) * (TILE / 2 / 16) + (ks & 3) * 2); };
                for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart&, int chunks) {
                    const int ms = (k.M + 15) / 16, vn = (k.V + 15) / 16 * 16;
                    const bool zero = entering(call, k, it, STATES) == nullptr, exact = !HALF && exact_state<STATES>(k), fp32 = k.out_dtype == MKDA_F32;
                    constexpr uint32_t F16 = HALF ? ~(1u << 7 | 1u << 10) : ~0u;         // both operands fp16
                    const uint32_t id_p0 = umma::idesc_bf16(128, C) & F16, id_in = umma::idesc_bf16(128, vn) & F16, id_pc = umma::idesc_bf16(128, vn, 0, 1) & F16,
                                   id_x = umma::idesc_bf16(128, ms * 16, 0, 1) & F16;
#pragma unroll 1
                    for (int t = 0; t < chunks; ++t, ++n) {
                        const uint32_t ta = n * PER, tb = ta + (STATES ? 0 : 1), tc = tb + 1, par = n & 1;
                        const bool from_zero = zero && t == 0;
                        if (!STATES) mbar_wait(&sh.full[slot_of(ta)], parity_of(ta), tries);
                        mbar_wait(&sh.full[slot_of(tb)], parity_of(tb), tries);
                        if (!STATES) {
                            // P0 goes where the last stretch's P is the left operand of a product with another accumulator, and products are ordered among themselves by a common
                            // accumulator only (8192 packed tokens x 16 heads, forward and backward, 171 us, 169 without the wait; 32749 x 32 forward 441 and 440)
                            if (n) wait_mma(&sh.o_done, par ^ 1u, tries);
                            const uint64_t ad = k_desc | tile_at(ta), bd = k_desc | tile_at(tb);
#pragma unroll 1
                            for (int ks = 0; ks < ms; ++ks) umma::mma_bf16(tmem + P, ad + k_step(ks), bd + k_step(ks), id_p0, ks != 0);
                            umma::commit(&sh.p0_done);
                        }
                        wait_mma(&sh.s_ready, par, tries);
                        const uint64_t bm = mn_desc | tile_at(tb);
                        // The first half of X lies in front of the product with the state, which waits for the last stretch's output to be read; the second half's parts of f c are
                        // made beside it
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            if (!STATES && q == 2) {
                                if (n) wait_mma(&sh.o_free, par ^ 1u, tries);
                                if (!from_zero) {
                                    const uint64_t ad = k_desc | tile_at(ta), m = k_desc | state_at;
#pragma unroll 1
                                    for (int ks = 0; ks < ms; ++ks) {
                                        umma::mma_bf16_fill(tmem + O, ad + k_step(ks), m + TILE / 16 + k_step(ks), id_in, ks != 0);
                                        umma::mma_bf16_lastuse(tmem + O, ad + k_step(ks), m + k_step(ks), id_in, 1u);
                                    }
                                }
                                umma::commit(&sh.in_done);
                                umma::commit(&sh.empty[slot_of(ta)]);
                            }
                            wait_mma(&sh.f_ready[q & 1], (2 * n + (q >> 1)) & 1, tries);
#pragma unroll 1
                            for (int ks = 0; ks < 2; ++ks) {       // 16 tokens: the smallest of the three parts of f c first
                                const uint32_t at = tmem + F + 64 * (q & 1) + 8 * ks;
                                const uint64_t bd = bm + 128 * (2 * q + ks);
                                if (exact) umma::mma_bf16_ta(tmem + X, at + 32, bd, id_x, q + ks != 0);
                                umma::mma_bf16_ta(tmem + X, at + 16, bd, id_x, exact || q + ks != 0);
                                umma::mma_bf16_ta(tmem + X, at, bd, id_x, 1u);
                            }
                            umma::commit(&sh.f_free[q & 1]);
                        }
                        umma::commit(&sh.x_done);
                        if (STATES) umma::commit(&sh.empty[slot_of(tb)]);
                        if (!STATES) {
                            wait_mma(&sh.p_ready, par, tries);
                            wait_mma(&sh.o_scaled, par, tries);
                            mbar_wait(&sh.full[slot_of(tc)], parity_of(tc), tries);
                            const uint64_t cd = mn_desc | tile_at(tc);
#pragma unroll 1
                            for (int ks = 0; ks < 8; ++ks) {
                                const uint32_t at = tmem + P + 16 * ks;
                                umma::mma_bf16_ta(tmem + O, at + 8, cd + 128 * ks, id_pc, ks != 0 || !from_zero);
                                umma::mma_bf16_ta(tmem + O, at, cd + 128 * ks, id_pc, 1u);
                            }
                            umma::commit(&sh.o_done);
                        }
                        if (STATES || !fp32) umma::commit(&sh.empty[slot_of(tc)]);
                    }
                });
                if (n) mbar_wait(&sh.empty[slot_of(n * PER - 1)], parity_of(n * PER - 1), tries);      // the last arrival of a product
            }
            __syncwarp();
        } else if (!STATES && warp == WARP_STORE) {
            // The rows of a whole stretch are put down in the place of its b, which the products are through with, and leave as a tiled copy: stored from registers, 32 rows at a time, they
            // kept the load / store units busy for 3000 of 8000 cycles
            if (umma::elect_one()) {
                uint32_t n = 0;
                for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
#pragma unroll 1
                    for (int t = 0; t < chunks; ++t, ++n) {
                        const int c0 = first_of(k, chunks, t);
                        const uint32_t slot = slot_of(n * PER + 1);
                        mbar_wait(&sh.o_staged[n & 1], (n >> 1) & 1, tries);
                        const bool fp32 = k.out_dtype == MKDA_F32;
                        const int box = fp32 ? 32 : 64;
                        if (part.len - c0 >= C) {          // rows behind a short stretch's end are another sequence's
#pragma unroll 1
                            for (int m0 = 0; m0 < k.V; m0 += box) store_box(&maps.out[it.kind], m0, it.h, part.start + c0, staging(n, fp32, m0));
                            umma::bulk_store_commit();
                            umma::bulk_store_wait_read();
                        }
                        umma::arrive(&sh.empty[slot]);
                        if (fp32) umma::arrive(&sh.empty[slot_of(n * PER + 2)]);
                    }
                });
            }
            __syncwarp();
        }
    } else if (warp < WARP_FACTORS) {
        // ---- pairs and output: row i = this lane's token, half of the columns
        if (!STATES) {
            uint32_t n = 0;
            const int w = warp & 3, half = warp >> 2, i = 32 * w + lane, m_first = 64 * half;
            for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
                const float gamma = call.log_decay[it.h];
                group_sync(1);
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    const int away = u ? tid : k.back ? tid - C : C - tid;
                    const float power = away >= 0 && away <= C ? decay_power(gamma, away) : 0.f;
                    if (u == 0) sh.pair[tid] = away < C ? power * k.pair_scale : 0.f;
                    else if (tid <= C) sh.row[tid] = power * k.state_scale;
                }
                group_sync(1);
                const bool zero = entering(call, k, it, STATES) == nullptr, fp32 = k.out_dtype == MKDA_F32;
                const int m_end = min(k.V, m_first + 64);
#pragma unroll 1
                for (int t = 0; t < chunks; ++t, ++n) {
                    const int c0 = first_of(k, chunks, t), len = min(C, part.len - c0);
                    float up = 1.f;                        // fp16: what this row is scaled by
                    wait_mma(&sh.p0_done, n & 1, tries);
#pragma unroll 1
                    for (int pass = HALF ? 0 : 1; pass < 2; ++pass) {      // the first one only looks for the largest of the row
                        float top = 0.f;
#pragma unroll 1
                        for (int j0 = 64 * half; j0 < 64 * half + 64; j0 += 16) {      // 16 columns leave as 8 of hi and 8 of lo in their place
                            const uint32_t at = umma::tmem_addr(tmem, w, P + j0);
                            const int blk = j0 >> 5;
                            if (k.back ? blk < w || j0 >= len : blk > w) {
                                const uint32_t none[16] = {};
                                if (!HALF || pass) umma::tmem_st16(at, none);
                                continue;
                            }
                            float v[16];
                            umma::tmem_ld16(at, v);
                            const float* weight = sh.pair + C + j0 - i;
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[e] = weight[e] == 0.f ? 0.f : v[e] * weight[e];      // what does not count may not be a number
                            if (k.back && j0 + 16 > len) {     // columns behind the part's end
#pragma unroll
                                for (int e = 0; e < 16; ++e)
                                    if (j0 + e >= len) v[e] = 0.f;
                            }
                            if (HALF && !pass) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(fmaf(v[e], 0.f, v[e])));      // finite ones
                                continue;
                            }
                            uint32_t h[8], l[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                f32x2 x = pack2(v[2 * e], v[2 * e + 1]);
                                if (HALF) x = mul2(x, both(up));
                                h[e] = take_part<HALF>(x);
                                l[e] = as_part<HALF>(x);
                            }
                            umma::tmem_st8(at, h);
                            umma::tmem_st8(at + 8, l);
                        }
                        if (HALF && !pass) {               // nobody writes the next stretch's in front of the products of this one, which wait for all rows
                            const int mine = exponent_of(top);
                            sh.p_top[half][i] = (uint8_t)mine;
                            __syncwarp();
                            if (lane == 0) umma::arrive(&sh.e_ready[n & 1]);
                            mbar_wait(&sh.e_ready[n & 1], (n >> 1) & 1, tries);
                            // 2^40 at most, which leaves the state's part of the row room in fp32: what that takes from a pair, 2^-65, is nothing beside fp16's smallest number, 2^-24
                            up = fminf(scale_of(max(mine, (int)sh.p_top[half ^ 1][i]), 15), 0x1p40f);
                            __syncwarp();
                        }
                    }
                    umma::tmem_wait_st();
                    signal_tmem(&sh.p_ready, lane);
                    wait_mma(&sh.in_done, n & 1, tries);
                    if (!zero || t) {
                        float factor = sh.row[k.back ? max(len - 1 - i, 0) : i + 1];
                        if (HALF) {
                            factor *= 1.f / sh.s_scale[n & 1];
                            factor *= up;
                            if (fabsf(factor) > FLT_MAX) factor = copysignf(FLT_MAX, factor);      // 0 times infinity is not 0
                        }
                        const f32x2 f = both(factor);
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
                    wait_mma(&sh.o_done, n & 1, tries);
                    if (*reinterpret_cast<const volatile unsigned long long*>(sh.bad[n & 1])) {      // c had 0 in the place of what is not finite: the rows that it counts in are NaN
                        const int turn = k.back ? C - 1 - i : i;
#pragma unroll 1
                        for (int m0 = m_first; m0 < m_end; m0 += 16) {
                            if (!*reinterpret_cast<const volatile uint8_t*>(&sh.bad[n & 1][(m0 >> 5) + ((m0 >> 4) & 1) * 4])) continue;
                            const uint32_t at = umma::tmem_addr(tmem, w, O + m0);
                            float v[16];
                            umma::tmem_ld16(at, v);
                            uint32_t u[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) u[e] = turn >= sh.edge[n & 1][m0 + e] ? 0x7fffffffu : __float_as_uint(v[e]);
                            umma::tmem_st16(at, u);
                        }
                        umma::tmem_wait_st();
                    }
                    const float down = HALF ? 1.f / up : 1.f;
                    const size_t row = ((size_t)(part.start + c0 + i) * call.HV + it.h) * k.V;
                    if (len == C) {
#pragma unroll 1
                        for (int m0 = m_first; m0 < m_end; m0 += 16) {
                            float v[16];
                            umma::tmem_ld16(umma::tmem_addr(tmem, w, O + m0), v);
                            if (HALF)
#pragma unroll
                                for (int e = 0; e < 16; ++e) v[e] *= down;
                            uint8_t* const to = staging(n, fp32, m0);
                            if (fp32) {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    *reinterpret_cast<float4*>(to + umma::tile_chunk_offset(128, i, ((m0 & 31) >> 2) + e)) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                            } else {
                                uint32_t u[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) u[e] = as_part<HALF>(pack2(v[2 * e], v[2 * e + 1]));
                                *reinterpret_cast<uint4*>(to + umma::tile_chunk_offset(128, i, (m0 & 63) >> 3)) = make_uint4(u[0], u[1], u[2], u[3]);
                                *reinterpret_cast<uint4*>(to + umma::tile_chunk_offset(128, i, ((m0 & 63) >> 3) + 1)) = make_uint4(u[4], u[5], u[6], u[7]);
                            }
                        }
                        signal_tmem(&sh.o_free, lane);
                        umma::signal(&sh.o_staged[n & 1], lane);
                    } else {
#pragma unroll 1
                        for (int m0 = m_first; m0 < m_first + 64; m0 += 16) {
                            float v[16];
                            __syncwarp();
                            if (m0 < m_end) umma::tmem_ld16(umma::tmem_addr(tmem, w, O + m0), v);
                            if (m0 == m_first + 48) {
                                signal_tmem(&sh.o_free, lane);
                                signal_tmem(&sh.o_staged[n & 1], lane);
                            }
                            if (i >= len || m0 >= m_end) continue;
                            if (HALF)
#pragma unroll
                                for (int e = 0; e < 16; ++e) v[e] *= down;
                            if (fp32) {
                                float* to = static_cast<float*>(k.out) + row + m0;
#pragma unroll
                                for (int e = 0; e < 16; e += 4)
                                    if (m0 + e < m_end) *reinterpret_cast<float4*>(to + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                            } else {
                                uint16_t* to = static_cast<uint16_t*>(k.out) + row + m0;
                                uint32_t u[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) u[e] = as_part<HALF>(pack2(v[2 * e], v[2 * e + 1]));
                                *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
                                if (m0 + 8 < m_end) *reinterpret_cast<uint4*>(to + 8) = make_uint4(u[4], u[5], u[6], u[7]);
                            }
                        }
                    }
                    __syncwarp();
                }
            });
        }
    } else if (warp < WARP_STATE) {
        // ---- f c, transposed: row = channel of c, 16 of them a warp.  Blocks of 8 tokens x 8 channels come transposed out of shared memory, in the layout that 16 rows of tensor
        // memory take
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(FACTOR_REGS));
        uint32_t n = 0;
        const int me = tid - 32 * WARP_FACTORS, w = warp & 3, half = (warp - WARP_FACTORS) >> 2;
        uint32_t marked = 0;                               // whether sh.bad has a note of this warp for even and for odd stretches
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            const float gamma = call.log_decay[it.h];
            const bool exact = !HALF && exact_state<STATES>(k);
            int factors_of = -1;                           // tokens that the table is for
#pragma unroll 1
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
                mbar_wait(&sh.full[slot_of(tc)], parity_of(tc), tries);
                if (len < C) {                             // rows behind the part's end belong to somebody else: 0 times what is not finite is not 0
                    uint8_t* const b = ring + slot_of(tb) * TILE;
                    mbar_wait(&sh.full[slot_of(tb)], parity_of(tb), tries);
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
                // 16 tokens: blocks (tokens 0..7, channels 0..7), (0..7, 8..15), (8..15, 0..7), (8..15, 8..15), of each this lane's two tokens; and their f
                auto fetch = [&](int j0, uint32_t (&r)[4]) {
                    const int j = j0 + ((lane >> 4) << 3) + (lane & 7), k8 = (32 * w + 16 * half) / 8 + ((lane >> 3) & 1);
                    load_transposed(rows + umma::tile_chunk_offset(128, j, k8), r);
                };
                auto f_of = [&](int j0, int m) { return *reinterpret_cast<const f32x2*>(sh.factor + j0 + 8 * (m >> 1) + 2 * (lane & 3)); };
                float up[2] = {1.f, 1.f};                  // fp16: what this lane's two channels are scaled by
                if (HALF) {
                    float top[2] = {0.f, 0.f};
#pragma unroll 1
                    for (int j0 = 0; j0 < C; j0 += 16) {
                        uint32_t r[4];
                        fetch(j0, r);
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            float a, b;
                            unpack2(mul2(of_part<HALF>(r[m]), f_of(j0, m)), a, b);
                            top[m & 1] = fmaxf(top[m & 1], fmaxf(fabsf(fmaf(a, 0.f, a)), fabsf(fmaf(b, 0.f, b))));      // finite ones
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        top[m] = fmaxf(top[m], __shfl_xor_sync(0xffffffffu, top[m], 1));
                        top[m] = fmaxf(top[m], __shfl_xor_sync(0xffffffffu, top[m], 2));
                        up[m] = scale_to(top[m], 15);
                        if ((lane & 3) == 0) sh.f_scale[n & 1][32 * w + 16 * half + 8 * m + (lane >> 2)] = (uint8_t)exponent_of(up[m]);
                    }
                }
                uint32_t odd = 0;                          // not 0: a value of this thread is not finite
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    const uint32_t use = 2 * n + (q >> 1);         // of this buffer
                    uint32_t part_[3][8];
#pragma unroll
                    for (int g2 = 0; g2 < 2; ++g2) {
                        uint32_t r[4];
                        fetch(32 * q + 16 * g2, r);
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            if (!STATES) note_not_finite<HALF>(odd, r[m]);
                            f32x2 x = mul2(of_part<HALF>(r[m]), f_of(32 * q + 16 * g2, m));
                            if (HALF) x = mul2(x, both(up[m & 1]));
                            const int to = 2 * (2 * g2 + (m >> 1)) + (m & 1);
                            part_[0][to] = take_part<HALF>(x);
                            if (exact) {
                                part_[1][to] = take_part<HALF>(x);
                                part_[2][to] = as_part<HALF>(x);
                            } else {
                                part_[1][to] = as_part<HALF>(x);
                            }
                        }
                    }
                    if (use) wait_mma(&sh.f_free[q & 1], (use - 1) & 1, tries);
                    // The product with P would carry what is not finite to every token of the stretch: it gets 0 in its place, and the output's warps say where that counts.  They have read
                    // the notes of two stretches ago: behind them the products freed the buffer.
                    if (!STATES && q == 3 && __any_sync(0xffffffffu, (odd | marked) != 0)) {
                        const bool found = __any_sync(0xffffffffu, odd != 0);
                        uint8_t* const edge = sh.edge[n & 1] + 32 * w + 16 * half;
                        if (lane < 16) edge[lane] = C;
                        if (lane == 0) sh.bad[n & 1][warp - WARP_FACTORS] = found;
                        marked = found ? marked | 1u << (n & 1) : marked & ~(1u << (n & 1));
                        __syncwarp();
#pragma unroll 1
                        for (int e = lane; e < (found ? 16 * C : 0); e += 32) {      // two tokens at a time: 16 channels by half of the lanes each
                            const int j = e >> 4, ch = 32 * w + 16 * half + (e & 15);
                            uint16_t* const at = reinterpret_cast<uint16_t*>(c + umma::tile_chunk_offset(128, j, ch >> 3)) + (ch & 7);
                            constexpr uint32_t TOP = HALF ? 0x7c00 : 0x7f80;
                            int turn = (*at & TOP) == TOP ? k.back ? C - 1 - j : j : C;
                            if (turn < C) *at = 0;
                            turn = min(turn, __shfl_xor_sync(0xffffffffu, turn, 16));
                            if (lane < 16 && turn < edge[lane]) edge[lane] = (uint8_t)turn;
                        }
                        umma::fence_async_smem();
                    }
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        if (p < 2 || exact) tmem_st_16x16(umma::tmem_addr(tmem, w, F + 64 * (q & 1) + 16 * p) + ((uint32_t)(16 * half) << 16), part_[p]);
                    umma::tmem_wait_st();
                    signal_tmem(&sh.f_ready[q & 1], lane);
                }
            }
        });
    } else {
        // ---- the state: row = this lane's channel of c, half of the channels of b as columns, in registers.  What a stretch adds comes from an accumulator of its own: the tensor cores cut off what
        // does not fit into 32 bits, and over a long sequence's products that is an error of one sign (2.5e-6 of the state behind 32 k tokens, this way 0.4e-6).
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(STATE_REGS));
        uint32_t n = 0;
        const int w = warp & 3, half = (warp - WARP_STATE) >> 2, ch = 32 * w + lane, m_first = 64 * half;
        for_items<STATES>(plan, [&](const LinearKind& k, const Item& it, const LinearPart& part, int chunks) {
            const float* in = entering(call, k, it, STATES);
            const size_t size = (size_t)k.M * k.V;
            float* out = STATES ? k.parts + ((size_t)(it.n * call.S.segs + it.part + (k.back ? -1 : 1)) * call.HV + it.h) * size
                                : k.last && part.leaves_last ? k.last + ((size_t)it.n * call.HV + it.h) * size : nullptr;
            const float gamma = call.log_decay[it.h];
            Decay whole = {0.f, 0.f}, rest = {0.f, 0.f};   // lam to the tokens of a whole stretch and of the sequence's last one
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {
                whole = rest;
                rest = decay_parts(gamma, u ? part.len % C : C);
            }
            // the state enters and leaves through the accumulator of X, so that what touches memory is a short loop
            const size_t first = k.transposed ? (size_t)ch * k.M : ch, step = k.transposed ? 1 : k.V;
            f32x2 s[32];
            const int m_end = min(k.M, m_first + 64);
#pragma unroll
            for (int m = 0; m < 32; ++m) s[m] = 0ull;
            if (in) {
#pragma unroll 1
                for (int m0 = m_first; m0 < (m_end + 15) / 16 * 16; m0 += 8) {
                    uint32_t v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = ch < k.V && m0 + e < k.M ? __float_as_uint(in[first + (m0 + e) * step]) : 0u;
                    __syncwarp();
                    umma::tmem_st8(umma::tmem_addr(tmem, w, X + m0), v);
                }
                umma::tmem_wait_st();
            }
            auto state_pieces = [&](int g, f32x2 up) {     // 16 columns as the right operand of the next products
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f32x2 y = HALF ? mul2(s[8 * g + e + j], up) : s[8 * g + e + j];
                        h[j] = take_part<HALF>(y);
                        l[j] = as_part<HALF>(y);
                    }
                    uint8_t* const to = state_hi + umma::tile_chunk_offset(128, ch, 8 * half + 2 * g + e / 4);
                    *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(to + TILE) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            };
#pragma unroll 1
            for (int t = 0; t <= chunks; ++t) {
                const bool add = t || in, store = !STATES && t < chunks && add;
                f32x2 f = both(0.f), f_lo = both(0.f);
                if (t) {
                    const bool short_one = part.len - first_of(k, chunks, t - 1) < C;
                    f = both(short_one ? rest.hi : whole.hi);
                    f_lo = both(short_one ? rest.lo : whole.lo);
                    wait_mma(&sh.x_done, (n - 1) & 1, tries);
                }
                if (add) {
                    // what has come from memory into X is not scaled
                    const f32x2 down = both(HALF && t ? __uint_as_float((254u - sh.f_scale[(n - 1) & 1][ch]) << 23) : 1.f);
                    float top = 0.f;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        if (m_first + 16 * g >= m_end) break;
                        float x[16];
                        umma::tmem_ld16(umma::tmem_addr(tmem, w, X + m_first + 16 * g), x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            f32x2 y = pack2(x[2 * e], x[2 * e + 1]);
                            if (HALF) y = mul2(y, down);
                            s[8 * g + e] = fma2(s[8 * g + e], f, fma2(s[8 * g + e], f_lo, y));
                            if (HALF) {
                                float a, b;
                                unpack2(s[8 * g + e], a, b);
                                top = fmaxf(top, fmaxf(fabsf(fmaf(a, 0.f, a)), fabsf(fmaf(b, 0.f, b))));      // finite ones
                            }
                        }
                        if (!HALF && store) state_pieces(g, both(1.f));
                    }
                    if (HALF && store) {
                        top = warp_top(top);
                        if (lane == 0) sh.s_top[warp - WARP_STATE] = (uint8_t)exponent_of(top);
                        group_sync(3);
                        const float up = scale_of(top_of(sh.s_top), 15);
                        group_sync(3);
                        if (warp == WARP_STATE && lane == 0) sh.s_scale[n & 1] = up;
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (m_first + 16 * g >= m_end) break;
                            state_pieces(g, both(up));
                        }
                    }
                }
                if (t == chunks) break;
                umma::signal(&sh.s_ready, lane);
                ++n;
            }
            if (!out) return;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const f32x2 v[4] = {s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
                umma::tmem_st8(umma::tmem_addr(tmem, w, X + m_first + 8 * g), v);
            }
            umma::tmem_wait_st();
#pragma unroll 1
            for (int m0 = m_first; m0 < m_end; m0 += 8) {
                float v[8];
                __syncwarp();
                umma::tmem_ld8(umma::tmem_addr(tmem, w, X + m0), v);
                if (ch >= k.V) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (m0 + e < k.M) out[first + (m0 + e) * step] = v[e];
            }
            __syncwarp();
        });
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (warp == 0) umma::tmem_dealloc(tmem, 512);
}

}  // namespace lt

static long long linear_items(const LinearCall& call) { return (long long)call.S.N * (call.S.seg ? call.S.segs : 1) * call.HV * call.kinds; }
bool linear_tc_takes(const LinearCall& call) {
    if (call.dtype == MKDA_F32 || call.S.TT < 1 || linear_items(call) > 0x7fffffff) return false;
    for (int i = 0; i < call.kinds; ++i) {
        const LinearKind& k = call.kind[i];
        if (k.M % 8 || k.V % 8 || (!k.states && (k.a_stride % 8 || !aligned16(k.a))) || k.b_stride % 8 || k.c_stride % 8 || !aligned16(k.b) || !aligned16(k.c)) return false;
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
        plan.map_a[i] = k.states ? 0 : map(k.a, k.a_stride, k.a_per, k.M);
        plan.map_b[i] = map(k.b, k.b_stride, k.b_per, k.M);
        plan.map_c[i] = map(k.c, k.c_stride, k.c_per, k.V);
        if (rc == MKDA_OK && !states) rc = make_heads_map(&maps.out[i], k.out, call.S.TT, call.HV, k.V, (long long)call.HV * k.V, "linear", k.out_dtype == MKDA_F32 ? 4 : 2);
    }
    if (rc != MKDA_OK) return rc;
    plan.items = (uint32_t)linear_items(call);
    auto* kern = call.dtype == MKDA_F16 ? states ? lt::linear_tc_kernel<true, true> : lt::linear_tc_kernel<false, true> : states ? lt::linear_tc_kernel<true, false> : lt::linear_tc_kernel<false, false>;
    rc = ensure_smem(reinterpret_cast<const void*>(kern), lt::SMEM, "linear");
    if (rc != MKDA_OK) return rc;
    static const int regs = std::min({kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<true, true>)), kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<false, true>)),
                                      kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<true, false>)), kernel_registers(reinterpret_cast<const void*>(lt::linear_tc_kernel<false, false>))});
    if (regs < lt::LAUNCH_REGS) return set_error(MKDA_ERR_LAUNCH, "linear: built with fewer registers than its warps redistribute");
    launch(kern, dim3((unsigned)std::min<uint32_t>(plan.items, sm_count())), lt::THREADS, lt::SMEM, stream, plan, maps);
    return check_launch("linear");
}
int linear_tc_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, umma::g_timeout_flag, sizeof(unsigned int)) == cudaSuccess ? 0 : -1; }
int linear_tc_status_clear() {
    const unsigned int zero = 0;
    return cudaMemcpyToSymbol(umma::g_timeout_flag, &zero, sizeof(zero)) == cudaSuccess ? 0 : -1;
}

}  // namespace mkda
