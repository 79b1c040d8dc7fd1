// Linear attention with a decay for each head: what its kernels (linear.cu) share.
//
// With lam = exp(log_decay) of a head, the forward pass and the three gradients are one operator of three row tensors,
//   out[i] = sum_j lam^|i - j| (a[i] . b[j]) c[j],   over j <= i, or backwards in time over j >= i:
//   o: (q, k, v)     dq: (do, v, k)     dk: (v, do, q) backwards     dv: (k, q, do) backwards
// Over a stretch of L tokens (i, j counted from its first one) it is, with the state M = sum lam^.. b c^T in front of the stretch (behind it)
//   forwards   out[i] = sum_{j <= i} lam^(i - j) (a[i] . b[j]) c[j] + lam^(i + 1) M^T a[i]        M <- lam^L M + sum_j lam^(L - 1 - j) b[j] c[j]^T
//   backwards  out[i] = sum_{j >= i} lam^(j - i) (a[i] . b[j]) c[j] + lam^(L - 1 - i) M^T a[i]    M <- lam^L M + sum_j lam^(j + 1) b[j] c[j]^T
// M is the state S of the caller for o, its transpose for dq, the state's gradient for dv and its transpose for dk.
#pragma once
#include <cfloat>

#include "block.cuh"

namespace mkda {

struct LinearKind {
    const void* a; const void* b; const void* c;
    int states;                                            // nothing but the states that the parts of the sequences leave; a is not looked at
    long long a_stride, b_stride, c_stride;
    int a_per, b_per, c_per;                               // v-heads to a head
    int M, V;                                              // channels of a and b, of c and out
    void* out; int out_dtype;                              // [TT, HV, V]
    float pair_scale, in_scale, state_scale;               // of a pair's product, of what goes into the state, of what comes out of it
    int back;
    int transposed;                                        // states lie as [V][M] in memory
    const float* first; float* last;                       // [N, HV, ..]
    float* parts;                                          // [N, segs, HV, ..] cut sequences: the state that each part enters with
};
struct LinearCall {
    MkdaSeqs S;
    int HV, dtype, kinds;
    const float* log_decay;
    LinearKind kind[3];
};

// lam^n, rounded once
__device__ __forceinline__ float decay_power(float log_decay, long long n) { return n == 0 ? 1.f : (float)exp((double)log_decay * (double)n); }
// ... and in two parts, for what a state is multiplied by over and over: rounded once it is off by up to 2^-25 with one sign every time (behind 131072 tokens of 128 at a time 4e-5 of the state)
struct Decay { float hi, lo; };
__device__ __forceinline__ Decay decay_parts(float log_decay, long long n) {
    const double x = n == 0 ? 1.0 : exp((double)log_decay * (double)n);
    const float hi = (float)x;
    return {hi, (float)(x - (double)hi)};
}
// lam^n s + x; an infinite s stays so
__device__ __forceinline__ float decayed(const Decay& d, float s, float x) { return fmaf(d.hi, s, fmaf(d.lo, fabsf(s) <= FLT_MAX ? s : 0.f, x)); }

// What a block has to do: tokens [start, start + len) of sequence n, which are part `part` of it
struct LinearPart { int start, len; bool nothing, enters_first, leaves_last; };
__device__ __forceinline__ LinearPart linear_part(const MkdaSeqs& s, int n, int part, bool back) {
    const Span w = sequence(s, n);
    const int len = w.end - w.start;
    if (!s.seg) return {w.start, len, false, true, true};
    const int parts = part_count(len, s.seg);
    if (part >= parts) return {0, 0, true, false, false};
    const int at = part * s.seg;
    return {w.start + at, min(s.seg, len - at), false, false, back ? part == 0 : part == parts - 1};
}

// linear_tc.cu: rows of 16 bits on the tensor cores, where tiled copies can fetch them.  `states`: nothing but what the parts of cut sequences make of a zero state.
bool linear_tc_takes(const LinearCall& call);
int launch_linear_tc(const LinearCall& call, bool states, cudaStream_t stream);

}  // namespace mkda
