/* C ABI of libmkda, second part: the operators that stand around the delta-rule layer in a block of a model (short causal convolution,
 * selective scan, RMS norm with the residual's addition).  The conventions of mkda.h hold: plain parameter structs and a stream, every buffer
 * belongs to the caller, nothing is allocated, errors are return codes with a text behind mkda_last_error().
 *
 *  - Tokens are addressed in the flattened [TT = B*T] space.  Activations are rows of D channels with a stride in elements between tokens
 *    (the last axis contiguous), outputs and gradients contiguous [TT, D].
 *  - Activations, their gradients and the convolution's states may have any address that their type allows, any row stride and any width.  Where 16-byte accesses do not fit, the
 *    16-bit rows of a convolution and the rows of a norm are read by the aligned words of 8 or 16 bytes that hold them and shifted into place: up to 14 bytes in front of and
 *    behind a row are read too (and not used), so those words must be readable; nothing outside a row is written.  Other rows go element by element.
 *  - Must be 16-byte aligned, or the call is refused: A, h0, ht, ckpt, state, dht, dh0, seg_h, seg_g, part_A, part_B and part_C of the scan, and `part` of the norm.
 *  - Parameters (weight, bias, A, D, dt_bias) and states of the scan are fp32; a state of the convolution has the type of x.
 */
#ifndef MKDA_BLOCK_H_
#define MKDA_BLOCK_H_

#include "mkda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MKDA_SCAN_CHECKPOINT 16
#define MKDA_SCAN_MAX_STATES 64
#define MKDA_NORM_MAX_WIDTH 32768
#define MKDA_SEQS_MAX_TOKENS 2147418111

/* The sequences of a call: N rows of T tokens (cu == NULL), or packed with boundaries cu[0..N] (int32 on the device, 0 <= cu[n] <= cu[n+1] <= TT). */
typedef struct {
    int TT; int N; int T;      /* TT up to MKDA_SEQS_MAX_TOKENS */
    int has_empty;             /* some sequence may have no token */
    const int* cu;
    const int* order;          /* [N] the sequences in the order in which they are started on, or NULL */
    const int* ckpt_off;       /* [N] first checkpoint of each sequence (ceil(length / MKDA_SCAN_CHECKPOINT) each), or NULL with cu == NULL */
    int seg; int segs;         /* scan: sequences are cut into parts of seg tokens (a multiple of 64) that run side by side, segs of them in the longest; seg = 0: not cut.
                                  Every sequence has a row of blocks for each of the segs parts, also for those without tokens */
} MkdaSeqs;

/* Depthwise causal convolution: y[t] = act(bias + sum_w weight[w] x[t - W + 1 + w]), W in 2..4.  What lies in front of a sequence's first
 * token comes from its state [W-1][D] (the tokens in front, the latest last) or is zero. */
typedef struct {
    MkdaSeqs S; int D; int W; int dtype; int silu;
    const void* x; long long x_stride;
    const float* weight;       /* [D,W] */
    const float* bias;         /* [D] or NULL */
    const void* state;         /* [N,W-1,D] or NULL */
    void* y;                   /* [TT,D] */
    void* last;                /* [N,W-1,D] the state behind each sequence, or NULL */
} MkdaConvFwd;
int mkda_conv_fwd(const MkdaConvFwd* p, void* stream);

typedef struct {
    MkdaSeqs S; int D; int W; int dtype; int silu;
    const void* x; long long x_stride;
    const float* weight; const float* bias; const void* state;
    const void* dy;            /* [TT,D] contiguous */
    const void* dlast;         /* [N,W-1,D] or NULL */
    void* dx;                  /* [TT,D] */
    void* dstate;              /* [N,W-1,D] or NULL */
    int part_rows;             /* R, what mkda_conv_bwd_part_rows says: the tokens are cut into R runs, each with a row of partial sums */
    float* part;               /* [R][W+1][D]: of the weight's W columns, then of the bias */
} MkdaConvBwd;
int mkda_conv_bwd(const MkdaConvBwd* p, void* stream);
int mkda_conv_bwd_part_rows(int TT, int D);

/* One token of each of N sequences; the state is shifted in place. */
typedef struct {
    int N; int D; int W; int dtype; int silu;
    const void* x; long long x_stride;
    const float* weight; const float* bias;
    void* state;               /* [N,W-1,D], read and written */
    void* y;                   /* [N,D] */
} MkdaConvStep;
int mkda_conv_step(const MkdaConvStep* p, void* stream);

/* Selective scan: d = dt + dt_bias (through softplus where asked), h[n] = exp(d A[n]) h[n] + d x B[n], y = sum_n C[n] h[n] + D x, times silu(z).
 * Channel c belongs to the group c / (D / G) of B and C.  1 to MKDA_SCAN_MAX_STATES states per channel. */
typedef struct {
    MkdaSeqs S; int D; int NST; int G; int dtype; int softplus;
    const void* x; const void* dt; const void* z; const void* B; const void* C;          /* z may be NULL */
    long long x_stride; long long dt_stride; long long z_stride; long long B_stride; long long C_stride;
    const float* A;            /* [D,NST] */
    const float* skip;         /* [D] or NULL */
    const float* dt_bias;      /* [D] or NULL */
    const float* h0;           /* [N,D,NST] or NULL */
    void* y;                   /* [TT,D] */
    float* ht;                 /* [N,D,NST] or NULL */
    float* seg_h; float* seg_d;           /* cut sequences: [segs][N][D][P] what each part makes of nothing, [segs][N][D] its sum of d (workspace) */
    float* ckpt;               /* states in front of every MKDA_SCAN_CHECKPOINT-th token of each sequence, [checkpoints][D][P], or NULL; P = NST padded to 8, 16, 32 or 64 */
} MkdaScanFwd;
int mkda_scan_fwd(const MkdaScanFwd* p, void* stream);

typedef struct {
    MkdaScanFwd f;             /* the forward call: y, ht, h0, seg_h and seg_d are not looked at, ckpt is read; f.S.seg need not be the forward call's */
    const void* dy;            /* [TT,D] */
    const float* dht;          /* [N,D,NST] or NULL */
    void* dx; void* ddt; void* dz;        /* [TT,D]; dz only with z */
    float* dh0;                /* [N,D,NST] or NULL */
    float* seg_g; float* seg_d;           /* as in the forward call, of the gradient */
    int slots;                 /* the sequences (or their parts) are dealt to so many rows of blocks */
    int channel_blocks;        /* what mkda_scan_bwd_channel_blocks says */
    float* part_B; float* part_C;         /* [G][blocks][TT][P]: per block of channels; only rows of tokens of sequences are written */
    float* part_A;             /* [slots][D][P] */
    float* part_skip;          /* [slots][D] or NULL */
    float* part_bias;          /* [slots][D] or NULL */
    int first_block; int blocks;          /* of each group's channel_blocks / G blocks of channels, the call is for `blocks` from the first_block-th on; blocks = 0: for all */
} MkdaScanBwd;
int mkda_scan_bwd(const MkdaScanBwd* p, void* stream);
/* Blocks of channels of the backward kernel for D channels in G groups (each group has as many) and NST states; the padded number of states P. */
int mkda_scan_bwd_channel_blocks(int D, int G, int NST);
int mkda_scan_padded_states(int NST);

typedef struct {
    int N; int D; int NST; int G; int dtype; int softplus;
    const void* x; const void* dt; const void* z; const void* B; const void* C;
    long long x_stride; long long dt_stride; long long z_stride; long long B_stride; long long C_stride;
    const float* A; const float* skip; const float* dt_bias;
    float* state;              /* [N,D,NST], read and written */
    void* y;                   /* [N,D] */
} MkdaScanStep;
int mkda_scan_step(const MkdaScanStep* p, void* stream);

/* s = x + residual, held in the residual's type, which is x's or fp32; y = s / sqrt(mean s^2 + eps) * weight, rows of `width` channels.
 * Without a residual s = x.  out_e4m3: y leaves as e4m3 with scales such that a row (group = 0) or each `group` = 128 channels of it reach 448. */
typedef struct {
    int rows; int width; int dtype; int res_dtype; float eps;
    const void* x; long long x_stride;
    const void* residual; long long res_stride;           /* or NULL */
    const void* weight; int weight_dtype;                 /* or NULL */
    void* sum;                 /* [rows,width] in res_dtype, with a residual */
    void* y;                   /* [rows,width] in dtype, or e4m3 */
    int out_e4m3; int group;
    float* scale;              /* [rows] or [rows,width/group] */
} MkdaNormFwd;
int mkda_norm_fwd(const MkdaNormFwd* p, void* stream);

typedef struct {
    int rows; int width; int dtype; float eps;
    const void* s; long long s_stride; int s_dtype;       /* what was normalised, in dtype or fp32 */
    const void* weight; int weight_dtype;
    const void* dy;            /* [rows,width] in dtype, contiguous */
    const void* dsum;          /* [rows,width] in s_dtype, or NULL */
    void* dx;                  /* [rows,width] in dtype */
    void* dres;                /* [rows,width] in s_dtype, or NULL */
    int part_rows;             /* what mkda_norm_bwd_part_rows says */
    float* part;               /* [part_rows,width] partial sums of the weight's gradient, or NULL */
} MkdaNormBwd;
int mkda_norm_bwd(const MkdaNormBwd* p, void* stream);
int mkda_norm_bwd_part_rows(int rows, int width);

/* Second stage of the sums above, up to five in one launch, fixed order.  Of each of `groups` stacks of `rows` rows (one behind the other, `pitch` floats apart)
 * column c < cols goes to out[g * out_group + (c / inner) * out_outer + (c % inner) * out_inner] where c % inner < valid.  A job without `out` is skipped. */
typedef struct {
    const float* in; int rows; int groups; long long pitch; long long cols; int inner; int valid;
    long long out_group; long long out_outer; long long out_inner;
    void* out; int out_dtype;
} MkdaSumJob;
typedef struct {
    MkdaSumJob job[5];
} MkdaSumRows;
int mkda_sum_rows(const MkdaSumRows* p, void* stream);

#define MKDA_BLOCK_STRUCTS(X) \
    X(MkdaSeqs) X(MkdaConvFwd) X(MkdaConvBwd) X(MkdaConvStep) X(MkdaScanFwd) X(MkdaScanBwd) X(MkdaScanStep) X(MkdaNormFwd) X(MkdaNormBwd) \
    X(MkdaSumJob) X(MkdaSumRows)
int mkda_block_struct_sizes(int* out, int n);

#ifdef __cplusplus
}
#endif
#endif /* MKDA_BLOCK_H_ */
