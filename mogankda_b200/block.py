"""The operators that stand around the delta-rule layer in a block of a model: the short causal convolution in front of q, k and v (or of a
scan), the selective scan, the RMS norm and the layer norm with the residual's addition; and its sibling without the delta rule, the linear attention with a decay
for each head, with rotary positions of several axes in front of it.

Conventions of the layer hold: CUDA tensors only, bfloat16, float16 or float32, arithmetic in 32 bits, launches on
``torch.cuda.current_stream()`` of the tensors' device, packed sequences addressed by ``cu_seqlens`` (B == 1; tokens behind the last boundary give zeros,
and have zero gradients), ``initial_state`` / final state with one row per sequence.  Activations may be slices of a wider projection: rows with any stride
are read where they lie as long as one stride leads from token to token, other layouts are copied.  Gradients exist for every floating
argument of the functions without ``_step``; a gradient that is differentiated again (``create_graph``) raises, unless it is a constant.  Results do not depend on
the order of execution.
"""
import torch

from . import _lib
from .index import get_bounds


def _sequences(x, cu_seqlens, dim=3):
    if cu_seqlens is None:
        return None, None
    if not x.is_cuda:
        raise RuntimeError("mogankda_b200 kernels need CUDA tensors (there is no CPU fallback)")
    if x.dim() != dim or x.shape[0] != 1:
        raise ValueError(f"The batch size is expected to be 1 rather than {x.shape[0]} when using `cu_seqlens`.")
    if cu_seqlens.dim() != 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must be a vector of int32 or int64")
    b = get_bounds(x.shape[1], cu_seqlens, x.device)
    return b.table, b.dims


def _silu(activation):
    if activation not in (None, "silu"):
        raise ValueError(f"unknown activation {activation!r}")
    return int(activation == "silu")


def causal_conv1d(x, weight, bias=None, *, activation=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Depthwise causal convolution over the tokens, ``y[t] = act(bias + sum_w weight[:, w] x[t - W + 1 + w])``.

    x [B,T,D]; weight [D,W] with 2 to 4 taps, bias [D] (any of the three types); activation None or "silu".  ``initial_state`` [N,W-1,D] in the type of x:
    the tokens in front of each sequence, the latest last (zeros without it) - what ``cp_context.conv_halo_tokens`` asks of the previous rank,
    behind zeros where there are fewer.  Returns ``(y, final_state)``: y like x, and the last W - 1 tokens of each sequence or None."""
    table, dims = _sequences(x, cu_seqlens)
    return _lib.host().conv(x, weight, bias, initial_state, table, dims, _silu(activation), output_final_state)


def causal_conv1d_step(x, state, weight, bias=None, *, activation=None):
    """One more token of each of N running sequences: x [N,D], state [N,W-1,D] (contiguous, in the type of x), which is shifted IN PLACE.
    Returns y [N,D].  No backward pass."""
    return _lib.host().conv_step(x, state, weight, bias, _silu(activation))


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, *, dt_softplus=False, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Selective state space scan, a diagonal state of N numbers per channel:

        d = dt + dt_bias (through softplus with ``dt_softplus``);  h = exp(d A) h + d x B;  y = sum_n C h + D x;  y silu(z) with ``z``

    x, dt, z [B,T,D] and B, C [B,T,N] or [B,T,G,N] share a type (channel c reads group c // (D / G)); A [D,N], 1 to 64 states, D and dt_bias [D]
    of any of the three types.  ``initial_state`` [sequences,D,N] float32.  Returns ``(y, final_state)``: y like x; the state float32 or None.
    A call that wants gradients keeps the state in front of every 16th token (P / 4 bytes per token and channel; P: N padded to 8, 16, 32 or 64).  Its backward pass leaves dB and
    dC per block of 512 / P channels, 8 P bytes per token and block, before it adds them up (4 bytes per token and channel at 16 states, 64 at 64); more than 1 GiB of it is
    worked off by ranges of blocks that fill the GPU.  An infinite A is taken as the largest number of its sign: -inf keeps nothing of a state wherever d > 0.  Gradients around an
    infinite x or dt may be NaN."""
    table, dims = _sequences(x, cu_seqlens)
    return _lib.host().scan(x, dt, A, B, C, D, z, dt_bias, initial_state, table, dims, dt_softplus, output_final_state)


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, *, dt_softplus=False):
    """One more token of each of N running sequences: x, dt, z [N,D], B, C [N,states] or [N,G,states], state [N,D,states] float32 (contiguous), which is
    updated IN PLACE.  Returns y [N,D].  No backward pass.  Where d is 0, A has to be above -2.3e38 (A log2 e a finite number)."""
    return _lib.host().scan_step(x, dt, A, B, C, D, z, dt_bias, state, dt_softplus)


def rms_norm(x, weight=None, *, residual=None, eps=1e-6, out_dtype=None, scale_group=None):
    """RMS norm of the rows of x [..,H], H up to 32768: ``y = s / sqrt(mean s^2 + eps) * weight`` with s = x, or with ``residual`` s = x + residual as the
    residual's type holds it (that of x, or float32).  Statistics in 32 bits, y rounded once.

    Returns y; with ``residual`` ``(y, s)``.  ``out_dtype=torch.float8_e4m3fn`` returns ``(y8, scale)`` or ``(y8, scale, s)``: y8 * scale is y, with one scale
    per row ([..,1]) or with ``scale_group=128`` per 128 channels ([..,H/128]), max |y| / 448 (at least 2^-126); it has no gradient."""
    e4m3 = out_dtype == torch.float8_e4m3fn
    if not e4m3 and out_dtype not in (None, x.dtype):
        raise ValueError(f"out_dtype must be the type of x or torch.float8_e4m3fn, got {out_dtype}")
    if scale_group not in (None, 128) or (scale_group and not e4m3):
        raise ValueError("scale_group is 128 or None, and belongs to an output in 8 bits")
    got = _lib.host().norm(x, weight, residual, eps, e4m3, scale_group or 0)
    if got[-1] is None:
        got = got[:-1]
    return got if len(got) > 1 else got[0]


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Linear attention with a decay for each head, the delta-rule layer's sibling without the delta rule:

        S[t] = exp(log_decay) S[t - 1] + k[t] v[t]^T;  o[t] = scale S[t]^T q[t]

    q, k [B,T,HK,K] and v [B,T,HV,V] share a type, K and V up to 128; HV is a multiple of HK: v-head h reads head h // (HV // HK) of q and k.  ``log_decay`` [HV] (any of the
    three types, natural logarithm, at most 0) has no gradient: a call that wants one is refused.  ``scale`` is K ** -0.5 by default; ``initial_state`` [N,HV,K,V] float32.
    Returns ``(o, final_state)``: o [B,T,HV,V] in the type of q; the state float32 or None.

    Pairs of tokens up to 128 apart are computed as products of q and k, earlier ones through the state, which is held in fp32.  In 16 bits the weights of pairs, and the state where it meets q,
    go into these products as two 16-bit parts each (off by 2^-16 of the value at most in bfloat16; in float16 by 2^-22 of it, or 2^-39 of the largest of a token's pairs or of the state), and what goes into the state
    as three (bfloat16; two where ``output_final_state`` is not asked for, so that o may differ in its last bit by that flag; float16 always two).  o is rounded once.  Long sequences of few
    heads are cut into parts that run side by side, by a rule on sizes: results on both sides of it agree to rounding.  What is not finite stays in its sequence and reaches no
    token in front of it (in the gradients: behind it); where the definition has an infinity, a result may be NaN.

    Workspace: a cut call holds the states that its parts enter with, 4 K V bytes a part and v-head, 256 MB at most, and twice that in the backward pass; with HV > HK the backward pass holds the
    gradients of q and k per v-head, 8 HV K bytes a token."""
    table, dims = _sequences(q, cu_seqlens, 4)
    return _lib.host().linear(q, k, v, log_decay, initial_state, table, dims, scale, output_final_state)


def linear_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One more token of each of N running sequences: q, k [N,HK,K], v [N,HV,V], state [N,HV,K,V] float32 (contiguous), which is updated IN PLACE.  Returns o
    [N,HV,V].  No backward pass."""
    return _lib.host().linear_step(q, k, v, log_decay, state, scale)


def rotary(q, k, positions, inv_freq, *, axes=None, interleaved=False):
    """Rotary positions: pair f of the channels of each head is turned by ``positions * inv_freq[f]``.

    q [..,HQ,D] and k [..,HK,D] (or None) share a type, D up to 512; ``inv_freq`` [F] float32, 2 F <= D: the pairs are channels (f, f + F), with ``interleaved``
    (2 f, 2 f + 1), and channels behind the first 2 F stay as they are.  ``positions`` int32 or int64 with the leading axes of q; with ``axes``, F whole numbers, ``positions`` is
    [A,..] and frequency f goes by ``positions[axes[f]]`` (time, height and width of a video's tokens: ``axes=[0] * 16 + [1] * 24 + [2] * 24``, or any other order).
    Angles are formed in 64 bits, so that far positions keep theirs.  Returns q, or ``(q, k)``, as new tensors; gradients for q and k, none for ``inv_freq``."""
    got = _lib.host().rotary(q, k, positions, inv_freq, axes, interleaved)
    return got if k is not None else got[0]


def layer_norm(x, weight=None, bias=None, *, residual=None, groups=1, eps=1e-5):
    """Layer norm of the rows of x [..,H]: ``y = (s - mean s) / sqrt(var s + eps) * weight + bias`` with s = x, or with ``residual`` s = x + residual as the residual's type holds it
    (that of x, or float32).  ``groups`` > 1: each of so many equal parts of a row, up to 32768 channels, by itself, as for the heads of a token's outputs; ``weight`` and ``bias`` are
    [H] all the same.  Statistics in 32 bits, y rounded once.  Returns y; with ``residual`` ``(y, s)``."""
    got = _lib.host().layer_norm(x, weight, bias, residual, groups, eps)
    return got if residual is not None else got[0]
