"""PyTorch front end of the linear-attention block's kernels (csrc/csn_linear_attention.cu, csn_linear_attention_tc.cu,
csn_layer_norm.cu, bound by csn_torch.cpp): linear attention with a decay for each head and its step, and
layer norm of 16-bit rows.

Like the gated block's ops (``gated.py``) these read and write float32, bfloat16 and float16 tensors as they are, of
one type in a call, with float32 states, and take strided rows in place: only the last axis has to be
contiguous, so slices of one projection's output are not copied.  Every op runs on the current stream of its
tensors' device.  Gradients are first-order, and forward-mode tangents are refused.

The reference has no counterpart; its state per head is python/clifford_cl6.py:150-171's rotor recurrence.
"""
from __future__ import annotations

from . import gated


def linear_attention(q, k, v, log_decay, s0=None, cu_seqlens=None, scale=None):
    """Attention without a softmax, whose memory of head h fades by exp(log_decay[h]) a step, (o, s_last):

        S_t = exp(log_decay) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t

    q [B, T, H, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv], o [B, T, H, Dv]; or [L, ...] rows with ``cu_seqlens`` (int32
    row numbers [S + 1] on the device, rising): sequence s has the rows cu_seqlens[s] .. cu_seqlens[s+1] - 1 and
    may have none; rows of no sequence come out as 0.  Hk divides H, and each head of k and v serves H / Hk
    neighbouring heads of q.  Head sizes of 1 to 128.  log_decay: float32 [H], at most 0 (-inf: no memory),
    without a gradient.  s0: the states before the first steps ([B, H, Dk, Dv] or [S, ...], zero if absent);
    s_last: the float32 states after the last ones, s0 for a sequence without steps.  scale: Dk ** -0.5 if absent.
    Differentiable in q, k, v and s0.

    Sums and states are float32.  16-bit tensors go through the tensor cores in blocks of 128 steps (one more rounding
    to 16 bits of q k^T inside a block and of the state where it meets q, none of the state that is carried); there an
    infinity or NaN in k or v can reach the outputs of its whole block, one in q, k, v or the gradient of o the gradients of its
    block, and what depends on it may be NaN where it would be infinite; other blocks, heads and sequences that do not depend on
    it keep their bits.  16-bit rows that do not start on 16 bytes, and expanded ones, are copied first."""
    return (gated._module or gated._ext()).linear_attention(q, k, v, log_decay, s0, cu_seqlens, scale)


def linear_attention_step(q, k, v, log_decay, s, scale=None):
    """One step of :func:`linear_attention` for B streams: s [B, H, Dk, Dv] (float32, contiguous) is advanced in place
    and o [B, H, Dv] returned; q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv].  One launch and, but for o, no
    allocation.  For generation: not differentiable."""
    return (gated._module or gated._ext()).linear_attention_step(q, k, v, log_decay, s, scale)


def layer_norm_rows(x, weight, bias, eps):
    """ops.layer_norm of bfloat16 or float16 rows."""
    return (gated._module or gated._ext()).layer_norm_rows(x, weight, bias, eps)
