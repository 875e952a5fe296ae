"""PyTorch front end of the gated recurrent block's kernels (csrc/csn_gated_scan.cu, csn_ffn.cu,
csn_dropout.cu, bound by csn_torch.cpp): the channelwise recurrence and its step, the gated feed-forward product, and
dropout on the residual path.

Unlike the rotor ops these read and write float32, bfloat16 and float16 tensors as they are (all
tensors of a call of one type; recurrence states are float32) and take strided rows in place: only
the last axis has to be contiguous, so slices of one projection's output are not copied.  Every op
runs on the current stream of its tensors' device.  Gradients are first-order: a second backward
pass through them raises, and so does an input with a forward-mode tangent.

The reference has no counterpart of these; its matrix recurrence is python/clifford_cl6.py:150-171
and its gated product python/clifford_model.py:42-43.
"""
from __future__ import annotations

import importlib.util
import threading

from . import _lib

_lock = threading.Lock()
_module = None


def _ext():
    """The compiled binding (csrc/csn_torch.cpp), loaded once; there is no other path."""
    global _module
    if _module is None:
        with _lock:
            if _module is None:
                _lib.load()
                path = _lib.LIB_PATH.with_name("_gated.so")
                if not path.exists():
                    raise RuntimeError(f"{path} is missing: build it with __graft_entry__.build() or "
                                       "`python -m csn_b200._build` (there is no CPU fallback)")
                spec = importlib.util.spec_from_file_location("csn_b200._gated", path)
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
                _module = module
    return _module


# ------------------------------------------------------------- gated recurrence
def gated_scan(f, x, h0=None, gate=None, cu_seqlens=None):
    """The gated linear recurrence over channels, (y, h_last):

        a_t = sigmoid(f_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t silu(gate_t)

    (y = h without a gate).  f, x, gate: [B, T, C], or [L, C] with ``cu_seqlens`` (int32 row numbers
    [S + 1] on the device, rising from 0): sequence s has the rows cu_seqlens[s] .. cu_seqlens[s+1] - 1
    and may have none; rows of no sequence come out as 0.  h0: the states before the first steps
    ([B, C] or [S, C], zero if absent); h_last: the float32 states after the last ones, h0 for a
    sequence without steps.  Differentiable in f, x, h0 and gate."""
    return (_module or _ext()).gated_scan(f, x, h0, gate, cu_seqlens)


def gated_step(f, x, h, gate=None):
    """One step of :func:`gated_scan` for B streams: h [B, C] (float32, contiguous) is advanced in
    place and y [B, C] returned; f, x, gate [B, C].  One launch and, but for y, no allocation.  For
    generation: not differentiable."""
    return (_module or _ext()).gated_step(f, x, h, gate)


# ---------------------------------------------------- gated feed-forward product
def silu_gated_linear(x, w_gate, w_up):
    """silu(x w_gate^T) * (x w_up^T) in one kernel: x [..., C], w_gate and w_up [F, C], result [..., F]
    (what :func:`silu_gate` makes of the library product of both weights).  bfloat16 or float16 on the
    tensor cores, sums in float32, one rounding at the end.  The backward pass forms both products
    again, or, for C >= 1536, takes them from float32 copies that the forward pass keeps (8 bytes an
    element of the result until then; torch.ops.csn.silu_gated_linear_fwd never keeps them, and
    activation checkpointing drops them).  At most 2^21 rows, C and F.  float32 layers use ``silu_gate(linear(x, cat))``."""
    return (_module or _ext()).silu_gated_linear(x, w_gate, w_up)


# ------------------------------------------------------------------------ dropout
def dropout_add(x, residual, p: float, rng):
    """residual + dropout(x, p) in one kernel each way, without a stored mask (residual None: dropout
    alone).  rng: int64 [2] on the device, (seed, offset): the mask is a function of these and of the
    place alone (Philox4x32-10, see csn_dropout_add in include/csn_b200.h), so equal numbers give equal
    masks and a captured graph draws a new one when the numbers are changed between replays
    (csn_b200.modules.DropoutAdd draws them itself).  p is taken in steps of 2^-16 and kept places
    are scaled by one over the probability of being kept."""
    return (_module or _ext()).dropout_add(x, residual, p, rng)
