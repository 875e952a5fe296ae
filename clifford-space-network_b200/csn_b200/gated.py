"""PyTorch front end of the gated recurrent block's kernels (csrc/csn_gated_scan.cu, csn_ffn.cu,
csn_dropout.cu): the channelwise recurrence and its step, the gated feed-forward product, and
dropout on the residual path.

Unlike the rotor ops these read and write float32, bfloat16 and float16 tensors as they are (all
tensors of a call of one type; recurrence states are float32) and take strided rows in place: only
the last axis has to be contiguous, so slices of one projection's output are not copied.  Every op
runs on the current stream of its tensors' device.  Gradients are first-order: a second backward
pass through them raises.

The reference has no counterpart of these; its matrix recurrence is python/clifford_cl6.py:150-171
and its gated product python/clifford_model.py:42-43.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _require_cuda

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MARK = 64  # steps between two kept states of the scan (csn_gated_scan_marks)
_NAMES = {t: str(t).replace("torch.", "") for t in DTYPES}

# a generation step is one small kernel, so what its call costs on the host is what it costs: the
# index forms of current_device() and current_stream() take a tenth of the time
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


def _launch(name, index, *args):
    """Calls an entry point on the current stream of device `index`; None is a null pointer."""
    if _current_device() == index:
        rc = getattr(_lib.load(), name)(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(_lib.load(), name)(*args, _current_stream(index))
    if rc:
        raise _lib.CsnError(name, rc, _lib.load().csn_last_error().decode(errors="replace"))


@functools.lru_cache(maxsize=1024)
def _size(query, *sizes):
    """A size query of the library, which is a function of its arguments alone."""
    return getattr(_lib.load(), query)(*sizes)


def _first_order(backward):
    """once_differentiable, without its cost where no second backward pass can follow."""
    once = once_differentiable(backward)

    @functools.wraps(backward)
    def call(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call


def _device_of(name, first, *rest):
    """The index of the device that all tensors are on."""
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            index = -1
            break
    if index < 0:
        _require_cuda(first, *rest)
        raise ValueError(f"{name}: tensors are on different devices")
    return index


def _dtype_of(name, allowed, first, *rest):
    """The dtype code of tensors that have to share one of the allowed types."""
    dtype = first.dtype
    if dtype in allowed:
        for t in rest:
            if t is not None and t.dtype != dtype:
                break
        else:
            return DTYPES[dtype]
    raise ValueError(f"{name}: tensors of one type among {', '.join(_NAMES[d] for d in allowed)} expected, got "
                     f"{', '.join(str(t.dtype) for t in (first, *rest) if t is not None)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t with a contiguous last axis (itself where it has one)."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _packed(t):
    """t contiguous and 16-byte aligned (itself where it is)."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _row_strides(*ts):
    """Strides of every axis but the last of each tensor, as a host array; 0 where an axis has one
    entry (its stride means nothing) or a tensor is absent.  [rows, C] gives (0, row)."""
    out = []
    for t in ts:
        if t is None:
            out += (0, 0)
            continue
        n, st = t.shape, t.stride()
        if len(n) == 2:
            out += (0, st[0] if n[0] > 1 else 0)
        else:
            out += (st[0] if n[0] > 1 else 0, st[1] if n[1] > 1 else 0)
    return _STRIDES[len(out)](*out)


_STRIDES = {n: ctypes.c_int64 * n for n in (3, 6, 8)}


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------- gated recurrence
def _scan_sizes(f, cu):
    n = f.shape
    return (n[0], n[1], n[2]) if cu is None else (cu.shape[0] - 1, n[0], n[1])


def _scan_workspace(f, S, T, C, cu, backward):
    nb = _size("csn_gated_scan_workspace_bytes", S, T, C, int(cu is not None), DTYPES[f.dtype], backward)
    return (f.new_empty((nb,), dtype=torch.uint8) if nb else None), nb


def _gated_scan_fwd(f, x, h0, gate, cu, keep):
    """(y, h_last, marks or None) of rows as they lie; h0 float32."""
    f, x, gate, h0 = _rows(f), _rows(x), _rows(gate), _packed(h0)
    S, T, C = _scan_sizes(f, cu)
    index = f.get_device()
    y = f.new_empty(f.shape)
    h_last = f.new_empty((S, C), dtype=torch.float32)
    marks = None
    if keep:
        marks = f.new_empty((_size("csn_gated_scan_marks", S, T, C, int(cu is not None)),), dtype=torch.float32)
    ws, nb = _scan_workspace(f, S, T, C, cu, 0)
    _launch("csn_gated_scan_fwd", index, _ptr(f), _ptr(x), _ptr(gate), _row_strides(f, x, gate), _ptr(h0), _ptr(cu),
            _ptr(y), _ptr(h_last), _ptr(marks), S, T, C, DTYPES[f.dtype], _ptr(ws), nb)
    return y, h_last, marks


def _gated_scan_bwd(f, x, gate, cu, marks, dy, dh_last, need):
    """Gradients (df, dx, dh0, dgate); dh0 where `need` asks for it, dgate where there is a gate."""
    if dy is None:  # only the last states are used
        dy = f.new_zeros((1,) * f.dim()).expand(f.shape)
    f, x, gate, dy, dh_last = _rows(f), _rows(x), _rows(gate), _rows(dy), _packed(dh_last)
    S, T, C = _scan_sizes(f, cu)
    df, dx = f.new_empty(f.shape), f.new_empty(f.shape)
    dh0 = f.new_empty((S, C), dtype=torch.float32) if need[2] else None
    dgate = f.new_empty(f.shape) if gate is not None else None
    ws, nb = _scan_workspace(f, S, T, C, cu, 1)
    _launch("csn_gated_scan_bwd", f.get_device(), _ptr(f), _ptr(x), _ptr(gate), _ptr(dy),
            _row_strides(f, x, gate, dy), _ptr(cu), _ptr(marks), _ptr(dh_last), _ptr(df), _ptr(dx), _ptr(dgate),
            _ptr(dh0), S, T, C, DTYPES[f.dtype], _ptr(ws), nb)
    return df, dx, dh0, dgate


class GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, x, h0, gate, cu):
        ctx.set_materialize_grads(False)
        y, h_last, marks = _gated_scan_fwd(f, x, h0, gate, cu, True)
        ctx.save_for_backward(f, x, gate, cu, marks)
        return y, h_last

    @staticmethod
    @_first_order
    def backward(ctx, dy, dh_last):
        if dy is None and dh_last is None:
            return None, None, None, None, None
        f, x, gate, cu, marks = ctx.saved_tensors
        return (*_gated_scan_bwd(f, x, gate, cu, marks, dy, dh_last, ctx.needs_input_grad), None)


def _check_scan(f, x, h0, gate, cu):
    _device_of("gated_scan", f, x, h0, gate, cu)
    _dtype_of("gated_scan", DTYPES, f, x, gate)
    n = f.shape
    if len(n) != (3 if cu is None else 2) or x.shape != n or (gate is not None and gate.shape != n):
        raise ValueError("gated_scan: f, x and gate [B, T, C], or [L, C] with cu_seqlens, of one shape expected, got "
                         f"{', '.join(str(tuple(t.shape)) for t in (f, x, gate) if t is not None)}")
    if cu is not None and (cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 2 or not cu.is_contiguous()):
        raise ValueError("gated_scan: cu_seqlens is a contiguous int32 vector of at least 2 row numbers")
    S, _, C = _scan_sizes(f, cu)
    if h0 is not None and (tuple(h0.shape) != (S, C) or not h0.is_floating_point()):
        raise ValueError(f"gated_scan: h0 [{S}, {C}] of a floating type expected, got {tuple(h0.shape)} {h0.dtype}")


def gated_scan(f, x, h0=None, gate=None, cu_seqlens=None):
    """The gated linear recurrence over channels, (y, h_last):

        a_t = sigmoid(f_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t silu(gate_t)

    (y = h without a gate).  f, x, gate: [B, T, C], or [L, C] with ``cu_seqlens`` (int32 row numbers
    [S + 1] on the device, rising from 0): sequence s has the rows cu_seqlens[s] .. cu_seqlens[s+1] - 1
    and may have none; rows of no sequence come out as 0.  h0: the states before the first steps
    ([B, C] or [S, C], zero if absent); h_last: the float32 states after the last ones, h0 for a
    sequence without steps.  Differentiable in f, x, h0 and gate."""
    _check_scan(f, x, h0, gate, cu_seqlens)
    if h0 is not None and h0.dtype != torch.float32:
        h0 = h0.to(torch.float32)
    if not _wants_grad(f, x, h0, gate):
        return _gated_scan_fwd(f, x, h0, gate, cu_seqlens, False)[:2]
    return GatedScanFunction.apply(f, x, h0, gate, cu_seqlens)


def gated_step(f, x, h, gate=None):
    """One step of :func:`gated_scan` for B streams: h [B, C] (float32, contiguous) is advanced in
    place and y [B, C] returned; f, x, gate [B, C].  One launch and, but for y, no allocation.  For
    generation: not differentiable."""
    index = _device_of("gated_step", f, x, h, gate)
    code = _dtype_of("gated_step", DTYPES, f, x, gate)
    n = f.shape
    if len(n) != 2 or x.shape != n or h.shape != n or (gate is not None and gate.shape != n):
        raise ValueError("gated_step: f, x, h and gate [B, C] of one shape expected")
    if h.dtype != torch.float32 or not h.is_contiguous() or h.data_ptr() % 16:
        raise ValueError("gated_step: h is a contiguous float32 state, 16-byte aligned")
    if _wants_grad(f, x, h, gate):
        raise ValueError("gated_step: not differentiable; call it under torch.no_grad() or use gated_scan")
    f, x, gate = _rows(f), _rows(x), _rows(gate)
    y = f.new_empty(n)
    strides = _STRIDES[3](f.stride(0), x.stride(0), 0 if gate is None else gate.stride(0))
    _launch("csn_gated_step", index, _ptr(f), _ptr(x), _ptr(gate), strides, _ptr(h), _ptr(y), n[0], n[1], code)
    return y


# ---------------------------------------------------- gated feed-forward product
HALF_TYPES = (torch.bfloat16, torch.float16)


def _tiled(t):
    """(rows, row stride) of a 16-bit matrix whose rows start on 16 bytes: t itself where its rows do,
    otherwise a copy with padded rows."""
    t = _rows(t)
    n, c = t.shape
    ld = t.stride(0) if n > 1 else (c + 7) // 8 * 8
    if t.data_ptr() % 16 == 0 and ld % 8 == 0 and ld >= c:
        return t, ld
    ld = (c + 7) // 8 * 8
    room = t.new_empty((n, ld))
    room[:, :c].copy_(t)
    return room, ld


def _silu_gated_linear_fwd(x, wg, wu):
    R, C, F = x.shape[0], x.shape[1], wg.shape[0]
    (x, ldx), (wg, ldg), (wu, ldu) = _tiled(x), _tiled(wg), _tiled(wu)
    y = x.new_empty((R, F))
    _launch("csn_silu_gated_linear_fwd", x.get_device(), _ptr(x), ldx, _ptr(wg), ldg, _ptr(wu), ldu, _ptr(y), R, C, F,
            DTYPES[x.dtype])
    return y


def _silu_gated_linear_bwd(x, wg, wu, dy, need):
    R, C, F = x.shape[0], x.shape[1], wg.shape[0]
    (x, ldx), (wg, ldg), (wu, ldu), dy = _tiled(x), _tiled(wg), _tiled(wu), _rows(dy)
    dx = x.new_empty((R, C)) if need[0] else None
    dwg = x.new_empty((F, C)) if need[1] else None
    dwu = x.new_empty((F, C)) if need[2] else None
    nb = _size("csn_silu_gated_linear_bwd_workspace_bytes", R, C, F)
    ws = x.new_empty((nb,), dtype=torch.uint8)
    _launch("csn_silu_gated_linear_bwd", x.get_device(), _ptr(x), ldx, _ptr(wg), ldg, _ptr(wu), ldu, _ptr(dy),
            dy.stride(0), _ptr(dx), _ptr(dwg), _ptr(dwu), R, C, F, DTYPES[x.dtype], _ptr(ws), nb)
    return dx, dwg, dwu


class SiluGatedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu):
        ctx.save_for_backward(x, wg, wu)
        return _silu_gated_linear_fwd(x, wg, wu)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        return _silu_gated_linear_bwd(*ctx.saved_tensors, dy, ctx.needs_input_grad)


def silu_gated_linear(x, w_gate, w_up):
    """silu(x w_gate^T) * (x w_up^T) in one kernel: x [..., C], w_gate and w_up [F, C], result [..., F]
    (what :func:`silu_gate` makes of the library product of both weights).  bfloat16 or float16 on the
    tensor cores, sums in float32, one rounding at the end; the backward pass forms both products
    again instead of keeping them.  float32 layers use ``silu_gate(linear(x, cat))``."""
    _device_of("silu_gated_linear", x, w_gate, w_up)
    _dtype_of("silu_gated_linear", HALF_TYPES, x, w_gate, w_up)
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError("silu_gated_linear: x [..., C] and w_gate, w_up [F, C] expected, got "
                         f"{tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    C, F = w_gate.shape[1], w_gate.shape[0]
    x2 = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), C)
    y = (SiluGatedLinearFunction.apply(x2, w_gate, w_up) if _wants_grad(x, w_gate, w_up)
         else _silu_gated_linear_fwd(x2, w_gate, w_up))
    return y if x.dim() == 2 else y.view(*x.shape[:-1], F)


# ------------------------------------------------------------------------ dropout
def _dropout_add(x, residual, cut, rng):
    x, residual = _packed(x), _packed(residual)
    y = x.new_empty(x.shape)
    _launch("csn_dropout_add", x.get_device(), _ptr(x), _ptr(residual), _ptr(rng), _ptr(y), x.numel(), cut,
            DTYPES[x.dtype])
    return y


class DropoutAddFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, cut, rng):
        ctx.save_for_backward(rng)  # changing rng in place before the backward pass raises there
        ctx.cut = cut
        return _dropout_add(x, residual, cut, rng)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        dx = _dropout_add(dy, None, ctx.cut, rng) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None


def dropout_add(x, residual, p: float, rng):
    """residual + dropout(x, p) in one kernel each way, without a stored mask (residual None: dropout
    alone).  rng: int64 [2] on the device, (seed, offset): the mask is a function of these and of the
    place alone (Philox4x32-10, see csn_dropout_add in include/csn_b200.h), so equal numbers give equal
    masks and a captured graph draws a new one when the numbers are changed between replays
    (csn_b200.modules.DropoutAdd counts for itself).  p is taken in steps of 2^-16 and kept places
    are scaled by one over the probability of being kept."""
    _device_of("dropout_add", x, residual, rng)
    _dtype_of("dropout_add", DTYPES, x, residual)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"dropout_add: x and residual of one shape expected, got {tuple(x.shape)}, "
                         f"{tuple(residual.shape)}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout_add: 0 <= p <= 1 expected, got {p}")
    if rng.dtype != torch.int64 or tuple(rng.shape) != (2,) or not rng.is_contiguous():
        raise ValueError("dropout_add: rng is a contiguous int64 tensor (seed, offset)")
    cut = round(p * 65536)
    if not _wants_grad(x, residual):
        return _dropout_add(x, residual, cut, rng)
    return DropoutAddFunction.apply(x, residual, cut, rng)
