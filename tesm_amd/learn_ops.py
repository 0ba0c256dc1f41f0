"""Operators that learn, over the C-ABI: a gated linear recurrence, float projections, the loss of given tokens.

Reached as ``hip_ops.gated_scan`` and so on.  Every operator has three forms:

* the plain call, with autograd where an input requires a gradient (once differentiable; forward-mode tangents are refused);
* ``keep=True`` (under ``torch.no_grad()``): the call also returns what its backward pass needs, as its last result;
* ``.._backward``: that backward pass by hand, the form for captured graphs.  A stream that is being captured records no
  autograd graph of these operators: the call is refused there (a leaf's gradient would be accumulated on the stream that its
  first graph was made on, which a capture cannot wait for).

As elsewhere every call queues HIP kernels on the current stream and returns tensors allocated here, workspaces included, so
that graphs captured from it share nothing.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, hip_ops
from .hip_ops import (_as_rows, _f32, _out_rows, _ptr, _same_dtype, _sequences, dt_code, on_device, raw_stream,
                      require_device)

_ACTS = {None: 0, "silu": 1, "gelu": 2}


def _act_code(act: Optional[str], what: str, pair: bool = False) -> int:
    if act not in _ACTS or (pair and act is None):
        names = ", ".join(repr(a) for a in _ACTS if a is not None or not pair)
        raise ValueError(f"{what}: act must be one of {names}; got {act!r}")
    return _ACTS[act]


def _records(what: str, keep: bool, *ts) -> bool:
    """Whether the call is one for autograd; refused where it cannot be."""
    _no_tangents(what, *ts)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in ts):
        return False
    if keep:
        raise RuntimeError(f"{what}: keep=True is for backward passes called by hand: run under torch.no_grad()")
    _no_capture(what)
    return True


def _no_tangents(what: str, *ts) -> None:
    """Forward-mode derivatives are refused: the results would have none, without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{what}: no forward-mode derivatives: an operand has a tangent")


def _by_hand(what: str, *ts) -> None:
    """A call without derivatives of its own."""
    _no_tangents(what, *ts)
    hip_ops._no_grad(what, *ts)


def _no_capture(what: str) -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: no autograd graph while a stream is captured: capture the call with keep=True and "
                           f"{what}_backward under torch.no_grad()")


def _workspace(nbytes: int, dev):
    return torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None


def _rows(t: Optional[torch.Tensor], lead: int):
    """``_as_rows`` for rows of the last dimension, contiguous ones at once (short calls are bound by the host)."""
    if t is not None and t.is_contiguous():
        return t, t.shape[-1] or 1
    return _as_rows(t, lead)


def _empty_as(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, of t's shape and dtype."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _needed(what: str, name: str, *ts) -> None:
    for t in ts:
        if t is None:
            raise ValueError(f"{what}: needs {name}")


def _like(what: str, name: str, t: Optional[torch.Tensor], shape, dtype) -> None:
    if t is not None and (t.shape != torch.Size(shape) or t.dtype != dtype):
        raise ValueError(f"{what}: {name} must be a {dtype} tensor of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


# ---------------------------------------------------------------------------
# gated linear recurrence
# ---------------------------------------------------------------------------
class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, value, write, decay, bias, state, seq_starts):
        ctx.set_materialize_grads(False)
        h, last, kept = _scan_forward(value, write, decay, bias, state, seq_starts, None, True)
        ctx.save_for_backward(value, write, decay, bias, state, seq_starts, kept)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_state):
        _no_capture("gated_scan")
        value, write, decay, bias, state, seq_starts, kept = ctx.saved_tensors
        if grad is None:
            grad = torch.zeros_like(value)
        dv, dw, dd, db, ds = _scan_backward(grad, value, write, decay, bias, state, seq_starts, kept, grad_state,
                                            ctx.needs_input_grad[3])
        if db is not None:
            db = db.to(bias.dtype).view(bias.shape)
        return dv, dw, dd, db, ds, None


def _gates(value, write, decay, bias, state, seq_starts, what, zero_rest=False):
    """The call's checked operands: the descriptor, its tensors (kept alive by the caller) and the number of sequences."""
    if value.dim() != 3 or write.shape != value.shape or decay.shape != value.shape:
        raise ValueError(f"{what}: value, write and decay must all be (B, L, C)")
    _same_dtype(what, value.dtype, write=write, decay=decay)
    B, L, C = value.shape
    code = dt_code(value.dtype)
    seq_starts, S = _sequences(seq_starts, B, what)
    _like(what, "state", state, (S, C), torch.float32)
    bias = _f32(bias, C, "decay_bias", what)
    state = state.contiguous() if state is not None else None
    (value, ld_v), (write, ld_w), (decay, ld_d) = _rows(value, 2), _rows(write, 2), _rows(decay, 2)
    require_device(value, write, decay, bias, state, seq_starts)
    d = _lib.Gates(code, B, L, C, S, value.data_ptr(), ld_v, write.data_ptr(), ld_w, decay.data_ptr(), ld_d, _ptr(bias),
                   _ptr(seq_starts), _ptr(state), int(zero_rest and S > 0))
    return d, (value, write, decay, bias, state, seq_starts), S


def _scan_forward(value, write, decay, bias, state, seq_starts, out, keep):
    what = "gated_scan"
    g, held, S = _gates(value, write, decay, bias, state, seq_starts, what, seq_starts is not None and out is None)
    B, L, C = value.shape
    dev = value.device
    if out is None:  # (rows of no sequence are set to zero by the call, where it has a sequence)
        out = _empty_as(value) if S else torch.zeros((B, L, C), dtype=value.dtype, device=dev)
        ld = max(C, 1)
    else:
        require_device(value, out)
        ld = _out_rows(out, (B, L, C), value.dtype, 2, what)
    last = torch.empty((S, C), dtype=torch.float32, device=dev)
    lib = _lib.load()
    kept = torch.empty((lib.tesm_hip_gated_scan_slots(ctypes.byref(g)), C), dtype=torch.float32, device=dev) if keep else None
    d = _lib.Recurrence(g, out.data_ptr(), ld, last.data_ptr(), _ptr(kept))
    ref = ctypes.byref(d)
    nbytes = lib.tesm_hip_gated_scan_ws_bytes(ref)
    ws = _workspace(nbytes, dev)
    on_device(dev.index, lib.tesm_hip_gated_scan, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return out, last, kept


def gated_scan(value: torch.Tensor, write: torch.Tensor, decay: torch.Tensor, decay_bias: Optional[torch.Tensor] = None, *,
               state: Optional[torch.Tensor] = None, seq_starts: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, keep: bool = False):
    """Gated linear recurrence over time; returns ``(h (B, L, C), state (S, C) float32)``.

    Per channel ``h_t = sigmoid(decay_t + decay_bias) h_(t-1) + sigmoid(write_t) tanh(value_t)``: the gates of TESM's own
    state scan, from their values before the activations.  value, write, decay (B, L, C) share a dtype and may be column slices of
    wider rows; ``decay_bias`` (C); ``state`` (S, C) float32: the states before each sequence (zeros by default).  The state
    returned is the one behind each sequence.  With ``seq_starts`` (S + 1, on the device) the operands are (1, rows, C) and hold S
    sequences one behind the other, sequence s in rows ``seq_starts[s] .. seq_starts[s + 1] - 1`` (starts outside the rows count as
    the nearest, one below an earlier one as that one); rows in front of the first and behind the last one stay as they are in
    ``out`` (zero without ``out``).  A decay of -infinity forgets, one of +infinity with a write of -infinity leaves the state
    as it is; states are float32, finite ones, and results repeat bit for bit.

    ``keep=True`` also returns what ``gated_scan_backward`` needs (float32, one row per 64).  ``out`` takes no gradients and must not
    overlap an operand.  Fewer than 2^31 rows, C below 2^24, fewer than 2^23 tiles of 64 rows of a sequence by 64 channels.
    """
    if _records("gated_scan", keep, value, write, decay, decay_bias, state):
        if out is not None:
            raise RuntimeError("gated_scan: out takes no gradients: run under torch.no_grad()")
        return _GatedScan.apply(value, write, decay, decay_bias, state, seq_starts)
    _by_hand("gated_scan", out)
    h, last, kept = _scan_forward(value, write, decay, decay_bias, state, seq_starts, out, keep)
    return (h, last, kept) if keep else (h, last)


def _scan_backward(grad, value, write, decay, bias, state, seq_starts, kept, grad_state, need_bias):
    what = "gated_scan_backward"
    _needed(what, "the gradient of h", grad)
    _needed(what, "kept, as the forward call with keep=True returned it", kept)
    g, held, S = _gates(value, write, decay, bias, state, seq_starts, what, seq_starts is not None)
    B, L, C = value.shape
    dev = value.device
    _like(what, "the gradient", grad, value.shape, value.dtype)
    _like(what, "grad_state", grad_state, (S, C), torch.float32)
    lib = _lib.load()
    _like(what, "kept", kept, (lib.tesm_hip_gated_scan_slots(ctypes.byref(g)), C), torch.float32)
    grad, ld_g = _rows(grad, 2)
    grad_state = grad_state.contiguous() if grad_state is not None else None
    kept = kept.contiguous()
    require_device(value, grad, grad_state, kept)
    new = torch.empty if S else torch.zeros
    dv, dw, dd = (new((B, L, C), dtype=value.dtype, device=dev) for _ in range(3))
    db = torch.empty((C,), dtype=torch.float32, device=dev) if need_bias else None
    ds = torch.empty((S, C), dtype=torch.float32, device=dev) if state is not None else None
    ld = max(C, 1)
    d = _lib.RecurrenceGrad(g, kept.data_ptr(), grad.data_ptr(), ld_g, _ptr(grad_state), dv.data_ptr(), ld, dw.data_ptr(), ld,
                            dd.data_ptr(), ld, _ptr(db), _ptr(ds))
    ref = ctypes.byref(d)
    nbytes = lib.tesm_hip_gated_scan_backward_ws_bytes(ref)
    ws = _workspace(nbytes, dev)
    on_device(dev.index, lib.tesm_hip_gated_scan_backward, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return dv, dw, dd, db, ds


def gated_scan_backward(grad: torch.Tensor, value: torch.Tensor, write: torch.Tensor, decay: torch.Tensor,
                        decay_bias: Optional[torch.Tensor] = None, *, kept: torch.Tensor, state: Optional[torch.Tensor] = None,
                        seq_starts: Optional[torch.Tensor] = None, grad_state: Optional[torch.Tensor] = None):
    """The gradients ``(value, write, decay, decay_bias, state)`` of ``gated_scan``, called with the same operands and ``keep=True``.

    ``grad`` (B, L, C): the gradient of h; ``grad_state`` (S, C) float32: that of the final states (zero by default).  The bias's
    and the state's are float32, None where there was none.  Rows of no sequence get zeros.
    """
    _by_hand("gated_scan_backward", grad, value, write, decay, decay_bias, state, grad_state)
    return _scan_backward(grad, value, write, decay, decay_bias, state, seq_starts, kept, grad_state, decay_bias is not None)


def gated_scan_step(value: torch.Tensor, write: torch.Tensor, decay: torch.Tensor, decay_bias: Optional[torch.Tensor] = None, *,
                    state: torch.Tensor, out: Optional[torch.Tensor] = None):
    """One token of ``gated_scan`` for B sequences: returns h (B, C); ``state`` (B, C) float32 is updated in place.

    value, write, decay (B, C) share a dtype and may be column slices of wider rows.  ``out`` must not overlap an operand.  B < 65536.
    """
    what = "gated_scan_step"
    _needed(what, "the state", state)
    if value.dim() != 2 or write.shape != value.shape or decay.shape != value.shape:
        raise ValueError(f"{what}: value, write and decay must all be (B, C)")
    _by_hand(what, value, write, decay, decay_bias, state, out)
    _same_dtype(what, value.dtype, write=write, decay=decay)
    B, C = value.shape
    code = dt_code(value.dtype)
    _like(what, "state", state, (B, C), torch.float32)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous (it is updated in place)")
    decay_bias = _f32(decay_bias, C, "decay_bias", what)
    (value, ld_v), (write, ld_w), (decay, ld_d) = _rows(value, 1), _rows(write, 1), _rows(decay, 1)
    require_device(value, write, decay, decay_bias, state, out)
    dev = value.device
    if out is None:
        out = _empty_as(value)
        ld = max(C, 1)
    else:
        ld = _out_rows(out, (B, C), value.dtype, 1, what)
    d = _lib.RecurrenceStep(code, B, C, value.data_ptr(), ld_v, write.data_ptr(), ld_w, decay.data_ptr(), ld_d, _ptr(decay_bias),
                            state.data_ptr(), out.data_ptr(), ld)
    on_device(dev.index, _lib.load().tesm_hip_gated_scan_step, ctypes.byref(d), raw_stream(dev.index))
    return out


# ---------------------------------------------------------------------------
# float projections
# ---------------------------------------------------------------------------
def _dense(x, weight, up, bias, residual, act, what):
    """The checked operands: a descriptor without outputs, its tensors, rows and the results' shape."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: x must be (.., K) and the weight (N, K); got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if K < 1:
        raise ValueError(f"{what}: rows without values")
    code = dt_code(x.dtype)
    _same_dtype(what, x.dtype, weight=weight, up=up, bias=bias, residual=residual)
    if up is not None and up.shape != weight.shape:
        raise ValueError(f"{what}: the two weights must share a shape, got {tuple(weight.shape)} and {tuple(up.shape)}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{what}: bias must hold {N} values, got {tuple(bias.shape)}")
    lead = x.shape[:-1]
    shape = (*lead, N)
    if residual is not None and residual.shape != torch.Size(shape):
        raise ValueError(f"{what}: residual must be {shape}, got {tuple(residual.shape)}")
    M = math.prod(lead)
    (x, ld_x), (residual, ld_r) = _rows(x, len(lead)), _rows(residual, len(lead))
    (weight, ld_w), (up, ld_u) = _rows(weight, 1), _rows(up, 1)
    bias = bias.contiguous() if bias is not None else None
    require_device(x, weight, up, bias, residual)
    d = _lib.Dense(code, act, M, K, N, x.data_ptr(), ld_x, weight.data_ptr(), ld_w, _ptr(up), ld_u, _ptr(bias), _ptr(residual), ld_r,
                   None, 0, None, None)
    return d, (x, weight, up, bias, residual), M, shape


def _kept_dtype(dtype):
    return torch.float32 if dtype == torch.float32 else torch.uint8


def _kept_shape(M, N, dtype):
    """What is kept of each product: float32, or 3 bytes a value (and what keeps a pair's second one's on 16 bytes)."""
    return (M, N) if dtype == torch.float32 else ((3 * M * N + 15) // 16 * 16,)


def _dense_forward(x, weight, up, bias, residual, act, keep, what):
    d, held, M, shape = _dense(x, weight, up, bias, residual, act, what)
    dev, N = x.device, shape[-1]
    y = x.new_empty(shape)
    d.y, d.ld_y = y.data_ptr(), max(N, 1)
    kept = None
    if keep and up is not None:
        kept = torch.empty((2, *_kept_shape(M, N, x.dtype)), dtype=_kept_dtype(x.dtype), device=dev).unbind()
        d.z, d.z_up = kept[0].data_ptr(), kept[1].data_ptr()
    elif keep and act:
        kept = torch.empty(_kept_shape(M, N, x.dtype), dtype=_kept_dtype(x.dtype), device=dev)
        d.z = kept.data_ptr()
    lib, ref = _lib.load(), ctypes.byref(d)
    nbytes = lib.tesm_hip_dense_ws_bytes(ref)
    ws = _workspace(nbytes, dev)
    on_device(dev.index, lib.tesm_hip_dense_forward, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return y, kept


def _dense_backward(grad, x, weight, up, kept, act, need_x, need_w, need_b, what):
    _needed(what, "the gradient of the result", grad)
    if up is not None:
        _needed(what, "kept, the two tensors that the forward call with keep=True returned",
                *(kept if isinstance(kept, (tuple, list)) and len(kept) == 2 else (None,)))
    elif act:
        _needed(what, "kept, as the forward call with keep=True returned it", kept)
    d, held, M, shape = _dense(x, weight, up, None, None, act, what)
    dev, (N, K) = x.device, weight.shape
    _like(what, "the gradient", grad, shape, x.dtype)
    kept = tuple(kept) if up is not None else (kept,) if act else ()
    for t in kept:
        _like(what, "kept", t, _kept_shape(M, N, x.dtype), _kept_dtype(x.dtype))
        if not t.is_contiguous():
            raise ValueError(f"{what}: kept must be what the forward call returned")
    grad, ld_g = _rows(grad, len(shape) - 1)
    require_device(x, grad, *kept)
    if kept:
        d.z = kept[0].data_ptr()
    if up is not None:
        d.z_up = kept[1].data_ptr()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    dw = torch.empty((N, K), dtype=x.dtype, device=dev) if need_w else None
    du = torch.empty((N, K), dtype=x.dtype, device=dev) if need_w and up is not None else None
    db = torch.empty((N,), dtype=x.dtype, device=dev) if need_b else None
    g = _lib.DenseGrad(d, grad.data_ptr(), ld_g, _ptr(dx), _ptr(dw), _ptr(du), _ptr(db))
    lib, ref = _lib.load(), ctypes.byref(g)
    nbytes = lib.tesm_hip_dense_backward_ws_bytes(ref)
    ws = _workspace(nbytes, dev)
    on_device(dev.index, lib.tesm_hip_dense_backward, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return dx, dw, du, db


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        h, kept = _dense_forward(x, w_gate, w_up, None, None, act, True, "gated_linear")
        ctx.act = act
        ctx.save_for_backward(x, w_gate, w_up, *kept)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_capture("gated_linear")
        x, w_gate, w_up, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dg, du, _ = _dense_backward(grad, x, w_gate, w_up, kept, ctx.act, need[0], need[1] or need[2], False, "gated_linear")
        return dx, dg, du, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, act: str = "silu", keep: bool = False):
    """A feed-forward block's gated pair in one kernel: ``act(x w_gate^T) * (x w_up^T)``, (.., N).

    x (.., K), w_gate and w_up (N, K) share a dtype; ``act`` is "silu" or "gelu" (the error function's form, by a polynomial that is
    1.5e-7 off at most).  Sums and the activation are float32, the result is rounded once.  float32 operands go through the matrix
    units in three bfloat16 parts, to the error of a float32 sum; an infinity among them may give NaN, and values below 2^-100 in
    magnitude keep fewer bits.  Of few rows (up to 32, float32 64) the weights are streamed once.
    Rows of more than 2^21 values may be refused.  ``keep=True`` also returns what ``gated_linear_backward`` needs (both products,
    in 24 bits where x is bfloat16).
    """
    code = _act_code(act, "gated_linear", pair=True)
    if _records("gated_linear", keep, x, w_gate, w_up):
        return _GatedLinear.apply(x, w_gate, w_up, code)
    h, kept = _dense_forward(x, w_gate, w_up, None, None, code, keep, "gated_linear")
    return (h, kept) if keep else h


def gated_linear_backward(grad: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, kept, act: str = "silu",
                          need_x: bool = True, need_weights: bool = True):
    """The gradients ``(x, w_gate, w_up)`` of ``gated_linear``, called with the same operands and ``keep=True``; those not asked
    for are None.  The gradients of the two products go into those with x and the weights in 16 bits (float32: all 24), the sums are
    float32, and the results are rounded once; where bfloat16 operands hold an infinity, gradients made with it may be NaN."""
    _by_hand("gated_linear_backward", grad, x, w_gate, w_up)
    return _dense_backward(grad, x, w_gate, w_up, kept, _act_code(act, "gated_linear_backward", pair=True), need_x, need_weights, False,
                           "gated_linear_backward")[:3]


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, kept = _dense_forward(x, weight, None, bias, residual, act, True, "fused_linear")
        ctx.act = act
        ctx.save_for_backward(x, weight, kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_capture("fused_linear")
        x, weight, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, _, db = _dense_backward(grad, x, weight, None, kept, ctx.act, need[0], need[1], need[2], "fused_linear")
        return dx, dw, db, grad if need[3] else None, None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
                 residual: Optional[torch.Tensor] = None, keep: bool = False):
    """A projection with what follows it in one kernel: ``act(x weight^T + bias) + residual``, (.., N).

    x (.., K), weight (N, K), bias (N) and residual (.., N) share a dtype; ``act`` is None, "silu" or "gelu".  Precision and few
    rows as in ``gated_linear``.  ``keep=True`` also returns what ``fused_linear_backward`` needs (the sum in front of the activation, in 24
    bits where x is bfloat16; None without an activation).
    """
    code = _act_code(act, "fused_linear")
    if _records("fused_linear", keep, x, weight, bias, residual):
        return _FusedLinear.apply(x, weight, bias, residual, code)
    y, kept = _dense_forward(x, weight, None, bias, residual, code, keep, "fused_linear")
    return (y, kept) if keep else y


def fused_linear_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, kept=None,
                          act: Optional[str] = None, need_x: bool = True, need_weight: bool = True):
    """The gradients ``(x, weight, bias)`` of ``fused_linear``, called with the same operands and ``keep=True`` (the residual's is
    ``grad`` itself); the bias's is None without one, those not asked for are.  Roundings as in ``gated_linear_backward``."""
    _by_hand("fused_linear_backward", grad, x, weight, bias)
    dx, dw, _, db = _dense_backward(grad, x, weight, None, kept, _act_code(act, "fused_linear_backward"), need_x, need_weight,
                                    bias is not None, "fused_linear_backward")
    return dx, dw, db


# ---------------------------------------------------------------------------
# log probabilities of given tokens
# ---------------------------------------------------------------------------
def _logits(logits, targets, what):
    if logits.dim() < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: logits must be (.., V) and targets (..); got {tuple(logits.shape)} and {tuple(targets.shape)}")
    if targets.dtype != torch.int64:
        raise TypeError(f"{what}: targets must be int64, got {targets.dtype}")
    if logits.shape[-1] < 1:
        raise ValueError(f"{what}: rows without logits")
    code = dt_code(logits.dtype)
    logits, ld = _rows(logits, logits.dim() - 1)
    targets = targets.contiguous()
    require_device(logits, targets)
    return code, logits, ld, targets


def _logp_forward(logits, targets, top, ignore_index, keep):
    what = "token_log_probs"
    top, V, lead = int(top), logits.shape[-1] if logits.dim() else 0, targets.shape
    if not 0 <= top <= min(64, max(V, 1)):
        raise ValueError(f"{what}: 0 to {min(64, max(V, 1))} alternatives, got {top}")
    code, x, ld, targets = _logits(logits, targets, what)
    dev, rows = x.device, targets.numel()
    logp = torch.empty(lead, dtype=torch.float32, device=dev)  # (no views of one buffer: autograd would refuse to change them in place)
    entropy = torch.empty_like(logp)
    best = torch.empty((*lead, top), dtype=torch.float32, device=dev) if top else None
    tokens = torch.empty((*lead, top), dtype=torch.int64, device=dev) if top else None
    kept = torch.empty((rows, 4), dtype=torch.float32, device=dev) if keep else None
    d = _lib.Logp(code, rows, V, top, x.data_ptr(), ld, targets.data_ptr(), int(ignore_index), logp.data_ptr(), entropy.data_ptr(),
                  _ptr(best), _ptr(tokens), _ptr(kept))
    lib, ref = _lib.load(), ctypes.byref(d)
    nbytes = lib.tesm_hip_token_log_probs_ws_bytes(ref)
    ws = _workspace(nbytes, dev)
    on_device(dev.index, lib.tesm_hip_token_log_probs, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return logp, entropy, best, tokens, kept


def _logp_backward(grad, grad_entropy, logits, targets, kept, ignore_index):
    what = "token_log_probs_backward"
    _needed(what, "kept, as the forward call with keep=True returned it", kept)
    lead = targets.shape
    _like(what, "the log probabilities' gradient", grad, lead, torch.float32)
    _like(what, "the entropies' gradient", grad_entropy, lead, torch.float32)
    code, x, ld, targets = _logits(logits, targets, what)
    _like(what, "kept", kept, (targets.numel(), 4), torch.float32)
    grad = grad.contiguous() if grad is not None else None
    grad_entropy = grad_entropy.contiguous() if grad_entropy is not None else None
    kept = kept.contiguous()
    require_device(x, grad, grad_entropy, kept)
    dev, V = x.device, x.shape[-1]
    out = torch.empty(logits.shape, dtype=x.dtype, device=dev)
    d = _lib.LogpGrad(code, targets.numel(), V, x.data_ptr(), ld, targets.data_ptr(), int(ignore_index), kept.data_ptr(), _ptr(grad),
                      _ptr(grad_entropy), out.data_ptr(), V)
    on_device(dev.index, _lib.load().tesm_hip_token_log_probs_backward, ctypes.byref(d), raw_stream(dev.index))
    return out


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, ignore_index):
        ctx.set_materialize_grads(False)
        logp, entropy, best, tokens, kept = _logp_forward(logits, targets, top, ignore_index, True)
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(logits, targets, kept)
        if top:
            ctx.mark_non_differentiable(best, tokens)
        return logp, entropy, best, tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_entropy, _best, _tokens):
        _no_capture("token_log_probs")
        logits, targets, kept = ctx.saved_tensors
        return _logp_backward(grad, grad_entropy, logits, targets, kept, ctx.ignore_index), None, None, None


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, ignore_index: int = -100, keep: bool = False):
    """Log probabilities of given tokens: ``(log_probs (..), entropy (..), top_log_probs (.., top), top_tokens (.., top))``.

    ``logits`` (.., V), ``targets`` (..) int64.  ``log_probs`` is ``log_softmax(logits)`` at the target, 0 where the target is
    ``ignore_index``; ``entropy`` that of the row's distribution, of every row; both float32, exact to a float32 rounding and the sum's
    own error at every offset of the logits.  With ``top`` (at most 64) the row's largest log probabilities and their tokens follow in
    falling order, equal ones by token (None without).  A logit of -infinity is a masked token.  Rows with a NaN or +infinite logit, or
    none above -infinity, give NaN, and so does any other target outside the vocabulary, which sets bit 2 of ``device_status``.
    Fewer than 2^24 rows.
    Gradients flow through ``log_probs`` and ``entropy``.  ``keep=True`` also returns what ``token_log_probs_backward`` needs.
    """
    if _records("token_log_probs", keep, logits):
        return _TokenLogProbs.apply(logits, targets, int(top), int(ignore_index))
    out = _logp_forward(logits, targets, top, ignore_index, keep)
    return out if keep else out[:4]


def token_log_probs_backward(grad: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor], logits: torch.Tensor,
                             targets: torch.Tensor, *, kept: torch.Tensor, ignore_index: int = -100):
    """The gradient of the logits of ``token_log_probs``, called with the same operands and ``keep=True``; ``grad`` and
    ``grad_entropy`` (..) float32 are those of its first two results (None: zero)."""
    _by_hand("token_log_probs_backward", grad, grad_entropy, logits)
    return _logp_backward(grad, grad_entropy, logits, targets, kept, ignore_index)
