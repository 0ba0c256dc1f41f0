"""Tensor-level wrappers over the C-ABI (device memory and streams come from torch).

Every function queues HIP kernels on the current torch stream of the tensors'
device and returns torch tensors allocated here.  Nothing computes on the host
and nothing falls back to torch ops: a missing library raises.

Row-major 2-D operands may have a row stride (``x.stride(0)``) larger than their
width as long as the last dimension is contiguous, so slices of a wider
projection output are passed without copies.
"""
from __future__ import annotations

import array
import ctypes
import functools
import math
from typing import Optional

import torch

from . import _lib

_DT = {torch.float32: 0, torch.bfloat16: 1}


def dt_code(dtype: torch.dtype) -> int:
    try:
        return _DT[dtype]
    except KeyError:
        raise TypeError(f"hip backend supports float32 and bfloat16, got {dtype}") from None


def _p(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """2-D view with a contiguous last dimension (copies only if needed)."""
    if x.dim() != 2:
        raise ValueError("expected a 2-D tensor")
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def require_device(*ts):
    """Every tensor handed to a kernel must live on one ROCm device: a host pointer would be
    dereferenced by the GPU."""
    first, dev = None, -1
    for t in ts:
        if t is None:
            continue
        d = t.get_device()  # the index, -1 on the host: cheaper per call than building and comparing devices
        if d < 0 or not t.is_cuda:
            raise RuntimeError(f"hip backend ops need tensors on a ROCm device, got one on {t.device}")
        if first is None:
            first, dev = t, d
        elif d != dev:
            raise RuntimeError(f"hip backend ops need all tensors on one device, got {first.device} and {t.device}")


def raw_stream(index: int) -> int:
    """The raw handle of device ``index``'s current stream (``torch.cuda.current_stream(..).cuda_stream``
    without building a Stream object, which costs over a microsecond per call)."""
    return torch._C._cuda_getCurrentRawStream(index)


def on_device(index: int, fn, *args) -> None:
    """``fn(*args)`` with device ``index`` current (switched only if it is not already), its return code checked."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _lib.check(rc)


def kpad(K: int) -> int:
    return int(_lib.load().tesm_hip_kpad(K))


@functools.lru_cache(maxsize=1024)
def round_dtype(v: float, dtype: torch.dtype) -> float:
    """The float value that torch uses for a Python scalar compared against a ``dtype`` tensor."""
    return float(torch.tensor(v, dtype=torch.float32).to(dtype).float())


# ---------------------------------------------------------------------------
# BitLinear pieces
# ---------------------------------------------------------------------------
def quant_act(x: torch.Tensor, eps: float = 1e-5, layout: int = 1, ldq: Optional[int] = None):
    """Per-token int8 codes of ``x`` (M, K): returns (codes (M, ldq), s_x (M), rowsum (M))."""
    lib = _lib.load()
    x = _rows(x)
    require_device(x)
    M, K = x.shape
    ldq = kpad(K) if ldq is None else ldq
    q = torch.empty((M, ldq), dtype=torch.int8, device=x.device)
    s = torch.empty((M,), dtype=torch.float32, device=x.device)
    rs = torch.empty((M,), dtype=torch.int32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(lib.tesm_hip_quant_act_i8(_p(x), dt_code(x.dtype), M, K, x.stride(0), eps, layout, _p(q), ldq,
                                             _p(s), _p(rs), _stream(x)))
    return q, s, rs


def absmean_scale(w: torch.Tensor, eps: float = 1e-5):
    """(s_w, c_w) device scalars: s_w = 1/max(mean|w|, eps), c_w = 1/s_w, rounded to w's dtype."""
    lib = _lib.load()
    w = w.contiguous()
    require_device(w)
    ws = torch.empty((int(lib.tesm_hip_absmean_ws_bytes()),), dtype=torch.uint8, device=w.device)
    s_w = torch.empty((1,), dtype=torch.float32, device=w.device)
    c_w = torch.empty((1,), dtype=torch.float32, device=w.device)
    with torch.cuda.device(w.device):
        _lib.check(lib.tesm_hip_absmean_scale(_p(w), dt_code(w.dtype), w.numel(), eps, _p(ws), _p(s_w), _p(c_w),
                                              _stream(w)))
    return s_w, c_w


def pack_weight(w: torch.Tensor, s_w: torch.Tensor, per_row: bool = False, ldp: Optional[int] = None):
    """Ternary codes of ``w`` (N, K) at scale ``s_w`` packed 4 per byte: (N, ldp) uint8.

    ``ldp`` defaults to kpad(K)/4 (the layout the products read); pass
    ``ldp=ceil(K/4)`` for the canonical export layout.
    """
    lib = _lib.load()
    w = _rows(w)
    require_device(w, s_w)
    N, K = w.shape
    ldp = kpad(K) // 4 if ldp is None else ldp
    packed = torch.empty((N, ldp), dtype=torch.uint8, device=w.device)
    s_w = s_w.to(torch.float32).contiguous()
    with torch.cuda.device(w.device):
        _lib.check(lib.tesm_hip_pack_w_i2(_p(w), dt_code(w.dtype), N, K, w.stride(0), _p(s_w), int(per_row),
                                          _p(packed), ldp, _stream(w)))
    return packed


def unpack_weight(packed: torch.Tensor, K: int):
    lib = _lib.load()
    packed = _rows(packed)
    require_device(packed)
    N = packed.shape[0]
    codes = torch.empty((N, K), dtype=torch.int8, device=packed.device)
    with torch.cuda.device(packed.device):
        _lib.check(lib.tesm_hip_unpack_w_i2(_p(packed), N, K, packed.stride(0), _p(codes), K, _stream(packed)))
    return codes


def bitlinear(q, s_x, rowsum, packed, c_w, N: int, K: int, out_dtype: torch.dtype, bias=None,
              c_w_per_row: bool = False, acc_dump: bool = False, out: Optional[torch.Tensor] = None):
    """out (M, N) = (q . codes) / s_x * c_w (+ bias); optionally also the int32 accumulators."""
    lib = _lib.load()
    M = q.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=q.device)
    acc = torch.empty((M, N), dtype=torch.int32, device=q.device) if acc_dump else None
    require_device(q, s_x, rowsum, packed, c_w, bias, out, acc)
    with torch.cuda.device(q.device):
        _lib.check(lib.tesm_hip_bitlinear_i2(_p(q), q.stride(0), _p(s_x), _p(rowsum), _p(packed), packed.stride(0),
                                             _p(c_w), int(c_w_per_row), _p(bias), M, N, K, _p(out),
                                             dt_code(out.dtype), out.stride(0), _p(acc), _stream(q)))
    return (out, acc) if acc_dump else out


@functools.lru_cache(maxsize=256)
def _bitlinear_ws_bytes(M: int, K: int) -> int:
    return int(_lib.load().tesm_hip_bitlinear_fwd_ws_bytes(M, K))


def bitlinear_fwd(x, packed, c_w, N: int, eps: float = 1e-5, bias=None, c_w_per_row: bool = False,
                  fuse: bool = True, out: Optional[torch.Tensor] = None):
    """BitLinear forward from raw activations x (M, K): codes + product in one C-ABI call (fused
    for decode-size M when ``fuse``); out (M, N) in x's dtype."""
    lib = _lib.load()
    x = _rows(x)
    M, K = x.shape
    dev = x.device
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=dev)
    require_device(x, packed, c_w, bias, out)
    nbytes = _bitlinear_ws_bytes(M, K)
    from .tesm import workspace
    raw = raw_stream(dev.index)
    ws = workspace(dev, nbytes, raw=raw)
    # (pointers as plain integers: the signatures convert them, a c_void_p object per argument would cost more)
    on_device(dev.index, lib.tesm_hip_bitlinear_fwd, x.data_ptr(), dt_code(x.dtype), x.stride(0), eps,
              packed.data_ptr(), packed.stride(0), c_w.data_ptr(), int(c_w_per_row),
              bias.data_ptr() if bias is not None else None, M, N, K, out.data_ptr(), dt_code(out.dtype),
              out.stride(0), int(fuse), ws.data_ptr(), nbytes, raw)
    return out


# ---------------------------------------------------------------------------
# diagnostics: launch log, device status, decision taps
# ---------------------------------------------------------------------------
class launch_log:
    """Context manager recording the kernel instantiations launched inside it::

        with hip_ops.launch_log() as log:
            layer(u)
        assert "scan_lb_kernel<1,1,1,16,8>" in log.kernels
    """

    def __enter__(self):
        self.kernels = []
        _lib.check(_lib.load().tesm_hip_launch_log(1))
        return self

    def __exit__(self, *exc):
        lib = _lib.load()
        n = int(lib.tesm_hip_launch_log_read(None, 0, 0))
        buf = ctypes.create_string_buffer(n + 1)
        lib.tesm_hip_launch_log_read(buf, n + 1, 1)
        lib.tesm_hip_launch_log(0)
        self.kernels = [k for k in buf.value.decode().split("\n") if k]
        return False


def stream_copy(dst: torch.Tensor, src: torch.Tensor) -> None:
    """Copy src's bytes into dst with the library's streaming copy kernel (a bandwidth reference)."""
    require_device(dst, src)
    if not (dst.is_contiguous() and src.is_contiguous()):
        raise ValueError("stream_copy: tensors must be contiguous")
    n = src.numel() * src.element_size()
    if dst.numel() * dst.element_size() < n:
        raise ValueError("stream_copy: destination too small")
    with torch.cuda.device(src.device):
        _lib.check(_lib.load().tesm_hip_stream_copy(_p(dst), _p(src), n, _stream(src)))


def device_status(clear: bool = True) -> int:
    """The device status word of the current device (bit 0: a scan look-back gave up; bit 1: a parent of
    ``reorder_rows`` was none of the beams); synchronises."""
    v = ctypes.c_uint32(0)
    lib = _lib.load()
    _lib.check(lib.tesm_hip_device_status(ctypes.byref(v), int(clear)))
    return int(v.value)


def debug_scan_spin_limit(limit: int) -> None:
    _lib.check(_lib.load().tesm_hip_debug_scan_spin_limit(int(limit)))


def set_taps(**bufs) -> None:
    """Point the decision taps at device tensors (q_te, s_te, q_c, s_c, q_y, s_y, tern, wts); no
    arguments stops tapping."""
    lib = _lib.load()
    if not bufs:
        _lib.check(lib.tesm_hip_debug_taps(None))
        return
    require_device(*bufs.values())
    t = _lib.Taps(**{k: (v.data_ptr() if v is not None else None) for k, v in bufs.items()})
    _lib.check(lib.tesm_hip_debug_taps(ctypes.byref(t)))


# ---------------------------------------------------------------------------
# scan / RoPE / entanglement
# ---------------------------------------------------------------------------
def scan(decay: torch.Tensor, update: torch.Tensor, chunk_size: int = 16, h0: Optional[torch.Tensor] = None,
         out_dtype: Optional[torch.dtype] = None):
    """States of h_t = d_t h_{t-1} + u_t for (B, L, C) inputs; returns (states, h_final fp64)."""
    lib = _lib.load()
    if decay.shape != update.shape or decay.dim() != 3:
        raise ValueError("decay and update must both be (B, L, C)")
    if decay.dtype != update.dtype:
        raise TypeError("decay and update must share a dtype")
    decay, update = decay.contiguous(), update.contiguous()
    require_device(decay, update, h0)
    B, L, C = decay.shape
    out_dtype = out_dtype or decay.dtype
    states = torch.empty((B, L, C), dtype=out_dtype, device=decay.device)
    h_final = torch.empty((B, C), dtype=torch.float64, device=decay.device)
    if h0 is not None:
        h0 = h0.to(dtype=torch.float64).contiguous()
    nbytes = int(lib.tesm_hip_scan_ws_bytes(B, L, C, chunk_size))
    ws = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device=decay.device)
    with torch.cuda.device(decay.device):
        _lib.check(lib.tesm_hip_scan(_p(decay), C, _p(update), C, dt_code(decay.dtype), B, L, C, chunk_size, _p(h0),
                                     _p(states), C, dt_code(out_dtype), _p(h_final), _p(ws), nbytes, _stream(decay)))
    return states, h_final


def rope_table(L: int, R: int, dtype: torch.dtype, device, base: float = 10000.0, pos_offset: int = 0):
    """(L, R/2, 2) float32 (cos, sin) of positions pos_offset..pos_offset+L-1, rounded to ``dtype``."""
    lib = _lib.load()
    tab = torch.empty((max(L, 1), R // 2, 2), dtype=torch.float32, device=device)
    with torch.cuda.device(tab.device):
        _lib.check(lib.tesm_hip_rope_table(_p(tab), L, R, pos_offset, float(base), dt_code(dtype), _stream(tab)))
    return tab


def window_bias(bias, H: int, W: int, dt, device):
    """The window bias as the entanglement kernels take it: float32 (H, W) on ``device``, each value rounded
    to the layer dtype ``dt`` first (the reference adds the bias in that dtype)."""
    return bias.reshape(H, W).to(device=device, dtype=dt).to(torch.float32).contiguous()


def _ready_bias(bias, H: int, W: int, dt, device, bias_rounded: bool):
    if not bias_rounded:
        return window_bias(bias, H, W, dt, device)
    if bias.dtype != torch.float32 or bias.numel() != H * W or not bias.is_contiguous() or bias.device != device:
        raise ValueError("bias_rounded=True needs the float32 (H, W) contiguous tensor window_bias() returns, "
                         "on the states' device")
    return bias


def local_ent(q, k, rope, S, bias, W: int, thr: float, ent_scale: float, q_add=None, mimo: bool = False, H: int = 1,
              outputs=("avg",), want_tern: bool = False, bias_rounded: bool = False):
    """Window entanglement over (B, L, H*R) queries/keys and (B, L, H*D) states.

    ``bias`` is (H, W) (or (W,)) in any float dtype; it is rounded to the states' dtype (with
    ``bias_rounded`` it is already ``window_bias()``'s result and is passed as it is, so the call
    launches no conversion).  ``thr`` is rounded to that dtype too.  Returns a dict of the requested
    outputs among ``avg``, ``e``, ``c``, ``e_tanh`` (and ``tern`` if ``want_tern``).
    """
    lib = _lib.load()
    B, L, HR = q.shape
    D = S.shape[-1] // H
    R = HR // H
    dt = S.dtype
    q = q.reshape(B * L, HR)
    k = k.reshape(B * L, HR)
    q, k = _rows(q), _rows(k)
    S2 = _rows(S.reshape(B * L, H * D))
    qa = _rows(q_add.reshape(B * L, HR)) if q_add is not None else None
    # small parameter: accepted from any device, copied next to the states
    bias_f = _ready_bias(bias, H, W, dt, S.device, bias_rounded)
    weff = W if mimo else min(W, L)
    outs = {name: torch.empty((B, L, H * D), dtype=dt, device=S.device) for name in outputs}
    tern = torch.empty((B, L, H, weff), dtype=torch.int8, device=S.device) if want_tern else None
    nbytes = int(lib.tesm_hip_local_ent_ws_bytes(B, L, H, weff))
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=S.device)
    require_device(q, k, rope, qa, bias_f, S2, tern, ws, *outs.values())
    with torch.cuda.device(S.device):
        _lib.check(lib.tesm_hip_local_ent(
            _p(q), q.stride(0), _p(k), k.stride(0), _p(rope), _p(qa), qa.stride(0) if qa is not None else 0,
            _p(bias_f), _p(S2), S2.stride(0), dt_code(dt), int(mimo), B, L, H, R, D, W, round_dtype(thr, dt),
            float(ent_scale), _p(outs.get("avg")), _p(outs.get("e")), _p(outs.get("c")), _p(outs.get("e_tanh")),
            H * D, _p(tern), _p(ws), nbytes, _stream(S)))
    if want_tern:
        outs["tern"] = tern
    return outs



def local_ent_quant(q, k, rope, S, bias, W: int, thr: float, ent_scale: float, eps: float = 1e-5, q_add=None,
                    want_floats: bool = False, want_tern: bool = False, bias_rounded: bool = False):
    """Fused SISO entanglement + int8 codes of tanh(E) and C (the state_proj / ent_proj inputs).
    ``bias`` as in ``local_ent`` (one head).

    Returns a dict with ``te`` and ``c`` = (codes (M, kpad(D)) layout 1, scales (M), rowsums (M)),
    plus ``e_tanh`` / ``c_float`` / ``tern`` when asked for.
    """
    lib = _lib.load()
    B, L, R = q.shape
    D = S.shape[-1]
    dt = S.dtype
    q2, k2 = _rows(q.reshape(B * L, R)), _rows(k.reshape(B * L, R))
    S2 = _rows(S.reshape(B * L, D))
    qa = _rows(q_add.reshape(B * L, R)) if q_add is not None else None
    bias_f = _ready_bias(bias, 1, W, dt, S.device, bias_rounded)
    M, ldq = B * L, kpad(D)
    dev = S.device
    te = (torch.empty((M, ldq), dtype=torch.int8, device=dev), torch.empty(M, device=dev),
          torch.empty(M, dtype=torch.int32, device=dev))
    cc = (torch.empty((M, ldq), dtype=torch.int8, device=dev), torch.empty(M, device=dev),
          torch.empty(M, dtype=torch.int32, device=dev))
    et = torch.empty((B, L, D), dtype=dt, device=dev) if want_floats else None
    cf = torch.empty((B, L, D), dtype=dt, device=dev) if want_floats else None
    tern = torch.empty((B, L, min(W, L)), dtype=torch.int8, device=dev) if want_tern else None
    require_device(q2, k2, rope, qa, bias_f, S2, *te, *cc, et, cf, tern)
    d = _lib.EntQuant()
    d.dt = dt_code(dt)
    d.B, d.L, d.R, d.D, d.W = B, L, R, D, W
    d.thr, d.ent_scale, d.eps = round_dtype(thr, dt), float(ent_scale), float(eps)
    d.q, d.ld_q, d.k, d.ld_k = q2.data_ptr(), q2.stride(0), k2.data_ptr(), k2.stride(0)
    d.rope = rope.data_ptr()
    d.q_add, d.ld_qadd = (qa.data_ptr(), qa.stride(0)) if qa is not None else (None, 0)
    d.bias, d.S, d.ld_s = bias_f.data_ptr(), S2.data_ptr(), S2.stride(0)
    d.q_te, d.s_te, d.rs_te = (t.data_ptr() for t in te)
    d.q_c, d.s_c, d.rs_c = (t.data_ptr() for t in cc)
    d.ldq = ldq
    d.e_tanh = et.data_ptr() if et is not None else None
    d.c_out = cf.data_ptr() if cf is not None else None
    d.ld_out = D
    d.tern = tern.data_ptr() if tern is not None else None
    with torch.cuda.device(dev):
        _lib.check(lib.tesm_hip_local_ent_quant(ctypes.byref(d), _stream(S)))
    out = {"te": te, "c": cc}
    if want_floats:
        out["e_tanh"], out["c_float"] = et, cf
    if want_tern:
        out["tern"] = tern
    return out


def output_gate(te, cc, sp_packed, sp_cw, ep_packed, ep_cw, local, gate, d_state: int, eps: float = 1e-5,
                quantize: bool = True, want_y: bool = True):
    """y = local + sigmoid(gate) * state_proj(tanh E) + ent_proj(C) from code triples ``te``/``cc``.

    ``local``/``gate`` are (M, d_model) views (row stride allowed).  With ``quantize`` the kernel
    also returns y's out_proj codes (codes, scales, rowsums).
    """
    lib = _lib.load()
    local, gate = _rows(local), _rows(gate)
    M, dm = local.shape
    dt = local.dtype
    dev = local.device
    y = torch.empty((M, dm), dtype=dt, device=dev) if (want_y or not quantize) else None
    qy = None
    if quantize:
        ldq = kpad(dm)
        qy = (torch.empty((M, ldq), dtype=torch.int8, device=dev), torch.empty(M, device=dev),
              torch.empty(M, dtype=torch.int32, device=dev))
    require_device(*te, *cc, sp_packed, sp_cw, ep_packed, ep_cw, local, gate, y, *(qy or ()))
    d = _lib.OutputGate()
    d.dt = dt_code(dt)
    d.M, d.d_model, d.d_state, d.eps = M, dm, d_state, float(eps)
    d.q_te, d.ldq_te, d.s_te, d.rs_te = te[0].data_ptr(), te[0].stride(0), te[1].data_ptr(), te[2].data_ptr()
    d.q_c, d.ldq_c, d.s_c, d.rs_c = cc[0].data_ptr(), cc[0].stride(0), cc[1].data_ptr(), cc[2].data_ptr()
    d.state_proj = _lib.Linear(sp_packed.data_ptr(), sp_packed.stride(0), sp_cw.data_ptr(), 0)
    d.ent_proj = _lib.Linear(ep_packed.data_ptr(), ep_packed.stride(0), ep_cw.data_ptr(), 0)
    d.local, d.ld_local, d.gate, d.ld_gate = local.data_ptr(), local.stride(0), gate.data_ptr(), gate.stride(0)
    d.y, d.ld_y = (y.data_ptr(), dm) if y is not None else (None, 0)
    if qy is not None:
        d.q_y, d.ldq_y, d.s_y, d.rs_y = qy[0].data_ptr(), qy[0].stride(0), qy[1].data_ptr(), qy[2].data_ptr()
    with torch.cuda.device(dev):
        _lib.check(lib.tesm_hip_output_gate_i2(ctypes.byref(d), _stream(local)))
    return y, qy


# ---------------------------------------------------------------------------
# selective state space pieces: short causal convolution, selective scan, their one-token step
# ---------------------------------------------------------------------------
def _no_grad(what: str, *ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what}: the hip kernels are forward-only: run under torch.no_grad()")


def _row_pitch(x: torch.Tensor, lead: int):
    """The pitch in elements of ``x``'s rows (the first ``lead`` dimensions flattened into one row axis, the others
    one contiguous row), or None where ``x`` is not laid out in such rows."""
    shape, strides = x.shape, x.stride()
    width = 1
    for d in range(len(shape) - 1, lead - 1, -1):
        n = shape[d]
        if n != 1 and strides[d] != width:
            return None if x.numel() else max(math.prod(shape[lead:]), 1)
        width *= n
    pitch, span = -1, 0  # from the last row dimension that has more than one entry
    for d in range(lead - 1, -1, -1):
        n = shape[d]
        if n == 1:
            continue
        if n == 0 or width == 0:
            return max(width, 1)
        if pitch < 0:
            pitch = span = strides[d]
        elif strides[d] != span:
            return None
        span *= n
    if pitch < 0:
        return width
    return pitch if pitch >= width else None


def _as_rows(x: Optional[torch.Tensor], lead: int):
    """``x`` and its row pitch, copied only where it is not laid out in rows."""
    if x is None:
        return None, 0
    pitch = _row_pitch(x, lead)
    if pitch is None:
        x = x.contiguous()
        pitch = _row_pitch(x, lead)
    return x, pitch


def _out_rows(out: torch.Tensor, shape, dtype, lead: int, what: str) -> int:
    pitch = _row_pitch(out, lead) if out.dtype == dtype and out.shape == torch.Size(shape) else None
    if pitch is None:
        raise ValueError(f"{what}: out must be a {dtype} tensor of shape {tuple(shape)} in contiguous rows, each at the "
                         "same distance from the last")
    return pitch


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _f32(t: Optional[torch.Tensor], n: int, name: str, what: str):
    if t is None:
        return None
    if t.numel() != n:
        raise ValueError(f"{what}: {name} must hold {n} values, got {tuple(t.shape)}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _sequences(seq_starts: Optional[torch.Tensor], B: int, what: str):
    """``seq_starts`` as the kernels take it (int32, contiguous), and the number of sequences."""
    if seq_starts is None:
        return None, B
    if B != 1:
        raise ValueError(f"{what}: packed sequences lie in one row axis: with seq_starts the first dimension must be 1")
    if seq_starts.dim() != 1 or seq_starts.numel() < 1 or seq_starts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: seq_starts must be a 1-D int32 or int64 tensor of one entry more than sequences")
    S = seq_starts.numel() - 1
    if seq_starts.dtype == torch.int64:  # (starts past int32 are past the rows as well, and must not wrap)
        seq_starts = seq_starts.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return seq_starts.contiguous(), S


def _same_dtype(what: str, dtype: torch.dtype, **ts) -> None:
    for name, t in ts.items():
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, expected {dtype} as the first argument")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, silu: bool = True,
                state: Optional[torch.Tensor] = None, seq_starts: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None):
    """Short causal convolution over time, one filter per channel; returns ``(y (B, L, C), state (S, W - 1, C))``.

    ``y[b, t, c] = silu(bias[c] + sum_j weight[c, j] x[b, t - W + 1 + j, c])`` (``silu=False``: no activation) for x
    (B, L, C) and ``weight`` (C, W), 2 <= W <= 8, summed in float32.  With ``seq_starts`` (S + 1, on the device, not
    decreasing) x is (1, rows, C) and holds S sequences one behind the other, sequence s in rows
    ``seq_starts[s] .. seq_starts[s + 1] - 1`` (starts past the rows count as their end); rows in front of the first and
    behind the last one stay as they are in ``out`` (zero without ``out``).  ``state`` (S, W - 1, C): the rows before each
    sequence, oldest first, zeros by default.  The state returned holds each sequence's last W - 1 rows.  ``out`` may be
    columns beside x in wider rows, but an output that overlaps an input is refused.  x, state and y share a dtype; weight
    and bias share one (float32 or bfloat16) of their own.
    """
    if x.dim() != 3 or weight.dim() != 2 or weight.shape[0] != x.shape[2]:
        raise ValueError("causal_conv: x must be (B, L, C) and weight (C, W)")
    _no_grad("causal_conv", x, weight, bias, state, out)
    B, L, C = x.shape
    W = weight.shape[1]
    if not 2 <= W <= 8:
        raise ValueError(f"causal_conv: the filter must have 2 to 8 taps, got {W}")
    seq_starts, S = _sequences(seq_starts, B, "causal_conv")
    _same_dtype("causal_conv", x.dtype, state=state)
    _same_dtype("causal_conv", weight.dtype, bias=bias)
    if bias is not None and bias.numel() != C:
        raise ValueError(f"causal_conv: bias must hold {C} values, got {tuple(bias.shape)}")
    if state is not None and state.shape != (S, W - 1, C):
        raise ValueError(f"causal_conv: state must be {(S, W - 1, C)}, got {tuple(state.shape)}")
    codes = dt_code(x.dtype), dt_code(weight.dtype)
    weight = weight.contiguous()
    bias = bias.contiguous() if bias is not None else None
    state = state.contiguous() if state is not None else None
    x, ld = _as_rows(x, 2)
    require_device(x, weight, bias, state, seq_starts, out)
    if out is None:
        out = (torch.zeros if seq_starts is not None else torch.empty)((B, L, C), dtype=x.dtype, device=x.device)
    if out.data_ptr() == x.data_ptr() and x.numel():
        raise ValueError("causal_conv: out must not be x")
    new = torch.empty((S, W - 1, C), dtype=x.dtype, device=x.device)
    # (fields in the descriptor's order)
    d = _lib.Conv(*codes, B, L, C, W, S, int(silu), x.data_ptr(), ld, weight.data_ptr(), _ptr(bias), _ptr(seq_starts),
                  _ptr(state), out.data_ptr(), _out_rows(out, (B, L, C), x.dtype, 2, "causal_conv"), new.data_ptr())
    on_device(x.device.index, _lib.load().tesm_hip_causal_conv, ctypes.byref(d), raw_stream(x.device.index))
    return out, new


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, softplus: bool = True,
                   state: Optional[torch.Tensor] = None, seq_starts: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None):
    """Selective state space scan; returns ``(y (B, L, H, P), state (S, H, P, N) float32)``.

    Per head h with its group's B and C (H heads share G groups), over rows t:
    ``d = softplus(dt + dt_bias)`` (``softplus=False``: ``dt + dt_bias``), ``state = exp(d A) state + d x B^T``,
    ``y = state C + D x``, times ``silu(z)`` with ``z``.  x, z: (B, L, H, P); dt: (B, L, H); B, C: (B, L, G, N),
    N <= 256; A, D, dt_bias: (H); ``state`` (S, H, P, N) float32: the states before each sequence (zeros by default).
    ``seq_starts`` and ``out`` as in ``causal_conv``.  x, dt, B, C, z and y share a dtype and may be column slices of
    wider rows.  States and sums are float32; with bfloat16 operands the decayed scores and the states that rows read go
    into their products as two bfloat16 parts (16 bits).  A NaN or an infinity in row t reaches no row before it; an infinite
    x or state may leave NaN where the formula's value is infinite, and so may states beyond 2^118 in magnitude.  Fewer than
    65536 sequences, H * P and row pitches below 2^24.
    """
    if x.dim() != 4 or dt.dim() != 3 or B.dim() != 4 or dt.shape != x.shape[:3] or B.shape[:2] != x.shape[:2] or \
            C.shape != B.shape or (z is not None and z.shape != x.shape):
        raise ValueError("selective_scan: x and z must be (B, L, H, P), dt (B, L, H), B and C (B, L, G, N)")
    _no_grad("selective_scan", x, dt, A, B, C, D, z, dt_bias, state, out)
    nb, L, H, P = x.shape
    G, N = B.shape[2:]
    if H < 1 or P < 1 or G < 1 or N < 1 or H % G:
        raise ValueError(f"selective_scan: {H} heads of {P} channels do not share {G} groups of {N} states evenly")
    if N > 256:
        raise ValueError(f"selective_scan: at most 256 states, got {N}")
    _same_dtype("selective_scan", x.dtype, dt=dt, B=B, C=C, z=z)
    seq_starts, S = _sequences(seq_starts, nb, "selective_scan")
    if state is not None and (state.shape != (S, H, P, N) or state.dtype != torch.float32):
        raise ValueError(f"selective_scan: state must be float32 {(S, H, P, N)}, got {state.dtype} {tuple(state.shape)}")
    A, D, dt_bias = (_f32(t, H, n, "selective_scan") for t, n in ((A, "A"), (D, "D"), (dt_bias, "dt_bias")))
    state = state.contiguous() if state is not None else None
    code = dt_code(x.dtype)
    (x, ld_x), (dt, ld_dt), (B, ld_b), (C, ld_c), (z, ld_z) = (_as_rows(x, 2), _as_rows(dt, 2), _as_rows(B, 2),
                                                              _as_rows(C, 2), _as_rows(z, 2))
    dev = x.device
    require_device(x, dt, A, B, C, D, z, dt_bias, state, seq_starts, out)
    if out is None:
        out = (torch.zeros if seq_starts is not None else torch.empty)((nb, L, H, P), dtype=x.dtype, device=dev)
    px, pb, pc, pz, py = x.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), out.data_ptr()
    if py in (px, pb, pc, pz) and x.numel():
        raise ValueError("selective_scan: out must not be one of the operands")
    new = torch.empty((S, H, P, N), dtype=torch.float32, device=dev)
    # (fields in the descriptor's order)
    d = _lib.Ssm(code, nb, L, H, P, G, N, S, int(softplus), px, ld_x, dt.data_ptr(), ld_dt, A.data_ptr(), pb, ld_b, pc, ld_c,
                 _ptr(D), pz, ld_z, _ptr(dt_bias), _ptr(seq_starts), _ptr(state), py,
                 _out_rows(out, (nb, L, H, P), x.dtype, 2, "selective_scan"), new.data_ptr())
    lib = _lib.load()
    ref = ctypes.byref(d)
    nbytes = lib.tesm_hip_selective_scan_ws_bytes(ref)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None
    on_device(dev.index, lib.tesm_hip_selective_scan, ref, _ptr(ws), nbytes, raw_stream(dev.index))
    return out, new


def selective_scan_step(row: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, state: torch.Tensor,
                        conv_weight: Optional[torch.Tensor] = None, conv_bias: Optional[torch.Tensor] = None,
                        conv_state: Optional[torch.Tensor] = None, *, n_groups: int = 1,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None, softplus: bool = True, silu: bool = True,
                        out: Optional[torch.Tensor] = None, conv_state_out: Optional[torch.Tensor] = None):
    """One token of ``causal_conv`` and ``selective_scan``: returns ``(y (B, H, P), conv_state)``.

    ``row`` (B, H * P + 2 * G * N) holds the token's x, B and C before the convolution, whose result stays in float32;
    without ``conv_weight`` the row is used as it is.  ``state`` (B, H, P, N) float32 is updated in place;
    ``conv_state`` (B, W - 1, H * P + 2 * G * N) is read, and the state after the token is returned in a tensor of its
    own (``conv_state_out``, which must not be ``conv_state``; captured graphs alternate between two).  dt (B, H),
    z (B, H, P); the rest as in ``selective_scan``.  An output that overlaps another argument
    is refused.  B < 65536, P <= 4096.
    """
    if state.dim() != 4 or row.dim() != 2 or row.shape[0] != state.shape[0] or dt.shape != state.shape[:2] or \
            (z is not None and z.shape != state.shape[:3]):
        raise ValueError("selective_scan_step: row must be (B, channels), dt (B, H), z (B, H, P) and state (B, H, P, N)")
    _no_grad("selective_scan_step", row, dt, A, state, conv_weight, conv_bias, conv_state, D, z, dt_bias, out,
             conv_state_out)
    nb, H, P, N = state.shape
    G, width = int(n_groups), row.shape[1]
    if G < 1 or H < 1 or P < 1 or N < 1 or H % G or width != H * P + 2 * G * N:
        raise ValueError(f"selective_scan_step: a row of {H} heads x {P} channels and {G} groups x 2 x {N} states has "
                         f"{H * P + 2 * G * N} values, got {width}")
    if N > 256:
        raise ValueError(f"selective_scan_step: at most 256 states, got {N}")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("selective_scan_step: state must be a contiguous float32 tensor (it is updated in place)")
    _same_dtype("selective_scan_step", row.dtype, dt=dt, z=z, conv_state=conv_state)
    A, D, dt_bias = (_f32(t, H, n, "selective_scan_step") for t, n in ((A, "A"), (D, "D"), (dt_bias, "dt_bias")))
    code = w_code = dt_code(row.dtype)
    W, dev = 0, row.device
    if conv_weight is not None:
        W = conv_weight.shape[-1]
        if conv_weight.shape != (width, W) or not 2 <= W <= 8:
            raise ValueError(f"selective_scan_step: conv_weight must be ({width}, 2 to 8), got {tuple(conv_weight.shape)}")
        if conv_bias is not None and (conv_bias.numel() != width or conv_bias.dtype != conv_weight.dtype):
            raise ValueError(f"selective_scan_step: conv_bias must hold {width} values of conv_weight's dtype")
        if conv_state is None or conv_state.shape != (nb, W - 1, width):
            raise ValueError(f"selective_scan_step: conv_state must be {(nb, W - 1, width)}")
        conv_weight, conv_state = conv_weight.contiguous(), conv_state.contiguous()
        conv_bias = conv_bias.contiguous() if conv_bias is not None else None
        if conv_state_out is None:
            conv_state_out = torch.empty_like(conv_state)
        elif conv_state_out.shape != conv_state.shape or conv_state_out.dtype != row.dtype or \
                not conv_state_out.is_contiguous() or (nb and conv_state_out.data_ptr() == conv_state.data_ptr()):
            raise ValueError("selective_scan_step: conv_state_out must be another contiguous tensor like conv_state")
        w_code = dt_code(conv_weight.dtype)
    elif conv_bias is not None or conv_state is not None or conv_state_out is not None:
        raise ValueError("selective_scan_step: conv_bias and conv_state need conv_weight")
    (row, ld_row), (dt, ld_dt), (z, ld_z) = _as_rows(row, 1), _as_rows(dt, 1), _as_rows(z, 1)
    require_device(row, dt, A, state, conv_weight, conv_bias, conv_state, conv_state_out, D, z, dt_bias, out)
    if out is None:
        out = torch.empty((nb, H, P), dtype=row.dtype, device=dev)
        ld_y = H * P
    else:
        ld_y = _out_rows(out, (nb, H, P), row.dtype, 1, "selective_scan_step")
    # (fields in the descriptor's order)
    d = _lib.SsmStep(code, w_code, nb, H, P, G, N, W, int(softplus), int(silu), row.data_ptr(), ld_row, _ptr(conv_weight),
                     _ptr(conv_bias), _ptr(conv_state), _ptr(conv_state_out), dt.data_ptr(), ld_dt, A.data_ptr(), _ptr(D),
                     _ptr(z), ld_z, _ptr(dt_bias), state.data_ptr(), out.data_ptr(), ld_y)
    on_device(dev.index, _lib.load().tesm_hip_selective_scan_step, ctypes.byref(d), raw_stream(dev.index))
    return out, conv_state_out


# ---------------------------------------------------------------------------
# beam search: the choice of the next tokens, and the states that follow the beams
# ---------------------------------------------------------------------------
def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None, pad_token: int = 0, eos_token: Optional[int] = None):
    """The n best continuations of every request's K beams: ``(scores, parents, tokens, finished)``, each (B, n).

    ``logits`` (B, K, V) and ``scores`` (B, K) float32: beam k offers token v at
    ``scores[b, k] + log_softmax(logits[b, k])[v]``.  The n (default K) best offers come in falling order, equal ones in
    the order of ``k * V + v``.  NaN logits, rows with a +infinite logit and beams whose score is not finite offer
    -infinity.  A beam with ``finished`` (B, K) bool offers ``pad_token`` alone, at its own score; the last result says
    whether the parent was finished or the token is ``eos_token`` (None where neither argument is given).  parents and
    tokens are int64.  K and n are at most 64, B * K < 65536, V < 2^30.
    """
    if logits.dim() != 3 or scores.shape != logits.shape[:2]:
        raise ValueError("beam_select: logits must be (B, K, V) and scores (B, K)")
    _no_grad("beam_select", logits, scores)
    B, K, V = logits.shape
    n = K if n is None else int(n)
    if not (1 <= K <= 64 and 1 <= n <= 64 and n <= K * V):
        raise ValueError(f"beam_select: 1 to 64 beams and candidates, at most K * V of them; got K={K}, V={V}, n={n}")
    if scores.dtype != torch.float32:
        raise TypeError(f"beam_select: scores must be float32, got {scores.dtype}")
    if finished is not None and (finished.shape != scores.shape or finished.dtype not in (torch.bool, torch.uint8)):
        raise ValueError("beam_select: finished must be a (B, K) bool tensor")
    for name, t in (("pad_token", pad_token if finished is not None else None), ("eos_token", eos_token)):
        if t is not None and not 0 <= t < V:
            raise ValueError(f"beam_select: {name} {t} is outside the vocabulary of {V}")
    code = dt_code(logits.dtype)
    logits, ld = _as_rows(logits, 2)
    scores = scores.contiguous()
    finished = finished.contiguous() if finished is not None else None
    require_device(logits, scores, finished)
    dev = logits.device
    out = torch.empty((B, n), dtype=torch.float32, device=dev)
    parents, tokens = torch.empty((2, B, n), dtype=torch.int64, device=dev).unbind()
    done = torch.empty((B, n), dtype=torch.bool, device=dev) if finished is not None or eos_token is not None else None
    # (fields in the descriptor's order)
    d = _lib.Beam(code, B, K, V, n, logits.data_ptr(), ld, scores.data_ptr(), _ptr(finished), int(pad_token),
                  -1 if eos_token is None else int(eos_token), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), _ptr(done))
    lib = _lib.load()
    ref = ctypes.byref(d)
    nbytes = lib.tesm_hip_beam_select_ws_bytes(ref)
    ws = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device=dev)
    on_device(dev.index, lib.tesm_hip_beam_select, ref, ws.data_ptr(), nbytes, raw_stream(dev.index))
    return out, parents, tokens, done


def reorder_rows(tensors, parents: torch.Tensor) -> None:
    """Row ``b * K + k`` of every tensor becomes its old row ``b * K + parents[b, k]``, in place and in one launch.

    ``parents`` (B, K) int64, B < 65536, K <= 64; each tensor has B * K rows (its first dimension), each row contiguous; any
    dtype.  Tensors that overlap are refused.  A parent outside 0 .. K - 1 leaves its row as it is and sets bit 1 of
    ``device_status``.
    """
    if parents.dim() != 2 or parents.dtype != torch.int64:
        raise ValueError("reorder_rows: parents must be a (B, K) int64 tensor")
    B, K = parents.shape
    if not 1 <= K <= 64:
        raise ValueError(f"reorder_rows: 1 to 64 beams, got {K}")
    tensors = list(tensors)
    grad = torch.is_grad_enabled()
    rows, dev = B * K, parents.device
    table = []  # (address, pitch, row bytes) of each: a decode step hands over every layer's caches, so the loop is lean
    index = parents.get_device()
    for t in tensors:
        shape = t.shape
        if not shape or shape[0] != rows:
            raise ValueError(f"reorder_rows: a tensor of shape {tuple(shape)} does not have {rows} rows")
        if grad and t.requires_grad:
            _no_grad("reorder_rows", t)
        pitch = nbytes = t.nbytes // rows if rows else 0
        if not t.is_contiguous():
            pitch = _row_pitch(t, 1)
            if pitch is None:
                raise ValueError("reorder_rows: the rows of a tensor must be contiguous and must not overlap")
            pitch *= t.element_size()
        if t.get_device() != index:
            require_device(parents, t)
        if nbytes:  # (empty ones share whatever address they have)
            table += (t.data_ptr(), pitch, nbytes)
    count = len(table) // 3
    if len(set(table[::3])) != count:
        raise ValueError("reorder_rows: a tensor is given twice")
    parents = parents.contiguous()
    require_device(parents)
    table = array.array("q", table)
    on_device(dev.index, _lib.load().tesm_hip_reorder_rows, table.buffer_info()[0], count, parents.data_ptr(), B, K,
              raw_stream(dev.index))
