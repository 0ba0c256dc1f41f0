"""The state operators where their range ends: narrow states, far values, masks, memory on either side of the outputs.
Tolerances are those of the operators' own tests (``test_gpu_ssm``, ``test_gpu_beam``) unless a test derives another."""
import ctypes

import pytest
import torch

from hip_helpers import DEV, TOL, need_gpu, normwise, to_np
from oracle import tesm_torch as ot
from tesm_amd import TESM_SISO, _lib, hip_ops, tesm
from test_gpu_beam import INF, _case, _model, check_select
from test_gpu_ssm import (HALF, PACKED, SCANS, U, _check_scan, _dev, _randn, _run_scan, _scan_case, _silu, _within,
                          scan_ref)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


# ---------------------------------------------------------------------------
# scan: at most 32 states, whole chunks up to the arrays' ends
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [5, 16, 32])
@pytest.mark.parametrize("L", [32, 64, 1024])
def test_scan_of_few_states_in_whole_chunks(dtype, N, L):
    c = _scan_case(N + L, 1, L, 2, 32, 1, N, dtype)
    _check_scan(c, *_run_scan(c))


@pytest.mark.parametrize("N", [16, 32])
def test_scan_of_few_states_packed_in_whole_chunks(N):
    c = _scan_case(N, 1, 1056, 2, 24, 2, N, torch.bfloat16, starts=[0, 32, 96, 96, 1056])
    _check_scan(c, *_run_scan(c))


# ---------------------------------------------------------------------------
# activations and gates far from zero.  e^-v overflows below v = -88.7: silu(v) is 0 there.  Elsewhere silu is off by 8 u of
# its value, with bfloat16 operands by |v| u more (the exponent is one rounded product); a reciprocal below 2^-126 may
# come out as 0, which is off by at most 89 * 2^-126 < 2^-119.
# ---------------------------------------------------------------------------
FAR = [80.0, 85.0, 87.0, 88.0, 89.0, 92.0, 95.0, 100.0, 110.0, 200.0, 500.0, 1000.0, 1e4, 1e9, 1e30, 3e38]


def _far(dtype):
    v = torch.tensor(FAR)
    more = torch.cat([torch.linspace(-130.0, -80.0, 400), torch.linspace(-2e4, -130.0, 400)])
    return torch.cat([v, -v, more]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [1, 5, None])
def test_conv_of_far_values(dtype, C):
    v = _far(dtype)
    x = v[:, None, None].expand(-1, 1, C).contiguous() if C else v.view(1, 1, -1)
    w = torch.tensor([0.0, 1.0], dtype=dtype).expand(x.shape[2], 2)
    y, _ = hip_ops.causal_conv(_dev(x), _dev(w))
    want = _silu(x.double())
    _within(y, want, ((8 + x.double().abs().clamp(max=1e3)) * U + HALF[dtype]) * want.abs() + 2.0 ** -119, "conv")
    top = torch.full((1, 1, 8), float("inf"), dtype=dtype)
    assert bool((hip_ops.causal_conv(_dev(top), _dev(torch.ones(8, 2, dtype=dtype)))[0] == float("inf")).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_gate_of_far_values(dtype):
    # (values whose gate is a normal number or below 2^-126 by far: the scan's bound has no term for what lies between)
    v = torch.tensor([f for f in FAR if f < 87 or f > 90]).to(dtype)
    v = torch.cat([v[v < 1e31], -v])
    c = _scan_case(101, 1, 70, 2, 40, 1, 16, dtype)
    c["z"] = v[torch.arange(c["z"].numel()) % v.numel()].view(c["z"].shape).contiguous()
    _check_scan(c, *_run_scan(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
def test_scan_of_masked_step_sizes(dtype, bias):
    """Step sizes masked by the type's lowest value, by -infinity or by large negative numbers are 0: those rows leave
    the state as it is."""
    c = _scan_case(102, 2, 75, 3, 32, 1, 32, dtype, bias=bias)
    for i, low in enumerate((torch.finfo(dtype).min, float("-inf"), -1e30, -1e4, -95.0)):
        c["dt"][:, 3 + i::7] = low
    c["dt"][1, 40:] = torch.finfo(dtype).min
    _check_scan(c, *_run_scan(c))


def _check_step(c, W):
    """One token with the filter (0, .., 0, 1), so that the convolved values are silu(row), against 64 bits."""
    B, H, P, G, N, dtype = (c[k] for k in ("B", "H", "P", "G", "N", "dtype"))
    width = H * P + 2 * G * N
    w = torch.zeros(width, W, dtype=dtype)
    w[:, -1] = 1
    hd = _dev(c["h"]).clone()
    y, _ = hip_ops.selective_scan_step(_dev(c["row"]), _dev(c["dt"]), _dev(c["A"]), hd, _dev(w), None,
                                       torch.zeros(B, W - 1, width, dtype=dtype, device=DEV), n_groups=G, z=_dev(c["z"]))
    v = _silu(c["row"].double())
    dv = (8 + c["row"].double().abs().clamp(max=1e3)) * U * v.abs() + 2.0 ** -119
    cut = [H * P, G * N, G * N]
    (x, b, cc), (dx, db, dc) = v.split(cut, 1), dv.split(cut, 1)
    x, dx = (t.reshape(B, H, P) for t in (x, dx))
    b, cc, db, dc = (t.reshape(B, G, N).repeat_interleave(H // G, 1)[:, :, None] for t in (b, cc, db, dc))
    raw = c["dt"].double()
    d = torch.where(raw < -30, raw.exp(), torch.nn.functional.softplus(raw, threshold=700))
    a = (d * c["A"].double()).exp()[..., None, None]
    add = (d[..., None] * x)[..., None] * b
    hn = a * c["h"].double() + add
    mass = (a * c["h"].double()).abs() + add.abs()
    dh = d[..., None, None] * (dx[..., None] * b.abs() + x.abs()[..., None] * db) + 48 * U * mass
    _within(hd, hn, dh + 1e-36, "step state")
    gate = _silu(c["z"].double())
    dg = (8 + c["z"].double().abs().clamp(max=1e3)) * U * gate.abs() + 2.0 ** -119
    core = (hn * cc).sum(-1)
    ym = (hn.abs() * cc.abs()).sum(-1)
    tol = gate.abs() * ((dh * cc.abs() + hn.abs() * dc).sum(-1) + (N + 16) * U * ym) + dg * ym
    _within(y, core * gate, tol + HALF[dtype] * (core * gate).abs() + 1e-36, "step y")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [16, 33])
def test_step_of_far_values(dtype, N):
    g = torch.Generator().manual_seed(103)
    B, H, P, G = 3, 4, 40, 2
    c = dict(B=B, H=H, P=P, G=G, N=N, dtype=dtype)
    width = H * P + 2 * G * N
    c["row"] = _randn(g, B, width, dtype=dtype)
    low = -_far(dtype)[:len(FAR)]
    c["row"][:, ::3] = low[torch.arange(c["row"][:, ::3].numel()) % len(FAR)].view(B, -1)
    c["dt"] = _randn(g, B, H, dtype=dtype)
    c["dt"][0, 1], c["dt"][1, 2], c["dt"][2, 0], c["dt"][2, 3] = torch.finfo(dtype).min, float("-inf"), -95.0, 120.0
    c["A"] = -(0.3 + 4 * torch.rand(H, generator=g))
    v = _far(dtype)
    v = v[v < 1e31]
    c["z"] = v[torch.arange(B * H * P) % v.numel()].view(B, H, P).contiguous()
    c["h"] = _randn(g, B, H, P, N)
    _check_step(c, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_output_gate_of_far_values(dtype):
    """Gates below -88.7 are 0 like those whose sigmoid is lost beside the other addend."""
    g = torch.Generator().manual_seed(104)
    M, dm, D = 32, 64, 64
    codes = [hip_ops.quant_act(_randn(g, M, D, dtype=dtype).to(DEV)) for _ in range(2)]
    packed = []
    for _ in range(2):
        w = _randn(g, dm, D).to(DEV)
        s, cw = hip_ops.absmean_scale(w)
        packed += [hip_ops.pack_weight(w, s), cw]
    low = -_far(dtype)[:len(FAR)][torch.arange(M * dm) % len(FAR)].view(M, dm).to(DEV)
    local = _randn(g, M, dm, dtype=dtype).to(DEV)
    for quantize in (True, False):
        y, _ = hip_ops.output_gate(*codes, *packed, local, low, D, quantize=quantize)
        want, _ = hip_ops.output_gate(*codes, *packed, local, torch.full_like(low, -80.0), D, quantize=quantize)
        # sigmoid(-80) = 1.8e-35: no bit of a sum of ordinary numbers
        assert torch.equal(y, want)
        # and gates far above 0 are 1 like those of 80, infinite ones aside; NaN stays NaN
        high = -low
        high[0, 0] = float("nan")
        y, _ = hip_ops.output_gate(*codes, *packed, local, high, D, quantize=quantize)
        want, _ = hip_ops.output_gate(*codes, *packed, local, torch.full_like(low, 80.0), D, quantize=quantize)
        assert bool(y[0, 0].isnan()) and torch.equal(y.flatten()[1:], want.flatten()[1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay_bias", [-95.0, -110.0, -1000.0])
def test_layer_of_closed_decay_gates(dtype, decay_bias):
    cfg = dict(d_model=64, d_state=32, ent_rank=8, entanglement_window=8, entanglement_threshold=0.08,
               entanglement_scale=0.2, decay_init_bias=decay_bias, max_seq_len=64)
    torch.manual_seed(0)
    ref = ot.TESM_SISO(**cfg).eval()
    torch.manual_seed(0)
    m = TESM_SISO(**cfg).to(DEV).to(dtype).eval()
    u = torch.randn(2, 40, 64, generator=torch.Generator().manual_seed(1))
    y, _ = m(u.to(DEV).to(dtype))
    want, _ = ref.to(dtype)(u.to(dtype))
    assert bool(y.isfinite().all())
    assert normwise(to_np(y), to_np(want)) <= TOL[dtype]


# ---------------------------------------------------------------------------
# beam selection: logits of any magnitude
# ---------------------------------------------------------------------------
MASKS = [-1e4, -1e6, -1.1e6, -1e9, -3e9, -1e10, -1e20, -1e30, -3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("allowed", [1, 40, 3000])
def test_select_of_masked_rows(dtype, mask, allowed):
    """A few allowed tokens among ones masked by a large negative number: anywhere in the row, all in one part of it."""
    logits, scores, g = _case(200 + allowed, 4, 3, 20000, dtype)
    keep = torch.zeros(20000, dtype=torch.bool)
    keep[torch.randperm(20000, generator=g)[:allowed]] = True
    logits[:2, :, ~keep] = mask
    logits[2, :, allowed:] = mask
    logits[3, :2, :-allowed] = mask
    check_select(logits, scores, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [3e9, -3e9, 1e10, -1e10, 1e20, -1e20, 3e38, -3e38])
def test_select_of_rows_far_from_zero(dtype, top):
    """Rows whose largest logits are far from zero, equal or spread over a few steps of the type."""
    logits, scores, g = _case(210, 4, 2, 9000, dtype)
    step = abs(top) * torch.finfo(dtype).eps
    logits[0] = top
    logits[1] = (top + step * torch.randint(-3, 1, logits[1].shape, generator=g).double()).to(dtype)
    logits[2, :, ::5] = top
    logits[3, 0], logits[3, 1, 100:] = top, -INF
    check_select(logits, scores, 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [500, 20000])
@pytest.mark.parametrize("offset", [100.0, 1000.0, 10000.0, 1.1e6, 1e7])
def test_select_of_shifted_rows(dtype, V, offset):
    """A beam's offers do not depend on an offset of its logits: the scores keep their bound at every offset."""
    logits, scores, _ = _case(220, 4, 4, V, torch.float32)
    logits[:, 1] += offset
    logits[:, 2] -= offset
    logits[1, 3, ::2] += offset
    check_select(logits.to(dtype), scores, 8)


# ---------------------------------------------------------------------------
# outputs beside their inputs in one buffer, and on top of them
# ---------------------------------------------------------------------------
def test_outputs_in_columns_beside_the_inputs():
    g = torch.Generator().manual_seed(230)
    B, L, H, P, G, N = 2, 70, 4, 32, 1, 32
    C = H * P
    wide = torch.zeros(B, L, 3 * C, device=DEV)
    x, w = _randn(g, B, L, C).to(DEV), _randn(g, C, 4).to(DEV)
    wide[..., :C] = x
    y, new = hip_ops.causal_conv(wide[..., :C], w, out=wide[..., C:2 * C])
    want, want_new = hip_ops.causal_conv(x, w)
    assert torch.equal(y, want) and torch.equal(new, want_new) and torch.equal(wide[..., :C], x)
    with pytest.raises(RuntimeError, match="y overlaps x"):
        hip_ops.causal_conv(wide[..., :C], w, out=wide[..., C - 1:2 * C - 1])

    c = _scan_case(231, B, L, H, P, G, N, torch.float32)
    wide[..., :C] = _dev(c["x"]).flatten(2)
    args = [_dev(c[k]) for k in ("dt", "A", "B", "C")]
    y, h = hip_ops.selective_scan(wide[..., :C].unflatten(-1, (H, P)), *args, out=wide[..., 2 * C:].unflatten(-1, (H, P)))
    want, want_h = hip_ops.selective_scan(_dev(c["x"]), *args)
    assert torch.equal(y, want) and torch.equal(h, want_h)
    with pytest.raises(RuntimeError, match="y overlaps x"):
        hip_ops.selective_scan(wide[..., :C].unflatten(-1, (H, P)), *args, out=wide[..., 8:C + 8].unflatten(-1, (H, P)))

    width = C + 2 * G * N
    both = torch.zeros(B, width + C, device=DEV)
    both[:, :width] = _randn(g, B, width).to(DEV)
    row, dt, h = both[:, :width].clone(), _dev(c["dt"][:, 0]), torch.zeros(B, H, P, N, device=DEV)
    y, _ = hip_ops.selective_scan_step(both[:, :width], dt, args[1], h, out=both[:, width:].unflatten(-1, (H, P)))
    want, _ = hip_ops.selective_scan_step(row, dt, args[1], torch.zeros_like(h))
    assert torch.equal(y, want)
    keep = both.clone()
    with pytest.raises(RuntimeError, match="y overlaps row"):
        hip_ops.selective_scan_step(both[:, :width], dt, args[1], h, out=both[:, :C].unflatten(-1, (H, P)))
    assert torch.equal(both, keep)


def test_reorder_of_column_slices_of_one_buffer():
    g = torch.Generator().manual_seed(240)
    wide = torch.randn(6, 100, generator=g)
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]])
    rows = torch.tensor([2, 0, 0, 4, 4, 5])
    dev = wide.to(DEV)
    hip_ops.reorder_rows([dev[:, 40:90], dev[:, :17], torch.zeros(6, 0, device=DEV), dev[:, 17:30]], parents.to(DEV))
    want = wide.clone()
    for lo, hi in ((0, 30), (40, 90)):
        want[:, lo:hi] = wide[rows, lo:hi]
    assert torch.equal(dev.cpu(), want)
    with pytest.raises(RuntimeError, match="overlap"):
        hip_ops.reorder_rows([dev[:, 40:90], dev[:, :17], dev[:, 16:30]], parents.to(DEV))
    assert torch.equal(dev.cpu(), want)


# ---------------------------------------------------------------------------
# beam search from one token
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [{}, dict(use_mimo=True, n_heads=2), dict(entanglement_window=0)])
def test_beam_search_from_one_token_needs_no_earlier_prompt(kw):
    """The decode step is then the first call of all: its workspace holds the cross-layer query's buffers."""
    m = _model(torch.float32, **kw)
    ids = torch.randint(0, 300, (3, 1), generator=torch.Generator().manual_seed(1)).to(DEV)
    m(torch.zeros(8, 40, dtype=torch.int64, device=DEV))  # (a prompt leaves a workspace large enough for any step)
    want = m.beam_search(ids, 4, 5)
    torch.cuda.synchronize()
    tesm._WORKSPACES.clear()
    m = _model(torch.float32, **kw)
    got = m.beam_search(ids, 4, 5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------
# scan: rows that clear the state
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("step", [1e4, 1e8, 1e10, 1e12, 1e20, 1e30])
def test_scan_of_step_sizes_that_clear_the_state(dtype, step):
    """A huge step size with x = 0 leaves a state of 0: the rows behind it, in its chunk and later, know nothing of it."""
    c = _scan_case(300, 1, 140, 3, 32, 1, 32, dtype, softplus=False, bias=False, gate=False)
    c["dt"][0, ::9] = step
    c["x"][0, ::9] = 0
    c["A"][2] = -0.3
    _check_scan(c, *_run_scan(c))


# ---------------------------------------------------------------------------
# memory on either side of the outputs
# ---------------------------------------------------------------------------
class Guarded:
    """Buffers of exactly the sizes asked for, each inside a larger one filled with a byte that must stay."""
    PAD, BYTE = 1 << 16, 0xA5

    def __init__(self):
        self.all = []

    def bytes(self, n, fill=0):
        whole = torch.full((n + 2 * self.PAD,), self.BYTE, dtype=torch.uint8, device=DEV)
        whole[self.PAD:self.PAD + n] = fill
        self.all.append((whole, n))
        return whole[self.PAD:self.PAD + n]

    def like(self, shape, dtype):
        n = torch.Size(shape).numel() * dtype.itemsize
        return self.bytes(n).view(dtype).view(shape)

    def check(self):
        for whole, n in self.all:
            assert bool((whole[:self.PAD] == self.BYTE).all()) and bool((whole[self.PAD + n:] == self.BYTE).all())


ORDERS = [[0, 1000] * 8, [900, 100, 1000, 0, 700, 699, 5, 5, 1000, 3], [-5, 2000, -7, 1 << 30, 12, -(1 << 30), 64, 1000],
          [1000, 0], [0, 1000], [1000] * 5, [-3] * 5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts", ORDERS)
@pytest.mark.parametrize("H,P,G,N", [(2, 16, 1, 16), (4, 64, 2, 64)])
def test_scan_of_any_starts_writes_its_own_memory_only(dtype, starts, H, P, G, N):
    """What starts that are in no order give is not looked at; workspace, outputs and states are of the exact size."""
    M, S, code = 1000, len(starts) - 1, hip_ops.dt_code(dtype)
    c = _scan_case(72, 1, M, H, P, G, N, dtype, starts=starts)
    mem, ins = Guarded(), {k: _dev(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0")}
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    y, h = mem.like((M, H * P), dtype), mem.like((S, H, P, N), torch.float32)
    p = {k: v.data_ptr() for k, v in ins.items()}
    d = _lib.Ssm(code, 1, M, H, P, G, N, S, 1, p["x"], H * P, p["dt"], H, p["A"], p["B"], G * N, p["C"], G * N, p["D"], p["z"], H * P,
                 p["dt_bias"], at.data_ptr(), p["h0"], y.data_ptr(), H * P, h.data_ptr())
    lib = _lib.load()
    nbytes = lib.tesm_hip_selective_scan_ws_bytes(ctypes.byref(d))
    ws = mem.bytes(nbytes)
    keep = {k: v.clone() for k, v in ins.items()}
    _lib.check(lib.tesm_hip_selective_scan(ctypes.byref(d), ws.data_ptr() if nbytes else None, nbytes, hip_ops.raw_stream(0)))
    torch.cuda.synchronize()
    mem.check()
    assert all(torch.equal(v, keep[k]) for k, v in ins.items())
    if starts == sorted(starts) and starts[0] >= 0 and starts[-1] <= M:
        _check_scan(c, y.view(1, M, H, P), h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts", ORDERS)
@pytest.mark.parametrize("C", [3, 40])
def test_conv_of_any_starts_writes_its_own_memory_only(dtype, starts, C):
    M, S, W, code = 1000, len(starts) - 1, 4, hip_ops.dt_code(dtype)
    g = torch.Generator().manual_seed(73)
    x, w, state = (_randn(g, *n, dtype=dtype).to(DEV) for n in ((M, C), (C, W), (S, W - 1, C)))
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    mem = Guarded()
    y, new = mem.like((M, C), dtype), mem.like((S, W - 1, C), dtype)
    d = _lib.Conv(code, code, 1, M, C, W, S, 1, x.data_ptr(), C, w.data_ptr(), None, at.data_ptr(), state.data_ptr(), y.data_ptr(), C,
                  new.data_ptr())
    keep = x.clone(), state.clone()
    _lib.check(_lib.load().tesm_hip_causal_conv(ctypes.byref(d), hip_ops.raw_stream(0)))
    torch.cuda.synchronize()
    mem.check()
    assert torch.equal(x, keep[0]) and torch.equal(state, keep[1])


# ---------------------------------------------------------------------------
# scan: bfloat16 operands, products of float32 accuracy.  Rows hold what float32 operands' do and their own rounding, and on
# the way 2^-14 of the contributions' magnitudes: 2^-15 for the second bfloat16 part of the decayed scores and of the state,
# and below 2^-15 for the decays, whose sums, below 512, are each off by 2^-16 in the exponent of 2.
# ---------------------------------------------------------------------------
def _check_scan_closely(c, y):
    nb, L = c["x"].shape[:2]
    spans = [(i * L, i * L + L) for i in range(nb)] if c["starts"] is None else list(zip(c["starts"][:-1], c["starts"][1:]))
    want, mass, _, _ = scan_ref(c, spans, nb * L)
    longest = max([b - a for a, b in spans], default=0)
    count = c["N"] + 3 * min(longest, 64) + 6 * (longest // 32 + 1) + 64
    tol = (2.0 ** -14 + count * U) * mass + (HALF[torch.bfloat16] + 8 * U) * want.abs() + 1e-36
    for lo, hi in spans:
        _within(y.reshape(want.shape)[lo:hi], want[lo:hi], tol[lo:hi], "scan rows %d..%d" % (lo, hi))


@pytest.mark.parametrize("B,L,H,P,G,N", SCANS)
@pytest.mark.parametrize("full", [True, False])
def test_scan_rounds_bfloat16_rows_once(B, L, H, P, G, N, full):
    c = _scan_case(B + L + H + P + N, B, L, H, P, G, N, torch.bfloat16, init=full, gate=full, skip=full, bias=full)
    _check_scan_closely(c, _run_scan(c)[0])


@pytest.mark.parametrize("starts", PACKED + [[0, 1000, 1003, 1700]])
def test_scan_rounds_bfloat16_rows_once_packed(starts):
    c = _scan_case(310, 1, starts[-1] + 5, 4, 32, 2, 64, torch.bfloat16, starts=starts)
    _check_scan_closely(c, _run_scan(c)[0])
