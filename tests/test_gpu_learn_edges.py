"""The operators that learn where their range ends: strides, masks, empty parts, memory beside the outputs, other streams, captured graphs,
autograd, and a block of all of them.  Tolerances are those carried by ``learn_refs`` unless a test derives another."""
import math

import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_refs import HALF, U, dense_ref, logp_ref, scan_ref, within
from tesm_amd import TESMConfig, TESMLMHeadModel, hip_ops
from test_gpu_learn import BOTH, _dev, _gen, _randn, check_dense, check_scan, dense_case, logp_case, run_scan, scan_case

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


def _column_slice(t, at, more=7, fill=NAN):
    """``t`` on the device as columns of wider rows, between rows and columns of ``fill``."""
    if t is None:
        return None
    rows = t.reshape(-1, t.shape[-1])
    wide = torch.full((rows.shape[0] + 2, rows.shape[1] + more), fill, dtype=t.dtype, device=DEV)
    wide[1:-1, at:at + rows.shape[1]] = rows.to(DEV)
    if t.dim() == 1:
        return wide[1, at:at + rows.shape[1]]
    view = wide[1:-1, at:at + rows.shape[1]]
    return view if t.dim() == 2 else view.unflatten(0, t.shape[:-1])


# ---------------------------------------------------------------------------
# recurrence
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("at", [0, 1, 2, 5])
@pytest.mark.parametrize("C", [1, 66, 130])
def test_scan_of_columns(dtype, at, C):
    c = scan_case(at + C, 2, 70, C, dtype)
    check_scan(c, *run_scan(c, lambda t: _column_slice(t, at) if t is not None and t.dim() == 3 else _dev(t)))


@pytest.mark.parametrize("dtype", BOTH)
def test_scan_of_other_layouts(dtype):
    c = scan_case(3, 3, 40, 20, dtype)
    check_scan(c, *run_scan(c, lambda t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) if t is not None and t.dim() == 3 else _dev(t)))
    check_scan(c, *run_scan(c, lambda t: t.to(DEV).mT.contiguous().mT if t is not None and t.dim() == 3 else _dev(t)))


ORDERS = [[0, 64, 128, 200], [5, 5, 6, 100], [-9, 70, 500, 900], [150, 90, 120, 180], [200, 200], [0, 0, 0, 1], [-5, -1, 0], [300, 400],
          [120, 3, 400, 17]]


def _ordered(starts, L):
    """What starts count as: the nearest row, and no start below an earlier one."""
    out, m = [], 0
    for s in starts:
        m = max(m, min(max(s, 0), L))
        out.append(m)
    return out


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("starts", ORDERS)
@pytest.mark.parametrize("C", [3, 130])
def test_scan_of_any_starts(dtype, wide, starts, C):
    """Rows of no sequence stay as they are in ``out``, are 0 without it, and get no gradient; what lies beside ``out`` stays."""
    L, order = 200, _ordered(starts, 200)
    c = scan_case(sum(starts) + C, 1, L, C, dtype, starts=order)
    for k in ("value", "write", "decay", "grad"):  # (what no sequence holds is not read)
        c[k][0, :order[0]] = NAN
        c[k][0, order[-1]:] = NAN
    args = [_dev(c[k]) for k in ("value", "write", "decay", "bias")]
    how = dict(state=_dev(c["state"]), seq_starts=torch.tensor(starts, dtype=wide, device=DEV))
    out = torch.full((L + 2, C + 5), 7.0, dtype=dtype, device=DEV)
    h, last, kept = hip_ops.gated_scan(*args, keep=True, **how)
    h2, last2 = hip_ops.gated_scan(*args, out=out[None, 1:-1, 2:-3], **how)
    grads = hip_ops.gated_scan_backward(_dev(c["grad"]), *args, kept=kept, grad_state=_dev(c["grad_state"]), **how)
    inside = torch.zeros(L, dtype=torch.bool)
    inside[order[0]:order[-1]] = True
    assert torch.equal(last, last2) and torch.equal(h2[0, inside], h[0, inside])
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[1:-1, 2:-3][inside] = False
    assert bool((out[keep] == 7.0).all())
    for t in (h, *grads[:3]):
        assert bool((t[0, ~inside] == 0).all())
    for k in ("value", "write", "decay", "grad"):
        c[k] = torch.where(inside[:, None], c[k], torch.zeros_like(c[k]))
    h = h.cpu()
    check_scan(c, h, last, [torch.where(inside[:, None], g.cpu(), 0.0) if i < 3 else g for i, g in enumerate(grads)])


@pytest.mark.parametrize("dtype", BOTH)
def test_scan_of_closed_gates(dtype):
    """Infinite and very large gates: forgetting, holding, writing nothing."""
    c = scan_case(21, 1, 400, 8, dtype)
    c["decay"][0, 10::40] = -INF
    c["decay"][0, 50:120, 1::2], c["write"][0, 50:120, 1::2] = INF, -INF
    c["value"][0, 130:140], c["value"][0, 150:160] = INF, -INF
    c["write"][0, 170:180] = INF
    c["decay"][0, 200:220], c["write"][0, 200:220] = torch.finfo(dtype).min, torch.finfo(dtype).max
    c["decay"][0, 230:260, 3], c["write"][0, 230:260, 3] = 1e30, -1e30
    h, last, grads = run_scan(c)
    check_scan(c, h, last, grads)
    assert all(bool(g.isfinite().all()) for g in grads)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("name", ["value", "write", "decay"])
def test_scan_of_a_nan(dtype, name):
    """It stays in its channel, in the rows behind it (states) and in front of it (gradients)."""
    c = scan_case(22, 1, 1300, 5, dtype)
    c[name][0, 1100, 2] = NAN
    check_scan(c, *run_scan(c))


@pytest.mark.parametrize("dtype", BOTH)
def test_scan_of_nothing(dtype):
    for B, L, C in [(0, 5, 4), (2, 0, 4), (2, 5, 0)]:
        c = scan_case(1, B, L, C, dtype)
        h, last, grads = run_scan(c)
        assert h.shape == (B, L, C) and all(g.shape == w for g, w in zip(grads, [h.shape] * 3 + [(C,), (B, C)]))
        if not L:
            assert torch.equal(last, _dev(c["state"])) and torch.equal(grads[4], _dev(c["grad_state"])) and not grads[3].any()
    c = scan_case(1, 1, 9, 4, dtype, starts=[0])
    h, last, grads = run_scan(c)
    assert not h.any() and last.shape == (0, 4) and not any(g.any() for g in grads if g.numel())
    x = torch.empty(0, 4, dtype=dtype, device=DEV)
    assert hip_ops.gated_scan_step(x, x, x, state=torch.empty(0, 4, device=DEV)).shape == (0, 4)


def test_scan_that_gives_up_says_so():
    """A negative limit of polls lets every tile behind the first give up at once, so every wave still runs to its end."""
    c = scan_case(5, 1, 640, 130, torch.float32)
    args = [_dev(c[k]) for k in ("value", "write", "decay", "bias")]
    hip_ops.device_status(clear=True)
    hip_ops.debug_scan_spin_limit(-1)
    try:
        h, last = hip_ops.gated_scan(*args)
        torch.cuda.synchronize()
    finally:
        hip_ops.debug_scan_spin_limit(1 << 20)
    assert hip_ops.device_status(clear=True) & 1
    assert torch.isfinite(h[0, :64]).all() and torch.isnan(h[0, 64:]).all() and torch.isnan(last).all()
    assert torch.isfinite(hip_ops.gated_scan(*args)[0]).all() and hip_ops.device_status() == 0


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("at", [0, 3])
@pytest.mark.parametrize("B,C", [(1, 1), (3, 65), (40, 700)])
def test_step(dtype, at, B, C):
    """One token after another, out of columns, against the rows of the whole."""
    c = scan_case(B + C, B, 4, C, dtype)
    r = scan_ref(c["value"], c["write"], c["decay"], c["bias"], c["state"], None)
    state = _dev(c["state"])
    for t in range(4):
        out = torch.full((B, C + 6), 7.0, dtype=dtype, device=DEV)
        h = hip_ops.gated_scan_step(*(_column_slice(c[k][:, t], at) for k in ("value", "write", "decay")), _dev(c["bias"]), state=state,
                                    out=out[:, at:at + C])
        within(h, r["h"][0][:, t], r["h"][1][:, t], "h")
        out[:, at:at + C] = 7.0
        assert bool((out == 7.0).all())
    within(state, *r["last"], "state")


def test_step_of_closed_gates():
    c = scan_case(2, 2, 1, 6, torch.float32)
    c["decay"][:, :, 0], c["decay"][:, :, 1], c["write"][:, :, 1] = -INF, INF, -INF
    c["value"][:, :, 2], c["decay"][:, :, 3], c["write"][:, :, 4] = -INF, NAN, 1e30
    state = _dev(c["state"])
    h = hip_ops.gated_scan_step(*(_dev(c[k][:, 0]) for k in ("value", "write", "decay")), state=state)
    r = scan_ref(c["value"], c["write"], c["decay"], None, c["state"], None)
    within(h, r["h"][0][:, 0], r["h"][1][:, 0], "h")
    assert torch.equal(state[:, 1].cpu(), c["state"][:, 1]) and torch.equal(state[:, :3], h[:, :3])


# ---------------------------------------------------------------------------
# projections
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("at", [0, 1, 4])
@pytest.mark.parametrize("M,K,N", [(1, 33, 20), (20, 64, 48), (70, 104, 72), (200, 67, 130)])
@pytest.mark.parametrize("pair", [False, True])
def test_products_of_columns(dtype, at, M, K, N, pair):
    """Operands between NaN, at any alignment, in rows of any pitch."""
    check_dense(dense_case(at + M, M, K, N, dtype, pair=pair, bias=not pair, residual=not pair), "silu", lambda t: _column_slice(t, at))


@pytest.mark.parametrize("dtype", BOTH)
def test_products_of_other_layouts(dtype):
    c = dense_case(1, 60, 40, 24, dtype, bias=True, residual=True)
    check_dense(c, "gelu", lambda t: t.to(DEV).t().contiguous().t() if t is not None and t.dim() == 2 else _dev(t))
    x = _dev(c["x"]).view(3, 4, 5, 40)
    y = hip_ops.fused_linear(x, _dev(c["w"]), _dev(c["bias"]))
    assert torch.equal(y, hip_ops.fused_linear(_dev(c["x"]), _dev(c["w"]), _dev(c["bias"])).view(3, 4, 5, 24))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("M,K,N", [(1000, 500, 4000), (2000, 100, 4000), (2100, 1000, 1000), (1500, 1300, 2000), (777, 2500, 333)])
def test_products_of_many_tiles(dtype, pair, M, K, N):
    """Every tile size, whole and split contractions."""
    check_dense(dense_case(M + K, M, K, N, dtype, pair=pair, bias=not pair), "gelu")


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 512, 16384), (20, 512, 16384), (20, 516, 16384), (40, 70, 50), (64, 300, 33), (65, 300, 33)])
def test_products_of_few_rows(dtype, pair, M, K, N):
    """Weights streamed once, or in tiles where those are expected to take less time."""
    check_dense(dense_case(M + N, M, K, N, dtype, pair=pair, bias=not pair, residual=not pair), "silu")


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("pair", [False, True])
def test_products_of_nothing(dtype, pair):
    for M, N in [(0, 4), (5, 0), (0, 0)]:
        x, w, b = (torch.randn(*s, device=DEV).to(dtype) for s in ((M, 8), (N, 8), (N,)))
        grad = torch.randn(M, N, device=DEV).to(dtype)
        if pair:
            y, kept = hip_ops.gated_linear(x, w, w, keep=True)
            grads = hip_ops.gated_linear_backward(grad, x, w, w, kept=kept)
        else:
            y, kept = hip_ops.fused_linear(x, w, b, act="gelu", keep=True)
            grads = hip_ops.fused_linear_backward(grad, x, w, b, kept=kept, act="gelu")
        shapes = [(M, 8), (N, 8), (N, 8) if pair else (N,)]
        assert y.shape == (M, N) and [tuple(g.shape) for g in grads] == shapes and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M", [3, 100])
def test_products_keep_nans_and_infinities_in_their_rows(dtype, M):
    """Row 1 holds a NaN, row 2 (bfloat16) an infinity: other rows and their gradients are as without them."""
    c = dense_case(4, M, 72, 40, dtype)
    x, w = _dev(c["x"]), _dev(c["w"])
    y = hip_ops.fused_linear(x, w, act="silu")
    x[1, 5] = NAN
    x[2, 6] = INF
    z, kept = hip_ops.fused_linear(x, w, act="silu", keep=True)
    others = torch.arange(M, device=DEV)[(torch.arange(M, device=DEV) != 1) & (torch.arange(M, device=DEV) != 2)]
    assert torch.equal(z[others], y[others]) and bool(z[1].isnan().all())
    if dtype == torch.bfloat16:
        want = torch.where(c["w"][:, 6] > 0, INF, 0.0)  # (silu of -infinity: 0 times infinity is NaN in torch as well)
        assert torch.equal(z[2].cpu().float().nan_to_num(0.0, INF), want)


def test_backward_of_what_is_asked_for():
    for pair in (False, True):
        c = dense_case(6, 90, 48, 40, torch.bfloat16, pair=pair, bias=not pair)
        x, w, up, b, g = (_dev(c[k]) for k in ("x", "w", "up", "bias", "grad"))
        if pair:
            _, kept = hip_ops.gated_linear(x, w, up, keep=True)
            call = lambda **kw: hip_ops.gated_linear_backward(g, x, w, up, kept=kept, **kw)
            names = ("need_x", "need_weights")
        else:
            call = lambda **kw: hip_ops.fused_linear_backward(g, x, w, b, **kw)
            names = ("need_x", "need_weight")
        dx, dw, third = call()
        a = call(**{names[0]: False})
        assert a[0] is None and torch.equal(a[1], dw) and torch.equal(a[2], third)
        a = call(**{names[1]: False})
        assert a[1] is None and torch.equal(a[0], dx) and (a[2] is None if pair else torch.equal(a[2], third))


def test_refusals_on_the_device():
    x, w = torch.randn(3, 8, device=DEV), torch.randn(4, 8, device=DEV)
    g = torch.randn(2, 5, 6, device=DEV)
    with pytest.raises(ValueError, match="gradient"):
        hip_ops.fused_linear_backward(torch.randn(3, 5, device=DEV), x, w)
    with pytest.raises(ValueError, match="kept"):
        hip_ops.fused_linear_backward(torch.randn(3, 4, device=DEV), x, w, act="silu", kept=x)
    with pytest.raises(ValueError, match="kept"):
        hip_ops.gated_linear_backward(torch.randn(3, 4, device=DEV), x, w, w, kept=(x, x))
    with pytest.raises(ValueError, match="kept"):
        hip_ops.gated_scan_backward(g, g, g, g, kept=torch.randn(1, 6, device=DEV))
    with pytest.raises(ValueError, match="kept"):
        hip_ops.token_log_probs_backward(None, None, x, torch.zeros(3, dtype=torch.int64, device=DEV), kept=torch.randn(3, 3, device=DEV))
    with pytest.raises(ValueError, match="out must"):
        hip_ops.gated_scan(g, g, g, out=torch.empty(2, 6, 5, device=DEV).mT)
    with pytest.raises(RuntimeError, match="h overlaps value"):
        hip_ops.gated_scan(g, g, g, out=g)
    with pytest.raises(RuntimeError, match="h overlaps"):
        hip_ops.gated_scan_step(g[0], g[0], g[0], state=torch.zeros(5, 6, device=DEV), out=g[0])


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("at", [0, 1, 3])
@pytest.mark.parametrize("rows,V", [(3, 10), (2, 4097), (600, 300)])
def test_logp_of_columns(dtype, at, rows, V):
    x, t, g, e = logp_case(rows + V + at, rows, V, dtype)
    r = logp_ref(x, t, 3, -100, g, e)
    xd, td = _column_slice(x, at), _dev(t)
    logp, entropy, best, tokens, kept = hip_ops.token_log_probs(xd, td, top=3, keep=True)
    d = hip_ops.token_log_probs_backward(_dev(g), _dev(e), xd, td, kept=kept)
    assert torch.equal(tokens.cpu(), r["tokens"])
    for got, name in ((logp, "logp"), (entropy, "entropy"), (best, "top"), (d, "dx")):
        within(got, *r[name], name)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("V", [5, 900, 70000])
def test_logp_of_broken_rows(dtype, V):
    """A NaN, +infinity, nothing above -infinity: NaN in that row alone.  No such token: NaN, and the status word says so."""
    x, t, g, e = logp_case(V, 7, V, dtype)
    t[:] = torch.arange(7) % V
    x[1, V - 1], x[2, 3] = NAN, INF
    x[3] = -INF
    t[4], t[5] = V, -1
    hip_ops.device_status(clear=True)
    logp, entropy, best, tokens, kept = hip_ops.token_log_probs(_dev(x), _dev(t), top=2, keep=True)
    d = hip_ops.token_log_probs_backward(_dev(g), _dev(e), _dev(x), _dev(t), kept=kept)
    assert hip_ops.device_status(clear=True) == 4
    assert bool(logp[1:6].isnan().all()) and bool(entropy[1:4].isnan().all()) and bool(d[1:4].isnan().all())
    good = [0, 6]
    r = logp_ref(x[good], t[good], 2, -100, g[good], e[good])
    for got, name in ((logp, "logp"), (entropy, "entropy"), (best, "top"), (d, "dx")):
        within(got[good], *r[name], name)
    within(entropy[4:6], *(v[4:6] for v in logp_ref(x, torch.zeros(7, dtype=torch.int64), 0)["entropy"]), "entropy")
    assert bool((tokens >= 0).all()) and bool((tokens < V).all())


def test_logp_of_nothing_and_of_ignored_rows():
    x = torch.randn(0, 9, device=DEV)
    logp, entropy, best, tokens = hip_ops.token_log_probs(x, torch.zeros(0, dtype=torch.int64, device=DEV), top=4)
    assert logp.shape == (0,) and tokens.shape == (0, 4)
    x, t = torch.randn(5, 9, device=DEV), torch.full((5,), 3, dtype=torch.int64, device=DEV)
    logp, _, _, _, kept = hip_ops.token_log_probs(x, t, ignore_index=3, keep=True)
    assert not logp.any()
    assert not hip_ops.token_log_probs_backward(torch.ones(5, device=DEV), None, x, t, kept=kept, ignore_index=3).any()
    assert not hip_ops.token_log_probs_backward(None, None, x, t, kept=kept).any()
    assert hip_ops.device_status() == 0


# ---------------------------------------------------------------------------
# rows past 32-bit offsets
# ---------------------------------------------------------------------------
def test_scan_past_32_bits():
    L, C, n = 70000, 32768, 90
    g = torch.Generator(device=DEV).manual_seed(1)
    v, w, f = (torch.randn(L, C, generator=g, device=DEV, dtype=torch.bfloat16)[None] for _ in range(3))
    starts = [0, L - n, L]
    h, last = hip_ops.gated_scan(v, w, f, seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    cols = torch.tensor([0, 1, 5000, C - 2, C - 1])
    part = [t[:, L - n:, cols.to(DEV)].cpu() for t in (v, w, f)]
    r = scan_ref(*part, None, None, None)
    within(h[:, L - n:, cols.to(DEV)], *r["h"], "h")
    within(last[1:, cols.to(DEV)], *r["last"], "state")
    # behind the first 400 rows the start's decays keep nothing that counts: e^-280, for decays of sigmoid(N(0, 1))
    r = scan_ref(*(t[:, L - n - 490:L - n, cols.to(DEV)].cpu() for t in (v, w, f)), None, None, None)
    within(h[:, L - n - 90:L - n, cols.to(DEV)], *(x[:, 400:] for x in r["h"]), "h")


def test_products_past_32_bits():
    M, K, N = (1 << 31) // 1024 + 200, 24, 1032
    g = torch.Generator(device=DEV).manual_seed(2)
    x, grad = (torch.randn(M, n, generator=g, device=DEV, dtype=torch.bfloat16) for n in (K, N))
    w = torch.randn(N, K, generator=g, device=DEV, dtype=torch.bfloat16)
    y, kept = hip_ops.fused_linear(x, w, act="silu", keep=True)
    dx, _, _ = hip_ops.fused_linear_backward(grad, x, w, kept=kept, act="silu", need_weight=False)
    del kept
    last = slice(M - 300, M)
    r = dense_ref(x[last].cpu(), w.cpu(), None, None, None, "silu", grad[last].cpu())
    within(y[last], *r["y"], "y")
    within(dx[last], *r["dx"], "dx")


def test_log_probs_past_32_bits():
    rows, V = 43000, 50001
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(rows, V, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    grad = torch.randn(rows, generator=g, device=DEV)
    logp, entropy, _, _, kept = hip_ops.token_log_probs(x, t, keep=True)
    d = hip_ops.token_log_probs_backward(grad, None, x, t, kept=kept)
    for some in (slice(rows - 20, rows), slice(0, 5)):
        r = logp_ref(x[some].cpu(), t[some].cpu(), 0, -100, grad[some].cpu(), None)
        within(logp[some], *r["logp"], "logp")
        within(entropy[some], *r["entropy"], "entropy")
        within(d[some], *r["dx"], "dx")


# ---------------------------------------------------------------------------
# calls beside calls: repeats, streams, graphs
# ---------------------------------------------------------------------------
def _everything(dtype, seed, dev=_dev):
    """One call of every operator and of its backward pass; returns a function that makes them all."""
    s = scan_case(seed, 1, 700, 130, dtype, starts=[0, 300, 690])
    s_args = [dev(s[k]) for k in ("value", "write", "decay", "bias")]
    s_how = dict(state=dev(s["state"]), seq_starts=torch.tensor(s["starts"], dtype=torch.int32, device=DEV))
    s_grad, s_last = dev(s["grad"]), dev(s["grad_state"])
    p = dense_case(seed + 1, 700, 130, 72, dtype, pair=True)
    px, pw, pu, pg = (dev(p[k]) for k in ("x", "w", "up", "grad"))
    m = dense_case(seed + 2, 300, 72, 40, dtype, bias=True, residual=True)
    mx, mw, mb, mr, mg = (dev(m[k]) for k in ("x", "w", "bias", "residual", "grad"))
    f = dense_case(seed + 3, 5, 200, 90, dtype, pair=True)
    fx, fw, fu = (dev(f[k]) for k in ("x", "w", "up"))
    x, t, g, e = (dev(v) for v in logp_case(seed + 4, 9, 40000, dtype))

    def call():
        h, last, kept = hip_ops.gated_scan(*s_args, keep=True, **s_how)
        out = [h, last, *hip_ops.gated_scan_backward(s_grad, *s_args, kept=kept, grad_state=s_last, **s_how)]
        state = last.clone()
        out += [hip_ops.gated_scan_step(*(a[0, :2] for a in s_args[:3]), s_args[3], state=state), state]
        y, kept = hip_ops.gated_linear(px, pw, pu, keep=True)
        out += [y, *hip_ops.gated_linear_backward(pg, px, pw, pu, kept=kept)]
        y, kept = hip_ops.fused_linear(mx, mw, mb, act="gelu", residual=mr, keep=True)
        out += [y, *hip_ops.fused_linear_backward(mg, mx, mw, mb, kept=kept, act="gelu"), hip_ops.gated_linear(fx, fw, fu)]
        logp, entropy, best, tokens, kept = hip_ops.token_log_probs(x, t, top=5, keep=True)
        return out + [logp, entropy, best, tokens, hip_ops.token_log_probs_backward(g, e, x, t, kept=kept)]
    return call


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", BOTH)
def test_results_repeat_bit_for_bit(dtype):
    call = _everything(dtype, 31)
    first = call()
    for _ in range(5):
        assert _same(first, call())


def test_two_streams_at_once():
    a, b = _everything(torch.bfloat16, 41), _everything(torch.bfloat16, 51)
    want = a(), b()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(one):
            x = a()
        with torch.cuda.stream(two):
            y = b()
        torch.cuda.synchronize()
        assert _same(x, want[0]) and _same(y, want[1])


@pytest.mark.parametrize("dtype", BOTH)
def test_two_captured_graphs(dtype):
    """Replays in turn, with eager calls and synchronizations between them, against the eager results."""
    calls = [_everything(dtype, 61), _everything(dtype, 71)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(c())
        graphs.append(graph)
    for i in (0, 1, 1, 0, 0, 1):
        for o in outs[i]:
            o.zero_()
        graphs[i].replay()
        if i:
            torch.cuda.synchronize()
        assert _same(calls[1 - i](), want[1 - i])
        assert _same(outs[i], want[i])
    graphs[0].replay()
    graphs[1].replay()
    assert _same(outs[0], want[0]) and _same(outs[1], want[1])


def test_autograd_is_refused_while_a_stream_is_captured():
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    x, t = torch.randn(4, 8, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.enable_grad(), torch.cuda.graph(graph):
        y = x + 1
        for call in (lambda: hip_ops.fused_linear(x, w), lambda: hip_ops.gated_linear(x, w, w),
                     lambda: hip_ops.gated_scan(w[None], w[None], w[None]), lambda: hip_ops.token_log_probs(w[:4], t)):
            with pytest.raises(RuntimeError, match="no autograd graph while"):
                call()
    graph.replay()
    assert torch.equal(y, x + 1)


# ---------------------------------------------------------------------------
# autograd
# ---------------------------------------------------------------------------
def _leaf(t):
    return t.to(DEV).requires_grad_() if t is not None else None


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("starts", [None, [0, 30, 140]])
def test_autograd_of_the_recurrence(dtype, starts):
    c = scan_case(8, 2 if starts is None else 1, 150, 20, dtype, starts=starts)
    leaves = [_leaf(c[k]) for k in ("value", "write", "decay", "bias", "state")]
    how = dict(seq_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV))
    h0, last0, grads = run_scan(c)
    with torch.enable_grad():
        h, last = hip_ops.gated_scan(*leaves[:4], state=leaves[4], **how)
        torch.autograd.backward([h, last], [_dev(c["grad"]), _dev(c["grad_state"])])
    assert torch.equal(h, h0) and torch.equal(last, last0)
    assert all(torch.equal(a.grad, b.to(a.dtype)) for a, b in zip(leaves, grads))
    # the states alone, and a gradient whose rows are one
    for a in leaves:
        a.grad = None
    with torch.enable_grad():
        _, last = hip_ops.gated_scan(*leaves[:4], state=leaves[4], **how)
        last.sum().backward()
    c["grad"], c["grad_state"] = torch.zeros_like(c["grad"]), torch.ones_like(c["grad_state"])
    check_scan(c, h0, last0, [a.grad for a in leaves])
    for a in leaves:
        a.grad = None
    with torch.enable_grad():
        hip_ops.gated_scan(*leaves[:4], state=leaves[4], **how)[0].sum().backward()
    c["grad"], c["grad_state"] = torch.ones_like(c["grad"]), torch.zeros_like(c["grad_state"])
    check_scan(c, h0, last0, [a.grad for a in leaves])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("act", ["silu", "gelu", None])
def test_autograd_of_projections(dtype, act):
    c = dense_case(9, 50, 40, 24, dtype, bias=True, residual=True)
    leaves = [_leaf(c[k]) for k in ("x", "w", "bias", "residual")]
    r = dense_ref(c["x"], c["w"], None, c["bias"], c["residual"], act, c["grad"])
    with torch.enable_grad():
        y = hip_ops.fused_linear(*leaves[:3], act=act, residual=leaves[3])
        y.backward(_dev(c["grad"]))
    within(y, *r["y"], "y")
    for a, name in zip(leaves, ("dx", "dw", "db")):
        within(a.grad, *r[name], name)
    assert torch.equal(leaves[3].grad, _dev(c["grad"]))
    if act:
        c = dense_case(10, 50, 40, 24, dtype, pair=True)
        leaves = [_leaf(c[k]) for k in ("x", "w", "up")]
        r = dense_ref(c["x"], c["w"], c["up"], None, None, act, torch.ones_like(c["grad"]))
        with torch.enable_grad():
            hip_ops.gated_linear(*leaves, act=act).sum().backward()
        for a, name in zip(leaves, ("dx", "dw", "du")):
            within(a.grad, *r[name], name)
    # a weight that takes no gradient, and both weights the same
    x, w = _leaf(c["x"]), _dev(c["w"])
    with torch.enable_grad():
        hip_ops.fused_linear(x, w).sum().backward()
    assert x.grad is not None and w.grad is None


@pytest.mark.parametrize("dtype", BOTH)
def test_one_weight_for_both_of_a_pair(dtype):
    c = dense_case(12, 40, 24, 16, dtype, pair=True)
    c["up"] = c["w"]
    r = dense_ref(c["x"], c["w"], c["w"], None, None, "silu", c["grad"])
    x, w = _leaf(c["x"]), _leaf(c["w"])
    with torch.enable_grad():
        hip_ops.gated_linear(x, w, w).backward(_dev(c["grad"]))
    both = r["dw"][0] + r["du"][0]
    within(w.grad, both, r["dw"][1] + r["du"][1] + HALF[dtype] * both.abs(), "dw + du")


@pytest.mark.parametrize("dtype", BOTH)
def test_autograd_of_log_probs(dtype):
    x, t, g, e = logp_case(13, 6, 500, dtype)
    a = _leaf(x)
    r = logp_ref(x, t, 4, -100, g, e)
    with torch.enable_grad():
        logp, entropy, best, tokens = hip_ops.token_log_probs(a, _dev(t), top=4)
        assert not best.requires_grad and not tokens.requires_grad
        torch.autograd.backward([logp, entropy], [_dev(g), _dev(e)])
    within(a.grad, *r["dx"], "dx")
    a.grad = None
    with torch.enable_grad():
        (-hip_ops.token_log_probs(a, _dev(t))[0].sum()).backward()
    within(a.grad, *logp_ref(x, t, 0, -100, -torch.ones(6), None)["dx"], "dx")


def test_second_derivatives_are_refused():
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    with torch.enable_grad():
        g, = torch.autograd.grad(hip_ops.fused_linear(w, w, act="silu").sum(), w, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            g.sum().backward()


# ---------------------------------------------------------------------------
# all of them: a recurrent block, its loss and the gradients of its weights
# ---------------------------------------------------------------------------
def _block(p, x, starts, targets, ops):
    gates = ops["linear"](x, p["w_in"], p["b_in"])
    v, w, f = gates.chunk(3, -1)
    h, last = ops["scan"](v, w, f, p["decay_bias"], p["state"], starts)
    x = ops["linear"](h, p["w_out"], None, x)
    x = ops["linear"](ops["gated"](x, p["w_gate"], p["w_up"]), p["w_down"], p["b_down"], x)
    logp, entropy = ops["logp"](ops["linear"](x, p["w_vocab"], None), targets)
    return -logp.sum() - 0.1 * entropy.sum(), last


def _plain_scan(v, w, f, bias, state, starts):
    a, u = torch.sigmoid(f + bias), torch.sigmoid(w) * torch.tanh(v)
    rows, last = [], []
    for s in range(len(starts) - 1):
        x = state[s]
        for t in range(starts[s], starts[s + 1]):
            x = a[0, t] * x + u[0, t]
            rows.append(x)
        last.append(x)
    return torch.stack(rows)[None], torch.stack(last)


def _plain_logp(logits, targets):
    lp = logits.log_softmax(-1)
    return lp.gather(-1, targets[..., None])[..., 0], -(lp.exp() * lp).sum(-1)


PLAIN = dict(scan=_plain_scan, logp=_plain_logp,
             linear=lambda x, w, b, r=None: x @ w.t() + (0 if b is None else b) + (0 if r is None else r),
             gated=lambda x, g, u: torch.nn.functional.silu(x @ g.t()) * (x @ u.t()))
OWN = dict(scan=lambda v, w, f, b, s, starts: hip_ops.gated_scan(v, w, f, b, state=s, seq_starts=starts),
           linear=lambda x, w, b, r=None: hip_ops.fused_linear(x, w, b, residual=r), gated=hip_ops.gated_linear,
           logp=lambda x, t: hip_ops.token_log_probs(x, t)[:2])


@pytest.mark.parametrize("dtype,most", [(torch.float32, 2.0 ** -17), (torch.bfloat16, 2.0 ** -4)])
def test_a_block_that_learns(dtype, most):
    """Loss and gradients against the plain block in 64 bits.  On the longest way through the block and back a value is rounded 14 times
    and meets as many rounded operands: 28 half steps of bfloat16, 2^-3.2, if all of them pulled one way; half of that is allowed.
    float32: 28 sums of up to 300 terms, 2^-24 sqrt(300) each, 2^-15 in all; a quarter of that is."""
    L, D, F, V, starts = 300, 64, 96, 200, [0, 170, 300]
    g = _gen(17)
    shapes = dict(w_in=(3 * D, D), b_in=(3 * D,), decay_bias=(D,), state=(2, D), w_out=(D, D), w_gate=(F, D), w_up=(F, D), w_down=(D, F),
                  b_down=(D,), w_vocab=(V, D))
    p = {k: (torch.randn(s, generator=g) / math.sqrt(s[-1] if len(s) > 1 else 1)).to(torch.float32 if k in ("decay_bias", "state") else dtype)
         for k, s in shapes.items()}
    x, targets = torch.randn(1, L, D, generator=g).to(dtype), torch.randint(0, V, (1, L), generator=g)
    own = {k: _leaf(v) for k, v in p.items()}
    plain = {k: v.double().requires_grad_() for k, v in p.items()}
    with torch.enable_grad():
        want, want_last = _block(plain, x.double(), starts, targets, PLAIN)
        (want + want_last.sum()).backward()
        got, last = _block(own, _dev(x), torch.tensor(starts, dtype=torch.int32, device=DEV), _dev(targets), OWN)
        (got + last.sum()).backward()
    assert abs(got.item() - want.item()) <= most * abs(want.item())
    for k in shapes:
        a, b = own[k].grad.double().cpu(), plain[k].grad
        assert (a - b).norm() <= most * b.norm(), (k, ((a - b).norm() / b.norm()).item())


# ---------------------------------------------------------------------------
# scores of a model's own tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("L", [1, 2, 17])
def test_score(L):
    cfg = TESMConfig.tiny()
    torch.manual_seed(0)
    model = TESMLMHeadModel(cfg).to(DEV).eval()
    ids = torch.randint(0, cfg.vocab_size, (3, L), generator=_gen(L)).to(DEV)
    ids[1, L - 1:] = cfg.label_ignore_index
    logp, entropy, best, tokens = model.score(ids, top=3)
    assert logp.shape == (3, L - 1) and tokens.shape == (3, L - 1, 3)
    logits = model(ids.clamp(min=0))[0].logits[:, :-1]
    r = logp_ref(logits.cpu(), ids[:, 1:].cpu(), 3, cfg.label_ignore_index)
    for a, name in ((logp, "logp"), (entropy, "entropy"), (best, "top")):
        within(a, *r[name], name)
    assert torch.equal(tokens.cpu(), r["tokens"])
    assert model.score(ids)[2] is None
