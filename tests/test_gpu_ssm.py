"""Short convolution, selective scan and their one-token step against the definitions in 64 bits, row by row.

Tolerances are bounds, elementwise.  ``u`` = 2^-24 is half a float32 step, ``e`` half a step of the layer type
(2^-8 relative for bfloat16).  ``mass`` is the sum of the magnitudes of a result's contributions.  A sum of n terms in
float32 is off by at most n u mass; chunked products add their decays' errors (an exponential of a few ulps for every
chunk passed).  With bfloat16 operands each contribution is rounded to bfloat16 once on the way (the decayed score inside
a chunk, the state read across chunks: e mass in all); states are sums of products whose scaled operand is held whole, as
three bfloat16 parts.  The result is rounded once: e |y|.
"""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from tesm_amd import hip_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _dev(t):
    return t.to(DEV) if t is not None else None


def _within(got, want, tol, what):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol)
    bad &= ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol)[bad].max())} x"


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------
def conv_ref(x, w, b, silu, state, spans):
    """(y, mass, state) in 64 bits over rows (M, C); ``spans``: the rows of every sequence."""
    M, C = x.shape
    W = w.shape[1]
    y, mass = torch.zeros(M, C, dtype=torch.float64), torch.zeros(M, C, dtype=torch.float64)
    new = torch.zeros(len(spans), W - 1, C, dtype=torch.float64)
    for s, (lo, hi) in enumerate(spans):
        before = state[s].double() if state is not None else torch.zeros(W - 1, C, dtype=torch.float64)
        rows = torch.cat([before, x[lo:hi].double()])
        new[s] = rows[rows.shape[0] - (W - 1):]
        for t in range(hi - lo):
            win = rows[t:t + W] * w.double().t()
            y[lo + t] = win.sum(0) + (b.double() if b is not None else 0)
            mass[lo + t] = win.abs().sum(0) + (b.double().abs() if b is not None else 0)
    return (_silu(y) if silu else y), mass, new


def _conv_check(x, w, b, silu, state, starts, out, y, new, lens, dtype):
    spans, at = [], 0
    if starts is None:
        B, L = x.shape[:2]
        spans = [(i * L, i * L + L) for i in range(B)]
    else:
        spans = list(zip(starts[:-1], starts[1:]))
    C, W = w.shape
    want, mass, want_new = conv_ref(x.reshape(-1, C), w, b, silu, state, spans)
    # silu's slope is at most 1.1; its own exponential and reciprocal are good to 8 u
    tol = 1.1 * (W + 1) * U * mass + (8 * U + HALF[dtype]) * want.abs() + 1e-37
    got = y.reshape(-1, C)
    for lo, hi in spans:
        _within(got[lo:hi], want[lo:hi], tol[lo:hi], "conv")
    assert torch.equal(new.cpu().double(), want_new)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C,W", [(1, 1, 8, 4), (2, 3, 5, 4), (3, 70, 64, 4), (1, 129, 257, 2), (2, 33, 1032, 8), (4, 2, 96, 6),
                                     (2, 300, 40, 3)])
@pytest.mark.parametrize("init,silu,bias", [(False, True, True), (True, False, False)])
def test_conv(dtype, B, L, C, W, init, silu, bias):
    g = torch.Generator().manual_seed(B * 1000 + L + C + W)
    x, w = _randn(g, B, L, C, dtype=dtype), _randn(g, C, W, dtype=dtype)
    b = _randn(g, C, dtype=dtype) if bias else None
    state = _randn(g, B, W - 1, C, dtype=dtype) if init else None
    y, new = hip_ops.causal_conv(_dev(x), _dev(w), _dev(b), silu=silu, state=_dev(state))
    assert y.shape == x.shape and y.dtype == dtype
    _conv_check(x, w, b, silu, state, None, None, y, new, None, dtype)


PACKED = [[0, 0, 1, 4, 4, 70, 135, 136], [3, 20, 20, 84, 200], [0, 64, 128, 129], [0, 5], [0, 0], [2, 2, 2]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts", PACKED)
@pytest.mark.parametrize("C,init", [(24, True), (9, False), (512, True)])
def test_conv_packed_leaves_other_rows(dtype, starts, C, init):
    g = torch.Generator().manual_seed(len(starts) + C)
    M, S, W = starts[-1] + 7, len(starts) - 1, 4
    x, w, b = _randn(g, 1, M, C, dtype=dtype), _randn(g, C, W, dtype=torch.float32), _randn(g, C, dtype=torch.float32)
    state = _randn(g, S, W - 1, C, dtype=dtype) if init else None
    out = torch.full((1, M, C), 7.0, dtype=dtype, device=DEV)
    y, new = hip_ops.causal_conv(_dev(x), _dev(w), _dev(b), state=_dev(state),
                                 seq_starts=torch.tensor(starts, dtype=torch.int32, device=DEV), out=out)
    assert y is out
    _conv_check(x, w, b, True, state, starts, out, y, new, None, dtype)
    assert bool((out[0, :starts[0]] == 7).all()) and bool((out[0, starts[-1]:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off,C", [(0, 64), (1, 64), (8, 40), (3, 33)])
def test_conv_of_column_slices(dtype, off, C):
    """x and out are columns of wider rows, at aligned and unaligned places."""
    g = torch.Generator().manual_seed(off + C)
    wide = _randn(g, 2, 50, 128, dtype=dtype)
    w = _randn(g, C, 4, dtype=dtype)
    out = torch.full((2, 50, 136), 3.0, dtype=dtype, device=DEV)
    x = wide[..., off:off + C]
    y, new = hip_ops.causal_conv(_dev(wide)[..., off:off + C], _dev(w), None, out=out[..., off:off + C])
    _conv_check(x, w, None, True, None, None, out, y, new, None, dtype)
    assert bool((out[..., :off] == 3).all()) and bool((out[..., off + C:] == 3).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_non_finite_rows_reach_only_their_window(dtype):
    g = torch.Generator().manual_seed(5)
    x, w = _randn(g, 1, 40, 16, dtype=dtype), _randn(g, 16, 4, dtype=dtype)
    bad = x.clone()
    bad[0, 20] = float("nan")
    bad[0, 30] = float("inf")
    y, _ = hip_ops.causal_conv(_dev(x), _dev(w))
    yb, _ = hip_ops.causal_conv(_dev(bad), _dev(w))
    keep = [t for t in range(40) if not 20 <= t <= 23 and not 30 <= t <= 33]
    assert torch.equal(y[0, keep], yb[0, keep])
    assert bool(yb[0, 20:24].isnan().all())


def test_conv_continues_where_it_stopped():
    """A prompt in two parts, the state handed on, gives the bits of the whole prompt."""
    g = torch.Generator().manual_seed(6)
    x, w = _randn(g, 2, 37, 24, dtype=torch.bfloat16).to(DEV), _randn(g, 24, 4, dtype=torch.bfloat16).to(DEV)
    y, new = hip_ops.causal_conv(x, w)
    for cut in (1, 2, 16, 36):
        ya, sa = hip_ops.causal_conv(x[:, :cut], w)
        yb, sb = hip_ops.causal_conv(x[:, cut:], w, state=sa)
        assert torch.equal(torch.cat([ya, yb], 1), y) and torch.equal(sb, new)


# ---------------------------------------------------------------------------
# scan
# ---------------------------------------------------------------------------
def scan_ref(c, spans, M):
    """(y, tolerance of y before its rounding as mass and count, h, h's mass) in 64 bits over rows."""
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    f = {k: (c[k].reshape(M, *c[k].shape[2:]).double() if c[k] is not None else None) for k in ("x", "dt", "B", "C", "z")}
    raw = f["dt"] + (c["dt_bias"].double() if c["dt_bias"] is not None else 0)
    d = torch.nn.functional.softplus(raw, threshold=700) if c["softplus"] else raw
    d = torch.where(raw < -30, raw.exp(), d) if c["softplus"] else d
    a = (d * c["A"].double()).exp()
    y, mass = torch.zeros(M, H, P, dtype=torch.float64), torch.zeros(M, H, P, dtype=torch.float64)
    hs, ms = [], []
    for s, (lo, hi) in enumerate(spans):
        h = c["h0"][s].double() if c["h0"] is not None else torch.zeros(H, P, N, dtype=torch.float64)
        m = h.abs()
        for t in range(lo, hi):
            b, cc = (f[k][t].repeat_interleave(H // G, 0) for k in ("B", "C"))
            add = (d[t][:, None] * f["x"][t])[..., None] * b[:, None]
            h = a[t][:, None, None] * h + add
            m = a[t][:, None, None] * m + add.abs()
            y[t] = (h * cc[:, None]).sum(-1)
            mass[t] = (m * cc[:, None].abs()).sum(-1)
        hs.append(h)
        ms.append(m)
    if c["D"] is not None:
        skip = c["D"].double()[:, None] * f["x"]
        y, mass = y + skip, mass + U / HALF[c["dtype"]] * skip.abs()
    if f["z"] is not None:
        gate = _silu(f["z"])
        y, mass = y * gate, mass * gate.abs()
    empty = torch.zeros(0, H, P, N, dtype=torch.float64)
    return y, mass, torch.stack(hs) if hs else empty, torch.stack(ms) if ms else empty


def _scan_case(seed, B, L, H, P, G, N, dtype, starts=None, init=True, gate=True, skip=True, bias=True, softplus=True):
    g = torch.Generator().manual_seed(seed)
    S = B if starts is None else len(starts) - 1
    c = dict(H=H, P=P, G=G, N=N, dtype=dtype, softplus=softplus, starts=starts)
    c["x"] = _randn(g, B, L, H, P, dtype=dtype)
    c["dt"] = (_randn(g, B, L, H) if softplus else 0.3 * torch.rand(B, L, H, generator=g)).to(dtype)
    c["B"], c["C"] = _randn(g, B, L, G, N, dtype=dtype), _randn(g, B, L, G, N, dtype=dtype)
    c["A"] = -(0.3 + 4 * torch.rand(H, generator=g))
    c["D"] = _randn(g, H) if skip else None
    c["z"] = _randn(g, B, L, H, P, dtype=dtype) if gate else None
    c["dt_bias"] = (-4 + 3 * torch.rand(H, generator=g)) if bias else None
    c["h0"] = _randn(g, S, H, P, N) if init else None
    return c


def _run_scan(c, **kw):
    starts = torch.tensor(c["starts"], dtype=torch.int32, device=DEV) if c["starts"] is not None else None
    return hip_ops.selective_scan(_dev(c["x"]), _dev(c["dt"]), _dev(c["A"]), _dev(c["B"]), _dev(c["C"]), D=_dev(c["D"]),
                                  z=_dev(c["z"]), dt_bias=_dev(c["dt_bias"]), softplus=c["softplus"], state=_dev(c["h0"]),
                                  seq_starts=starts, **kw)


def _check_scan(c, y, h):
    nb, L = c["x"].shape[:2]
    M = nb * L
    spans = [(i * L, i * L + L) for i in range(nb)] if c["starts"] is None else list(zip(c["starts"][:-1], c["starts"][1:]))
    want, mass, want_h, mass_h = scan_ref(c, spans, M)
    e = HALF[c["dtype"]]
    longest = max([b - a for a, b in spans], default=0)
    # dot products over states and rows of a chunk, six roundings for each chunk of 32 rows passed, softplus and decays
    count = c["N"] + 3 * min(longest, 64) + 6 * (longest // 32 + 1) + 64
    between = e if c["dtype"] == torch.bfloat16 else 0.0
    tol = (between * 1.01 + count * U) * mass + (e + 8 * U) * want.abs() + 1e-36
    got = y.reshape(M, c["H"], c["P"])
    for lo, hi in spans:
        _within(got[lo:hi], want[lo:hi], tol[lo:hi], "scan rows %d..%d" % (lo, hi))
    _within(h, want_h, count * U * mass_h + 1e-36, "scan state")


SCANS = [  # B, L, H, P, G, N
    (1, 1, 1, 1, 1, 1), (2, 1, 4, 64, 1, 128), (1, 7, 2, 64, 1, 16), (1, 64, 2, 64, 1, 128), (2, 65, 3, 32, 3, 64),
    (1, 130, 4, 64, 2, 128), (1, 200, 5, 40, 1, 56), (2, 77, 2, 128, 1, 32), (1, 300, 6, 64, 2, 256), (1, 33, 3, 97, 1, 5),
    (3, 128, 8, 16, 4, 100), (1, 31, 2, 8, 2, 147), (1, 1100, 1, 32, 1, 128),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,P,G,N", SCANS)
@pytest.mark.parametrize("full", [True, False])
def test_scan(dtype, B, L, H, P, G, N, full):
    c = _scan_case(B + L + H + P + N, B, L, H, P, G, N, dtype, init=full, gate=full, skip=full, bias=full, softplus=True)
    y, h = _run_scan(c)
    assert y.dtype == dtype and y.shape == c["x"].shape and h.dtype == torch.float32
    _check_scan(c, y, h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_without_softplus(dtype):
    c = _scan_case(9, 2, 90, 3, 64, 1, 64, dtype, softplus=False, bias=False)
    _check_scan(c, *_run_scan(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts", PACKED + [[0, 1000, 1003, 1700], [0] + list(range(1, 71))])
@pytest.mark.parametrize("H,P,G,N,init", [(4, 64, 2, 128, True), (3, 24, 1, 33, False)])
def test_scan_packed_leaves_other_rows(dtype, starts, H, P, G, N, init):
    M = starts[-1] + 5
    c = _scan_case(len(starts) + H, 1, M, H, P, G, N, dtype, starts=starts, init=init)
    out = torch.full((1, M, H, P), 7.0, dtype=dtype, device=DEV)
    y, h = _run_scan(c, out=out)
    assert y is out
    _check_scan(c, y, h)
    assert bool((out[0, :starts[0]] == 7).all()) and bool((out[0, starts[-1]:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_scan_of_column_slices(dtype, off):
    """x, B, C, z and y as columns of wider rows, at aligned and unaligned places."""
    B, L, H, P, G, N = 2, 70, 3, 32, 1, 48
    c = _scan_case(21 + off, B, L, H, P, G, N, dtype)
    wide = torch.full((B, L, off + H * P + 2 * G * N + 8), 5.0, dtype=dtype, device=DEV)
    wide[..., off:off + H * P] = _dev(c["x"]).flatten(2)
    wide[..., off + H * P:off + H * P + G * N] = _dev(c["B"]).flatten(2)
    wide[..., off + H * P + G * N:off + H * P + 2 * G * N] = _dev(c["C"]).flatten(2)
    out = torch.full((B, L, H * P + 24), 5.0, dtype=dtype, device=DEV)
    y, h = hip_ops.selective_scan(wide[..., off:off + H * P].unflatten(-1, (H, P)), _dev(c["dt"]), _dev(c["A"]),
                                  wide[..., off + H * P:off + H * P + G * N].unflatten(-1, (G, N)),
                                  wide[..., off + H * P + G * N:off + H * P + 2 * G * N].unflatten(-1, (G, N)), D=_dev(c["D"]),
                                  z=_dev(c["z"]), dt_bias=_dev(c["dt_bias"]), state=_dev(c["h0"]),
                                  out=out[..., off:off + H * P].unflatten(-1, (H, P)))
    _check_scan(c, y, h)
    assert bool((out[..., :off] == 5).all()) and bool((out[..., off + H * P:] == 5).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_scan_non_finite_rows_leave_earlier_rows(dtype, bad):
    """A row that is no number reaches its own channel from that row on, and nothing else."""
    c = _scan_case(31, 1, 150, 2, 64, 1, 64, dtype)
    y, h = _run_scan(c)
    c["x"] = c["x"].clone()
    c["x"][0, 90, 1, 5] = bad
    yb, hb = _run_scan(c)
    assert torch.equal(y[:, :90], yb[:, :90])
    others = [p for p in range(64) if p != 5]
    assert torch.equal(y[:, :, 0], yb[:, :, 0]) and torch.equal(y[:, :, 1, others], yb[:, :, 1, others])
    assert not bool(yb[0, 90, 1, 5].isfinite())
    assert not bool(hb[0, 1, 5].isfinite().any()) and torch.equal(h[:, 0], hb[:, 0])
    for name in ("B", "C", "dt", "z"):
        c = _scan_case(31, 1, 150, 2, 64, 1, 64, dtype)
        c[name] = c[name].clone()
        c[name][0, 90] = bad
        assert torch.equal(y[:, :90], _run_scan(c)[0][:, :90]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_strong_decays(dtype):
    """Decays from e^-400 a row to none at all, in one chunk: no overflow, no difference of large sums left over."""
    c = _scan_case(41, 1, 140, 4, 32, 1, 32, dtype, softplus=False, bias=False)
    c["dt"][0, ::7] = 100.0
    c["dt"][0, 1::7] = 0.0
    c["dt"][0, 2::7] = 1e-3
    c["x"][0, ::7] *= 2.0 ** -6
    c["A"] = torch.tensor([-4.0, -0.5, -1e-3, 0.0])
    _check_scan(c, *_run_scan(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_growing_states_and_large_values(dtype):
    """Rates above zero (the state grows by e^4 over a chunk), and channels near 2^100: no scale on the way overflows."""
    c = _scan_case(42, 1, 200, 4, 32, 1, 32, dtype, softplus=False, bias=False, gate=False)
    c["A"] = torch.tensor([0.8, 0.4, 1e-3, -0.8])
    c["x"][0, :, 2:] *= 2.0 ** 100
    _check_scan(c, *_run_scan(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_state_holds_float32(dtype):
    """One row's addend, decayed over two chunks.  In units of 2^-24: the decay inside the chunk and the second chunk's, 2 for
    the exponential's value and 1 for its rounded argument each; d's and x's products 2; the scale's reciprocal and its two
    uses 4; the three parts of the addend's product 6 (the matrix unit may cut instead of rounding); the scale's product 1:
    19, and with as much again for what the library's exponential adds, 32."""
    c = _scan_case(43, 1, 50, 4, 64, 1, 128, dtype, init=False, softplus=False, bias=False, gate=False, skip=False)
    x = torch.zeros_like(c["x"])
    x[0, 5] = c["x"][0, 5]
    c["x"], c["A"] = x, -0.05 * torch.arange(1.0, 5.0)
    c["dt"] = torch.full_like(c["dt"], 0.25)
    c["A"] = c["A"].bfloat16().float()
    h = _run_scan(c)[1].cpu().double()
    decay = (c["A"].double() * 0.25 * 44).exp()
    want = 0.25 * decay[:, None, None] * c["x"][0, 5].double()[..., None] * c["B"][0, 5, 0].double()
    assert bool(((h[0] - want).abs() <= 32 * U * want.abs()).all())


def test_scan_of_decreasing_starts_stays_in_its_memory():
    """Starts that decrease are no valid input: what they give is not looked at, but nothing else is touched."""
    c = _scan_case(72, 1, 1000, 2, 16, 1, 16, torch.float32, starts=[0, 1000])
    y, h = _run_scan(c)
    bad = dict(c, starts=[0, 1000] * 8, h0=torch.zeros(15, 2, 16, 16))
    keep = [t.clone() for t in (y, h)]
    _run_scan(bad)
    assert torch.equal(y, keep[0]) and torch.equal(h, keep[1])
    again = _run_scan(c)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_same_bits_twice_and_for_equal_sequences(dtype):
    c = _scan_case(51, 1, 333, 4, 64, 1, 128, dtype)
    for k in ("x", "dt", "B", "C", "z", "h0"):
        c[k] = c[k].expand(3, *c[k].shape[1:]).contiguous()
    y, h = _run_scan(c)
    y2, h2 = _run_scan(c)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2]) and torch.equal(h[0], h[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_empty(dtype):
    c = _scan_case(61, 2, 0, 2, 8, 1, 16, dtype)
    y, h = _run_scan(c)
    assert y.shape == (2, 0, 2, 8) and torch.equal(h.cpu(), c["h0"])
    c = _scan_case(61, 0, 5, 2, 8, 1, 16, dtype)
    y, h = _run_scan(c)
    assert y.shape == (0, 5, 2, 8) and h.shape == (0, 2, 8, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_and_scan_on_two_streams_at_once(dtype):
    """Calls under way together keep to workspaces of their own; a captured convolution repeats."""
    cs = [_scan_case(91 + i, 1, 900, 4, 64, 1, 128, dtype) for i in range(2)]
    args = [{k: (_dev(v) if torch.is_tensor(v) else v) for k, v in c.items()} for c in cs]
    w = _randn(torch.Generator().manual_seed(3), 4 * 64, 4, dtype=dtype).to(DEV)

    def call(a):
        x, _ = hip_ops.causal_conv(a["x"].view(1, 900, 256), w)
        return hip_ops.selective_scan(x.view(1, 900, 4, 64), a["dt"], a["A"], a["B"], a["C"], dt_bias=a["dt_bias"])
    want = [call(a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, capture_error_mode="relaxed"):
        held = call(args[0])
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for a, st in zip(args, streams):
            with torch.cuda.stream(st):
                got.append(call(a))
        gr.replay()
        torch.cuda.synchronize()
        for o, v in zip(got + [held], want + want[:1]):
            assert torch.equal(o[0], v[0]) and torch.equal(o[1], v[1])


def test_scan_launches():
    """Whole slices and states take the kernels without edges; long sequences are divided, short ones are not."""
    def names(*a):
        c = _scan_case(5, *a, torch.bfloat16)
        with hip_ops.launch_log() as log:
            _run_scan(c)
        return [k for k in log.kernels if "ssm_" in k]
    short, long, ragged = names(1, 64, 2, 64, 1, 128), names(1, 700, 2, 64, 1, 128), names(1, 700, 2, 40, 1, 100)
    assert len(short) == 1 and len(long) == 3 and len(ragged) == 3
    assert "ssm_carry_kernel" in long[1] and "ssm_carry_kernel" in ragged[1] and long[2] == short[0] != ragged[2]


def test_scan_reads_starts_that_run_past_the_rows_as_the_last_row():
    c = _scan_case(71, 1, 50, 2, 16, 1, 16, torch.float32, starts=[0, 30, 50])
    y, h = _run_scan(c)
    c["starts"] = [-4, 30, 90]
    y2, h2 = _run_scan(c)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_captured_and_replayed(dtype):
    """Two graphs captured on one stream, replayed in turn with eager calls between."""
    cs = [_scan_case(81 + i, 1, 700 + 64 * i, 4, 64, 1, 64, dtype) for i in range(2)]
    args = [{k: (_dev(v) if torch.is_tensor(v) else v) for k, v in c.items()} for c in cs]

    def call(a):
        return hip_ops.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], D=a["D"], z=a["z"], dt_bias=a["dt_bias"],
                                      state=a["h0"])
    want = [call(a) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, capture_error_mode="relaxed"):
            outs.append(call(a))
        graphs.append(gr)
    for _ in range(3):
        for i in (0, 1):
            outs[i][0].zero_()
            outs[i][1].zero_()
            graphs[i].replay()
            eager = call(args[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(eager[0], want[1 - i][0])
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------
STEPS = [(1, 1, 1, 1, 1, 4), (1, 24, 64, 1, 128, 4), (3, 4, 40, 2, 56, 2), (2, 3, 97, 1, 5, 3), (5, 8, 16, 4, 256, 8), (2, 2, 128, 2, 147, 4),
         (4, 6, 64, 3, 16, 4)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,P,G,N,W", STEPS)
@pytest.mark.parametrize("conv", [True, False])
def test_step(dtype, B, H, P, G, N, W, conv):
    g = torch.Generator().manual_seed(B + H + P + N)
    width = H * P + 2 * G * N
    wide = _randn(g, B, width + 3, dtype=dtype)
    row, dt, z = wide[:, :width], _randn(g, B, H, dtype=dtype), _randn(g, B, H, P, dtype=dtype)
    A, D, bias = -(0.3 + 4 * torch.rand(H, generator=g)), _randn(g, H), -3 + 2 * torch.rand(H, generator=g)
    h = _randn(g, B, H, P, N)
    w, wb, cs = _randn(g, width, W, dtype=dtype), _randn(g, width, dtype=dtype), _randn(g, B, W - 1, width, dtype=dtype)
    hd = _dev(h).clone()
    extra = (_dev(w), _dev(wb), _dev(cs)) if conv else ()
    y, new = hip_ops.selective_scan_step(_dev(wide)[:, :width], _dev(dt), _dev(A), hd, *extra, n_groups=G, D=_dev(D), z=_dev(z),
                                         dt_bias=_dev(bias))
    v = row.double()
    dv = torch.zeros_like(v)
    if conv:
        win = torch.cat([cs, row[:, None]], 1).double() * w.double().t()
        v = _silu(win.sum(1) + wb.double())
        dv = 1.1 * (W + 1) * U * (win.abs().sum(1) + wb.double().abs()) + 8 * U * v.abs()
        assert torch.equal(new.cpu(), torch.cat([cs, row[:, None]], 1)[:, 1:])
    else:
        assert new is None
    cut = [H * P, G * N, G * N]
    (x, b, c), (dx, db, dc) = v.split(cut, 1), dv.split(cut, 1)
    x, dx = (t.reshape(B, H, P) for t in (x, dx))
    b, c, db, dc = (t.reshape(B, G, N).repeat_interleave(H // G, 1)[:, :, None] for t in (b, c, db, dc))
    d = torch.nn.functional.softplus(dt.double() + bias.double())
    a = (d * A.double()).exp()[..., None, None]
    add = (d[..., None] * x)[..., None] * b
    hn = a * h.double() + add
    mass = (a * h.double()).abs() + add.abs()
    # the convolved values' own error, then a rounding for each of: exponent (|d A| < 30 in steps of u), product, sum
    dh = d[..., None, None] * (dx[..., None] * b.abs() + x.abs()[..., None] * db) + 48 * U * mass
    _within(hd, hn, dh + 1e-36, "step state")
    gate = _silu(z.double())
    want = ((hn * c).sum(-1) + D.double()[:, None] * x) * gate
    ym = (hn.abs() * c.abs()).sum(-1) + (D.double()[:, None] * x).abs()
    tol = gate.abs() * ((dh * c.abs() + hn.abs() * dc).sum(-1) + D.double().abs()[:, None] * dx + (N + 16) * U * ym)
    _within(y, want, tol + (HALF[dtype] + 8 * U) * want.abs() + 1e-36, "step y")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_follows_the_scan(dtype):
    """Tokens one by one from a prompt's states give the whole prompt's rows, within the scan's own bounds."""
    B, L, H, P, G, N, cut = 2, 90, 4, 64, 2, 64, 70
    c = _scan_case(91, B, L, H, P, G, N, dtype, init=False)
    first = dict(c, **{k: c[k][:, :cut] for k in ("x", "dt", "B", "C", "z")})
    y, h = _run_scan(first)
    ys = [y]
    for t in range(cut, L):
        row = torch.cat([c["x"][:, t].flatten(1), c["B"][:, t].flatten(1), c["C"][:, t].flatten(1)], 1)
        yt, _ = hip_ops.selective_scan_step(_dev(row), _dev(c["dt"][:, t]), _dev(c["A"]), h, n_groups=G, D=_dev(c["D"]),
                                            z=_dev(c["z"][:, t]), dt_bias=_dev(c["dt_bias"]))
        ys.append(yt[:, None])
    _check_scan(c, torch.cat(ys, 1), h)


def test_step_other_stream_and_graph():
    """On a side stream, and captured with two conv states in turn: every replay is the next token."""
    g = torch.Generator().manual_seed(7)
    B, H, P, G, N, W, T = 2, 4, 32, 1, 64, 4, 6
    width = H * P + 2 * G * N
    rows, dts = _randn(g, T, B, width).to(DEV), _randn(g, T, B, H).to(DEV)
    w, A = _randn(g, width, W).to(DEV), -torch.rand(H, generator=g).to(DEV)
    h, cs = torch.zeros(B, H, P, N, device=DEV), torch.zeros(B, W - 1, width, device=DEV)
    want = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in range(T):
            y, cs = hip_ops.selective_scan_step(rows[t], dts[t], A, h, w, None, cs)
            want.append(y.clone())
    torch.cuda.current_stream().wait_stream(side)
    row, dt = rows[0].clone(), dts[0].clone()
    h2, two, outs, graphs = torch.zeros_like(h), [torch.zeros_like(cs) for _ in range(2)], [], []
    for i in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, capture_error_mode="relaxed"):
            outs.append(hip_ops.selective_scan_step(row, dt, A, h2, w, None, two[i], conv_state_out=two[1 - i])[0])
        graphs.append(gr)
    for t in range(T):
        row.copy_(rows[t])
        dt.copy_(dts[t])
        graphs[t % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[t % 2], want[t])
    assert torch.equal(h2, h)
