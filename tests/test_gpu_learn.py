"""The operators that learn (gated recurrence, float projections, log probabilities) against their 64-bit forms."""
import math

import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_refs import HALF, U, dense_ref, logp_ref, scan_ref, within
from tesm_amd import hip_ops

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


def _dev(t):
    return t.to(DEV) if t is not None else None


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


# ---------------------------------------------------------------------------
# recurrence
# ---------------------------------------------------------------------------
def scan_case(seed, B, L, C, dtype, starts=None, state=True, bias=True):
    g = _gen(seed)
    S = B if starts is None else len(starts) - 1
    c = {k: _randn(g, B, L, C, dtype=dtype) for k in ("value", "write", "decay", "grad")}
    c["bias"] = 1 + 5 * torch.rand(C, generator=g) if bias else None
    c["state"] = 0.5 * _randn(g, S, C) if state else None
    c["grad_state"] = _randn(g, S, C) if state else None
    c["starts"] = starts
    return c


def run_scan(c, dev=_dev):
    args = [dev(c[k]) for k in ("value", "write", "decay", "bias")]
    how = dict(state=dev(c["state"]), seq_starts=None if c["starts"] is None else torch.tensor(c["starts"], dtype=torch.int32, device=DEV))
    h, last, kept = hip_ops.gated_scan(*args, keep=True, **how)
    grads = hip_ops.gated_scan_backward(dev(c["grad"]), *args, kept=kept, grad_state=dev(c["grad_state"]), **how)
    return h, last, grads


def check_scan(c, h, last, grads):
    r = scan_ref(c["value"], c["write"], c["decay"], c["bias"], c["state"], c["starts"], c["grad"], c["grad_state"])
    within(h, *r["h"], "h")
    within(last, *r["last"], "state")
    for got, name in zip(grads, ("dv", "dw", "dd", "db", "ds")):
        if got is None:
            assert (name == "db" and c["bias"] is None) or (name == "ds" and c["state"] is None)
            continue
        within(got, *r[name], name)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,L,C", [(1, 1, 1), (2, 5, 3), (1, 16, 64), (3, 17, 66), (1, 127, 128), (2, 128, 130), (1, 129, 65), (2, 300, 96)])
def test_scan(dtype, B, L, C):
    c = scan_case(B + L + C, B, L, C, dtype)
    check_scan(c, *run_scan(c))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("L", [2047, 2048, 2049, 4500])
def test_scan_over_groups_of_tiles(dtype, L):
    """Chains longer than 16 tiles hand on their state as well."""
    c = scan_case(L, 1, L, 6, dtype, state=False)
    check_scan(c, *run_scan(c))


@pytest.mark.parametrize("bias,state", [(False, True), (True, False), (False, False)])
def test_scan_without_options(bias, state):
    c = scan_case(9, 2, 150, 10, torch.bfloat16, bias=bias, state=state)
    check_scan(c, *run_scan(c))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("starts", [[0, 1, 1, 130, 400, 400], [3, 3, 131, 259, 390], [0, 400], [0, 0], [7, 8]])
def test_scan_of_packed_sequences(dtype, starts):
    c = scan_case(sum(starts), 1, 400, 34, dtype, starts=starts)
    check_scan(c, *run_scan(c))


# ---------------------------------------------------------------------------
# projections
# ---------------------------------------------------------------------------
def dense_case(seed, M, K, N, dtype, pair=False, bias=False, residual=False):
    g = _gen(seed)
    c = dict(x=_randn(g, M, K, dtype=dtype), w=(_randn(g, N, K) / math.sqrt(K)).to(dtype),
             up=(_randn(g, N, K) / math.sqrt(K)).to(dtype) if pair else None,
             bias=_randn(g, N, dtype=dtype) if bias else None, residual=_randn(g, M, N, dtype=dtype) if residual else None,
             grad=_randn(g, M, N, dtype=dtype))
    return c


def check_dense(c, act, dev=_dev):
    r = dense_ref(c["x"], c["w"], c["up"], c["bias"], c["residual"], act, c["grad"])
    x, w, up, grad = (dev(c[k]) for k in ("x", "w", "up", "grad"))
    if up is not None:
        y, kept = hip_ops.gated_linear(x, w, up, act=act, keep=True)
        assert torch.equal(y, hip_ops.gated_linear(x, w, up, act=act))
        dx, dw, du = hip_ops.gated_linear_backward(grad, x, w, up, kept=kept, act=act)
        within(du, *r["du"], "du")
    else:
        b, res = dev(c["bias"]), dev(c["residual"])
        y, kept = hip_ops.fused_linear(x, w, b, act=act, residual=res, keep=True)
        assert torch.equal(y, hip_ops.fused_linear(x, w, b, act=act, residual=res))
        dx, dw, db = hip_ops.fused_linear_backward(grad, x, w, b, kept=kept, act=act)
        if b is not None:
            within(db, *r["db"], "db")
    within(y, *r["y"], "y")
    within(dx, *r["dx"], "dx")
    within(dw, *r["dw"], "dw")


SIZES = [(1, 8, 16), (1, 7, 5), (3, 33, 17), (16, 64, 48), (17, 100, 33), (32, 520, 24), (33, 8, 8), (40, 31, 70), (64, 96, 128),
         (130, 72, 136), (129, 257, 131), (300, 64, 256)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_gated(dtype, M, K, N):
    check_dense(dense_case(M + K + N, M, K, N, dtype, pair=True), "silu")


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(dtype, M, K, N):
    check_dense(dense_case(M * K + N, M, K, N, dtype, bias=True, residual=True), "gelu")


@pytest.mark.parametrize("act,bias,residual", [(None, False, False), (None, True, False), ("silu", False, True), ("gelu", True, False)])
@pytest.mark.parametrize("M,K,N", [(20, 40, 24), (70, 40, 26), (256, 512, 256)])
def test_linear_options(act, bias, residual, M, K, N):
    check_dense(dense_case(5, M, K, N, torch.bfloat16, bias=bias, residual=residual), act)


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("M,K,N", [(1024, 288, 4224), (3000, 160, 768)])
def test_large_tiles(pair, M, K, N):
    """Products that fill the card take the larger tiles."""
    with hip_ops.launch_log() as log:
        check_dense(dense_case(M, M, K, N, torch.bfloat16, pair=pair), "silu")
    assert any("product_kernel" in k for k in log.kernels)


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def check_logp(logits, targets, top, grad=None, grad_entropy=None, ignore=-100):
    r = logp_ref(logits, targets, top, ignore, grad, grad_entropy)
    x, t = _dev(logits), _dev(targets)
    logp, entropy, best, tokens, kept = hip_ops.token_log_probs(x, t, top=top, ignore_index=ignore, keep=True)
    finite = ~r["logp"][0].isinf()
    assert torch.equal(logp.cpu().isinf(), ~finite)
    within(logp.cpu()[finite], *(v[finite] for v in r["logp"]), "logp")
    within(entropy, *r["entropy"], "entropy")
    if top:
        assert torch.equal(tokens.cpu(), r["tokens"])
        fin = ~r["top"][0].isinf()
        assert torch.equal(best.cpu().isinf(), ~fin)
        within(best.cpu()[fin], *(v[fin] for v in r["top"]), "top")
    else:
        assert best is None and tokens is None
    if grad is not None or grad_entropy is not None:
        d = hip_ops.token_log_probs_backward(_dev(grad), _dev(grad_entropy), x, t, kept=kept, ignore_index=ignore)
        within(d, *r["dx"], "dx")


def logp_case(seed, rows, V, dtype, scale=2.5):
    g = _gen(seed)
    targets = torch.randint(0, V, (rows,), generator=g)
    targets[rows // 2::5] = -100
    return (scale * _randn(g, rows, V)).to(dtype), targets, _randn(g, rows), _randn(g, rows)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (2, 5, 5), (3, 63, 7), (1, 64, 64), (5, 1000, 20), (2, 8191, 1), (7, 8193, 64), (1, 50001, 20)])
def test_logp(dtype, rows, V, top):
    x, t, g, e = logp_case(rows + V, rows, V, dtype)
    check_logp(x, t, top, g, e)


@pytest.mark.parametrize("dtype", BOTH)
def test_logp_of_many_rows(dtype):
    x, t, g, e = logp_case(4, 1500, 700, dtype)
    check_logp(x, t, 0, g, None)
    check_logp(x, t, 3, None, e)


@pytest.mark.parametrize("offset", [0.0, 300.0, -300.0, 1e4, -1e4, 3e6, -3e6])
def test_logp_of_far_rows(offset):
    x, t, g, e = logp_case(11, 4, 3000, torch.float32)
    check_logp((x.double() + offset).float(), t, 10, g, e)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("low", [-math.inf, "lowest", -1e9])
def test_logp_of_masked_rows(dtype, low):
    x, t, g, e = logp_case(12, 6, 2100, dtype)
    low = torch.finfo(dtype).min if low == "lowest" else low
    x[:, 3::2] = low
    x[2, 1:] = low
    x[3, :2099] = low
    t = torch.where(t >= 0, (t // 2) * 2, t)
    t[2], t[3] = 0, 2099
    t[4] = 5  # a masked token: its log probability is -infinity, or very low
    if low != -math.inf:
        g[4] = 0.0
    check_logp(x, t, 12, g, e)
