"""Gradients and results that lose no more bits than their type's own rounding takes (bounds: ``learn_bits``)."""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_bits import dense_bounds, f32_bound, off_in_norm
from learn_refs import act_ref, scan_ref, within
from tesm_amd import hip_ops
from test_gpu_learn import _dev, check_scan, dense_case, run_scan, scan_case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


def gradients(c, act):
    x, w, up, b, grad = (_dev(c[k]) for k in ("x", "w", "up", "bias", "grad"))
    if up is not None:
        _, kept = hip_ops.gated_linear(x, w, up, act=act, keep=True)
        return dict(zip(("dx", "dw", "du"), hip_ops.gated_linear_backward(grad, x, w, up, kept=kept, act=act)))
    _, kept = hip_ops.fused_linear(x, w, b, act=act, keep=True)
    got = dict(zip(("dx", "dw", "db"), hip_ops.fused_linear_backward(grad, x, w, b, kept=kept, act=act)))
    return got if b is not None else {k: got[k] for k in ("dx", "dw")}


SIZES = [(40, 31, 70), (70, 40, 26), (130, 72, 136), (300, 64, 256)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_gradients_of_a_pair(act, M, K, N):
    c = dense_case(M + N, M, K, N, BF, pair=True)
    r = dense_bounds(c, act)
    for name, got in gradients(c, act).items():
        within(got, *r[name], name)


@pytest.mark.parametrize("act", ["silu", "gelu", None])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_gradients_of_an_activation(act, M, K, N):
    c = dense_case(M * N, M, K, N, BF, bias=True)
    r = dense_bounds(c, act)
    for name, got in gradients(c, act).items():
        within(got, *r[name], name)


# ---------------------------------------------------------------------------
# float32 operands keep float32's precision
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("M,K,N", [(7, 100, 90), (40, 520, 72), (64, 1030, 300), (70, 104, 72), (200, 67, 130), (300, 500, 400), (999, 515, 1030),
                                   (2100, 1000, 600), (1000, 500, 2000)])
def test_float32_products(M, K, N):
    c = dense_case(M + K, M, K, N, torch.float32, pair=True)
    x, w, up, grad = (_dev(c[k]) for k in ("x", "w", "up", "grad"))
    xd, wd, ud, gd = (t.double() for t in (x, w, up, grad))
    assert off_in_norm(hip_ops.fused_linear(x, w), xd @ wd.t()) <= f32_bound(K)
    dx, dw, _ = hip_ops.fused_linear_backward(grad, x, w)
    assert off_in_norm(dx, gd @ wd) <= f32_bound(N)
    assert off_in_norm(dw, gd.t() @ xd) <= f32_bound(M)
    # a pair: both products, and 8 half steps for the activation (slope at most 1.1) and the product of the two
    val = act_ref(xd @ wd.t(), "silu")[0]
    assert off_in_norm(hip_ops.gated_linear(x, w, up), val * (xd @ ud.t())) <= 2.1 * f32_bound(K) + 8 * 2.0 ** -24


@pytest.mark.parametrize("scale", [2.0 ** -99, 2.0 ** 100])
@pytest.mark.parametrize("M,K,N", [(40, 104, 72), (200, 500, 130)])
def test_float32_products_of_far_scales(scale, M, K, N):
    """Parts of operands down to 2^-100 are numbers too (few of the random ones are below 2^-100 themselves, none of weight)."""
    c = dense_case(M, M, K, N, torch.float32)
    x, w = _dev(c["x"]) * scale, _dev(c["w"])
    assert off_in_norm(hip_ops.fused_linear(x, w) / scale, (x.double() / scale) @ w.double().t()) <= f32_bound(K)


# ---------------------------------------------------------------------------
# the recurrence's decays
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("far", [0.0, 40.0, 300.0, 5000.0])
def test_decays_near_zero_from_far_biases(dtype, far):
    """What counts is decay + bias, whose float32 sum is exact where they nearly cancel."""
    c = scan_case(7, 2, 150, 12, dtype)
    c["decay"] = ((c["decay"].float() - far).to(dtype))
    c["bias"] = far + c["bias"]
    check_scan(c, *run_scan(c))
    state = _dev(c["state"])
    r = scan_ref(c["value"][:, :1], c["write"][:, :1], c["decay"][:, :1], c["bias"], c["state"], None)
    hip_ops.gated_scan_step(*(_dev(c[k][:, 0]) for k in ("value", "write", "decay")), _dev(c["bias"]), state=state)
    within(state, *r["last"], "state")
