"""Calls of the operators that learn which their documents allow: sizes, results changed in place, memory held."""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_bits import dense_bounds
from learn_refs import HALF, logp_ref, within
from tesm_amd import hip_ops
from test_gpu_learn import BOTH, _dev, logp_case, scan_case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


@pytest.mark.parametrize("dtype", BOTH)
def test_projections_of_more_than_four_million_rows(dtype):
    """The sums over rows take more than 65535 runs of 64.  Gradients are -1, 0 or 1 in few rows, so that their sums are exact."""
    M, K, N = 65535 * 64 + 330, 8, 8
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    w, b = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((N, K), (N,)))
    grad = torch.randint(-1, 2, (M, N), generator=g, device=DEV).to(dtype)
    dx, _, db = hip_ops.fused_linear_backward(grad, x, w, b, need_weight=False)
    want = grad.double().sum(0)
    within(db, want, HALF[dtype] * want.abs(), "db")
    _, kept = hip_ops.fused_linear(x, w, b, act="silu", keep=True)
    dx, _, _ = hip_ops.fused_linear_backward(grad, x, w, b, kept=kept, act="silu", need_weight=False)
    for some in (slice(0, 100), slice(65535 * 64 - 50, M)):
        c = dict(x=x[some].cpu(), w=w.cpu(), up=None, bias=b.cpu(), residual=None, grad=grad[some].cpu())
        within(dx[some], *dense_bounds(c, "silu")["dx"], "dx")


def test_grids_of_too_many_threads_are_refused():
    """A launch counts its threads in 32 bits."""
    n = 1 << 23
    v = torch.zeros(n, 1, 2, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="too many tiles"):
        hip_ops.gated_scan(v, v, v)
    h, _, kept = hip_ops.gated_scan(v[1:], v[1:], v[1:], keep=True)  # (one tile less)
    assert not h.any()
    with pytest.raises(RuntimeError, match="too many tiles"):
        hip_ops.gated_scan_backward(v, v, v, v, kept=torch.zeros(n, 2, device=DEV))
    x, t = torch.zeros(1 << 24, 2, dtype=BF, device=DEV), torch.zeros(1 << 24, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="too many rows"):
        hip_ops.token_log_probs(x, t)
    with pytest.raises(RuntimeError, match="too many rows"):
        hip_ops.token_log_probs_backward(None, None, x, t, kept=torch.zeros(1 << 24, 4, device=DEV))
    logp = hip_ops.token_log_probs(x[1:], t[1:])[0]
    assert bool((logp + 0.6931472 <= 2.0 ** -22).all()) and bool((logp + 0.6931472 >= -2.0 ** -22).all())


@pytest.mark.parametrize("dtype", BOTH)
def test_log_probs_may_be_changed_in_place(dtype):
    """A policy's loss: advantages times the log probabilities, in place."""
    x, t, g, e = logp_case(3, 8, 300, dtype)
    a = x.to(DEV).requires_grad_()
    with torch.enable_grad():
        logp, entropy, _, _ = hip_ops.token_log_probs(a, _dev(t))
        logp *= _dev(g)
        entropy.mul_(_dev(e))
        (logp.sum() + entropy.sum()).backward()
    within(a.grad, *logp_ref(x, t, 0, -100, g, e)["dx"], "dx")


@pytest.mark.parametrize("dtype", BOTH)
def test_gradients_of_the_recurrence_hold_their_own_memory(dtype):
    c = scan_case(4, 2, 90, 16, dtype)
    args = [_dev(c[k]) for k in ("value", "write", "decay", "bias")]
    h, last, kept = hip_ops.gated_scan(*args, state=_dev(c["state"]), keep=True)
    grads = hip_ops.gated_scan_backward(_dev(c["grad"]), *args, kept=kept, state=_dev(c["state"]))
    held = [t.untyped_storage() for t in (h, last, *grads)]
    assert len({s.data_ptr() for s in held}) == len(held)
    assert [s.nbytes() for s in held] == [t.numel() * t.element_size() for t in (h, last, *grads)]
