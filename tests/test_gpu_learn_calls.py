"""Calls of the operators that learn which their documents allow: sizes, results changed in place, memory held."""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_bits import dense_bounds
from learn_refs import HALF, within
from tesm_amd import hip_ops
from test_gpu_learn import BOTH

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
