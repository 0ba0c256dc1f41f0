"""The state operators where their range ends: narrow states, far values, masks, memory on either side of the outputs.
Tolerances are those of the operators' own tests (``test_gpu_ssm``, ``test_gpu_beam``) unless a test derives another."""
import pytest
import torch

from hip_helpers import need_gpu
from test_gpu_ssm import _check_scan, _run_scan, _scan_case

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
