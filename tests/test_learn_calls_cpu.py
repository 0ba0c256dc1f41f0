"""Calls of the operators that learn which have to be refused before any kernel runs, or answered without one."""
import ctypes
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from tesm_amd import TESMLMHeadModel, _lib, hip_ops
from test_learn_ops_cpu import _refused


def _pair(act, z, z_up):
    return _lib.Dense(0, act, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, 1 << 22, 8, None, None, 0, None, 0, z, z_up)


@pytest.mark.parametrize("z,z_up", [(None, None), (1 << 23, 1 << 24)])
def test_a_pair_without_an_activation_has_no_backward_pass(z, z_up):
    """Its kernel reads what the forward call kept, which that refuses to make."""
    b = _lib.DenseGrad(_pair(0, z, z_up), 1 << 25, 16, 1 << 26, None, None, None)
    assert "activation" in _refused("tesm_hip_dense_backward", ctypes.byref(b), None, 0, None)


R = torch.randn


@pytest.mark.parametrize("call", [
    lambda: hip_ops.fused_linear_backward(R(3, 4), R(3, 8), R(4, 8), act="silu"),
    lambda: hip_ops.gated_linear_backward(R(3, 4), R(3, 8), R(4, 8), R(4, 8), kept=None),
    lambda: hip_ops.gated_linear_backward(R(3, 4), R(3, 8), R(4, 8), R(4, 8), kept=R(3, 4)),
    lambda: hip_ops.gated_linear_backward(R(3, 4), R(3, 8), R(4, 8), R(4, 8), kept=(R(3, 4),)),
    lambda: hip_ops.gated_linear_backward(R(3, 4), R(3, 8), R(4, 8), R(4, 8), kept=(R(3, 4), None)),
    lambda: hip_ops.gated_scan_backward(R(2, 5, 6), R(2, 5, 6), R(2, 5, 6), R(2, 5, 6), kept=None),
    lambda: hip_ops.token_log_probs_backward(R(3), None, R(3, 9), torch.zeros(3, dtype=torch.int64), kept=None),
])
def test_backward_passes_without_what_the_forward_pass_kept(call):
    with torch.no_grad(), pytest.raises(ValueError, match="needs kept"):
        call()


@pytest.mark.parametrize("call,name", [
    (lambda: hip_ops.fused_linear_backward(None, R(3, 8), R(4, 8)), "gradient"),
    (lambda: hip_ops.gated_scan_backward(None, R(2, 5, 6), R(2, 5, 6), R(2, 5, 6), kept=R(2, 6)), "gradient"),
    (lambda: hip_ops.gated_scan_step(R(2, 6), R(2, 6), R(2, 6), state=None), "state"),
])
def test_calls_without_what_they_need(call, name):
    with torch.no_grad(), pytest.raises(ValueError, match="needs the " + name):
        call()


def _calls_of(g, x, w, y):
    t = torch.zeros(3, dtype=torch.int64)
    return dict(
        gated_scan=lambda: hip_ops.gated_scan(R(2, 5, 6), R(2, 5, 6), g),
        gated_scan_backward=lambda: hip_ops.gated_scan_backward(g, R(2, 5, 6), R(2, 5, 6), R(2, 5, 6), kept=R(2, 6)),
        gated_scan_step=lambda: hip_ops.gated_scan_step(g[:, 0], R(2, 6), R(2, 6), state=R(2, 6)),
        gated_linear=lambda: hip_ops.gated_linear(R(3, 8), R(4, 8), w),
        gated_linear_backward=lambda: hip_ops.gated_linear_backward(y, R(3, 8), R(4, 8), R(4, 8), kept=(R(3, 4), R(3, 4))),
        fused_linear=lambda: hip_ops.fused_linear(x, R(4, 8)),
        fused_linear_backward=lambda: hip_ops.fused_linear_backward(R(3, 4), x, R(4, 8)),
        token_log_probs=lambda: hip_ops.token_log_probs(x, t),
        token_log_probs_backward=lambda: hip_ops.token_log_probs_backward(R(3), None, x, t, kept=R(3, 4)))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_refused(grad):
    """In a level of forward-mode derivatives operands without a tangent go on (here, to the refusal of host memory)."""
    leaves = [R(*s) for s in ((2, 5, 6), (3, 8), (4, 8), (3, 4))]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        duals = [forward_ad.make_dual(v, torch.ones_like(v)) for v in leaves]
        for name, call in _calls_of(*duals).items():
            with pytest.raises(RuntimeError, match=name + ": no forward-mode"):
                call()
        for call in _calls_of(*leaves).values():
            with pytest.raises(RuntimeError, match="ROCm device"):
                call()


def test_an_output_that_requires_a_gradient_is_refused():
    g = R(2, 5, 6)
    with pytest.raises(RuntimeError, match="under torch.no_grad"):
        hip_ops.gated_scan(g, g, g, out=R(2, 5, 6, requires_grad=True))


class _Model:
    """As much of a model as ``score`` sees: it keeps the ids that it is given."""

    def __init__(self, ignore):
        self.tesm_config = SimpleNamespace(label_ignore_index=ignore, vocab_size=11)

    def __call__(self, ids):
        self.ids = ids
        return SimpleNamespace(logits=torch.zeros(*ids.shape, 11)), None


@pytest.mark.parametrize("ignore", [-100, -1, 0, 10, 11, 1 << 40])
def test_scores_read_no_embedding_behind_the_vocabulary(ignore, monkeypatch):
    model, seen = _Model(ignore), {}

    def log_probs(logits, targets, *, top, ignore_index):
        seen.update(targets=targets, ignore=ignore_index)
        return torch.zeros(targets.shape), torch.zeros(targets.shape), None, None

    monkeypatch.setattr(hip_ops, "token_log_probs", log_probs)
    ids = torch.tensor([[3, ignore, 10, 0], [ignore, 1, 2, ignore]])
    TESMLMHeadModel.score(model, ids)
    assert int(model.ids.min()) >= 0 and int(model.ids.max()) < 11
    token = (ids >= 0) & (ids < 11)
    assert torch.equal(model.ids, torch.where(token, ids, 0))
    assert torch.equal(seen["targets"][:, :-1], ids[:, 1:]) and seen["ignore"] == ignore
