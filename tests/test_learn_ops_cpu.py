"""The operators that learn, as far as the host goes: their descriptors' layout, what they refuse, outputs that share memory; and the
gradients of the 64-bit forms that the GPU tests compare with, against differences."""
import ctypes
import os
import subprocess

import pytest
import torch

import learn_refs
from conftest import ROOT
from learn_refs import dense_ref, logp_ref, scan_ref
from test_boundary_cpu import _c_struct_fields
from tesm_amd import _lib, hip_ops


def test_descriptor_layout_matches_header(tmp_path):
    with open(os.path.join(ROOT, "include", "tesm_hip.h")) as f:
        text = f.read()
    structs = {"tesm_hip_gates": _lib.Gates, "tesm_hip_recurrence": _lib.Recurrence, "tesm_hip_recurrence_grad": _lib.RecurrenceGrad,
               "tesm_hip_recurrence_step": _lib.RecurrenceStep, "tesm_hip_dense": _lib.Dense, "tesm_hip_dense_grad": _lib.DenseGrad,
               "tesm_hip_logp": _lib.Logp, "tesm_hip_logp_grad": _lib.LogpGrad}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "tesm_hip.h"', "int main(void) {"]
    for cname, py in structs.items():
        fields = _c_struct_fields(text, cname)
        assert fields == [f[0] for f in py._fields_], cname
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {fld} %zu\\n", offsetof({cname}, {fld}));' for fld in fields]
    lines.append("return 0; }")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in out if l.strip()}
    for cname, py in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(py), cname
        for fld, _ in py._fields_:
            assert got[(cname, fld)] == getattr(py, fld).offset, (cname, fld)


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------
R = torch.randn
BF = torch.bfloat16


@pytest.mark.parametrize("kw,err,msg", [
    (dict(value=R(2, 5)), ValueError, "must all be"),
    (dict(write=R(2, 5, 7)), ValueError, "must all be"),
    (dict(decay=R(2, 4, 6)), ValueError, "must all be"),
    (dict(decay=R(2, 5, 6).to(BF)), TypeError, "decay"),
    (dict(value=R(2, 5, 6).half(), write=R(2, 5, 6).half(), decay=R(2, 5, 6).half()), TypeError, "float32"),
    (dict(decay_bias=R(5)), ValueError, "decay_bias"),
    (dict(state=R(3, 6)), ValueError, "state"),
    (dict(state=R(2, 6).to(BF)), ValueError, "state"),
    (dict(seq_starts=torch.tensor([0, 5])), ValueError, "first dimension"),
    (dict(seq_starts=torch.tensor([0.0, 5.0]), value=R(1, 5, 6), write=R(1, 5, 6), decay=R(1, 5, 6)), ValueError, "seq_starts"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_recurrence_refusals(kw, err, msg):
    a = dict(value=R(2, 5, 6), write=R(2, 5, 6), decay=R(2, 5, 6), decay_bias=R(6))
    a.update(kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.gated_scan(a.pop("value"), a.pop("write"), a.pop("decay"), a.pop("decay_bias"), **a)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(value=R(2, 5, 6)), ValueError, "must all be"),
    (dict(state=R(2, 7)), ValueError, "state"),
    (dict(state=R(6, 2).t()), ValueError, "contiguous"),
    (dict(state=R(2, 6).to(BF)), ValueError, "state"),
    (dict(write=R(2, 6).to(BF)), TypeError, "write"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_step_refusals(kw, err, msg):
    a = dict(value=R(2, 6), write=R(2, 6), decay=R(2, 6), state=R(2, 6))
    a.update(kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.gated_scan_step(a.pop("value"), a.pop("write"), a.pop("decay"), **a)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(x=R(3, 7)), ValueError, "must be"),
    (dict(weight=R(4, 5, 8)), ValueError, "must be"),
    (dict(x=R(3, 0), weight=R(4, 0)), ValueError, "without values"),
    (dict(weight=R(4, 8).to(BF)), TypeError, "weight"),
    (dict(x=R(3, 8).double(), weight=R(4, 8).double()), TypeError, "float32"),
    (dict(bias=R(5)), ValueError, "bias"),
    (dict(bias=R(4).to(BF)), TypeError, "bias"),
    (dict(residual=R(3, 5)), ValueError, "residual"),
    (dict(residual=R(4)), ValueError, "residual"),
    (dict(act="relu"), ValueError, "act must be"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_linear_refusals(kw, err, msg):
    a = dict(x=R(3, 8), weight=R(4, 8))
    a.update(kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.fused_linear(a.pop("x"), a.pop("weight"), **a)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(w_up=R(5, 8)), ValueError, "share a shape"),
    (dict(w_up=R(4, 8).to(BF)), TypeError, "up"),
    (dict(act=None), ValueError, "act must be"),
    (dict(act="tanh"), ValueError, "act must be"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_gated_refusals(kw, err, msg):
    a = dict(x=R(3, 8), w_gate=R(4, 8), w_up=R(4, 8))
    a.update(kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.gated_linear(a.pop("x"), a.pop("w_gate"), a.pop("w_up"), **a)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(targets=torch.zeros(4, dtype=torch.int64)), ValueError, "must be"),
    (dict(targets=torch.zeros(3, dtype=torch.int32)), TypeError, "int64"),
    (dict(logits=R(3, 0)), ValueError, "without logits"),
    (dict(logits=R(3, 9).half()), TypeError, "float32"),
    (dict(top=10), ValueError, "alternatives"),
    (dict(top=65, logits=R(3, 100)), ValueError, "alternatives"),
    (dict(top=-1), ValueError, "alternatives"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_log_probs_refusals(kw, err, msg):
    a = dict(logits=R(3, 9), targets=torch.zeros(3, dtype=torch.int64))
    a.update(kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.token_log_probs(a.pop("logits"), a.pop("targets"), **a)


def test_backward_refusals():
    g, x, w = R(2, 5, 6), R(3, 8), R(4, 8)
    t = torch.zeros(3, dtype=torch.int64)
    with torch.no_grad():
        with pytest.raises(ValueError, match="gradient"):
            hip_ops.token_log_probs_backward(R(4), None, R(3, 9), t, kept=R(3, 4))
        with pytest.raises(RuntimeError, match="ROCm device"):
            hip_ops.gated_scan_backward(g, g, g, g, kept=R(2, 6))
        with pytest.raises(RuntimeError, match="ROCm device"):
            hip_ops.fused_linear_backward(R(3, 4), x, w)
        with pytest.raises(RuntimeError, match="ROCm device"):
            hip_ops.gated_linear_backward(R(3, 4), x, w, w, kept=(R(3, 4), R(3, 4)))
    with pytest.raises(RuntimeError, match="forward-only"):
        hip_ops.fused_linear_backward(R(3, 4), x.requires_grad_(), w)


def test_keep_is_not_for_autograd():
    g, x, w = R(2, 5, 6, requires_grad=True), R(3, 8, requires_grad=True), R(4, 8)
    for call in (lambda: hip_ops.gated_scan(g, g, g, keep=True), lambda: hip_ops.fused_linear(x, w, keep=True),
                 lambda: hip_ops.gated_linear(x, w, w, keep=True),
                 lambda: hip_ops.token_log_probs(x, torch.zeros(3, dtype=torch.int64), keep=True)):
        with pytest.raises(RuntimeError, match="keep=True"):
            call()
    with pytest.raises(RuntimeError, match="out takes no gradients"):
        hip_ops.gated_scan(g, g, g, out=R(2, 5, 6))
    with pytest.raises(RuntimeError, match="forward-only"):
        hip_ops.gated_scan_step(g[:, 0], g[:, 0], g[:, 0], state=R(2, 6))


# ---------------------------------------------------------------------------
# the C entries (addresses are compared, and sizes looked at, before memory is)
# ---------------------------------------------------------------------------
def _refused(fn, *args):
    lib = _lib.load()
    assert getattr(lib, fn)(*args) != 0
    return lib.tesm_hip_last_error().decode()


def _gates(base=1 << 20, dt=0, B=1, L=8, C=16, S=1, ld=16, starts=None):
    return _lib.Gates(dt, B, L, C, S, base, ld, base + 4096, ld, base + 8192, ld, None, starts, None, 0)


@pytest.mark.parametrize("make,msg", [
    (lambda: _lib.Recurrence(_gates(), (1 << 20) + 64, 16, 1 << 22, None), "h overlaps value"),
    (lambda: _lib.Recurrence(_gates(), 1 << 22, 16, (1 << 22) + 256, None), "h overlaps h_out"),
    (lambda: _lib.Recurrence(_gates(), 1 << 22, 16, 1 << 23, (1 << 20) + 8192), "carries overlaps decay"),
    (lambda: _lib.Recurrence(_gates(), 1 << 22, 16, 1 << 23, (1 << 24) - 4), "carries overlaps workspace"),
])
def test_recurrence_overlaps(make, msg):
    d = make()
    assert msg in _refused("tesm_hip_gated_scan", ctypes.byref(d), 1 << 24, 1 << 16, None)


def test_recurrence_in_columns_does_not_overlap():
    """Three operands and the result in one buffer of 64 columns: passes the check, and is refused for being no device memory."""
    p = 1 << 20
    g = _lib.Gates(0, 1, 8, 16, 1, p, 64, p + 64, 64, p + 128, 64, None, None, None, 0)
    d = _lib.Recurrence(g, p + 192, 64, 1 << 22, None)
    assert "overlaps" not in _refused("tesm_hip_gated_scan", ctypes.byref(d), None, 0, None)


def test_backward_overlaps():
    d = _lib.RecurrenceGrad(_gates(), 1 << 22, 1 << 23, 16, None, 1 << 24, 16, (1 << 24) + 64, 16, 1 << 25, 16, None, None)
    assert "d_value overlaps d_write" in _refused("tesm_hip_gated_scan_backward", ctypes.byref(d), None, 0, None)
    s = _lib.RecurrenceStep(0, 2, 16, 1 << 20, 16, 1 << 21, 16, 1 << 22, 16, None, 1 << 23, (1 << 23) + 4, 16)
    assert "h overlaps state" in _refused("tesm_hip_gated_scan_step", ctypes.byref(s), None)
    m = _lib.Dense(0, 0, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, None, 0, None, None, 0, (1 << 20) + 32, 16, None, None)
    assert "y overlaps x" in _refused("tesm_hip_dense_forward", ctypes.byref(m), None, 0, None)
    m = _lib.Dense(0, 0, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, None, 0, None, None, 0, None, 0, None, None)
    b = _lib.DenseGrad(m, 1 << 22, 16, 1 << 23, (1 << 23) + 64, None, None)
    assert "d_x overlaps d_weight" in _refused("tesm_hip_dense_backward", ctypes.byref(b), None, 0, None)
    t = _lib.Logp(0, 3, 9, 0, 1 << 20, 9, 1 << 21, -100, 1 << 22, (1 << 22) + 8, None, None, None)
    assert "log_probs overlaps entropy" in _refused("tesm_hip_token_log_probs", ctypes.byref(t), None, 0, None)
    t = _lib.LogpGrad(0, 3, 9, 1 << 20, 9, 1 << 21, -100, 1 << 22, None, None, 1 << 20, 9)
    assert "d_logits overlaps logits" in _refused("tesm_hip_token_log_probs_backward", ctypes.byref(t), None)


@pytest.mark.parametrize("kw", [dict(dt=3), dict(L=1 << 31), dict(C=1 << 24, ld=1 << 24), dict(S=2), dict(ld=15), dict(L=-1),
                                dict(B=1 << 40, L=1 << 40, S=1 << 40)])
def test_recurrence_sizes(kw):
    d = _lib.Recurrence(_gates(**kw), 1 << 40, kw.get("ld", 16), 1 << 50, None)
    _refused("tesm_hip_gated_scan", ctypes.byref(d), None, 0, None)


@pytest.mark.parametrize("at,kw", [("dt", 2), ("act", 3), ("M", 1 << 31), ("K", 0), ("K", 1 << 24), ("N", 1 << 24), ("ld_x", 7), ("M", -1)])
def test_product_sizes(at, kw):
    m = _lib.Dense(0, 0, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, None, 0, None, None, 0, 1 << 23, 16, None, None)
    setattr(m, at, kw)
    _refused("tesm_hip_dense_forward", ctypes.byref(m), None, 0, None)


def test_pair_takes_no_bias():
    m = _lib.Dense(0, 1, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, 1 << 22, 8, 1 << 23, None, 0, 1 << 24, 16, None, None)
    assert "no bias" in _refused("tesm_hip_dense_forward", ctypes.byref(m), None, 0, None)


@pytest.mark.parametrize("at,v", [("dt", 2), ("V", 0), ("V", 1 << 30), ("top", 65), ("top", 10), ("rows", -1), ("ld", 8)])
def test_log_probs_sizes(at, v):
    t = _lib.Logp(0, 3, 9, 0, 1 << 20, 9, 1 << 21, -100, 1 << 22, 1 << 23, 1 << 24, 1 << 25, None)
    setattr(t, at, v)
    _refused("tesm_hip_token_log_probs", ctypes.byref(t), None, 0, None)


# ---------------------------------------------------------------------------
# the 64-bit gradients, against central differences of the 64-bit values (step 1e-5: off by 1e-10 of the third derivative, and by the
# values' last bits over the step, 1e-11)
# ---------------------------------------------------------------------------
def _along(values, at, grads, seed):
    """Each input in turn, along a direction: differences of ``values()`` against its gradient."""
    g = torch.Generator().manual_seed(seed)
    for name, t in at.items():
        d = R(t.shape, generator=g, dtype=torch.float64)
        t0, step = t.clone(), 1e-5
        t.copy_(t0 + step * d)
        up = values()
        t.copy_(t0 - step * d)
        down = values()
        t.copy_(t0)
        want = (grads[name][0] * d).sum().item()
        assert abs((up - down) / (2 * step) - want) < 1e-7 * (1 + abs(want)), name


@pytest.mark.parametrize("starts", [None, [0, 3, 3, 9], [1, 8]])
def test_recurrence_gradients(starts, monkeypatch):
    monkeypatch.setitem(learn_refs.HALF, torch.float64, 0.0)
    g = torch.Generator().manual_seed(1)
    B, L, C = (2, 5, 3) if starts is None else (1, 10, 3)
    S = B if starts is None else len(starts) - 1
    v, w, f, dh = (R(B, L, C, generator=g, dtype=torch.float64) for _ in range(4))
    b, st, dl = (R(*s, generator=g, dtype=torch.float64) for s in ((C,), (S, C), (S, C)))
    grads = scan_ref(v, w, f, b, st, starts, dh, dl)

    def values():
        r = scan_ref(v, w, f, b, st, starts)
        return ((r["h"][0] * dh).sum() + (r["last"][0] * dl).sum()).item()
    _along(values, dict(dv=v, dw=w, dd=f, db=b, ds=st), grads, 2)


@pytest.mark.parametrize("act,pair", [("silu", False), ("gelu", False), (None, False), ("silu", True), ("gelu", True)])
def test_product_gradients(act, pair, monkeypatch):
    monkeypatch.setitem(learn_refs.HALF, torch.float64, 0.0)
    g = torch.Generator().manual_seed(3)
    x, w, u, b, r, dy = (R(*s, generator=g, dtype=torch.float64) for s in ((4, 5), (6, 5), (6, 5), (6,), (4, 6), (4, 6)))
    up, bias, res = (u, None, None) if pair else (None, b, r)
    grads = dense_ref(x, w, up, bias, res, act, dy)
    at = dict(dx=x, dw=w, du=u) if pair else dict(dx=x, dw=w, db=b)
    _along(lambda: (dense_ref(x, w, up, bias, res, act)["y"][0] * dy).sum().item(), at, grads, 4)


def test_log_probs_gradients(monkeypatch):
    monkeypatch.setitem(learn_refs.HALF, torch.float64, 0.0)
    g = torch.Generator().manual_seed(5)
    x, a, e = (R(*s, generator=g, dtype=torch.float64) for s in ((4, 9), (4,), (4,)))
    x[1, 3] = -float("inf")
    t = torch.tensor([0, 8, -100, 4])
    grads = logp_ref(x, t, 0, -100, a, e)

    def values():
        r = logp_ref(x, t, 0)
        return ((r["logp"][0] * a).sum() + (r["entropy"][0] * e).sum()).item()
    _along(values, dict(dx=x), grads, 6)
