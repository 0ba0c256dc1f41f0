"""Refusals of the state operators (short convolution, selective scan, beam selection, reordering) and their
descriptors' layout: host logic only."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from test_boundary_cpu import _c_struct_fields
from tesm_amd import TESMConfig, TESMLMHeadModel, _lib, hip_ops


def test_descriptor_layout_matches_header(tmp_path):
    with open(os.path.join(ROOT, "include", "tesm_hip.h")) as f:
        text = f.read()
    structs = {"tesm_hip_conv": _lib.Conv, "tesm_hip_ssm": _lib.Ssm, "tesm_hip_ssm_step": _lib.SsmStep,
               "tesm_hip_beam": _lib.Beam, "tesm_hip_rows": _lib.Rows}
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


def _conv_args(**kw):
    a = dict(x=torch.randn(2, 5, 6), weight=torch.randn(6, 4), bias=torch.randn(6), state=torch.randn(2, 3, 6))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err,msg", [
    (dict(x=torch.randn(5, 6)), ValueError, "must be"),
    (dict(weight=torch.randn(5, 4)), ValueError, "must be"),
    (dict(weight=torch.randn(6, 1)), ValueError, "taps"),
    (dict(weight=torch.randn(6, 9)), ValueError, "taps"),
    (dict(bias=torch.randn(5)), ValueError, "bias"),
    (dict(bias=torch.randn(6).bfloat16()), TypeError, "bias"),
    (dict(state=torch.randn(2, 4, 6)), ValueError, "state"),
    (dict(state=torch.randn(2, 3, 6).bfloat16()), TypeError, "state"),
    (dict(x=torch.randn(2, 5, 6).half()), TypeError, "float32 and bfloat16|expected"),
    (dict(seq_starts=torch.tensor([0, 5], dtype=torch.int32)), ValueError, "first dimension"),
    (dict(x=torch.randn(1, 5, 6), seq_starts=torch.tensor([0.0, 5.0]), state=None), ValueError, "seq_starts"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_conv_refusals(kw, err, msg):
    a = _conv_args(**kw)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.causal_conv(a.pop("x"), a.pop("weight"), a.pop("bias"), **a)


def test_operators_refuse_grad_mode():
    a = _conv_args(x=torch.randn(2, 5, 6, requires_grad=True))
    with pytest.raises(RuntimeError, match="forward-only"):
        hip_ops.causal_conv(a.pop("x"), a.pop("weight"), a.pop("bias"), **a)
    s = _scan_args(A=torch.randn(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="forward-only"):
        hip_ops.selective_scan(*s)
    with pytest.raises(RuntimeError, match="forward-only"):
        hip_ops.reorder_rows([torch.randn(4, 3, requires_grad=True)], torch.zeros(2, 2, dtype=torch.int64))


def _scan_args(**kw):
    a = dict(x=torch.randn(2, 5, 4, 8), dt=torch.randn(2, 5, 4), A=torch.randn(4), B=torch.randn(2, 5, 2, 16),
             C=torch.randn(2, 5, 2, 16))
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,opt,err,msg", [
    (dict(x=torch.randn(2, 5, 32)), {}, ValueError, "must be"),
    (dict(dt=torch.randn(2, 5, 3)), {}, ValueError, "must be"),
    (dict(C=torch.randn(2, 5, 2, 15)), {}, ValueError, "must be"),
    (dict(A=torch.randn(3)), {}, ValueError, "A must hold"),
    (dict(B=torch.randn(2, 5, 3, 16), C=torch.randn(2, 5, 3, 16)), {}, ValueError, "groups"),
    (dict(B=torch.randn(2, 5, 2, 257), C=torch.randn(2, 5, 2, 257)), {}, ValueError, "256"),
    (dict(dt=torch.randn(2, 5, 4).bfloat16()), {}, TypeError, "dt"),
    ({}, dict(z=torch.randn(2, 5, 4, 7)), ValueError, "must be"),
    ({}, dict(D=torch.randn(5)), ValueError, "D must hold"),
    ({}, dict(state=torch.randn(2, 4, 8, 15)), ValueError, "state"),
    ({}, dict(state=torch.randn(2, 4, 8, 16).bfloat16()), ValueError, "state"),
    ({}, dict(seq_starts=torch.tensor([0, 5], dtype=torch.int32)), ValueError, "first dimension"),
    ({}, {}, RuntimeError, "ROCm device"),
])
def test_scan_refusals(kw, opt, err, msg):
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.selective_scan(*_scan_args(**kw), **opt)


def _step_args(**kw):
    a = dict(row=torch.randn(2, 4 * 8 + 2 * 2 * 16), dt=torch.randn(2, 4), A=torch.randn(4), state=torch.randn(2, 4, 8, 16),
             conv_weight=torch.randn(96, 4), conv_bias=torch.randn(96), conv_state=torch.randn(2, 3, 96))
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,opt,err,msg", [
    (dict(row=torch.randn(2, 95)), {}, ValueError, "values"),
    (dict(row=torch.randn(3, 96)), {}, ValueError, "must be"),
    ({}, dict(n_groups=3), ValueError, "values"),
    (dict(state=torch.randn(2, 4, 16, 8).transpose(2, 3)), {}, ValueError, "contiguous"),
    (dict(state=torch.randn(2, 4, 8, 16).double()), {}, ValueError, "float32"),
    (dict(conv_weight=torch.randn(96, 9)), {}, ValueError, "conv_weight"),
    (dict(conv_weight=None), {}, ValueError, "need conv_weight"),
    (dict(conv_state=torch.randn(2, 2, 96)), {}, ValueError, "conv_state"),
    (dict(conv_state=None), {}, ValueError, "conv_state"),
    ({}, dict(z=torch.randn(2, 4, 9)), ValueError, "must be"),
    ({}, {}, RuntimeError, "ROCm device"),
])
def test_step_refusals(kw, opt, err, msg):
    opt = dict(dict(n_groups=2), **opt)
    with torch.no_grad(), pytest.raises(err, match=msg):
        hip_ops.selective_scan_step(*_step_args(**kw), **opt)


def test_step_refuses_its_own_conv_state_as_output():
    a = _step_args()
    with torch.no_grad(), pytest.raises(ValueError, match="another"):
        hip_ops.selective_scan_step(*a, n_groups=2, conv_state_out=a[-1])


@pytest.mark.parametrize("kw,err,msg", [
    (dict(logits=torch.randn(4, 9)), ValueError, "must be"),
    (dict(scores=torch.randn(2, 3)), ValueError, "must be"),
    (dict(scores=torch.randn(2, 4).double()), TypeError, "float32"),
    (dict(n=65), ValueError, "1 to 64"),
    (dict(n=0), ValueError, "1 to 64"),
    (dict(logits=torch.randn(2, 4, 1), n=5), ValueError, "K \\* V"),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError, "finished"),
    (dict(finished=torch.zeros(2, 4, dtype=torch.bool), pad_token=9), ValueError, "pad_token"),
    (dict(eos_token=9), ValueError, "eos_token"),
    (dict(), RuntimeError, "ROCm device"),
])
def test_beam_select_refusals(kw, err, msg):
    a = dict(logits=torch.randn(2, 4, 9), scores=torch.randn(2, 4))
    a.update(kw)
    with pytest.raises(err, match=msg):
        hip_ops.beam_select(**a)


def test_reorder_refusals():
    par = torch.zeros(2, 3, dtype=torch.int64)
    ok = torch.randn(6, 4)
    for tensors, parents, msg in (([ok], par.int(), "int64"), ([ok], par.view(-1), "int64"),
                                  ([torch.randn(5, 4)], par, "6 rows"), ([torch.tensor(1.0)], par, "6 rows"),
                                  ([torch.randn(4, 6).t()], par, "contiguous"),
                                  ([torch.randn(1, 4).expand(6, 4)], par, "overlap"), ([ok, ok], par, "twice"),
                                  ([ok], torch.zeros(1, 65, dtype=torch.int64), "64")):
        with pytest.raises(ValueError, match=msg):
            hip_ops.reorder_rows(tensors, parents)
    with pytest.raises(RuntimeError, match="ROCm device"):
        hip_ops.reorder_rows([ok], par)


def test_c_entries_refuse_bad_descriptors():
    """The C entries check sizes, pitches and workspaces before anything is queued (no device is needed)."""
    lib = _lib.load()
    err = lambda: lib.tesm_hip_last_error()
    for name in ("tesm_hip_causal_conv", "tesm_hip_selective_scan_step"):
        assert getattr(lib, name)(None, None) == 1 and b"null" in err()
    assert lib.tesm_hip_selective_scan(None, None, 0, None) == 1
    assert lib.tesm_hip_beam_select(None, None, 0, None) == 1
    c = _lib.Conv(B=2, L=3, C=4, W=9, S=2, ld_x=4, ld_y=4)
    assert lib.tesm_hip_causal_conv(ctypes.byref(c), None) == 3 and b"W" in err()
    c.W, c.S = 4, 3
    assert lib.tesm_hip_causal_conv(ctypes.byref(c), None) == 1 and b"S = B" in err()
    c.S, c.ld_x = 2, 3
    assert lib.tesm_hip_causal_conv(ctypes.byref(c), None) == 1 and b"ld_x" in err()
    s = _lib.Ssm(B=2, L=3, H=4, P=8, G=3, N=16, S=2)
    assert lib.tesm_hip_selective_scan(ctypes.byref(s), None, 0, None) == 1 and b"groups" in err()
    s.G, s.N = 2, 257
    assert lib.tesm_hip_selective_scan(ctypes.byref(s), None, 0, None) == 3 and b"256" in err()
    t = _lib.SsmStep(B=-1, H=4, P=8, G=2, N=16)
    assert lib.tesm_hip_selective_scan_step(ctypes.byref(t), None) == 1
    b = _lib.Beam(B=1, K=65, V=9, n=4, ld=9)
    assert lib.tesm_hip_beam_select(ctypes.byref(b), None, 0, None) == 3
    b.K, b.ld = 4, 8
    assert lib.tesm_hip_beam_select(ctypes.byref(b), None, 0, None) == 1 and b"ld" in err()
    b.V = b.ld = 1 << 30
    assert lib.tesm_hip_beam_select(ctypes.byref(b), None, 0, None) == 1 and b"sizes" in err()
    assert lib.tesm_hip_reorder_rows(None, 1, None, 2, 4, None) == 1
    assert lib.tesm_hip_reorder_rows(None, 0, None, 2, 65, None) == 3


def test_beam_search_refuses_what_does_not_fit():
    cfg = TESMConfig(d_model=32, n_layer=1, d_intermediate=64, vocab_size=20, max_seq_len=12, d_state=16, ent_rank=8,
                     entanglement_window=4)
    m = TESMLMHeadModel(cfg).eval()
    ids = torch.zeros(1, 5, dtype=torch.int64)
    for kw, msg in ((dict(num_beams=0, max_new_tokens=2), "beams"), (dict(num_beams=21, max_new_tokens=2), "beams"),
                    (dict(num_beams=2, max_new_tokens=0), "positive"), (dict(num_beams=2, max_new_tokens=9), "max_seq_len")):
        with pytest.raises(ValueError, match=msg):
            m.beam_search(ids, **kw)


def test_row_pitch():
    """Which layouts count as rows: column slices of wider rows do, transposed or overlapping ones do not."""
    wide = torch.zeros(3, 5, 40)
    assert hip_ops._row_pitch(wide, 2) == 40
    assert hip_ops._row_pitch(wide[..., 4:12], 2) == 40
    assert hip_ops._row_pitch(wide[..., 4:12].unflatten(-1, (2, 4)), 2) == 40
    assert hip_ops._row_pitch(wide[:, :4], 2) is None
    assert hip_ops._row_pitch(wide[:1, :4], 2) == 40
    assert hip_ops._row_pitch(wide[:, 1:2], 2) == 200
    assert hip_ops._row_pitch(wide.transpose(1, 2), 2) is None
    assert hip_ops._row_pitch(torch.zeros(1, 1, 8).expand(3, 5, 8), 2) is None
    assert hip_ops._row_pitch(torch.zeros(5, 8)[::2], 1) == 16
    assert hip_ops._row_pitch(wide[..., ::2], 2) is None
    assert hip_ops._row_pitch(torch.zeros(0, 5, 8), 2) == 8
