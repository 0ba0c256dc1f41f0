"""Outputs of the state operators that share memory with an input or another output are refused, and column slices that
only interleave are not: the rows' arithmetic against every byte, then the C entries (no device is needed: addresses are
compared before memory is looked at)."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from tesm_amd import _lib, hip_ops

CSRC = os.path.join(ROOT, "tesm_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rows_overlap.h"

using namespace tesm;

static char memory[4096];

static bool every_byte(const RowSpan& a, const RowSpan& b) {
  static char mark[4096];
  memset(mark, 0, sizeof mark);
  for (int64_t i = 0; i < a.n; ++i) memset(mark + (static_cast<const char*>(a.p) - memory) + i * a.pitch, 1, a.width);
  for (int64_t i = 0; i < b.n; ++i)
    for (int64_t j = 0; j < b.width; ++j)
      if (mark[(static_cast<const char*>(b.p) - memory) + i * b.pitch + j]) return true;
  return false;
}

static long seen[2], wrong;
static void compare(const RowSpan& a, const RowSpan& b) {
  const bool want = every_byte(a, b);
  ++seen[want];
  if (rows_share(a, b) == want && rows_share(b, a) == want) return;
  if (wrong++ < 5)
    printf("%ld x %ld of %ld at %ld, %ld x %ld of %ld at %ld: %d\n", (long)a.n, (long)a.width, (long)a.pitch,
           (long)(static_cast<const char*>(a.p) - memory), (long)b.n, (long)b.width, (long)b.pitch,
           (long)(static_cast<const char*>(b.p) - memory), want);
}

int main() {
  srand(1);
  for (int step = 0; step < 400000; ++step) {
    RowSpan s[2];
    for (RowSpan& r : s) {
      r.n = rand() % 7;
      r.width = rand() % 9;
      r.pitch = r.width + rand() % 20;
      r.p = memory + 200 + rand() % 200;
    }
    if (step % 3 == 0) s[1].pitch = s[0].pitch > s[1].width ? s[0].pitch : (s[0].pitch = s[1].width);
    if (step % 7 == 0) s[0].n = 1, s[0].width = rand() % 60, s[0].pitch = s[0].width;
    compare(s[0], s[1]);
  }
  if (rows_share({nullptr, 3, 4, 4}, {memory, 3, 4, 4})) ++wrong;
  printf("%ld apart, %ld sharing, %ld wrong\n", seen[0], seen[1], wrong);
  // several at once: column slices of one pitch, and arrays of their own
  long many[2] = {0, 0};
  for (int step = 0; step < 200000; ++step) {
    std::vector<RowSpan> v(2 + rand() % 4);
    const int64_t n = 1 + rand() % 5, pitch = 12 + rand() % 20;
    for (RowSpan& r : v) {
      r.n = n;
      r.width = rand() % 7;
      r.pitch = rand() % 4 ? pitch : r.width + rand() % 20;
      r.p = memory + 200 + (rand() % 2 ? rand() % 30 : 200 * (rand() % 8) + rand() % 10);
    }
    bool want = false;
    for (size_t a = 0; a < v.size(); ++a)
      for (size_t b = a + 1; b < v.size(); ++b) want = want || every_byte(v[a], v[b]);
    ++many[want];
    if (any_rows_share(v) != want && wrong++ < 5) printf("several: %d\n", want);
  }
  printf("several: %ld apart, %ld sharing, %ld wrong\n", many[0], many[1], wrong);
  if (many[0] < 10000 || many[1] < 10000) return 2;
  return wrong || seen[0] < 10000 || seen[1] < 10000;
}
"""


def test_rows_against_every_byte(tmp_path):
    src = tmp_path / "rows.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "rows"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


AT = 1 << 40  # an address that nothing owns: whether ranges meet is all that is asked here


def _places(sizes):
    """One range behind the other, a page apart."""
    at, out = AT, {}
    for name, n in sizes.items():
        out[name] = at
        at += n + 4096
    return out


def _refused(entry, d, *more):
    rc = entry(ctypes.byref(d), *more)
    text = _lib.load().tesm_hip_last_error().decode()
    assert rc == 1
    return text


B, L, C, W = 2, 5, 64, 4
CONV = dict(x=B * L * C * 4, weight=C * W * 4, bias=C * 4, state=B * 3 * C * 4, y=B * L * C * 4, state_out=B * 3 * C * 4)


def _conv(**kw):
    d = _lib.Conv(dt=0, w_dt=0, B=B, L=L, C=C, W=W, S=B, silu=1, ld_x=C, ld_y=C, **_places(CONV))
    for k, v in kw.items():
        setattr(d, k, v)
    return _refused(_lib.load().tesm_hip_causal_conv, d, None)


def test_conv_refuses_overlaps():
    p = _places(CONV)
    assert "overlaps" not in _conv()
    for out in ("y", "state_out"):
        for name in CONV:
            if name != out:
                for at in (p[name], p[name] + CONV[name] - 4, p[name] - CONV[out] + 4):
                    assert "overlaps" in _conv(**{out: at}), (out, name, at)
    # x and y as halves of wider rows, apart and one column too near
    assert "overlaps" not in _conv(ld_x=2 * C, ld_y=2 * C, y=p["x"] + 4 * C, weight=AT << 1, bias=0, state=0, state_out=0)
    assert "y overlaps x" in _conv(ld_x=2 * C, ld_y=2 * C, y=p["x"] + 4 * C - 4, weight=AT << 1, bias=0, state=0, state_out=0)


H, P, G, N = 2, 8, 1, 16
SCAN = dict(x=B * L * H * P * 4, dts=B * L * H * 4, Bm=B * L * G * N * 4, Cm=B * L * G * N * 4, z=B * L * H * P * 4, h0=B * H * P * N * 4,
            A=H * 4, D=H * 4, dt_bias=H * 4, y=B * L * H * P * 4, h_out=B * H * P * N * 4)


def _scan(**kw):
    d = _lib.Ssm(dt=0, B=B, L=L, H=H, P=P, G=G, N=N, S=B, softplus=1, ld_x=H * P, ld_dt=H, ld_b=G * N, ld_c=G * N, ld_z=H * P,
                 ld_y=H * P, **_places(SCAN))
    for k, v in kw.items():
        setattr(d, k, v)
    return _refused(_lib.load().tesm_hip_selective_scan, d, None, 0, None)


@pytest.mark.parametrize("out", ["y", "h_out"])
def test_scan_refuses_overlaps(out):
    p = _places(SCAN)
    assert "overlaps" not in _scan()
    for name in SCAN:
        if name != out:
            for at in (p[name], p[name] + SCAN[name] - 4, p[name] - SCAN[out] + 4):
                assert "overlaps" in _scan(**{out: at}), (name, at)


WIDTH = H * P + 2 * G * N
STEP = dict(row=B * WIDTH * 4, conv_weight=WIDTH * W * 4, conv_bias=WIDTH * 4, conv_state=B * 3 * WIDTH * 4, dts=B * H * 4, A=H * 4,
            D=H * 4, z=B * H * P * 4, dt_bias=H * 4, conv_state_out=B * 3 * WIDTH * 4, state=B * H * P * N * 4, y=B * H * P * 4)


def _step(**kw):
    d = _lib.SsmStep(dt=0, w_dt=0, B=B, H=H, P=P, G=G, N=N, W=W, softplus=1, silu=1, ld_row=WIDTH, ld_dt=H, ld_z=H * P, ld_y=H * P,
                     **_places(STEP))
    for k, v in kw.items():
        setattr(d, k, v)
    return _refused(_lib.load().tesm_hip_selective_scan_step, d, None)


@pytest.mark.parametrize("out", ["y", "state", "conv_state_out"])
def test_step_refuses_overlaps(out):
    p = _places(STEP)
    assert "overlaps" not in _step()
    for name in STEP:
        if name != out:
            for at in (p[name], p[name] + STEP[name] - 4, p[name] - STEP[out] + 4):
                assert "overlaps" in _step(**{out: at}), (name, at)
    # the token's outputs in the columns beside its inputs
    wide = WIDTH + H * P
    assert "overlaps" not in _step(ld_row=wide, ld_y=wide, row=AT << 1, y=(AT << 1) + 4 * WIDTH)


def _reorder(rows, B=2, K=3):
    t = (_lib.Rows * len(rows))(*[_lib.Rows(p=AT + at, pitch=pitch, bytes=n) for at, pitch, n in rows])
    rc = _lib.load().tesm_hip_reorder_rows(ctypes.addressof(t), len(rows), AT << 1, B, K, None)
    assert rc == 1
    return _lib.load().tesm_hip_last_error().decode()


def test_reorder_refuses_overlaps():
    apart = [(0, 40, 40), (240, 64, 40), (280, 64, 24), (1000, 16, 16), (0, 8, 0)]
    assert "overlap" not in _reorder(apart) and "overlap" not in _reorder(apart[::-1])
    for more in ((0, 40, 40), (39, 8, 8), (276, 64, 8), (1090, 16, 16), (990, 4, 4)):
        assert "overlap" in _reorder(apart + [more]), more
        assert "overlap" in _reorder([more] + apart), more
    assert "overlap" in _reorder([(0, 16, 16), (0, 16, 16)]) and "overlap" in _reorder([(0, 16, 16), (8, 16, 16)], 1, 1)


def test_reorder_refuses_a_tensor_given_twice_beside_an_empty_one():
    ok, par = torch.randn(6, 4), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="twice"):
        hip_ops.reorder_rows([ok, torch.zeros(6, 0), ok], par)
    with pytest.raises(RuntimeError, match="ROCm device"):  # (two empty ones are none)
        hip_ops.reorder_rows([ok, torch.zeros(6, 0), torch.zeros(6, 0)], par)
