"""Outputs of the state operators that share memory with an input or another output are refused, and column slices that
only interleave are not: the rows' arithmetic against every byte, then the C entries (no device is needed: addresses are
compared before memory is looked at)."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT
from tesm_amd import _lib

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
