"""Every row that a thread of the selective scan's chunk kernel reads lies inside its segment, and every unit of a chunk
is staged once: the kernel's own index arithmetic (``ssm_chunk.h``) built for the host and enumerated."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "tesm_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>

#include "ssm_chunk.h"

using namespace tesm;

static int errors = 0;

// An operand of U units per row over segments of every length up to three chunks and a bit.
template <int U>
static void operand(const char* name) {
  using CU = ChunkUnits<U>;
  long reads = 0, outside = 0, wrong = 0, missed = 0;
  for (int rows = 1; rows <= 3 * kQ + 5; ++rows)
    for (int row0 = 0; row0 < rows; row0 += kQ) {
      const bool whole = row0 + kQ <= rows;
      const int left = rows - row0, last = left - 1;
      int staged[kQ][U] = {};
      for (int tid = 0; tid < kChunkThreads; ++tid)
        for (int i = 0; i < CU::kEach; ++i) {
          const int r = CU::row(tid, i), from = chunk_source(whole, r, last);
          ++reads;
          outside += from < 0 || row0 + from >= rows;
          if (!CU::stages(tid)) continue;
          if (r < 0 || r >= kQ) {
            ++wrong;
            continue;
          }
          ++staged[r][tid % U];
          wrong += r < left && from != r;
        }
      for (int r = 0; r < kQ; ++r)
        for (int u = 0; u < U; ++u) missed += staged[r][u] != 1;
    }
  if (outside || wrong || missed) {
    printf("%s: %ld of %ld reads outside the segment, %ld rows wrong, %ld units not staged once\n", name, outside, reads, wrong, missed);
    ++errors;
  }
}

// Rows that a wave's lanes read one by one: the gate's (16 q + lane % 16).
static void gate() {
  for (int rows = 1; rows <= 3 * kQ + 5; ++rows)
    for (int row0 = 0; row0 < rows; row0 += kQ)
      for (int r = 0; r < kQ; ++r) {
        const int from = chunk_source(row0 + kQ <= rows, r, rows - 1 - row0);
        if (from < 0 || row0 + from >= rows || (row0 + r < rows && from != r)) {
          printf("gate: row %d of %d read for %d\n", row0 + from, rows, row0 + r);
          ++errors;
        }
      }
}

int main() {
  operand<16>("x, bfloat16");
  operand<32>("x, float32");
  operand<4>("B and C, bfloat16, 32 states");
  operand<8>("B and C, bfloat16, 64 states");
  operand<16>("B and C, bfloat16, 128 states");
  operand<32>("B and C, bfloat16, 256 states");
  operand<8>("B and C, float32, 32 states");
  operand<16>("B and C, float32, 64 states");
  operand<32>("B and C, float32, 128 states");
  operand<64>("B and C, float32, 256 states");
  gate();
  return errors != 0;
}
"""


def test_rows_read_lie_inside_the_segment(tmp_path):
    src = tmp_path / "rows.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "rows"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_the_kernel_forms_its_rows_that_way():
    """The loads of x, B, C and the gate go through one address, whose row is ``chunk_source``'s."""
    with open(os.path.join(CSRC, "ssm.hip")) as f:
        text = f.read()
    body = text[text.index("auto load_rows = "):text.index("auto load_chunk = ")]
    assert body.count("chunk_source(whole.value, r, last)") == 1
    assert body.count("load_rows(") == 4 and body.count("XU::row(tid, i)") == 1 and body.count("BU::row(tid, i)") == 2
    assert "load16(" in body and body.count("load16(") == 1 and body.count("load_unit<DT>(") == 1
