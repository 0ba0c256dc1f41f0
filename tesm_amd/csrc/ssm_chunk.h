// Which rows of a chunk the threads of the selective scan's kernel read and stage: plain arithmetic with no device code,
// so that a program on the host can go over every thread.
#pragma once

namespace tesm {

constexpr int kQ = 32;              // rows per chunk
constexpr int kChunkThreads = 256;  // threads per workgroup

// An operand whose rows are U units of 16 bytes: unit `tid % U` of row(tid, i), i < kEach.
template <int U>
struct ChunkUnits {
  static constexpr int kEach = kQ * U >= kChunkThreads ? kQ * U / kChunkThreads : 1;
  static constexpr int row(int tid, int i) { return tid / U + i * (kChunkThreads / U); }
  // (rows of 4 units are fewer units than threads: the threads behind them have no row of the chunk)
  static constexpr bool stages(int tid) { return kQ * U >= kChunkThreads || tid < kQ * U; }
};

// The row read in the place of row r, from the chunk's first: in a whole chunk one of its kQ, in a segment's last chunk
// none behind the segment's last row (`last`).  What takes another row's place is cleared or left out when staged.
constexpr int chunk_source(bool whole, int r, int last) {
  const int end = whole ? kQ - 1 : last;
  return r < end ? r : end;
}

}  // namespace tesm
