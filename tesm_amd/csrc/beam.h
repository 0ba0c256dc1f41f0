// Beam search: selection over beams and vocabulary, and the reordering of the states that follow the beams.
#pragma once

#include "tesm_hip_internal.h"

namespace tesm {

constexpr int64_t kBeamMaxN = 64;      // candidates chosen per request, and beams
constexpr int kReorderTensors = 96;    // tensors per launch (their table travels as a kernel argument)

struct BeamArgs {
  int dt = 0;
  int64_t B = 0, K = 0, V = 0, n = 0;
  const void* logits = nullptr;        // beam r = b * K + k at logits[r * ld]
  int64_t ld = 0;
  const float* scores = nullptr;       // (B, K)
  const uint8_t* finished = nullptr;   // optional (B, K)
  int64_t pad = 0, eos = -1;
  float* out_scores = nullptr;         // (B, n)
  int64_t* parents = nullptr;          // (B, n)
  int64_t* tokens = nullptr;           // (B, n)
  uint8_t* finished_out = nullptr;     // optional (B, n)
};
int64_t beam_select_ws_bytes(const BeamArgs& a);
int launch_beam_select(const BeamArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);

struct ReorderRows {
  void* p;
  int64_t pitch, bytes;  // row pitch and row size in bytes
};
int launch_reorder_rows(const ReorderRows* t, int64_t count, const int64_t* parents, int64_t B, int64_t K,
                        hipStream_t st);
// Status word of the reordering on the current device (bit 1: a parent outside [0, K)); synchronous.
int reorder_status(unsigned* out, int clear);

}  // namespace tesm
