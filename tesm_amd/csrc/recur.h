// Gated linear recurrence of a recurrent layer: forward, backward, one token.
#pragma once

#include "tesm_hip_internal.h"

namespace tesm {

// Rows per tile, except for the forward pass's tallest ones: kept carries are one row of states per so many rows.  (32, with three workgroups per CU backward instead of two, cost a tile's
// fixed time twice as often: 4 x 2048 x 384 15.5 and 19.0 us instead of 11.2 and 15.1, 32768 x 8192 backward 1033 instead of 885.)
constexpr int kRecurRows = 64;

struct RecurArgs {
  int dt = 0;
  int64_t B = 0, L = 0, C = 0, S = 0;
  const void* value = nullptr;  // row r, channel c at value[r * ld_v + c]
  int64_t ld_v = 0;
  const void* write = nullptr;
  int64_t ld_w = 0;
  const void* decay = nullptr;
  int64_t ld_d = 0;
  const float* bias = nullptr;         // optional (C)
  const int32_t* seq_starts = nullptr;  // optional (S + 1)
  const float* h0 = nullptr;           // optional (S, C)
  int zero_rest = 0;                   // rows of no sequence: outputs set to zero instead of left
  void* h = nullptr;
  int64_t ld_h = 0;
  float* h_out = nullptr;    // (S, C)
  float* carries = nullptr;  // optional (recur_slots, C): the state in front of every kRecurRows rows of a sequence
};

struct RecurBwdArgs {
  RecurArgs in;              // h, h_out not used; carries those of the forward call
  const void* grad = nullptr;
  int64_t ld_g = 0;
  const float* grad_state = nullptr;  // optional (S, C)
  void* d_value = nullptr;
  int64_t ld_dv = 0;
  void* d_write = nullptr;
  int64_t ld_dw = 0;
  void* d_decay = nullptr;
  int64_t ld_dd = 0;
  float* d_bias = nullptr;  // optional (C)
  float* d_h0 = nullptr;    // optional (S, C)
};

struct RecurStepArgs {
  int dt = 0;
  int64_t B = 0, C = 0;
  const void* value = nullptr;
  int64_t ld_v = 0;
  const void* write = nullptr;
  int64_t ld_w = 0;
  const void* decay = nullptr;
  int64_t ld_d = 0;
  const float* bias = nullptr;
  float* state = nullptr;  // (B, C), updated in place
  void* h = nullptr;
  int64_t ld_h = 0;
};

int64_t recur_slots(const RecurArgs& a);  // rows of the kept carries, and places of tiles of kRecurRows rows (-1: bad sizes)
int64_t recur_ws_bytes(const RecurArgs& a);
int64_t recur_bwd_ws_bytes(const RecurArgs& a, bool bias);
int launch_gated_scan(const RecurArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);
int launch_gated_scan_bwd(const RecurBwdArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);
int launch_gated_scan_step(const RecurStepArgs& a, hipStream_t st);
// Status word of the recurrence's bounded waits on the current device (bit 0); synchronous.
int recur_status(unsigned* out, int clear);
// Poll limit of later launches (< 0: give up at once; a test of the failure report).
void recur_set_spin_limit(int limit);

}  // namespace tesm
