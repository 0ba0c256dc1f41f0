// Log probabilities of given tokens, entropies and best alternatives of rows of logits, and the gradient of the logits.
#pragma once

#include "tesm_hip_internal.h"

namespace tesm {

constexpr int64_t kLogpMaxTop = 64;

struct LogpArgs {
  int dt = 0;
  int64_t rows = 0, V = 0, top = 0;
  const void* logits = nullptr;  // (rows, ld)
  int64_t ld = 0;
  const int64_t* targets = nullptr;  // (rows)
  int64_t ignore = -100;
  float* logp = nullptr;      // (rows)
  float* entropy = nullptr;   // (rows)
  float* top_logp = nullptr;  // (rows, top)
  int64_t* top_tokens = nullptr;
  float* kept = nullptr;  // optional (rows, 4)
};

struct LogpBwdArgs {
  int dt = 0;
  int64_t rows = 0, V = 0;
  const void* logits = nullptr;
  int64_t ld = 0;
  const int64_t* targets = nullptr;
  int64_t ignore = -100;
  const float* kept = nullptr;       // (rows, 4)
  const float* grad_logp = nullptr;  // optional (rows)
  const float* grad_entropy = nullptr;  // optional (rows)
  void* grad_logits = nullptr;
  int64_t ld_g = 0;
};

int64_t logp_ws_bytes(const LogpArgs& a);
int launch_token_logp(const LogpArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);
int launch_token_logp_bwd(const LogpBwdArgs& a, hipStream_t st);
// Status word on the current device (bit 2: a target was neither a token nor the ignored value); synchronous.
int logp_status(unsigned* out, int clear);

}  // namespace tesm
