// Penalties for repeated tokens, biases and masks on logits (penalize.cu).
#pragma once

#include "common.cuh"

namespace b2a {

struct PenalizeParams {
  const void* logits;  // [R, V], row stride ld_logits
  long long ld_logits;
  int logits_bf16;
  void* out;  // [R, V] of the same type; may be the logits
  long long ld_out;
  const void* tokens;  // optional [R, L] int32 or int64, strides (row, token)
  long long tokens_row, tokens_step;
  int tokens_64, L;
  const int* lengths;         // optional [R]: tokens that a row has (else L)
  const int* prompt_lengths;  // optional [R]: the first of them count for `repetition` only (else none)
  const float* repetition;    // optional [R] each, else the value for all
  const float* frequency;
  const float* presence;
  float repetition_all, frequency_all, presence_all;
  const float* bias;  // optional [R, V], row stride ld_bias (0: one row for all)
  long long ld_bias;
  const unsigned* allowed;  // optional [R, ceil(V / 32)], row stride ld_allowed (0: one row for all)
  long long ld_allowed;
  int R, V;
  int* err;
};

// Returns 0, or a negative value on launch failure.
int launch_penalize(const PenalizeParams& p, cudaStream_t st);

}  // namespace b2a
