// Parameters and launcher of token sampling (sample.cu).
#pragma once

#include "common.cuh"

namespace b2a {

struct SampleParams {
  const void* logits;  // [R, V], row stride ld_logits, fp32 or bf16
  long long ld_logits;
  int logits_bf16;
  const float* noise;  // [R, V] of Exp(1), row stride ld_noise; may be null if no row draws (greedy)
  long long ld_noise;
  // Per-row settings [R] (device), or nullptr: the value for all rows.
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long* out;  // [R] token ids, -1 for a row without a usable logit
  int R, V;
  int cluster;  // CTAs per row (a power of two), set by launch_sample
  int slice;    // tokens per CTA, a multiple of 8
  int* err;
  long long wait_limit = kWaitLimitCycles;  // of every wait, in cycles
  int mute_pass;                            // launch_sample_mute only
};

// Returns 0 or a negative value on launch failure.
int launch_sample(SampleParams p, cudaStream_t st);

// For the failure path's test: fp32 logits, and the last CTA of each row's
// cluster stops sending its values at pass mute_pass.
int launch_sample_mute(SampleParams p, cudaStream_t st);

}  // namespace b2a
