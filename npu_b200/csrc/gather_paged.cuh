// Reading a stretch of each sequence out of a paged cache as packed bf16 rows
// (gather_paged.cu).
#pragma once

#include "common.cuh"

namespace b2a {

struct GatherPagedParams {
  const void* k_pages;  // [n_pages, Hkv, page, D] bf16 (e4m3 with scales), strides kps (page, head, slot)
  const void* v_pages;
  long long kps[3], vps[3];
  const float* k_scales;  // both or neither: [n_pages, Hkv, page], strides kss (page, head)
  const float* v_scales;
  long long kss[2], vss[2];
  const int* block_table;  // [B, table_width], row stride table_ld
  long long table_ld;
  int table_width, n_pages, page;
  const int* cu_seqlens;     // [B + 1]: sequence b's rows of the outputs
  const int* start_pos_arr;  // optional [B]: position of the first of them
  int start_pos;
  __nv_bfloat16* k_out;  // [N, Hkv, D] contiguous
  __nv_bfloat16* v_out;
  int out_v8;  // both are 32-byte aligned
  int B, Hkv;
  long long N;
  int* err;
};

// Returns 0, -3 for an unsupported head_dim, another negative value on launch
// failure.
int launch_gather_paged(int D, const GatherPagedParams& p, cudaStream_t st);

}  // namespace b2a
