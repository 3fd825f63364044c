// Attention prologue for packed sequences and a paged KV cache: per-head
// RMSNorm (optional), rotary embedding, and a scatter of k and v into the
// pages of each token's sequence. The packed, paged counterpart of
// rope_append.cuh.
#pragma once

#include "common.cuh"

namespace b2a {

struct RopeAppendPagedParams {
  const void* q;  // [N, Hq, D], strides qs (token, head); k, v [N, Hkv, D]
  const void* k;
  const void* v;
  long long qs[2], ks[2], vs[2];
  const void* cos;  // [max_pos, rope_dim] contiguous, fp32 or the source dtype
  const void* sin;
  int tab_fp32;
  int max_pos, rope_dim;
  const void* q_norm;  // optional [D] in the source dtype
  const void* k_norm;
  float norm_eps;
  __nv_bfloat16* q_out;  // [N, Hq, D] contiguous
  __nv_bfloat16* k_out;  // optional [N, Hkv, D] contiguous
  __nv_bfloat16* v_out;  // optional [N, Hkv, D] contiguous
  __nv_bfloat16* k_pages;  // [n_pages, Hkv, page, D], strides kps (page, head, slot)
  __nv_bfloat16* v_pages;
  long long kps[3], vps[3];
  const int* block_table;  // [B, table_width], row stride table_ld
  long long table_ld;
  int table_width, n_pages, page;
  const int* cu_seqlens;     // [B + 1]: sequence b owns tokens [cu[b], cu[b + 1])
  const int* start_pos_arr;  // optional [B]: position of each sequence's first token
  int start_pos;
  int* seqlens_out;  // optional [B]: start + number of tokens
  int B, Hq, Hkv;
  long long N;
  int src_bf16;
  int* err;
};

// Returns 0, -3 for an unsupported head_dim, another negative value on launch
// failure.
int launch_rope_append_paged(int D, const RopeAppendPagedParams& p, cudaStream_t st);

}  // namespace b2a
