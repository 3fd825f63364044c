// Parameters and launcher of single-token attention over a paged KV cache
// (decode_paged.cu).
#pragma once

#include "common.cuh"

namespace b2a {

struct DecodePagedParams {
  const __nv_bfloat16* q;  // [B, Hq, D]
  long long q_sb, q_sh;
  const int* block_table;  // [B, table_width], row stride table_ld
  long long table_ld;
  int table_width, n_pages, page;
  int box_rows;            // keys per TMA box: 64, 32 or 16, divides page
  const int* seqlens;      // [B], device
  void* o;                 // [B, Hq, D]
  long long o_sb, o_sh;
  int out_fp32;
  const void* gate;        // optional [B, Hq, D]: o = attention * sigmoid(gate)
  long long g_sb, g_sh;
  int gate_bf16;
  int vec4;                // o and gate take accesses of four elements
  int B, Hq, Hkv, group;
  float scale_log2;
  // Split form: the partial of pair x = b Hkv + g from CTA c is number x + c
  // (each step along the stretches raises one of the two): O [group, D]
  // before its division, and (m, l) [group, 2].
  float* part_o;
  float* part_ml;
  int* place;        // [B Hkv, 2]: the CTAs with a pair's first and last tile
  int n_ctas;
  int* err;
};

// Whether a call runs the split form (partials and a joining kernel), the
// CTAs it may use for the current device, and its workspace.
bool decode_paged_splits(int table_width, int page);
int decode_paged_max_ctas(int D, int sms);
inline size_t decode_paged_parts(int B, int Hkv, int n_ctas) { return (size_t)B * Hkv + n_ctas; }

// tk / tv: 5-D maps (64 columns, slot in the page, D / 64, head, page) with
// box (64, box_rows, D / 64, 1, 1). Returns 0 on success, -3 for an
// unsupported head_dim, another negative value on launch failure.
int launch_decode_paged(int D, const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p,
                        cudaStream_t st);

}  // namespace b2a
