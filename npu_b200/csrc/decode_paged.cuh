// Parameters and launcher of single-token attention over a paged KV cache
// (decode_paged.cu).
#pragma once

#include "common.cuh"

namespace b2a {

// What the plan of the shared form leaves when it is done (decode_shared.cuh).
constexpr uint32_t kPlanReady = 0x706c616eu;

// A sequence whose first `skip` keys (a multiple of 64) are attended together
// with others' (decode_shared.cu): where the partials of its query heads are.
struct alignas(16) SharedSeq {
  int skip;   // 0: none
  int block;  // row block
  int row;    // its first row there
  int pad;
};

__device__ __forceinline__ SharedSeq load_seq(const SharedSeq* p) {  // past L1, see decode_shared.cuh
  const int4 w = __ldcg(reinterpret_cast<const int4*>(p));
  return SharedSeq{w.x, w.y, w.z, w.w};
}

struct DecodePagedParams {
  const __nv_bfloat16* q;  // [B, Hq, D]
  long long q_sb, q_sh;
  const int* block_table;  // [B, table_width], row stride table_ld
  long long table_ld;
  int table_width, n_pages, page;
  const float* k_scales;  // both or neither: [n_pages, Hkv, page], strides kss (page, head); the pools are then e4m3
  const float* v_scales;
  long long kss[2], vss[2];
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
  // Shared form: with seqs, this call attends the keys from seqs[b].skip on, and
  // the joining kernel adds the partials of the shared ones, numbered and placed
  // alike (item block Hkv + g, rows of block_rows, CTAs up to shared_ctas).
  const SharedSeq* seqs;
  uint32_t* ready;
  const float* shared_o;
  const float* shared_ml;
  const int* shared_place;
  int block_rows, shared_ctas;
  int* err;
};

// CTAs an SM holds; NT: blocks of 8 query heads of a group. 8-bit keys at head
// dim 64 are bound by instructions and need few registers: a third CTA hides
// more of their latency.
constexpr int decode_paged_ctas_per_sm(int D, int NT, bool e4m3) {
  return D == 256 ? 1 : (D == 64 && NT == 1 && e4m3 ? 3 : 2);
}

// Whether a call runs the split form (partials and a joining kernel), the
// CTAs it may use for the current device, and its workspace.
bool decode_paged_splits(int table_width, int page);
int decode_paged_max_ctas(int D, int group, bool e4m3, int sms);
inline size_t decode_paged_parts(int B, int Hkv, int n_ctas) { return (size_t)B * Hkv + n_ctas; }

// tk / tv: 5-D maps (64 columns, slot in the page, D / 64, head, page) with
// box (64, box_rows, D / 64, 1, 1); of 8-bit pools 128 columns and D / 128 (head
// dim 64: 64 and 1). Returns 0 on success, -3 for an
// unsupported head_dim, another negative value on launch failure.
int launch_decode_paged(int D, const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p,
                        cudaStream_t st);

// For the tests (b2a_diag_paged_units); tile: 64 keys, or 128 (8-bit, without p.seqs).
int launch_decode_paged_units(const DecodePagedParams& p, int tile, const long long* units, int n, long long* out,
                              cudaStream_t st);

}  // namespace b2a
