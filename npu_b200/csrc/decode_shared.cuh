// Single-token attention for sequences that share a prefix of their keys
// (decode_shared.cu): the prefix once for all sequences of a group, joined
// with each sequence's attention over its own keys (decode_paged.cu).
#pragma once

#include "decode_paged.cuh"

namespace b2a {

// Sequences of a group share their first `eff` keys: those of sequence `ref`.
// What the plan writes is read past L1 (load_group, load_seq): a CTA of the next
// kernel starts while the planning one runs, perhaps on its SM, whose L1 may
// hold lines from before the last writes.
//
// Four kernels in a row: the plan, the shared keys, the sequences' own keys and the
// join. The third starts beside the second and waits for it at its end only, so that
// the two run side by side (waiting at the start: 20 % more for the call, up to 49 %
// where it is short). What it reads, the plan and what the kernels before the plan
// wrote, is ordered by `ready`: the plan, which has waited for those kernels, releases
// kPlanReady there as its last act, the third kernel acquires it, and waits for the
// second as usual if it finds anything else. The join sets the word back.
struct alignas(16) SharedGroup {
  int eff, ref;      // eff: a multiple of the key block, 0 for nothing shared
  int first, count;  // its sequences
  int block0;        // number of its first row block
  int pad;
  long long unit0;   // number of its first unit of work
};

__device__ __forceinline__ SharedGroup load_group(const SharedGroup* p) {
  static_assert(sizeof(SharedGroup) == 32, "two 16-byte loads");
  int4 w[2] = {__ldcg(reinterpret_cast<const int4*>(p)), __ldcg(reinterpret_cast<const int4*>(p) + 1)};
  return *reinterpret_cast<const SharedGroup*>(w);
}

struct SharedPlanParams {
  const int* prefix_lens;  // [n_groups]
  const int* cu_groups;    // [n_groups + 1], or null: all sequences are one group
  int n_groups;
  const int* seqlens;  // [B]
  int B, Hkv, group;
  long long cap;       // keys a table can name
  int max_blocks;      // row blocks the workspace has room for
  long long least_saved;  // keys: sharing that saves reading fewer is not worth its launches
  SharedGroup* groups;  // [n_groups]
  SharedSeq* seqs;      // [B]
  long long* total;     // units of work
  uint32_t* ready;      // see above
  int* err;
};

struct DecodeSharedParams {
  const int* block_table;
  long long table_ld;
  int table_width, n_pages, page, box_rows;
  int n_groups, Hkv, group;
  float scale_log2;
  const SharedGroup* groups;
  const long long* total;
  // The partial of item x = row block * Hkv + KV head from CTA c is number
  // x + c: O [rows, D] before its division and (m, l) [rows, 2], in the
  // workspace; place[x]: the CTAs with the item's first and last key block.
  float* part_o;
  float* part_ml;
  int* place;
  int n_ctas;
  int* err;
};

// Sequences of a row block, and its rows (128 per tile, 128 / group sequences
// of `group` rows in each).
int decode_shared_block_seqs(int D, int group);
int decode_shared_block_rows(int D);
int decode_shared_max_ctas(int sms);

// tq: q as 3-D map (64 of D columns, head, sequence), box (64, group,
// 128 / group); tk / tv: the pools' 5-D maps with box (64, box_rows, 1, 1, 1).
// Returns 0, -3 for an unsupported head_dim, another negative value on launch
// failure.
int launch_decode_shared(int D, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                         const SharedPlanParams& plan, const DecodeSharedParams& p, cudaStream_t st);

}  // namespace b2a
