// extern "C" boundary of the serving operators (include/b2attn.h): attention
// over packed sequences, the paged KV cache and sampling. Argument checks,
// tensor maps and launches; stateless like capi.cu.
#include <algorithm>
#include <cmath>
#include <climits>

#include "b2attn.h"
#include "capi_internal.cuh"
#include "decode_paged.cuh"
#include "decode_shared.cuh"
#include "gather_paged.cuh"
#include "penalize.cuh"
#include "prefill.cuh"
#include "rope_append_paged.cuh"
#include "sample.cuh"

using b2a::api_aligned;
using b2a::api_strides_ok;

namespace {

bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

// One packed tensor [rows, heads, D] (strides {row, head}) as the prefill
// kernels' 4-D map with a batch of one.
int packed_map(CUtensorMap* m, const void* base, int D, int rows, int heads, const long long* s, int box_rows) {
  const unsigned long long dims[4] = {(unsigned long long)D, (unsigned long long)rows, (unsigned long long)heads, 1};
  const unsigned long long strides[3] = {(unsigned long long)s[0] * 2, (unsigned long long)s[1] * 2,
                                         (unsigned long long)s[0] * 2};
  const unsigned box[4] = {64u, (unsigned)box_rows, 1u, 1u};
  return b2a::api_tensor_map(m, base, 4, dims, strides, box);
}

// A page pool [n_pages, heads, page, D] (strides {page, head, slot}): 64
// columns, slot, D / 64 column chunks, head, page.
int pool_map(CUtensorMap* m, const void* base, int D, int n_pages, int heads, int page, const long long* s,
             int box_rows, int box_chunks) {
  const unsigned long long dims[5] = {64, (unsigned long long)page, (unsigned long long)(D / 64),
                                      (unsigned long long)heads, (unsigned long long)n_pages};
  const unsigned long long strides[4] = {(unsigned long long)s[2] * 2, 128, (unsigned long long)s[1] * 2,
                                         (unsigned long long)s[0] * 2};
  const unsigned box[5] = {64u, (unsigned)box_rows, (unsigned)box_chunks, 1u, 1u};
  return b2a::api_tensor_map(m, base, 5, dims, strides, box);
}

// The same of an 8-bit pool: 128 columns (head dim 64: 64), slot, column chunks, head, page.
int pool_map_e4m3(CUtensorMap* m, const void* base, int D, int n_pages, int heads, int page, const long long* s,
                  int box_rows) {
  const unsigned columns = D < 128 ? D : 128;
  const unsigned long long dims[5] = {columns, (unsigned long long)page, (unsigned long long)D / columns,
                                      (unsigned long long)heads, (unsigned long long)n_pages};
  const unsigned long long strides[4] = {(unsigned long long)s[2], 128, (unsigned long long)s[1],
                                         (unsigned long long)s[0]};
  const unsigned box[5] = {columns, (unsigned)box_rows, (unsigned)D / columns, 1u, 1u};
  return b2a::api_tensor_map_bytes(m, base, 5, dims, strides, box);
}

// The scales of 8-bit pools (strides {page, head}): both there, and each page's 16-byte aligned for the copies of 16
// or more slots that paged decode makes.
int scales_ok(const void* k_scales, const void* v_scales, const long long* kss, const long long* vss) {
  if (!k_scales || !v_scales || !kss || !vss) return B2A_ERR_INVALID_ARG;
  if (!api_aligned(k_scales, 16) || !api_aligned(v_scales, 16) || !api_strides_ok(kss, 2, 4) ||
      !api_strides_ok(vss, 2, 4))
    return B2A_ERR_ALIGNMENT;
  return B2A_OK;
}

int status_of(int rc) { return rc == -3 ? B2A_ERR_HEAD_DIM : (rc ? B2A_ERR_LAUNCH : B2A_OK); }

struct SharedPrefix {
  const int* prefix_lens;
  const int* cu_groups;
  int n_groups;
  long long least_saved;  // bytes, below 0: kLeastSaved
};

// When a call shares by the default rule, in bytes of keys and values. The device knows what sharing would save to
// read and weighs it against not sharing with the same launches: kLeastSaved. The host knows only the sizes: the
// call is b2a_decode_paged's, with fewer launches, below kLeastPossible for all sequences but one of each group sharing
// all that their tables can name. Both from 168 shapes (4 to 128 sequences, 1, 3 or 8 groups behind 512 to 32000 keys,
// 32 / 4 and 32 / 8 heads of 128, 9 / 3 of 64, 16 / 2 of 256):
// - tables as long as their sequences: with 160 MB a call takes 1.4 % longer on average than by the better way, at worst
//   85.8 us for 65.9 (two sequences in each of 8 groups behind 32000 keys), with 134 MB 2.3 %, with 200 MB 1.8 % (worst
//   31.5 for 17.1), never sharing 7 %, always 15 %;
// - tables of 32768 keys, so that the device decides: 36 MB is within 1.5 % of the better of its two ways on average, 20
//   to 45 MB are alike, 100 MB loses 6 %. Against b2a_decode_paged such a call takes 6 us more where nothing is shared
//   (up to 13, or 1.6 times), and up to 1.75 times where the device shares to little use (8 groups of two).
constexpr long long kLeastSaved = 36LL << 20, kLeastPossible = 160'000'000LL;

// Where the shared form's scratch is, behind that of the sequences' own keys.
struct SharedLayout {
  int max_blocks, n_ctas;
  size_t groups, seqs, place, part_ml, part_o, bytes;
};
SharedLayout shared_layout(int B, int Hq, int Hkv, int D, int n_groups) {
  SharedLayout at;
  const int group = Hq / Hkv;
  // Row blocks: every group of two or more sequences may leave one unfilled.
  at.max_blocks = B / b2a::decode_shared_block_seqs(D, group) + std::min(n_groups, B / 2);
  at.n_ctas = b2a::decode_shared_max_ctas(b2a::api_sm_count());
  const size_t items = (size_t)at.max_blocks * Hkv, rows = (items + at.n_ctas) * b2a::decode_shared_block_rows(D);
  at.groups = 256;
  at.seqs = at.groups + b2a::api_align256((size_t)n_groups * sizeof(b2a::SharedGroup));
  at.place = at.seqs + b2a::api_align256((size_t)B * sizeof(b2a::SharedSeq));
  at.part_ml = at.place + b2a::api_align256(items * 2 * sizeof(int));
  at.part_o = at.part_ml + b2a::api_align256(rows * 2 * sizeof(float));
  at.bytes = at.part_o + rows * D * sizeof(float) + 256;  // and to its own 256-byte boundary
  return at;
}

int paged_attention(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                    const float* k_scales, const float* v_scales, const long long* kss, const long long* vss,
                    const SharedPrefix* shared, long long table_ld, int table_width, const int* seqlens,
                    const void* gate, void* o, int B, int Hq, int Hkv, int n_pages, int page, int D,
                    const long long* qs, const long long* ks, const long long* vs, const long long* gs,
                    const long long* os, int gate_bf16, float scale, int out_fp32, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (!q || !k_pages || !v_pages || !block_table || !seqlens || !o || !qs || !ks || !vs || !os || (gate && !gs))
    return B2A_ERR_INVALID_ARG;
  const int tile = k_scales ? 128 : 64;  // keys; lengths are rounded up to whole ones
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || n_pages <= 0 || page <= 0 || page % 16 || table_width <= 0 ||
      table_ld < table_width || (long long)table_width * page > INT_MAX - tile)
    return B2A_ERR_INVALID_ARG;
  if (!(scale > 0.f) || !std::isfinite(scale)) return B2A_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return B2A_ERR_HEAD_DIM;
  if (Hq % Hkv || Hq / Hkv > 16) return B2A_ERR_GQA;
  if (!api_aligned(q, 16) || !api_aligned(k_pages, 16) || !api_aligned(v_pages, 16) ||
      !api_aligned(o, out_fp32 ? 4 : 2) || !api_aligned(block_table, 4) || !api_aligned(seqlens, 4) ||
      !api_aligned(gate, gate_bf16 ? 2 : 4))
    return B2A_ERR_ALIGNMENT;
  const long long pool_mult = k_scales ? 16 : 8;
  if (!api_strides_ok(qs, 2, 8) || !api_strides_ok(ks, 3, pool_mult) || !api_strides_ok(vs, 3, pool_mult))
    return B2A_ERR_ALIGNMENT;
  const size_t own = b2a_decode_paged_workspace_bytes(B, Hq, Hkv, D);
  const size_t need = own + (shared ? shared_layout(B, Hq, Hkv, D, shared->n_groups).bytes : 0);
  if (!workspace || workspace_bytes < need || !api_aligned(workspace, 16)) return B2A_ERR_WORKSPACE;

  int* err = nullptr;
  int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::DecodePagedParams p{};
  // Keys per TMA box: a box never crosses a page, a warp's 16 keys never a box.
  p.box_rows = page % 64 == 0 ? 64 : (page % 32 == 0 ? 32 : 16);
  CUtensorMap tk, tv;
  auto map = [&](CUtensorMap* m, const void* pool, const long long* strides, int box_chunks) {
    return k_scales ? pool_map_e4m3(m, pool, D, n_pages, Hkv, page, strides, p.box_rows)
                    : pool_map(m, pool, D, n_pages, Hkv, page, strides, p.box_rows, box_chunks);
  };
  if ((rc = map(&tk, k_pages, ks, D / 64)) || (rc = map(&tv, v_pages, vs, D / 64))) return rc;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  if (k_scales) {
    std::copy_n(kss, 2, p.kss);
    std::copy_n(vss, 2, p.vss);
  }
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = qs[0];
  p.q_sh = qs[1];
  p.block_table = block_table;
  p.table_ld = table_ld;
  p.table_width = table_width;
  p.n_pages = n_pages;
  p.page = page;
  p.seqlens = seqlens;
  p.o = o;
  p.o_sb = os[0];
  p.o_sh = os[1];
  p.out_fp32 = out_fp32 ? 1 : 0;
  p.gate = gate;
  if (gate) {
    p.g_sb = gs[0];
    p.g_sh = gs[1];
    p.gate_bf16 = gate_bf16 ? 1 : 0;
  }
  auto by4 = [](const void* ptr, const long long* st, unsigned size) {
    return api_aligned(ptr, 4 * size) && st[0] % 4 == 0 && st[1] % 4 == 0;
  };
  p.vec4 = by4(o, os, out_fp32 ? 4 : 2) && (!gate || by4(gate, gs, gate_bf16 ? 2 : 4));
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.scale_log2 = scale * b2a::kApiLog2e;
  p.err = err;
  p.n_ctas = b2a::decode_paged_max_ctas(D, p.group, k_scales != nullptr, b2a::api_sm_count());
  const size_t rows = b2a::decode_paged_parts(B, Hkv, p.n_ctas) * p.group;
  char* scratch = static_cast<char*>(workspace);
  p.part_o = reinterpret_cast<float*>(scratch);
  scratch += b2a::api_align256(rows * D * sizeof(float));
  p.part_ml = reinterpret_cast<float*>(scratch);
  p.place = reinterpret_cast<int*>(scratch + b2a::api_align256(rows * 2 * sizeof(float)));
  // Few keys, or one sequence: every sequence reads its own (one launch). So too where sharing could not save enough;
  // how much it does save is known on the device, where the plan looks again.
  const long long bytes_a_key = 4LL * Hkv * D;
  const bool by_rule = shared && shared->least_saved < 0;
  const long long least = by_rule ? kLeastSaved : (shared ? shared->least_saved : 0);
  const long long possible = (long long)(B - (by_rule ? shared->n_groups : 1)) * table_width * page;  // keys
  if (shared && B > 1 && b2a::decode_paged_splits(table_width, page) &&
      possible >= (by_rule ? kLeastPossible : least) / bytes_a_key) {
    const SharedLayout at = shared_layout(B, Hq, Hkv, D, shared->n_groups);
    char* base = reinterpret_cast<char*>(b2a::api_align256(reinterpret_cast<uintptr_t>(workspace) + own));
    b2a::SharedPlanParams plan{};
    plan.prefix_lens = shared->prefix_lens;
    plan.cu_groups = shared->cu_groups;
    plan.n_groups = shared->n_groups;
    plan.seqlens = seqlens;
    plan.B = B;
    plan.Hkv = Hkv;
    plan.group = p.group;
    plan.cap = (long long)table_width * page;
    plan.max_blocks = at.max_blocks;
    plan.least_saved = std::max(1LL, least / bytes_a_key);
    plan.groups = reinterpret_cast<b2a::SharedGroup*>(base + at.groups);
    plan.seqs = reinterpret_cast<b2a::SharedSeq*>(base + at.seqs);
    plan.total = reinterpret_cast<long long*>(base);
    plan.ready = reinterpret_cast<uint32_t*>(base + 64);
    plan.err = err;
    b2a::DecodeSharedParams s{};
    s.block_table = block_table;
    s.table_ld = table_ld;
    s.table_width = table_width;
    s.n_pages = n_pages;
    s.page = page;
    s.box_rows = p.box_rows;
    s.n_groups = shared->n_groups;
    s.Hkv = Hkv;
    s.group = p.group;
    s.scale_log2 = p.scale_log2;
    s.groups = plan.groups;
    s.total = plan.total;
    s.part_o = reinterpret_cast<float*>(base + at.part_o);
    s.part_ml = reinterpret_cast<float*>(base + at.part_ml);
    s.place = reinterpret_cast<int*>(base + at.place);
    s.n_ctas = at.n_ctas;
    s.err = err;
    CUtensorMap tq, sk, sv;
    const unsigned long long dims[3] = {(unsigned long long)D, (unsigned long long)Hq, (unsigned long long)B};
    const unsigned long long strides[2] = {(unsigned long long)qs[1] * 2, (unsigned long long)qs[0] * 2};
    const unsigned box[3] = {64u, (unsigned)p.group, 128u / (unsigned)p.group};
    if ((rc = b2a::api_tensor_map(&tq, q, 3, dims, strides, box)) || (rc = map(&sk, k_pages, ks, 1)) ||
        (rc = map(&sv, v_pages, vs, 1)))
      return rc;
    rc = b2a::launch_decode_shared(D, tq, sk, sv, plan, s, static_cast<cudaStream_t>(stream));
    if (rc) return status_of(rc);
    p.seqs = plan.seqs;
    p.ready = plan.ready;
    p.shared_o = s.part_o;
    p.shared_ml = s.part_ml;
    p.shared_place = s.place;
    p.block_rows = b2a::decode_shared_block_rows(D);
    p.shared_ctas = s.n_ctas;
  }
  return status_of(b2a::launch_decode_paged(D, tk, tv, p, static_cast<cudaStream_t>(stream)));
}

int append_paged(const void* q, const void* k, const void* v, const long long* qs, const long long* ks,
                 const long long* vs, int src_bf16, const void* q_norm, const void* k_norm, float eps,
                 const void* cos_tab, const void* sin_tab, int tab_fp32, int max_pos, int rope_dim,
                 void* q_out, void* k_out, void* v_out, void* k_pages, void* v_pages, const long long* kps,
                 const long long* vps, float* k_scales, float* v_scales, const long long* kss,
                 const long long* vss, const int* block_table, long long table_ld, int table_width,
                 int n_pages, int page, const int* cu_seqlens, int B, int N, int Hq, int Hkv, int D,
                 int start_pos, const int* start_pos_per_batch, int* seqlens_out, void* stream) {
  if (!q || !k || !v || !qs || !ks || !vs || !q_out || !k_pages || !v_pages || !kps || !vps || !block_table ||
      !cu_seqlens)
    return B2A_ERR_INVALID_ARG;
  if (B <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || n_pages <= 0 || page <= 0 || table_width <= 0 ||
      table_ld < table_width || (!start_pos_per_batch && start_pos < 0))
    return B2A_ERR_INVALID_ARG;
  // The positions are read while the lengths are written.
  if (start_pos_per_batch && seqlens_out && start_pos_per_batch < seqlens_out + B &&
      seqlens_out < start_pos_per_batch + B)
    return B2A_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return B2A_ERR_HEAD_DIM;
  if (rope_dim != 0 && (rope_dim < 16 || rope_dim > D || (rope_dim & (rope_dim - 1)))) return B2A_ERR_INVALID_ARG;
  if (rope_dim && (!cos_tab || !sin_tab || max_pos <= 0)) return B2A_ERR_INVALID_ARG;
  if ((q_norm || k_norm) && !(eps >= 0.f && std::isfinite(eps))) return B2A_ERR_INVALID_ARG;
  if (!src_bf16 && !tab_fp32) tab_fp32 = 1;
  for (const void* ptr : {q, k, v, cos_tab, sin_tab, q_norm, k_norm, (const void*)q_out, (const void*)k_out,
                          (const void*)v_out, (const void*)k_pages, (const void*)v_pages})
    if (!api_aligned(ptr, 16)) return B2A_ERR_ALIGNMENT;
  const long long mult = src_bf16 ? 8 : 4, pool_mult = k_scales ? 16 : 8;
  if (!api_strides_ok(qs, 2, mult) || !api_strides_ok(ks, 2, mult) || !api_strides_ok(vs, 2, mult) ||
      !api_strides_ok(kps, 3, pool_mult) || !api_strides_ok(vps, 3, pool_mult) || !api_aligned(block_table, 4) ||
      !api_aligned(cu_seqlens, 4) || !api_aligned(start_pos_per_batch, 4) || !api_aligned(seqlens_out, 4))
    return B2A_ERR_ALIGNMENT;

  int* err = nullptr;
  const int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::RopeAppendPagedParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  std::copy_n(qs, 2, p.qs);
  std::copy_n(ks, 2, p.ks);
  std::copy_n(vs, 2, p.vs);
  p.cos = cos_tab;
  p.sin = sin_tab;
  p.tab_fp32 = tab_fp32;
  p.max_pos = max_pos;
  p.rope_dim = rope_dim;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.norm_eps = eps;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  std::copy_n(kps, 3, p.kps);
  std::copy_n(vps, 3, p.vps);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  if (k_scales) {
    std::copy_n(kss, 2, p.kss);
    std::copy_n(vss, 2, p.vss);
  }
  p.block_table = block_table;
  p.table_ld = table_ld;
  p.table_width = table_width;
  p.n_pages = n_pages;
  p.page = page;
  p.cu_seqlens = cu_seqlens;
  p.start_pos_arr = start_pos_per_batch;
  p.start_pos = start_pos;
  p.seqlens_out = seqlens_out;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.N = N;
  p.src_bf16 = src_bf16 ? 1 : 0;
  p.err = err;
  return status_of(b2a::launch_rope_append_paged(D, p, static_cast<cudaStream_t>(stream)));
}

}  // namespace

extern "C" {

int b2a_prefill_varlen(const void* q, const void* k, const void* v, const void* gate, void* o, float* lse,
                       const int* cu_q, const int* cu_k, int B, int Nq, int Nk, int Hq, int Hkv, int D,
                       const long long* qs, const long long* ks, const long long* vs, const long long* gs,
                       const long long* os, int gate_bf16, float scale, int causal, int out_fp32, void* stream) {
  if (B <= 0 || Nq < 0 || Nk < 0 || Hq <= 0 || Hkv <= 0 || !cu_q || !cu_k) return B2A_ERR_INVALID_ARG;
  if (!qs || !ks || !vs || !os || (gate && !gs)) return B2A_ERR_INVALID_ARG;
  if (!(scale > 0.f) || !std::isfinite(scale)) return B2A_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return B2A_ERR_HEAD_DIM;
  if (Hq % Hkv) return B2A_ERR_GQA;
  if (Nq == 0) return B2A_OK;
  // Without any key the maps describe q; nothing is loaded through them.
  const int kv_heads = Nk == 0 ? Hq : Hkv;
  const int kv_rows = Nk == 0 ? Nq : Nk;
  if (Nk == 0) {
    k = v = q;
    ks = vs = qs;
  }
  if (!q || !k || !v || !o) return B2A_ERR_INVALID_ARG;
  if (!api_aligned(q, 16) || !api_aligned(k, 16) || !api_aligned(v, 16) || !api_aligned(o, 16) ||
      !api_aligned(gate, 16) || !api_aligned(lse, 4) || !api_aligned(cu_q, 4) || !api_aligned(cu_k, 4))
    return B2A_ERR_ALIGNMENT;
  if (!api_strides_ok(qs, 2, 8) || !api_strides_ok(ks, 2, 8) || !api_strides_ok(vs, 2, 8) ||
      !api_strides_ok(os, 2, out_fp32 ? 4 : 8) || (gate && !api_strides_ok(gs, 2, gate_bf16 ? 8 : 4)))
    return B2A_ERR_ALIGNMENT;
  const b2a::PrefillPlan plan = b2a::prefill_plan_packed(D, Hq, Hkv, Nq, B);
  const int rows = plan.rows_per_item;
  const long long n_qblk = b2a::packed_blocks(Nq, B, rows);
  if (n_qblk * Hq > INT_MAX) return B2A_ERR_INVALID_ARG;

  int* err = nullptr;
  int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  CUtensorMap tq, tk, tv;
  const int kv_box = D == 256 ? 64 : 128;
  if ((rc = packed_map(&tq, q, D, Nq, Hq, qs, 128)) || (rc = packed_map(&tk, k, D, kv_rows, kv_heads, ks, kv_box)) ||
      (rc = packed_map(&tv, v, D, kv_rows, kv_heads, vs, kv_box)))
    return rc;
  const int esz = out_fp32 ? 4 : 2;
  b2a::PrefillParams p{};
  p.o = o;
  p.o_sh = os[1];
  p.o_st = os[0];
  p.lse = lse;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.Tq = Nq;
  p.Tk = Nk;
  p.scale_log2 = scale * b2a::kApiLog2e;
  p.causal = causal ? 1 : 0;
  p.out_fp32 = out_fp32 ? 1 : 0;
  p.n_qblk = (int)n_qblk;
  p.head_pairs = plan.head_pairs;
  p.err = err;
  p.gate = gate;
  if (gate) {
    p.g_sh = gs[1];
    p.g_st = gs[0];
    p.gate_bf16 = gate_bf16 ? 1 : 0;
  }
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.o_v8 = api_aligned(o, 32) && (os[0] * esz) % 32 == 0 && (os[1] * esz) % 32 == 0;
  return status_of(b2a::launch_prefill_packed(D, plan, tq, tk, tv, p, static_cast<cudaStream_t>(stream)));
}

size_t b2a_decode_paged_workspace_bytes(int B, int Hq, int Hkv, int D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 16 || !head_dim_ok(D)) return 0;
  // Of either cache: 8-bit calls use no fewer CTAs.
  const int group = Hq / Hkv, ctas = b2a::decode_paged_max_ctas(D, group, true, b2a::api_sm_count());
  const size_t rows = b2a::decode_paged_parts(B, Hkv, ctas) * group;
  return b2a::api_align256(rows * D * sizeof(float)) + b2a::api_align256(rows * 2 * sizeof(float)) +
         (size_t)B * Hkv * 2 * sizeof(int);
}

int b2a_decode_paged(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                     long long table_ld, int table_width, const int* seqlens, const void* gate, void* o, int B,
                     int Hq, int Hkv, int n_pages, int page, int D, const long long* qs, const long long* ks,
                     const long long* vs, const long long* gs, const long long* os, int gate_bf16, float scale,
                     int out_fp32, void* workspace, size_t workspace_bytes, void* stream) {
  return paged_attention(q, k_pages, v_pages, block_table, nullptr, nullptr, nullptr, nullptr, nullptr, table_ld,
                         table_width, seqlens, gate, o, B, Hq, Hkv, n_pages, page, D, qs, ks, vs, gs, os, gate_bf16,
                         scale, out_fp32, workspace, workspace_bytes, stream);
}

size_t b2a_decode_paged_shared_workspace_bytes(int B, int Hq, int Hkv, int D, int n_groups) {
  const size_t own = b2a_decode_paged_workspace_bytes(B, Hq, Hkv, D);
  return own == 0 || n_groups <= 0 ? 0 : own + shared_layout(B, Hq, Hkv, D, n_groups).bytes;
}

int b2a_decode_paged_shared(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                            long long table_ld, int table_width, const int* seqlens, const int* prefix_lens,
                            const int* cu_groups, int n_groups, long long least_saved_bytes, const void* gate, void* o,
                            int B, int Hq, int Hkv,
                            int n_pages, int page, int D, const long long* qs, const long long* ks,
                            const long long* vs, const long long* gs, const long long* os, int gate_bf16, float scale,
                            int out_fp32, void* workspace, size_t workspace_bytes, void* stream) {
  if (!prefix_lens || n_groups <= 0 || (!cu_groups && n_groups != 1)) return B2A_ERR_INVALID_ARG;
  if (!api_aligned(prefix_lens, 4) || !api_aligned(cu_groups, 4)) return B2A_ERR_ALIGNMENT;
  const SharedPrefix shared{prefix_lens, cu_groups, n_groups, least_saved_bytes};
  return paged_attention(q, k_pages, v_pages, block_table, nullptr, nullptr, nullptr, nullptr, &shared, table_ld,
                         table_width, seqlens, gate, o, B, Hq, Hkv, n_pages, page, D, qs, ks, vs, gs, os, gate_bf16,
                         scale, out_fp32, workspace, workspace_bytes, stream);
}

int b2a_decode_paged_e4m3(const void* q, const void* k_pages, const void* v_pages, const float* k_scales,
                          const float* v_scales, const long long* kss, const long long* vss, const int* block_table,
                          long long table_ld, int table_width, const int* seqlens, const void* gate, void* o, int B,
                          int Hq, int Hkv, int n_pages, int page, int D, const long long* qs, const long long* ks,
                          const long long* vs, const long long* gs, const long long* os, int gate_bf16, float scale,
                          int out_fp32, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = scales_ok(k_scales, v_scales, kss, vss)) return rc;
  return paged_attention(q, k_pages, v_pages, block_table, k_scales, v_scales, kss, vss, nullptr, table_ld, table_width,
                         seqlens, gate, o, B, Hq, Hkv, n_pages, page, D, qs, ks, vs, gs, os, gate_bf16, scale, out_fp32,
                         workspace, workspace_bytes, stream);
}

int b2a_rope_append_paged(const void* q, const void* k, const void* v, const long long* qs, const long long* ks,
                          const long long* vs, int src_bf16, const void* q_norm, const void* k_norm, float eps,
                          const void* cos_tab, const void* sin_tab, int tab_fp32, int max_pos, int rope_dim,
                          void* q_out, void* k_out, void* v_out, void* k_pages, void* v_pages, const long long* kps,
                          const long long* vps, const int* block_table, long long table_ld, int table_width,
                          int n_pages, int page, const int* cu_seqlens, int B, int N, int Hq, int Hkv, int D,
                          int start_pos, const int* start_pos_per_batch, int* seqlens_out, void* stream) {
  return append_paged(q, k, v, qs, ks, vs, src_bf16, q_norm, k_norm, eps, cos_tab, sin_tab, tab_fp32, max_pos, rope_dim,
                      q_out, k_out, v_out, k_pages, v_pages, kps, vps, nullptr, nullptr, nullptr, nullptr, block_table,
                      table_ld, table_width, n_pages, page, cu_seqlens, B, N, Hq, Hkv, D, start_pos,
                      start_pos_per_batch, seqlens_out, stream);
}

int b2a_rope_append_paged_e4m3(const void* q, const void* k, const void* v, const long long* qs, const long long* ks,
                               const long long* vs, int src_bf16, const void* q_norm, const void* k_norm, float eps,
                               const void* cos_tab, const void* sin_tab, int tab_fp32, int max_pos, int rope_dim,
                               void* q_out, void* k_out, void* v_out, void* k_pages, void* v_pages,
                               const long long* kps, const long long* vps, float* k_scales, float* v_scales,
                               const long long* kss, const long long* vss, const int* block_table, long long table_ld,
                               int table_width, int n_pages, int page, const int* cu_seqlens, int B, int N, int Hq,
                               int Hkv, int D, int start_pos, const int* start_pos_per_batch, int* seqlens_out,
                               void* stream) {
  if (const int rc = scales_ok(k_scales, v_scales, kss, vss)) return rc;
  return append_paged(q, k, v, qs, ks, vs, src_bf16, q_norm, k_norm, eps, cos_tab, sin_tab, tab_fp32, max_pos, rope_dim,
                      q_out, k_out, v_out, k_pages, v_pages, kps, vps, k_scales, v_scales, kss, vss, block_table,
                      table_ld, table_width, n_pages, page, cu_seqlens, B, N, Hq, Hkv, D, start_pos,
                      start_pos_per_batch, seqlens_out, stream);
}

int b2a_gather_paged(const void* k_pages, const void* v_pages, const long long* kps, const long long* vps,
                     const float* k_scales, const float* v_scales, const long long* kss, const long long* vss,
                     const int* block_table, long long table_ld, int table_width, int n_pages, int page,
                     const int* cu_seqlens, int B, int N, int Hkv, int D, int start_pos,
                     const int* start_pos_per_batch, void* k_out, void* v_out, void* stream) {
  if (!k_pages || !v_pages || !kps || !vps || !block_table || !cu_seqlens || !k_out || !v_out)
    return B2A_ERR_INVALID_ARG;
  if (!k_scales != !v_scales) return B2A_ERR_INVALID_ARG;
  if (B <= 0 || N <= 0 || Hkv <= 0 || n_pages <= 0 || page <= 0 || table_width <= 0 || table_ld < table_width ||
      (!start_pos_per_batch && start_pos < 0))
    return B2A_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return B2A_ERR_HEAD_DIM;
  if (k_scales)
    if (const int rc = scales_ok(k_scales, v_scales, kss, vss)) return rc;
  const unsigned long long bytes = 2ull * N * Hkv * D;  // of either output
  const uintptr_t ko = reinterpret_cast<uintptr_t>(k_out), vo = reinterpret_cast<uintptr_t>(v_out);
  if (ko < vo + bytes && vo < ko + bytes) return B2A_ERR_INVALID_ARG;
  for (const void* ptr : {k_pages, v_pages, (const void*)k_out, (const void*)v_out})
    if (!api_aligned(ptr, 16)) return B2A_ERR_ALIGNMENT;
  const long long mult = k_scales ? 16 : 8;
  if (!api_strides_ok(kps, 3, mult) || !api_strides_ok(vps, 3, mult) || !api_aligned(block_table, 4) ||
      !api_aligned(cu_seqlens, 4) || !api_aligned(start_pos_per_batch, 4))
    return B2A_ERR_ALIGNMENT;
  int* err = nullptr;
  const int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::GatherPagedParams p{};
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  std::copy_n(kps, 3, p.kps);
  std::copy_n(vps, 3, p.vps);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  if (k_scales) {
    std::copy_n(kss, 2, p.kss);
    std::copy_n(vss, 2, p.vss);
  }
  p.block_table = block_table;
  p.table_ld = table_ld;
  p.table_width = table_width;
  p.n_pages = n_pages;
  p.page = page;
  p.cu_seqlens = cu_seqlens;
  p.start_pos_arr = start_pos_per_batch;
  p.start_pos = start_pos;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.out_v8 = api_aligned(k_out, 32) && api_aligned(v_out, 32);
  p.B = B;
  p.Hkv = Hkv;
  p.N = N;
  p.err = err;
  return status_of(b2a::launch_gather_paged(D, p, static_cast<cudaStream_t>(stream)));
}

int b2a_penalize(const void* logits, long long ld_logits, int logits_bf16, const void* tokens, int tokens_64,
                 long long tokens_row, long long tokens_step, int L, const int* lengths, const int* prompt_lengths,
                 const float* repetition, float repetition_all, const float* frequency, float frequency_all,
                 const float* presence, float presence_all, const float* bias, long long ld_bias, const int* allowed,
                 long long ld_allowed, void* out, long long ld_out, int R, int V, void* stream) {
  if (!logits || !out || R <= 0 || V <= 0 || V > (1 << 30) || L < 0 || L > (1 << 30) || (L > 0 && !tokens))
    return B2A_ERR_INVALID_ARG;
  if (ld_logits < 0 || ld_out < (R > 1 ? V : 0) || tokens_row < 0 || tokens_step < 0 || ld_bias < 0 || ld_allowed < 0)
    return B2A_ERR_INVALID_ARG;
  if ((!repetition && !(repetition_all > 0.f && std::isfinite(repetition_all))) ||
      (!frequency && !std::isfinite(frequency_all)) || (!presence && !std::isfinite(presence_all)))
    return B2A_ERR_INVALID_ARG;
  const unsigned size = logits_bf16 ? 2 : 4;
  if (!api_aligned(logits, size) || !api_aligned(out, size) || !api_aligned(tokens, tokens_64 ? 8 : 4))
    return B2A_ERR_ALIGNMENT;
  for (const void* ptr : {(const void*)lengths, (const void*)prompt_lengths, (const void*)repetition,
                          (const void*)frequency, (const void*)presence, (const void*)bias, (const void*)allowed})
    if (!api_aligned(ptr, 4)) return B2A_ERR_ALIGNMENT;
  // In place, row by row, or apart: chunks of a row run in any order.
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(logits), y0 = reinterpret_cast<uintptr_t>(out);
  const uintptr_t x1 = x0 + ((unsigned long long)(R - 1) * ld_logits + V) * size;
  const uintptr_t y1 = y0 + ((unsigned long long)(R - 1) * ld_out + V) * size;
  if (x0 < y1 && y0 < x1 && !(x0 == y0 && (ld_logits == ld_out || R == 1))) return B2A_ERR_INVALID_ARG;
  // The rest is read by other chunks than the one that writes, too: apart. (tokens: the caller's
  // to see to.)
  auto meets_out = [&](const void* base, unsigned long long bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    return base && at < y1 && y0 < at + bytes;
  };
  const unsigned long long last = R - 1, words = (V + 31LL) / 32;
  if (meets_out(bias, (last * ld_bias + V) * 4) || meets_out(allowed, (last * ld_allowed + words) * 4))
    return B2A_ERR_INVALID_ARG;
  for (const void* rows : {(const void*)lengths, (const void*)prompt_lengths, (const void*)repetition,
                           (const void*)frequency, (const void*)presence})
    if (meets_out(rows, 4ull * R)) return B2A_ERR_INVALID_ARG;
  int* err = nullptr;
  const int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::PenalizeParams p{};
  p.logits = logits;
  p.ld_logits = ld_logits;
  p.logits_bf16 = logits_bf16 ? 1 : 0;
  p.out = out;
  p.ld_out = ld_out;
  p.tokens = L > 0 ? tokens : nullptr;
  p.tokens_row = tokens_row;
  p.tokens_step = tokens_step;
  p.tokens_64 = tokens_64 ? 1 : 0;
  p.L = L;
  p.lengths = lengths;
  p.prompt_lengths = prompt_lengths;
  p.repetition = repetition;
  p.frequency = frequency;
  p.presence = presence;
  p.repetition_all = repetition_all;
  p.frequency_all = frequency_all;
  p.presence_all = presence_all;
  p.bias = bias;
  p.ld_bias = ld_bias;
  p.allowed = reinterpret_cast<const unsigned*>(allowed);
  p.ld_allowed = ld_allowed;
  p.R = R;
  p.V = V;
  p.err = err;
  return status_of(b2a::launch_penalize(p, static_cast<cudaStream_t>(stream)));
}

int b2a_sample(const void* logits, long long ld_logits, int logits_bf16, const float* noise, long long ld_noise, int R,
               int V, const float* temperature, float temperature_all, const int* top_k, int top_k_all,
               const float* top_p, float top_p_all, const float* min_p, float min_p_all, long long* out,
               void* stream) {
  if (!logits || !out || R <= 0 || V <= 0 || ld_logits < 0 || ld_noise < 0) return B2A_ERR_INVALID_ARG;
  if ((!temperature && std::isnan(temperature_all)) || (!top_p && std::isnan(top_p_all)) ||
      (!min_p && std::isnan(min_p_all)))
    return B2A_ERR_INVALID_ARG;
  if (!api_aligned(logits, logits_bf16 ? 2 : 4) || !api_aligned(noise, 4) || !api_aligned(temperature, 4) ||
      !api_aligned(top_k, 4) || !api_aligned(top_p, 4) || !api_aligned(min_p, 4) || !api_aligned(out, 8))
    return B2A_ERR_ALIGNMENT;
  int* err = nullptr;
  const int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::SampleParams p{};
  p.logits = logits;
  p.ld_logits = ld_logits;
  p.logits_bf16 = logits_bf16 ? 1 : 0;
  p.noise = noise;
  p.ld_noise = ld_noise;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = temperature_all;
  p.top_k_all = top_k_all;
  p.top_p_all = top_p_all;
  p.min_p_all = min_p_all;
  p.out = out;
  p.R = R;
  p.V = V;
  p.err = err;
  return status_of(b2a::launch_sample(p, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
