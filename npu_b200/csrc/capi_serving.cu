// extern "C" boundary of the serving operators (include/b2attn.h): attention
// over packed sequences, the paged KV cache and sampling. Argument checks,
// tensor maps and launches; stateless like capi.cu.
#include <algorithm>
#include <cmath>
#include <climits>

#include "b2attn.h"
#include "capi_internal.cuh"
#include "decode_paged.cuh"
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
             int box_rows) {
  const unsigned long long dims[5] = {64, (unsigned long long)page, (unsigned long long)(D / 64),
                                      (unsigned long long)heads, (unsigned long long)n_pages};
  const unsigned long long strides[4] = {(unsigned long long)s[2] * 2, 128, (unsigned long long)s[1] * 2,
                                         (unsigned long long)s[0] * 2};
  const unsigned box[5] = {64u, (unsigned)box_rows, (unsigned)(D / 64), 1u, 1u};
  return b2a::api_tensor_map(m, base, 5, dims, strides, box);
}

int status_of(int rc) { return rc == -3 ? B2A_ERR_HEAD_DIM : (rc ? B2A_ERR_LAUNCH : B2A_OK); }

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
  const size_t rows = b2a::decode_paged_parts(B, Hkv, b2a::decode_paged_max_ctas(D, b2a::api_sm_count())) * (Hq / Hkv);
  return b2a::api_align256(rows * D * sizeof(float)) + b2a::api_align256(rows * 2 * sizeof(float)) +
         (size_t)B * Hkv * 2 * sizeof(int);
}

int b2a_decode_paged(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                     long long table_ld, int table_width, const int* seqlens, const void* gate, void* o, int B,
                     int Hq, int Hkv, int n_pages, int page, int D, const long long* qs, const long long* ks,
                     const long long* vs, const long long* gs, const long long* os, int gate_bf16, float scale,
                     int out_fp32, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_pages || !v_pages || !block_table || !seqlens || !o || !qs || !ks || !vs || !os || (gate && !gs))
    return B2A_ERR_INVALID_ARG;
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || n_pages <= 0 || page <= 0 || page % 16 || table_width <= 0 ||
      table_ld < table_width || (long long)table_width * page > INT_MAX - 64)
    return B2A_ERR_INVALID_ARG;
  if (!(scale > 0.f) || !std::isfinite(scale)) return B2A_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return B2A_ERR_HEAD_DIM;
  if (Hq % Hkv || Hq / Hkv > 16) return B2A_ERR_GQA;
  if (!api_aligned(q, 16) || !api_aligned(k_pages, 16) || !api_aligned(v_pages, 16) ||
      !api_aligned(o, out_fp32 ? 4 : 2) || !api_aligned(block_table, 4) || !api_aligned(seqlens, 4) ||
      !api_aligned(gate, gate_bf16 ? 2 : 4))
    return B2A_ERR_ALIGNMENT;
  if (!api_strides_ok(qs, 2, 8) || !api_strides_ok(ks, 3, 8) || !api_strides_ok(vs, 3, 8)) return B2A_ERR_ALIGNMENT;
  const size_t need = b2a_decode_paged_workspace_bytes(B, Hq, Hkv, D);
  if (!workspace || workspace_bytes < need || !api_aligned(workspace, 16)) return B2A_ERR_WORKSPACE;

  int* err = nullptr;
  int rc = b2a::api_prologue(&err);
  if (rc) return rc;
  b2a::DecodePagedParams p{};
  // Keys per TMA box: a box never crosses a page, a warp's 16 keys never a box.
  p.box_rows = page % 64 == 0 ? 64 : (page % 32 == 0 ? 32 : 16);
  CUtensorMap tk, tv;
  if ((rc = pool_map(&tk, k_pages, D, n_pages, Hkv, page, ks, p.box_rows)) ||
      (rc = pool_map(&tv, v_pages, D, n_pages, Hkv, page, vs, p.box_rows)))
    return rc;
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
  p.n_ctas = b2a::decode_paged_max_ctas(D, b2a::api_sm_count());
  const size_t rows = b2a::decode_paged_parts(B, Hkv, p.n_ctas) * p.group;
  char* scratch = static_cast<char*>(workspace);
  p.part_o = reinterpret_cast<float*>(scratch);
  scratch += b2a::api_align256(rows * D * sizeof(float));
  p.part_ml = reinterpret_cast<float*>(scratch);
  p.place = reinterpret_cast<int*>(scratch + b2a::api_align256(rows * 2 * sizeof(float)));
  return status_of(b2a::launch_decode_paged(D, tk, tv, p, static_cast<cudaStream_t>(stream)));
}

int b2a_rope_append_paged(const void* q, const void* k, const void* v, const long long* qs, const long long* ks,
                          const long long* vs, int src_bf16, const void* q_norm, const void* k_norm, float eps,
                          const void* cos_tab, const void* sin_tab, int tab_fp32, int max_pos, int rope_dim,
                          void* q_out, void* k_out, void* v_out, void* k_pages, void* v_pages, const long long* kps,
                          const long long* vps, const int* block_table, long long table_ld, int table_width,
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
  const long long mult = src_bf16 ? 8 : 4;
  if (!api_strides_ok(qs, 2, mult) || !api_strides_ok(ks, 2, mult) || !api_strides_ok(vs, 2, mult) ||
      !api_strides_ok(kps, 3, 8) || !api_strides_ok(vps, 3, 8) || !api_aligned(block_table, 4) ||
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
  p.k_pages = static_cast<__nv_bfloat16*>(k_pages);
  p.v_pages = static_cast<__nv_bfloat16*>(v_pages);
  std::copy_n(kps, 3, p.kps);
  std::copy_n(vps, 3, p.vps);
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
