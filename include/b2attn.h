/*
 * b2attn — C ABI of the B200 (sm_100a) attention engine.
 *
 * This is the boundary that replaces the reference's FlashAttention-2 device
 * path: the host wrapper NpuAttention.run_batch (npu/fa.py:206-323), which
 * packs Q/K/V, dispatches the AIE kernel entry points attn_block /
 * attn_finalise (npu/fa_kernel.cc:68-217, :219-227) and reads the output back.
 * Those entry points keep per-dispatch running state in static tile memory
 * (npu/fa_kernel.cc:59-64); every function here is instead stateless,
 * re-entrant and ordered on the caller's CUDA stream.
 *
 * Conventions
 *  - All tensor pointers are caller-owned device memory (b2a_prefill_host:
 *    host memory, plus a device workspace); nothing here allocates on the
 *    call path. Scratch comes from the caller (b2a_decode_workspace_bytes,
 *    b2a_prefill_host_workspace_bytes).
 *  - Element types: Q/K/V and the KV cache are bf16. Outputs are bf16 or fp32
 *    (out_fp32). Innermost (head_dim) stride is 1; every other stride is given
 *    in ELEMENTS and must be a multiple of 8 (16 bytes). Base pointers must be
 *    16-byte aligned.
 *  - `stream` is a cudaStream_t (NULL = legacy default stream).
 *  - Return value: B2A_OK (0) or a negative B2A_ERR_* code; no C++ exception
 *    crosses this boundary. Device-side faults that kernels detect (a bounded
 *    wait that ran out, a sequence length larger than the cache) are reported
 *    through b2a_get_device_error.
 *  - GQA: query head h reads KV head h / (Hq / Hkv) — the repeat_interleave
 *    mapping of smollm.py:205-207 and qwen/forward.py:194-197.
 */
#ifndef B2ATTN_H
#define B2ATTN_H

#include <stddef.h>

#if defined(__GNUC__)
#define B2A_API __attribute__((visibility("default")))
#else
#define B2A_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum {
  B2A_OK = 0,
  B2A_ERR_INVALID_ARG = -1,      /* null pointer, non-positive size, scale <= 0 */
  B2A_ERR_HEAD_DIM = -2,         /* head_dim not supported by this entry point */
  B2A_ERR_GQA = -3,              /* Hq not a multiple of Hkv, or group too large */
  B2A_ERR_ALIGNMENT = -4,        /* pointer or stride not 16-byte aligned */
  B2A_ERR_TMA = -5,              /* tensor-map encoding failed or unavailable */
  B2A_ERR_LAUNCH = -6,           /* kernel launch failed (cudaGetLastError) */
  B2A_ERR_WORKSPACE = -7,        /* decode workspace missing or too small */
  B2A_ERR_DEVICE = -8,           /* current device is not sm_100 */
  B2A_ERR_DEVICE_TIMEOUT = -9,   /* a kernel's bounded wait ran out */
  B2A_ERR_DEVICE_BAD_LEN = -10,  /* a sequence length exceeded the cache */
  B2A_ERR_CUDA = -11             /* another CUDA runtime error */
};

/* Human-readable text for a status code. Never NULL. */
B2A_API const char* b2a_strerror(int code);

/* ABI version (major * 100 + minor). */
B2A_API int b2a_version(void);

/*
 * Causal (or full) GQA attention prefill.
 * Replaces: NpuAttention.run_batch (npu/fa.py:206-323) driving attn_block /
 * attn_finalise (npu/fa_kernel.cc:68-227); arithmetic follows
 * flash_attention_ref (npu/fa_ref.py:42-131).
 *
 *   q   [B, Hq,  Tq, D]  strides q_strides  = {batch, head, row}
 *   k   [B, Hkv, Tk, D]  strides k_strides
 *   v   [B, Hkv, Tk, D]  strides v_strides
 *   o   [B, Hq,  Tq, D]  strides o_strides  (bf16, or fp32 if out_fp32)
 *   lse optional [B, Hq, Tq] fp32 contiguous: natural-log sum of
 *       exp(scale * s) over unmasked keys (-inf for fully masked rows).
 *
 * Query row r sits at absolute position start + r, where start is
 * start_pos_per_batch[b] (device int32 array) when that pointer is non-NULL,
 * else start_pos. With causal != 0, key c is masked iff c > start + r
 * (npu/fa_ref.py:57-60, :102-108). Rows with no unmasked key output 0
 * (npu/fa_ref.py:112-128). scale is the softmax scale (1/sqrt(D) in the
 * reference, npu/fa_ref.py:68). Tk may be 0: every row is then 0 and k / v
 * are not read (they may be NULL).
 * Supported D: 64, 128, 256.
 * With the environment variable B2A_PREFILL_SM_PAIRS set to a positive row
 * count, head dim 128 queries with an even GQA group and at least that many
 * rows run on SM pairs (a two-CTA cluster per 256 rows of two query heads,
 * tcgen05.mma.cta_group::2): same results bit for bit, measured slower than
 * the default one-SM kernel, so off unless asked for. Read on every call.
 */
B2A_API int b2a_prefill(const void* q, const void* k, const void* v, void* o, float* lse, int B, int Hq, int Hkv,
                int Tq, int Tk, int D, const long long* q_strides, const long long* k_strides,
                const long long* v_strides, const long long* o_strides, int start_pos,
                const int* start_pos_per_batch, float scale, int causal, int out_fp32, void* stream);

/*
 * Bytes of caller-provided device scratch that b2a_decode needs for the given
 * geometry and split length (0 split_len = the default chosen by b2a_decode).
 */
B2A_API size_t b2a_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int Lmax, int split_len);

/*
 * The split length b2a_decode uses when called with split_len = 0: keys per
 * split CTA such that the estimated work (B x Hkv x Lmax / 2 keys, since the
 * lengths are on the device) fills about one wave of CTAs, rounded to a
 * power of two in [512, 4096], and 2048 when that still leaves several
 * waves. Pass an explicit split_len when the lengths are known to be far
 * from half the cache.
 */
B2A_API int b2a_decode_default_split(int B, int Hkv, int Lmax);

/*
 * Single-token decode attention over a contiguous KV cache (split-KV
 * flash-decode + log-sum-exp combine, two launches on `stream`).
 * Replaces: the T=1 attention step of smollm.py:222-234 (and the bucketed
 * decode route through run_batch, smollm.py:144,212-221).
 *
 *   q        [B, Hq, D]        strides q_strides = {batch, head}
 *   k_cache  [B, Hkv, Lmax, D] strides k_strides = {batch, head, position}
 *   v_cache  [B, Hkv, Lmax, D] strides v_strides
 *   seqlens  [B] int32 device  keys 0 .. seqlens[b]-1 are attended (no mask)
 *   o        [B, Hq, D]        strides o_strides = {batch, head}
 *
 * split_len: keys per split CTA, a multiple of 64 (0 = default).
 * Supported D: 64, 128, 256; Hq / Hkv <= 16.
 */
B2A_API int b2a_decode(const void* q, const void* k_cache, const void* v_cache, const int* seqlens, void* o, int B,
               int Hq, int Hkv, int Lmax, int D, const long long* q_strides, const long long* k_strides,
               const long long* v_strides, const long long* o_strides, float scale, int split_len,
               int out_fp32, void* workspace, size_t workspace_bytes, void* stream);

/*
 * b2a_prefill / b2a_decode with the gated-attention epilogue of Qwen3.5/3.6
 * (qwen/forward.py:223-226): the output is attention * sigmoid(gate), fused
 * into the kernels' output stores (no extra pass over O).
 *   prefill: gate [B, Hq, Tq, D], element strides gate_strides = {batch,
 *            head, row}, 16-byte aligned, strides multiples of 16 bytes;
 *   decode:  gate [B, Hq, D], gate_strides = {batch, head}.
 * gate_bf16: 1 for bf16, 0 for fp32. The q projection of the reference holds
 * [q_h | gate_h] per head, so the gate is usually a strided view of it
 * (head stride 2 D). All other arguments as the ungated calls.
 */
B2A_API int b2a_prefill_gated(const void* q, const void* k, const void* v, const void* gate, void* o, float* lse,
                              int B, int Hq, int Hkv, int Tq, int Tk, int D, const long long* q_strides,
                              const long long* k_strides, const long long* v_strides,
                              const long long* gate_strides, const long long* o_strides, int gate_bf16,
                              int start_pos, const int* start_pos_per_batch, float scale, int causal,
                              int out_fp32, void* stream);

B2A_API int b2a_decode_gated(const void* q, const void* k_cache, const void* v_cache, const int* seqlens,
                             const void* gate, void* o, int B, int Hq, int Hkv, int Lmax, int D,
                             const long long* q_strides, const long long* k_strides, const long long* v_strides,
                             const long long* gate_strides, const long long* o_strides, int gate_bf16,
                             float scale, int split_len, int out_fp32, void* workspace, size_t workspace_bytes,
                             void* stream);

/*
 * b2a_decode followed by the output projection and residual add, fused into
 * the combine kernel: x[b, :] += o_b @ wo^T, where o_b is sequence b's
 * attention output [Hq * D] (rounded to x's dtype) and wo [dim, Hq * D] the
 * output projection weight (F.linear layout, row stride wo_ld elements, fp32
 * with wo_fp32 = 1 else bf16; 16-byte aligned, wo_ld a multiple of 16 bytes).
 * x: the residual stream [B, dim] (row stride x_sb elements, fp32 with
 * x_fp32 = 1 else bf16), updated in place; the attention output itself is not
 * stored. Replaces: the attention core plus `x = x + wo(o)` of the T=1 layer
 * step (smollm.py:222-236, where the output projection follows attention at
 * :235-236). The combine runs per (block of 32 outputs, sequence): every
 * output of x has one writer and a fixed summation order, so results are
 * reproducible. Hq * D <= ~51k (one sequence's attention output in shared
 * memory). Workspace as b2a_decode.
 */
B2A_API int b2a_decode_proj(const void* q, const void* k_cache, const void* v_cache, const int* seqlens,
                            const void* wo, long long wo_ld, int wo_fp32, int dim, void* x, long long x_sb,
                            int x_fp32, int B, int Hq, int Hkv, int Lmax, int D, const long long* q_strides,
                            const long long* k_strides, const long long* v_strides, float scale, int split_len,
                            void* workspace, size_t workspace_bytes, void* stream);

/* Size of the fixed device scratch buffer behind b2a_decode_noalloc. */
#define B2A_NOALLOC_SCRATCH_BYTES (16u * 1024u * 1024u)

/*
 * b2a_decode without caller scratch, for callers that cannot allocate device
 * memory (hosts that reserve all device memory up front and forbid later
 * cudaMalloc/cudaFree, plugin/FFI callers holding only input and output
 * pointers). No counterpart in the reference.
 * Same arguments and results as b2a_decode minus the workspace. Scratch is a
 * device array of B2A_NOALLOC_SCRATCH_BYTES inside this library, held by every
 * GPU that loads it until exit. With split_len = 0 the default split length
 * is doubled until the partial results fit; problems that need more even with
 * one split per sequence (or with the caller's split_len) return
 * B2A_ERR_WORKSPACE before any launch (use a larger split_len, or b2a_decode).
 * A non-sm_100 device returns B2A_ERR_DEVICE. The first call in a device's
 * context looks up the array's device address (cudaGetSymbolAddress): make it
 * outside any stream capture; a new context (after cudaDeviceReset) is
 * detected and looked up again. All calls on a device share the buffer, so
 * calls that overlap on the GPU race; nothing in it needs to start at zero.
 */
B2A_API int b2a_decode_noalloc(const void* q, const void* k_cache, const void* v_cache, const int* seqlens,
                               void* o, int B, int Hq, int Hkv, int Lmax, int D, const long long* q_strides,
                               const long long* k_strides, const long long* v_strides,
                               const long long* o_strides, float scale, int split_len, int out_fp32,
                               void* stream);

/*
 * Fused RoPE + in-place KV-cache append, one launch per layer and step.
 * Replaces: the per-step projection transposes, the two apply_rope calls,
 * torch.cat of the layer cache and repeat_interleave of smollm.py:186-208
 * (and the Tk buckets of smollm.py:17-20,144): the cache is a preallocated
 * device buffer written in place and read by b2a_prefill / b2a_decode
 * without expanding GQA heads.
 *
 *   q, k, v  [B, T, H, D] views (H = Hq, Hkv, Hkv), element strides
 *            {batch, token, head} in q/k/v_strides, D contiguous; fp32
 *            (src_bf16 = 0) or bf16 (src_bf16 = 1); 16-byte aligned, strides
 *            multiples of 16 bytes
 *   cos_tab, sin_tab [max_pos, D] contiguous, same dtype as q/k/v: the
 *            model's rotary tables (build_rope_cache, smollm.py:45-50)
 *   q_out    [B, Hq, T, D] bf16 contiguous: q rotated (the attention
 *            kernels' query layout)
 *   k_cache, v_cache [B, Hkv, Lmax, D] bf16, element strides {batch, head,
 *            position} in k/v_cache_strides (multiples of 8): rows
 *            p_b .. p_b + T - 1 receive k rotated and v, where p_b =
 *            start_pos_per_batch[b] (device int32) or start_pos
 *   seqlens_out [B] int32 device, optional: set to p_b + T
 *
 * Rotation is rotate-half (smollm.py:53-58), computed op by op in the source
 * dtype as the reference does, then rounded to bf16. Positions must satisfy
 * 0 <= p_b and p_b + T <= min(Lmax, max_pos): checked on the host for a
 * scalar start_pos (B2A_ERR_INVALID_ARG), on the device for per-batch
 * positions (rows out of range are skipped and the device error word reports
 * B2A_ERR_DEVICE_BAD_LEN). Supported D: 64, 128, 256.
 */
B2A_API int b2a_rope_append(const void* q, const void* k, const void* v, const long long* q_strides,
                            const long long* k_strides, const long long* v_strides, int src_bf16,
                            const void* cos_tab, const void* sin_tab, int max_pos, void* q_out, void* k_cache,
                            void* v_cache, const long long* k_cache_strides, const long long* v_cache_strides,
                            int B, int T, int Hq, int Hkv, int D, int Lmax, int start_pos,
                            const int* start_pos_per_batch, int* seqlens_out, void* stream);

/*
 * b2a_rope_append with the gated-attention prologue of Qwen3.5/3.6
 * (qwen/forward.py:178-204): each q and k head is RMS-normalised over its D
 * lanes with the weights q_norm / k_norm ([D], source dtype; either may be
 * null to skip; fp32 statistics, (x * rsqrt(mean(x^2) + eps)) * w as
 * qwen/forward.py:58-61) and then rotated on its first rope_dim lanes only
 * (partial rotate-half, qwen/forward.py:81-95; cos_tab/sin_tab are
 * [max_pos, rope_dim]). rope_dim is 0 (no rotation) or a power of two in
 * [16, D]. q may be a strided view of the [q_h | gate_h] per-head layout of
 * the gated q projection (head stride 2 D). Sources need 16-byte alignment
 * and strides that are multiples of 16 bytes; caches and q_out likewise.
 * Otherwise as b2a_rope_append (which is this call with rope_dim = D and no
 * norms).
 */
B2A_API int b2a_qk_norm_rope_append(const void* q, const void* k, const void* v, const long long* q_strides,
                                    const long long* k_strides, const long long* v_strides, int src_bf16,
                                    const void* q_norm, const void* k_norm, float eps, const void* cos_tab,
                                    const void* sin_tab, int max_pos, int rope_dim, void* q_out, void* k_cache,
                                    void* v_cache, const long long* k_cache_strides,
                                    const long long* v_cache_strides, int B, int T, int Hq, int Hkv, int D,
                                    int Lmax, int start_pos, const int* start_pos_per_batch, int* seqlens_out,
                                    void* stream);

/*
 * Prefill with inputs and result in HOST memory: the call surface of the
 * reference's NpuAttention.run_batch (npu/fa.py:206-323), which takes host
 * Q/K/V stacks and returns the host O stack.
 *
 *   q   [B, Hq,  Tq, D]  bf16, contiguous, host memory
 *   k   [B, Hkv, Tk, D]  bf16, contiguous, host memory (may be NULL if Tk == 0)
 *   v   [B, Hkv, Tk, D]
 *   o   [B, Hq,  Tq, D]  bf16 (fp32 if out_fp32), contiguous, host memory
 *   start_pos_per_batch  optional HOST int32 [B]; else start_pos for all
 *   workspace  device memory of b2a_prefill_host_workspace_bytes(...) bytes,
 *              256-byte aligned
 *
 * Same arithmetic, masking and results as b2a_prefill. The problem is cut
 * into n_chunks pieces of (batch, KV head) units (0 = 32): whole batches
 * when there are enough, else KV heads of one batch. Each piece is copied in
 * on a library-owned copy stream, computed on `stream`, and copied out on a
 * second copy stream, with two workspace slots alternating, so uploads,
 * kernels and downloads of neighbouring pieces overlap. The call is
 * asynchronous and ordered on `stream`: it returns once everything is
 * queued, and work queued on `stream` afterwards (a synchronize, an event)
 * sees the complete o. Host buffers must stay valid and unmodified until
 * then. Page-locked host memory is needed for the copies to overlap;
 * pageable buffers give the same result with the copies serialised.
 * Concurrent calls on one device are serialised while queueing and must not
 * share a workspace unless ordered on one stream.
 */
B2A_API size_t b2a_prefill_host_workspace_bytes(int B, int Hq, int Hkv, int Tq, int Tk, int D, int out_fp32,
                                                int n_chunks);
B2A_API int b2a_prefill_host(const void* q, const void* k, const void* v, void* o, int B, int Hq, int Hkv, int Tq,
                             int Tk, int D, int start_pos, const int* start_pos_per_batch, float scale, int causal,
                             int out_fp32, int n_chunks, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Serving sequences of different lengths together: attention over packed
 * prompts, a paged KV cache (append, single-token attention, reading back), bf16
 * or 8-bit, penalties on logits and sampling.
 *
 * Packed tensors hold the sequences' tokens one after another: sequence b owns
 * rows [cu[b], cu[b + 1]) of a tensor, cu int32 [B + 1] on the device, not
 * decreasing, from 0 or more to at most the tensor's rows. Rows outside every
 * sequence are neither read nor written. A paged cache is a pool
 * [n_pages, Hkv, page, D] (bf16; strides {page, head, slot}) and a block
 * table int32 [B, table_width] (row stride table_ld) on the device: key j of
 * sequence b is slot j % page of page table[b][j / page]. Entries past a
 * sequence's last page are not read. Pools may be any stored order with a
 * contiguous last dimension, [n_pages, page, Hkv, D] included.
 */

/*
 * b2a_prefill over packed sequences: q [Nq, Hq, D], k and v [Nk, Hkv, D],
 * o [Nq, Hq, D], optional gate as q (o = attention * sigmoid(gate)), optional
 * lse [Hq, Nq] fp32; *_strides = {row, head}. Sequence b's queries are rows
 * [cu_q[b], cu_q[b + 1]), its keys rows [cu_k[b], cu_k[b + 1]); with causal
 * its last query sees all its keys: row r sees keys up to
 * (keys - queries) + r, and a row that sees none gives 0. No replacement in
 * the reference, whose prompts run one at a time (smollm.py:168-253).
 * A pair of offsets that is not a stretch of the tensors leaves its sequence
 * out (with more than 256 sequences maybe others too) and reports
 * B2A_ERR_DEVICE_BAD_LEN. Supported D: 64, 128, 256.
 */
B2A_API int b2a_prefill_varlen(const void* q, const void* k, const void* v, const void* gate, void* o, float* lse,
                               const int* cu_q, const int* cu_k, int B, int Nq, int Nk, int Hq, int Hkv, int D,
                               const long long* q_strides, const long long* k_strides,
                               const long long* v_strides, const long long* gate_strides,
                               const long long* o_strides, int gate_bf16, float scale, int causal, int out_fp32,
                               void* stream);

/* Bytes of device scratch b2a_decode_paged needs for these sizes. */
B2A_API size_t b2a_decode_paged_workspace_bytes(int B, int Hq, int Hkv, int D);

/*
 * b2a_decode over a paged cache: q and o [B, Hq, D] (strides {batch, head}),
 * pools k_pages and v_pages [n_pages, Hkv, page, D], seqlens [B] int32: keys
 * 0 .. seqlens[b] - 1 are attended, none gives 0. Optional gate as
 * b2a_decode_gated. Slots past a sequence's end may hold anything. A length
 * below 0 or above table_width * page is cut to that range, a block table
 * entry outside the pool reads page 0; both report B2A_ERR_DEVICE_BAD_LEN.
 * page: a multiple of 16. Supported D: 64, 128, 256; Hq / Hkv <= 16.
 */
B2A_API int b2a_decode_paged(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                             long long table_ld, int table_width, const int* seqlens, const void* gate, void* o,
                             int B, int Hq, int Hkv, int n_pages, int page, int D, const long long* q_strides,
                             const long long* k_strides, const long long* v_strides, const long long* gate_strides,
                             const long long* o_strides, int gate_bf16, float scale, int out_fp32, void* workspace,
                             size_t workspace_bytes, void* stream);

/*
 * b2a_qk_norm_rope_append for packed tokens and a paged cache: q [N, Hq, D],
 * k and v [N, Hkv, D] views (strides {token, head}), cu_seqlens [B + 1].
 * Token n of sequence b is at position start + n - cu[b] (start =
 * start_pos_per_batch[b], device, or start_pos). Writes the rotated q to
 * q_out [N, Hq, D] and k, v to the sequence's pages (all bf16, q_out
 * contiguous); k_out / v_out, optional, contiguous [N, Hkv, D] bf16, receive
 * the same k and v packed (what b2a_prefill_varlen reads). seqlens_out [B],
 * optional: start + tokens; must not overlap start_pos_per_batch (refused),
 * which is read while it is written. cos_tab / sin_tab [max_pos, rope_dim] are fp32
 * (tab_fp32 = 1) or of the source type; computed in fp32, rounded once.
 * Tokens whose position or page is out of range are skipped (only k and v, if
 * it is only the page) and report B2A_ERR_DEVICE_BAD_LEN; so does a pair of
 * offsets that is not a stretch of the tokens, whose sequence is left out. Supported D: 64, 128, 256.
 */
B2A_API int b2a_rope_append_paged(const void* q, const void* k, const void* v, const long long* q_strides,
                                  const long long* k_strides, const long long* v_strides, int src_bf16,
                                  const void* q_norm, const void* k_norm, float eps, const void* cos_tab,
                                  const void* sin_tab, int tab_fp32, int max_pos, int rope_dim, void* q_out,
                                  void* k_out, void* v_out, void* k_pages, void* v_pages,
                                  const long long* k_page_strides, const long long* v_page_strides,
                                  const int* block_table, long long table_ld, int table_width, int n_pages,
                                  int page, const int* cu_seqlens, int B, int N, int Hq, int Hkv, int D,
                                  int start_pos, const int* start_pos_per_batch, int* seqlens_out, void* stream);

/*
 * b2a_rope_append_paged into an 8-bit cache: pools of e4m3 values (strides in
 * elements, multiples of 16) and, for each token and KV head, a scale in
 * k_scales / v_scales [n_pages, Hkv, page] fp32 (contiguous slots; strides
 * {page, head} multiples of 4, 16-byte aligned). A row y (k after norm and
 * rotation, v) is stored as e4m3(y r), r = 1 / s and s = max(max|y| / 448, 2^-100)
 * rounded to fp32, from the fp32 values; rows with an infinity or a NaN read back as NaN. k_out / v_out
 * receive the values before that rounding, as bf16.
 */
B2A_API int b2a_rope_append_paged_e4m3(const void* q, const void* k, const void* v, const long long* q_strides,
                                       const long long* k_strides, const long long* v_strides, int src_bf16,
                                       const void* q_norm, const void* k_norm, float eps, const void* cos_tab,
                                       const void* sin_tab, int tab_fp32, int max_pos, int rope_dim, void* q_out,
                                       void* k_out, void* v_out, void* k_pages, void* v_pages,
                                       const long long* k_page_strides, const long long* v_page_strides,
                                       float* k_scales, float* v_scales, const long long* k_scale_strides,
                                       const long long* v_scale_strides, const int* block_table, long long table_ld,
                                       int table_width, int n_pages, int page, const int* cu_seqlens, int B, int N,
                                       int Hq, int Hkv, int D, int start_pos, const int* start_pos_per_batch,
                                       int* seqlens_out, void* stream);

/*
 * b2a_decode_paged over an 8-bit cache as b2a_rope_append_paged_e4m3 writes it:
 * key and value are the e4m3 numbers times their row's scale, not rounded to
 * fewer bits on the way. Scales are positive; of v's, one below 2^-100 counts as
 * 2^-100 and one above 2^90 as NaN. Slots and scales past a sequence's end may hold
 * anything.
 */
B2A_API int b2a_decode_paged_e4m3(const void* q, const void* k_pages, const void* v_pages, const float* k_scales,
                                  const float* v_scales, const long long* k_scale_strides,
                                  const long long* v_scale_strides, const int* block_table, long long table_ld,
                                  int table_width, const int* seqlens, const void* gate, void* o, int B, int Hq,
                                  int Hkv, int n_pages, int page, int D, const long long* q_strides,
                                  const long long* k_strides, const long long* v_strides,
                                  const long long* gate_strides, const long long* o_strides, int gate_bf16,
                                  float scale, int out_fp32, void* workspace, size_t workspace_bytes, void* stream);

/*
 * b2a_decode_paged for sequences that share the first keys of their cache (a
 * system prompt, a document): the same result, the shared keys read once and
 * attended as one matrix product (P rounded to bf16 there, as in b2a_prefill).
 * Group g is the sequences [cu_groups[g], cu_groups[g + 1]) (device int32
 * [n_groups + 1]; NULL with n_groups = 1: all of them); their first
 * prefix_lens[g] keys (device int32 [n_groups]) are the same, whichever
 * sequence's table names them. Sequences in no group, alone in one, or shorter
 * than its prefix attend all their keys by themselves, as every sequence does
 * with the last prefix_lens[g] % 64 of them. A pair of offsets that is not a stretch
 * of the sequences, groups that overlap or a prefix outside 0 .. table_width * page
 * report B2A_ERR_DEVICE_BAD_LEN; nothing is shared then for such a group (the prefix
 * is cut). A call in which the host sees nothing to share (one sequence, a table of no
 * more than 512 keys, too little to save) does not read either array. Where sharing would save reading fewer than least_saved_bytes bytes of
 * keys and values nothing is shared (below 0: 36 MB, and 160 MB if all sequences
 * but one of each group shared all that the table can name, about where it begins
 * to pay). bf16 pools. Workspace: b2a_decode_paged_shared_workspace_bytes.
 */
B2A_API size_t b2a_decode_paged_shared_workspace_bytes(int B, int Hq, int Hkv, int D, int n_groups);
B2A_API int b2a_decode_paged_shared(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                                    long long table_ld, int table_width, const int* seqlens, const int* prefix_lens,
                                    const int* cu_groups, int n_groups, long long least_saved_bytes,
                                    const void* gate, void* o, int B, int Hq, int Hkv, int n_pages, int page, int D,
                                    const long long* q_strides, const long long* k_strides,
                                    const long long* v_strides, const long long* gate_strides,
                                    const long long* o_strides, int gate_bf16, float scale, int out_fp32,
                                    void* workspace, size_t workspace_bytes, void* stream);

/*
 * k and v of a stretch of each sequence out of a paged cache, as packed rows
 * k_out / v_out [N, Hkv, D] bf16 contiguous (what b2a_prefill_varlen reads):
 * row n of sequence b (cu[b] <= n < cu[b + 1]) is the key at position
 * start + n - cu[b]. bf16 pools (k_scales and v_scales NULL) or 8-bit ones (as
 * b2a_rope_append_paged_e4m3; a value is its e4m3 times its scale, rounded to
 * bf16 once). k_out and v_out must not overlap. Rows outside every sequence are not written; a position without
 * a page gives zeros, a pair of offsets that is not a stretch of the N rows
 * leaves its sequence out, and both report B2A_ERR_DEVICE_BAD_LEN.
 * Supported D: 64, 128, 256.
 */
B2A_API int b2a_gather_paged(const void* k_pages, const void* v_pages, const long long* k_page_strides,
                             const long long* v_page_strides, const float* k_scales, const float* v_scales,
                             const long long* k_scale_strides, const long long* v_scale_strides,
                             const int* block_table, long long table_ld, int table_width, int n_pages, int page,
                             const int* cu_seqlens, int B, int N, int Hkv, int D, int start_pos,
                             const int* start_pos_per_batch, void* k_out, void* v_out, void* stream);

/*
 * Penalties for repeated tokens, a bias and a mask on logits [R, V] (fp32, or
 * bf16 with logits_bf16 = 1; row stride ld_logits), before b2a_sample. Row r has
 * the tokens tokens[r, 0 .. lengths[r] - 1] (int32, or int64 with tokens_64 = 1;
 * strides tokens_row and tokens_step; lengths NULL: all L), of which the first
 * prompt_lengths[r] (NULL: none) are its prompt; ids outside 0 .. V - 1 count
 * for nothing. For token v, c = how often it is among those after the prompt:
 *   y = x > 0 ? x / repetition : x * repetition   if v is among all of them
 *   y = y - frequency c - (c > 0 ? presence : 0)
 *   y = y + bias[r, v]                            (bias optional, fp32)
 *   y = -inf  unless bit v % 32 of allowed[r, v / 32] is set (optional, int32)
 * each step rounded in fp32, the result to the logits' type. repetition,
 * frequency, presence: per-row device arrays [R], or NULL for the *_all value
 * (repetition_all above 0). ld_bias / ld_allowed 0: one row for all. out
 * [R, V] (row stride ld_out): the logits themselves, or apart from them, and apart
 * from every other input. A
 * length outside 0 .. L is cut and reports B2A_ERR_DEVICE_BAD_LEN. V, L <= 2^30.
 */
B2A_API int b2a_penalize(const void* logits, long long ld_logits, int logits_bf16, const void* tokens, int tokens_64,
                         long long tokens_row, long long tokens_step, int L, const int* lengths,
                         const int* prompt_lengths, const float* repetition, float repetition_all,
                         const float* frequency, float frequency_all, const float* presence, float presence_all,
                         const float* bias, long long ld_bias, const int* allowed, long long ld_allowed, void* out,
                         long long ld_out, int R, int V, void* stream);

/*
 * The next token of each row of logits [R, V] (fp32, or bf16 with
 * logits_bf16 = 1; row stride ld_logits) from given random numbers: noise
 * [R, V] fp32, independent draws of Exp(1), all above 0 (row stride ld_noise).
 *
 * With m the row's maximum, T its temperature: w_i = exp((x_i - m) / T).
 * Tokens are ranked by logit (descending, lowest index first among equals).
 * Token j is kept iff fewer than top_k tokens rank ahead of it (top_k <= 0:
 * no limit), the weight ahead of it is below top_p of the row's total weight
 * (top_p >= 1: no limit) and w_j >= min_p; the first is always kept. The
 * result is argmax w_i / noise_i over the kept tokens, lowest index on ties:
 * token i with probability w_i / (sum of the kept w). T <= 0 gives argmax x.
 * NaN logits count as -inf; a row without a logit above -inf gives -1.
 * temperature, top_k, top_p, min_p: per-row device arrays [R], or NULL for
 * the *_all value in every row. noise may be NULL: every row is then greedy.
 * Replaces: nothing in the reference, which takes the argmax on the host.
 */
B2A_API int b2a_sample(const void* logits, long long ld_logits, int logits_bf16, const float* noise,
                       long long ld_noise, int R, int V, const float* temperature, float temperature_all,
                       const int* top_k, int top_k_all, const float* top_p, float top_p_all, const float* min_p,
                       float min_p_all, long long* out, void* stream);

/*
 * Read (and optionally clear) the device error word the kernels set on the
 * current device. Synchronises `stream`. *status receives B2A_OK,
 * B2A_ERR_DEVICE_TIMEOUT or B2A_ERR_DEVICE_BAD_LEN.
 */
B2A_API int b2a_get_device_error(int* status, int clear, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B2ATTN_H */
