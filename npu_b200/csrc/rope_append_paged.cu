// Attention prologue over packed tokens and a paged cache
// (rope_append_paged.cuh).
//
// For token n of sequence b (cu[b] <= n < cu[b + 1]) at position
// p = start[b] + n - cu[b], with every head x of q and k:
//   y = x * rsqrt(mean(x^2) + eps) * w          (when a norm weight is given)
//   z_i = y_i cos_p,i - y_{i + r/2} sin_p,i     (i < r/2; r = rope_dim)
//   z_i = y_i cos_p,i + y_{i - r/2} sin_p,i     (r/2 <= i < r), z_i = y_i after
// q goes to q_out[n], k and v to slot p % page of page table[b][p / page].
// Everything is computed in fp32 and rounded to bf16 once, at the store (the
// attention kernels read bf16); products and sums are separate roundings, so
// fp32 sources give the same bits as the dense-cache kernel.
//
// Bound by memory: each source element is read once, each output element
// written once. D / 8 threads share one head's row, 8 elements (16 or 32
// bytes) each; a norm's sum of squares and the rotate-half partner are
// shuffles inside those lanes.
#include "rope_append_paged.cuh"

namespace b2a {

namespace {

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = a.z;
  x[3] = a.w;
  x[4] = b.x;
  x[5] = b.y;
  x[6] = b.z;
  x[7] = b.w;
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint4 v;
  v.x = pack_bf16x2(x[0], x[1]);
  v.y = pack_bf16x2(x[2], x[3]);
  v.z = pack_bf16x2(x[4], x[5]);
  v.w = pack_bf16x2(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = v;
}

// The sequence that owns token n: the largest b with cu[b] <= n (0 when there
// is none), by a search that narrows 32-fold per step. Warp-collective.
__device__ __forceinline__ int find_sequence(const int* cu, int B, long long n) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = B;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int at = lo + lane * step;
    const bool before = lane * step < len && (lane == 0 || cu[at] <= n);
    const unsigned m = __ballot_sync(0xffffffffu, before);
    const int hit = 31 - __clz(m);
    len = min(step, len - hit * step);
    lo += hit * step;
  }
  return lo;
}

template <typename Src, int D>
__global__ void __launch_bounds__(256) rope_append_paged_kernel(const RopeAppendPagedParams p) {
  constexpr int TPR = D / 8;  // threads per row
  constexpr int ROWS = 256 / TPR;
  __shared__ int s_first;
  const int heads = p.Hq + 2 * p.Hkv;
  const long long row0 = (long long)blockIdx.x * ROWS;
  if (threadIdx.x < 32) {
    const int b0 = find_sequence(p.cu_seqlens, p.B, row0 / heads);
    if (threadIdx.x == 0) s_first = b0;
  }
  if (blockIdx.x == 0 && p.seqlens_out)
    for (int b = threadIdx.x; b < p.B; b += 256)
      p.seqlens_out[b] = (p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + p.cu_seqlens[b + 1] - p.cu_seqlens[b];
  __syncthreads();

  const int part = threadIdx.x % TPR;
  const long long row = row0 + threadIdx.x / TPR;
  const long long n = row / heads;
  const int j = (int)(row - n * heads);
  bool active = n < p.N;
  int b = s_first;
  if (active) {
    while (b + 1 < p.B && p.cu_seqlens[b + 1] <= n) ++b;
    active = n >= p.cu_seqlens[b] && n < p.cu_seqlens[b + 1];
  }
  const int kind = j < p.Hq ? 0 : (j < p.Hq + p.Hkv ? 1 : 2);  // q, k, v
  const int h = kind == 0 ? j : (kind == 1 ? j - p.Hq : j - p.Hq - p.Hkv);
  const bool rotated = kind != 2 && p.rope_dim > 0;
  long long pos = 0;
  int page_id = -1;
  if (active) {
    pos = (long long)(p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (n - p.cu_seqlens[b]);
    bool ok = pos >= 0 && !(rotated && pos >= p.max_pos);
    if (ok && kind != 0) {
      const long long e = pos / p.page;
      if (e < p.table_width) page_id = p.block_table[b * p.table_ld + e];
      ok = page_id >= 0 && page_id < p.n_pages;
    }
    if (!ok) {
      if (p.err && part == 0) atomicOr(p.err, kErrBadArgs);
      active = false;
    }
  }

  const int i0 = 8 * part;
  float x[8];
  if (active) {
    const Src* src;
    if (kind == 0)
      src = static_cast<const Src*>(p.q) + n * p.qs[0] + h * p.qs[1];
    else if (kind == 1)
      src = static_cast<const Src*>(p.k) + n * p.ks[0] + h * p.ks[1];
    else
      src = static_cast<const Src*>(p.v) + n * p.vs[0] + h * p.vs[1];
    load8(src + i0, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  }

  if (p.q_norm || p.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __fmaf_rn(x[e], x[e], ss);
#pragma unroll
    for (int off = TPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    const void* wp = kind == 0 ? p.q_norm : (kind == 1 ? p.k_norm : nullptr);
    if (wp) {
      const float rms = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)D), p.norm_eps));
      float w[8];
      load8(static_cast<const Src*>(wp) + i0, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], rms), w[e]);
    }
  }

  if (p.rope_dim > 0) {
    const int xo = p.rope_dim / 16;  // lane distance of a rotate-half pair
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __shfl_xor_sync(0xffffffffu, x[e], xo);
    if (active && rotated && i0 < p.rope_dim) {
      const bool first = (part & xo) == 0;
      float c[8], s[8];
      if (p.tab_fp32) {
        load8(static_cast<const float*>(p.cos) + pos * p.rope_dim + i0, c);
        load8(static_cast<const float*>(p.sin) + pos * p.rope_dim + i0, s);
      } else {
        load8(static_cast<const __nv_bfloat16*>(p.cos) + pos * p.rope_dim + i0, c);
        load8(static_cast<const __nv_bfloat16*>(p.sin) + pos * p.rope_dim + i0, s);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(x[e], c[e]), __fmul_rn(first ? -y[e] : y[e], s[e]));
    }
  }
  if (!active) return;

  if (kind == 0) {
    store8(p.q_out + (n * p.Hq + h) * D + i0, x);
  } else {
    const long long slot = pos % p.page;
    const bool is_k = kind == 1;
    const long long* ps = is_k ? p.kps : p.vps;
    store8((is_k ? p.k_pages : p.v_pages) + page_id * ps[0] + h * ps[1] + slot * ps[2] + i0, x);
    __nv_bfloat16* packed = is_k ? p.k_out : p.v_out;
    if (packed) store8(packed + (n * p.Hkv + h) * D + i0, x);
  }
}

template <typename Src, int D>
int launch_t(const RopeAppendPagedParams& p, cudaStream_t st) {
  constexpr int ROWS = 256 / (D / 8);
  const long long rows = p.N * (p.Hq + 2 * p.Hkv);
  const long long blocks = (rows + ROWS - 1) / ROWS;
  if (blocks <= 0 || blocks > 0x7fffffffLL) return -2;
  rope_append_paged_kernel<Src, D><<<(unsigned)blocks, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

template <typename Src>
int launch_src(int D, const RopeAppendPagedParams& p, cudaStream_t st) {
  switch (D) {
    case 64: return launch_t<Src, 64>(p, st);
    case 128: return launch_t<Src, 128>(p, st);
    case 256: return launch_t<Src, 256>(p, st);
    default: return -3;
  }
}

}  // namespace

int launch_rope_append_paged(int D, const RopeAppendPagedParams& p, cudaStream_t st) {
  return p.src_bf16 ? launch_src<__nv_bfloat16>(D, p, st) : launch_src<float>(D, p, st);
}

}  // namespace b2a
