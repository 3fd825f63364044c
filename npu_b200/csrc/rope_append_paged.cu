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
// written once. D / 8 threads share one head's row. A thread holds four
// elements and their four rotate-half partners (8 contiguous elements past
// rope_dim), so the rotation needs no exchange between threads; a norm's sum
// of squares is a shuffle reduction over the row's threads. A warp takes
// kSteps rows per thread of one token, its loads issued before the token's
// sequence, position and page are looked up, so the two latencies overlap;
// the tables are read once per warp and reused for its heads.
#include "rope_append_paged.cuh"

namespace b2a {

namespace {

constexpr int kSteps = 4;  // rows a thread handles

// Four elements as loaded, and as floats.
template <typename Src>
struct Four;
template <>
struct Four<float> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
};
template <>
struct Four<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void get(float (&x)[4]) const {
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};

__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}

template <typename T>
__device__ __forceinline__ void load4(const void* p, long long at, float (&x)[4]) {
  Four<T> f;
  f.load(static_cast<const T*>(p) + at);
  f.get(x);
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
__global__ void __launch_bounds__(256) rope_append_paged_kernel(const RopeAppendPagedParams p, int chunks) {
  constexpr int LPR = D / 8;       // lanes per row
  constexpr int ROWS = 32 / LPR;   // rows of a warp at a time
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const int heads = p.Hq + 2 * p.Hkv;
  const long long warp = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (blockIdx.x == 0 && p.seqlens_out)
    for (int b = threadIdx.x; b < p.B; b += 256)
      p.seqlens_out[b] = (p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + p.cu_seqlens[b + 1] - p.cu_seqlens[b];
  const long long n = warp / chunks;  // token
  if (n >= p.N) return;
  const int j0 = (int)(warp - n * chunks) * (kSteps * ROWS) + lane / LPR;  // step k takes row j0 + k ROWS

  // This thread's two runs of four elements: o0 and its partner o1.
  const bool turns = 8 * part < p.rope_dim;
  const int o0 = turns ? 4 * part : 8 * part, o1 = turns ? 4 * part + p.rope_dim / 2 : 8 * part + 4;
  Four<Src> raw[kSteps][2];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int j = j0 + k * ROWS;
    const Src* src;
    if (j < p.Hq)
      src = static_cast<const Src*>(p.q) + n * p.qs[0] + j * p.qs[1];
    else if (j < p.Hq + p.Hkv)
      src = static_cast<const Src*>(p.k) + n * p.ks[0] + (j - p.Hq) * p.ks[1];
    else
      src = static_cast<const Src*>(p.v) + n * p.vs[0] + (j - p.Hq - p.Hkv) * p.vs[1];
    if (j < heads) {
      raw[k][0].load(src + o0);
      raw[k][1].load(src + o1);
    } else {
      raw[k][0].v = raw[k][1].v = {};
    }
  }

  // The token's sequence, position and page: the same for the whole warp.
  const int b = find_sequence(p.cu_seqlens, p.B, n);
  const int c0 = p.cu_seqlens[b], c1 = p.cu_seqlens[b + 1];
  if (n < c0 || n >= c1) return;  // a row outside every sequence
  const long long pos = (long long)(p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (n - c0);
  int page_id = -1;
  long long slot = 0;
  if (pos >= 0) {
    const long long e = pos / p.page;
    slot = pos - e * p.page;
    if (e < p.table_width) page_id = p.block_table[b * p.table_ld + e];
  }
  const bool in_table = pos >= 0 && (p.rope_dim == 0 || pos < p.max_pos);
  const bool in_pool = pos >= 0 && page_id >= 0 && page_id < p.n_pages;
  if ((!in_table || !in_pool) && p.err && lane == 0) atomicOr(p.err, kErrBadArgs);

  float cos0[4], cos1[4], sin0[4], sin1[4];
  if (turns && in_table) {
    const long long at = pos * p.rope_dim;
    if (p.tab_fp32) {
      load4<float>(p.cos, at + o0, cos0), load4<float>(p.cos, at + o1, cos1);
      load4<float>(p.sin, at + o0, sin0), load4<float>(p.sin, at + o1, sin1);
    } else {
      load4<__nv_bfloat16>(p.cos, at + o0, cos0), load4<__nv_bfloat16>(p.cos, at + o1, cos1);
      load4<__nv_bfloat16>(p.sin, at + o0, sin0), load4<__nv_bfloat16>(p.sin, at + o1, sin1);
    }
  }

#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int j = j0 + k * ROWS;
    const bool is_q = j < p.Hq, is_k = !is_q && j < p.Hq + p.Hkv;
    const int h = is_q ? j : (is_k ? j - p.Hq : j - p.Hq - p.Hkv);
    float x[4], y[4];
    raw[k][0].get(x);
    raw[k][1].get(y);
    if (p.q_norm || p.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = __fmaf_rn(x[e], x[e], __fmaf_rn(y[e], y[e], ss));
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      const void* wp = is_q ? p.q_norm : (is_k ? p.k_norm : nullptr);
      if (wp) {
        const float rms = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)D), p.norm_eps));
        float w0[4], w1[4];
        load4<Src>(wp, o0, w0), load4<Src>(wp, o1, w1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = __fmul_rn(__fmul_rn(x[e], rms), w0[e]);
          y[e] = __fmul_rn(__fmul_rn(y[e], rms), w1[e]);
        }
      }
    }
    if ((is_q || is_k) && turns && in_table) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[e], c = y[e];
        x[e] = __fadd_rn(__fmul_rn(a, cos0[e]), __fmul_rn(-c, sin0[e]));
        y[e] = __fadd_rn(__fmul_rn(c, cos1[e]), __fmul_rn(a, sin1[e]));
      }
    }
    if (j >= heads) continue;
    // A token without a place in the tables or the pool is not written where
    // it would need it.
    if (is_q) {
      __nv_bfloat16* dst = p.q_out + (n * p.Hq + h) * D;
      if (in_table) store4(dst + o0, x), store4(dst + o1, y);
    } else if (in_pool && (in_table || !is_k)) {
      const long long* ps = is_k ? p.kps : p.vps;
      __nv_bfloat16* dst = (is_k ? p.k_pages : p.v_pages) + page_id * ps[0] + h * ps[1] + slot * ps[2];
      store4(dst + o0, x), store4(dst + o1, y);
      __nv_bfloat16* packed = is_k ? p.k_out : p.v_out;
      if (packed) {
        packed += (n * p.Hkv + h) * D;
        store4(packed + o0, x), store4(packed + o1, y);
      }
    }
  }
}

template <typename Src, int D>
int launch_t(const RopeAppendPagedParams& p, cudaStream_t st) {
  constexpr int ROWS = 32 / (D / 8);
  const int chunks = (p.Hq + 2 * p.Hkv + kSteps * ROWS - 1) / (kSteps * ROWS);
  const long long blocks = (p.N * chunks + 7) / 8;
  if (blocks <= 0 || blocks > 0x7fffffffLL) return -2;
  rope_append_paged_kernel<Src, D><<<(unsigned)blocks, 256, 0, st>>>(p, chunks);
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
