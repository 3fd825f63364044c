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
// STEPS rows per thread of one token, its loads issued before the token's
// sequence, position and page are looked up, so the two latencies overlap;
// the tables are read once per warp and reused for its heads.
//
// Measured on one B200 (device time): 10209 prompt tokens, 16 / 2 heads of 256
// with norms and 64 turned lanes: 45 us, 5.0 TB/s (0.76 of the measured copy
// rate; issue slots at 64 % are the next bound), from fp32 sources 58 us, 5.9
// TB/s (0.90); 64 single tokens, 32 / 4 heads of 128: 3.0 us, one launch.
#include "capi_internal.cuh"
#include "rope_append_paged.cuh"

namespace b2a {

namespace {

// Four elements as loaded, and as two pairs of floats (the arithmetic below is
// on pairs: one instruction for two).
template <typename Src>
struct Four;
template <>
struct Four<float> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float2 (&x)[2]) const {
    x[0] = make_float2(v.x, v.y);
    x[1] = make_float2(v.z, v.w);
  }
};
template <>
struct Four<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void get(float2 (&x)[2]) const {
    x[0] = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u));
    x[1] = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  }
};

// a b rounded by itself: with its rounding spelled out the product is not
// contracted with the addition that follows.
__device__ __forceinline__ float2 product(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ void store4(__nv_bfloat16* p, const float2 (&x)[2]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0].x, x[0].y), pack_bf16x2(x[1].x, x[1].y));
}

template <typename T>
__device__ __forceinline__ void load4(const void* p, long long at, float2 (&x)[2]) {
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

// Whether offsets c0 and c1 are a stretch of the tokens.
__device__ __forceinline__ bool is_stretch(const RopeAppendPagedParams& p, int c0, int c1) {
  return c0 >= 0 && c1 >= c0 && c1 <= p.N;
}

constexpr int kWarps = 4;  // tokens of a block

// Warp x of block (i, y) takes token i kWarps + x and chunk y of its rows: the
// first q_chunks chunks are of q, the rest of k and v. A chunk is STEPS times
// the 32 / (D / 8) rows a warp holds at a time.
template <typename Src, int D, int STEPS>
__global__ void __launch_bounds__(32 * kWarps)
    rope_append_paged_kernel(const __grid_constant__ RopeAppendPagedParams p, int q_chunks) {
  constexpr int LPR = D / 8;       // lanes per row
  constexpr int ROWS = 32 / LPR;   // rows of a warp at a time
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const long long n = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);  // token
  grid_dep_wait();
  grid_dep_launch();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < p.B; b += 32 * kWarps) {
      const int c0 = p.cu_seqlens[b], c1 = p.cu_seqlens[b + 1];
      const bool good = is_stretch(p, c0, c1);
      if (!good && p.err) atomicOr(p.err, kErrBadArgs);
      if (p.seqlens_out)
        p.seqlens_out[b] = (p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (good ? c1 - c0 : 0);
    }
  if (n >= p.N) return;
  const bool q_rows = (int)blockIdx.y < q_chunks;  // q, else k and v
  // Step s takes row j0 + s ROWS of q, or of k and then v.
  const int j0 = ((int)blockIdx.y - (q_rows ? 0 : q_chunks)) * (STEPS * ROWS) + lane / LPR;
  const int rows = q_rows ? p.Hq : 2 * p.Hkv;

  // This thread's two runs of four elements: o0 and its partner o1.
  const bool turns = 8 * part < p.rope_dim;
  const int o0 = turns ? 4 * part : 8 * part, o1 = turns ? 4 * part + p.rope_dim / 2 : 8 * part + 4;
  Four<Src> raw[STEPS][2];
  {
    const Src* first = static_cast<const Src*>(q_rows ? p.q : p.k) + n * (q_rows ? p.qs[0] : p.ks[0]);
    const Src* v = static_cast<const Src*>(p.v) + n * p.vs[0];
    const long long step = q_rows ? p.qs[1] : p.ks[1];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int j = j0 + s * ROWS;
      const Src* src = first + j * step;
      if (!q_rows && j >= p.Hkv) src = v + (j - p.Hkv) * p.vs[1];
      if (j < rows) {
        raw[s][0].load(src + o0);
        raw[s][1].load(src + o1);
      } else {
        raw[s][0].v = raw[s][1].v = {};
      }
    }
  }

  // The token's sequence, position and page: the same for the whole warp.
  const int b = find_sequence(p.cu_seqlens, p.B, n);
  const int c0 = p.cu_seqlens[b], c1 = p.cu_seqlens[b + 1];
  if (n < c0 || n >= c1 || !is_stretch(p, c0, c1)) return;  // a row outside every sequence
  const long long at = (long long)(p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (n - c0);
  const bool counts = at >= 0 && at <= 0x7fffffff;
  const unsigned pos = counts ? (unsigned)at : 0u;
  const bool in_table = counts && (p.rope_dim == 0 || pos < (unsigned)p.max_pos);
  unsigned slot = 0;
  int page_id = -1;
  if (!q_rows) {
    const unsigned entry = pos / (unsigned)p.page;
    slot = pos - entry * p.page;
    if (counts && entry < (unsigned)p.table_width) page_id = p.block_table[b * p.table_ld + entry];
  }
  const bool in_pool = page_id >= 0 && page_id < p.n_pages;
  if ((!in_table || !(q_rows || in_pool)) && p.err && lane == 0) atomicOr(p.err, kErrBadArgs);

  float2 cos0[2], cos1[2], sin0[2], sin1[2];
  if (turns && in_table) {
    const long long t = (long long)pos * p.rope_dim;
    if (p.tab_fp32) {
      load4<float>(p.cos, t + o0, cos0), load4<float>(p.cos, t + o1, cos1);
      load4<float>(p.sin, t + o0, sin0), load4<float>(p.sin, t + o1, sin1);
    } else {
      load4<__nv_bfloat16>(p.cos, t + o0, cos0), load4<__nv_bfloat16>(p.cos, t + o1, cos1);
      load4<__nv_bfloat16>(p.sin, t + o0, sin0), load4<__nv_bfloat16>(p.sin, t + o1, sin1);
    }
  }
  const void* weights = q_rows ? p.q_norm : p.k_norm;
  float2 w0[2], w1[2];
  if (weights) load4<Src>(weights, o0, w0), load4<Src>(weights, o1, w1);

  // RMSNorm (with a weight) and rotation of one row's two runs.
  auto turn = [&](float2 (&x)[2], float2 (&y)[2], bool is_v) {
    if (weights) {
      const float2 s2 =
          __ffma2_rn(x[0], x[0], __ffma2_rn(x[1], x[1], __ffma2_rn(y[0], y[0], __fmul2_rn(y[1], y[1]))));
      float ss = s2.x + s2.y;
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (!is_v) {
        const float rms = rsqrtf(__fmaf_rn(ss, 1.f / D, p.norm_eps));
        const float2 rms2 = make_float2(rms, rms);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = __fmul2_rn(__fmul2_rn(x[e], rms2), w0[e]);
          y[e] = __fmul2_rn(__fmul2_rn(y[e], rms2), w1[e]);
        }
      }
    }
    if (turns && in_table && !is_v) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 a = x[e], c = y[e];
        x[e] = __fadd2_rn(product(a, cos0[e]), product(make_float2(-c.x, -c.y), sin0[e]));
        y[e] = __fadd2_rn(product(c, cos1[e]), product(a, sin1[e]));
      }
    }
  };

  // A token without a place in the tables or the pool is not written where it
  // would need it.
  if (q_rows) {
    __nv_bfloat16* dst = p.q_out + (n * p.Hq + j0) * D;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      float2 x[2], y[2];
      raw[s][0].get(x);
      raw[s][1].get(y);
      turn(x, y, false);
      if (in_table && j0 + s * ROWS < rows) {
        store4(dst + s * ROWS * D + o0, x);
        store4(dst + s * ROWS * D + o1, y);
      }
    }
  } else {
    __nv_bfloat16* k_dst = p.k_pages + page_id * p.kps[0] + slot * p.kps[2];
    __nv_bfloat16* v_dst = p.v_pages + page_id * p.vps[0] + slot * p.vps[2];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int j = j0 + s * ROWS;
      const bool is_v = j >= p.Hkv;
      const int h = is_v ? j - p.Hkv : j;
      float2 x[2], y[2];
      raw[s][0].get(x);
      raw[s][1].get(y);
      turn(x, y, is_v);
      if (!in_pool || !in_table || j >= rows) continue;
      __nv_bfloat16* dst = is_v ? v_dst + h * p.vps[1] : k_dst + h * p.kps[1];
      store4(dst + o0, x), store4(dst + o1, y);
      __nv_bfloat16* packed = is_v ? p.v_out : p.k_out;
      if (packed) {
        packed += (n * p.Hkv + h) * D;
        store4(packed + o0, x), store4(packed + o1, y);
      }
    }
  }
}

template <typename Src, int D, int STEPS>
int launch_steps(const RopeAppendPagedParams& p, cudaStream_t st) {
  constexpr int ROWS = 32 / (D / 8);
  const long long blocks = (p.N + kWarps - 1) / kWarps;
  const int q_chunks = (p.Hq + STEPS * ROWS - 1) / (STEPS * ROWS);
  const int chunks = q_chunks + (2 * p.Hkv + STEPS * ROWS - 1) / (STEPS * ROWS);
  if (blocks <= 0 || blocks > 0x7fffffffLL || chunks > 65535) return -2;
  return launch_dependent(rope_append_paged_kernel<Src, D, STEPS>, dim3((unsigned)blocks, (unsigned)chunks),
                          32 * kWarps, 0, st, 0, p, q_chunks) == cudaSuccess
             ? 0
             : -1;
}

// Four rows per thread spread a token's lookups over more rows; few tokens get
// one, so that their rows are in more warps at once.
template <typename Src, int D>
int launch_t(const RopeAppendPagedParams& p, cudaStream_t st) {
  const long long row_warps = p.N * ((p.Hq + 2 * p.Hkv) / (32 / (D / 8)) + 1);
  return row_warps >= 148 * 32 ? launch_steps<Src, D, 4>(p, st) : launch_steps<Src, D, 1>(p, st);
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
