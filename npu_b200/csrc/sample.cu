// Token sampling with temperature, top-k, top-p and min-p from given random
// numbers, sm_100a.
//
// With x the row's logits (NaN counts as -inf), m their maximum, T the
// temperature: w_i = exp((x_i - m) / T), S = sum w. Tokens are ranked by
// (x descending, index ascending). Token j is kept iff its rank is below
// top_k, the weight ranked ahead of it is below top_p S, and w_j >= min_p;
// rank 0 is always kept. The token is argmax w_i / e_i over the kept ones
// (lowest index on ties), e ~ Exp(1) given per token: the first arrival of
// independent exponential clocks with rates w_i, so token i is drawn with
// probability w_i / sum of the kept w. T <= 0: argmax x.
//
// Nothing is sorted. The kept tokens are a prefix of the ranking, so whether
// the winner j of a race is kept takes one pass: the count and the weight
// ranked ahead of it. If it is not kept, neither is anything ranked behind
// it, and the next race runs among the tokens ahead of j, whose winner the
// same pass has found. A race's winner is a draw by weight, so a rejected one
// takes about half of the unwanted weight with it: few passes are needed.
#include "sample.cuh"

namespace b2a {

namespace {

constexpr int kSampleThreads = 1024;

__device__ __forceinline__ float load_logit(const float* p, long long i) { return p[i]; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p, long long i) { return __bfloat162float(p[i]); }
// NaN counts as -inf, -0 as +0 (equal logits have to have equal bits below).
__device__ __forceinline__ float usable(float x) { return x == x ? __fadd_rn(x, 0.f) : -INFINITY; }

// exp(z) to about 2^-22: 2^t for t = z log2(e), corrected for t's rounding
// and the rounding of log2(e) (which alone would cost |z| 2^-24).
__device__ __forceinline__ float exp_weight(float z) {
  constexpr float kHi = 1.442695040888963f, kLo = 1.925963033e-8f;  // log2(e) in two fp32 terms
  z = fmaxf(z, -104.f);  // exp(-104) is below every fp32 number
  const float t = __fmul_rn(z, kHi);
  const float r = fmaf(z, kLo, fmaf(z, kHi, -t));
  const float w = ex2(t);
  return fmaf(w, r * 0.6931471805599453f, w);
}

__device__ __forceinline__ float weight(float x, float m, float T) {
  return x == m ? 1.f : (x == -INFINITY ? 0.f : exp_weight(__fdiv_rn(__fsub_rn(x, m), T)));
}

// A race entry: ratio (not negative) in the high word, the index's complement
// in the low one, so the larger entry is the larger ratio, then the lower index.
__device__ __forceinline__ unsigned long long entry(float ratio, int i) {
  return ((unsigned long long)__float_as_uint(ratio > 0.f ? ratio : 0.f) << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ int entry_index(unsigned long long e) { return (int)(0xffffffffu - (unsigned)e); }

struct Found {
  unsigned long long best;  // race winner
  float sum;
  int count;
};

__device__ __forceinline__ Found join(const Found& a, const Found& b) {
  return {a.best > b.best ? a.best : b.best, a.sum + b.sum, a.count + b.count};
}

// Every thread gets the block's value, joined in a fixed order.
__device__ __forceinline__ Found block_join(Found f, Found* scratch) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    f = join(f, {__shfl_xor_sync(0xffffffffu, f.best, off), __shfl_xor_sync(0xffffffffu, f.sum, off),
                 __shfl_xor_sync(0xffffffffu, f.count, off)});
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) scratch[warp] = f;
  __syncthreads();
  f = scratch[lane];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    f = join(f, {__shfl_xor_sync(0xffffffffu, f.best, off), __shfl_xor_sync(0xffffffffu, f.sum, off),
                 __shfl_xor_sync(0xffffffffu, f.count, off)});
  return f;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  __shared__ Found scratch[32];
  const int r = blockIdx.x;
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld_logits;
  const float* noise = p.noise + r * p.ld_noise;
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;

  // Maximum, and its lowest index.
  float mx = -INFINITY;
  int mi = p.V;
  for (int i = threadIdx.x; i < p.V; i += kSampleThreads) {
    const float x = usable(load_logit(logits, i));
    if (x > mx) mx = x, mi = i;
  }
  const unsigned bits = __float_as_uint(mx);
  const unsigned ordered = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  const unsigned long long top =
      block_join({((unsigned long long)ordered << 32) | (0xffffffffu - (unsigned)mi), 0.f, 0}, scratch).best;
  const unsigned top_bits = (unsigned)(top >> 32);
  const float m = __uint_as_float((top_bits & 0x80000000u) ? top_bits ^ 0x80000000u : ~top_bits);
  if (m == -INFINITY || !(temperature > 0.f) || !p.noise) {
    if (threadIdx.x == 0) p.out[r] = m == -INFINITY ? -1 : entry_index(top);
    return;
  }

  // The race over all tokens, and the total weight.
  Found f{0, 0.f, 0};
  for (int i = threadIdx.x; i < p.V; i += kSampleThreads) {
    const float x = usable(load_logit(logits, i));
    if (x == -INFINITY) continue;
    const float w = weight(x, m, temperature);
    f = join(f, {entry(__fdiv_rn(w, noise[i]), i), w, 0});
  }
  f = block_join(f, scratch);
  int j = entry_index(f.best);
  if (top_k > 0 || top_p < 1.f || min_p > 0.f) {
    const float mass = top_p < 1.f ? top_p * f.sum : INFINITY;
    while (true) {
      const float xj = usable(load_logit(logits, j));
      f = {0, 0.f, 0};
      for (int i = threadIdx.x; i < p.V; i += kSampleThreads) {
        const float x = usable(load_logit(logits, i));
        if (x > xj || (x == xj && i < j)) {
          const float w = weight(x, m, temperature);
          f = join(f, {entry(__fdiv_rn(w, noise[i]), i), w, 1});
        }
      }
      f = block_join(f, scratch);
      const bool kept = (top_k <= 0 || f.count < top_k) && f.sum < mass && weight(xj, m, temperature) >= min_p;
      if (kept || f.count == 0) break;
      j = entry_index(f.best);
    }
  }
  if (threadIdx.x == 0) p.out[r] = j;
}

}  // namespace

int launch_sample(const SampleParams& p, cudaStream_t st) {
  if (p.logits_bf16)
    sample_kernel<__nv_bfloat16><<<(unsigned)p.R, kSampleThreads, 0, st>>>(p);
  else
    sample_kernel<float><<<(unsigned)p.R, kSampleThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace b2a
