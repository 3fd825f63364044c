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
//
// A row is spread over a cluster of CTAs. Each copies its slice of the
// logits to shared memory once (one bulk copy), so every later pass reads
// shared memory, and asks for its slice of the noise in L2 at the same time;
// the passes' results are joined through the cluster's shared memory in a
// fixed order. The first race reads the noise once; later ones only for the
// tokens ahead of the pivot.
#include "sample.cuh"

namespace b2a {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kGroup = 8;                      // logits a thread handles at a time
constexpr int kMaxStageBytes = 200 * 1024;     // slices above this stay in global memory

__device__ __forceinline__ float usable(float x) { return x == x ? __fadd_rn(x, 0.f) : -INFINITY; }

// w(x) = exp(z), z = (x - m) / T rounded as the division rounds: the
// quotient's estimate q = d rT is corrected by its remainder. 2^t for
// t = z log2(e) is then corrected for t's rounding and for log2(e)'s (which
// alone would cost |z| 2^-24): about 2^-22 in all.
struct Weight {
  float m, T, rT;
  __device__ __forceinline__ float operator()(float x) const {
    constexpr float kHi = 1.442695040888963f, kLo = 1.925963033e-8f;  // log2(e) in two fp32 terms
    const float d = __fsub_rn(x, m);
    const float q = __fmul_rn(d, rT);
    float z = fmaf(fmaf(-q, T, d), rT, q);
    z = d > -INFINITY ? fmaxf(z, -104.f) : -104.f;  // exp(-104) is below every fp32 number
    const float t = __fmul_rn(z, kHi);
    const float r = fmaf(z, kLo, fmaf(z, kHi, -t));
    const float w = ex2(t);
    return x == m ? 1.f : fmaf(w, r * 0.6931471805599453f, w);
  }
};

// A race entry: ratio (not negative) in the high word, the index's complement
// in the low one, so the larger entry is the larger ratio, then the lower index.
__device__ __forceinline__ unsigned long long entry(float ratio, int i) {
  return ((unsigned long long)__float_as_uint(fmaxf(ratio, 0.f)) << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ int entry_index(unsigned long long e) { return (int)(0xffffffffu - (unsigned)e); }

struct Found {  // 24 bytes, its members 8-byte aligned in pairs
  unsigned long long best;  // race winner
  float x;                  // its logit
  float sum;                // weight
  int count;
  int pad;
};

__device__ __forceinline__ Found join(const Found& a, const Found& b) {
  const bool first = a.best >= b.best;
  return {first ? a.best : b.best, first ? a.x : b.x, a.sum + b.sum, a.count + b.count, 0};
}

__device__ __forceinline__ Found warp_join(Found f, int width) {
  for (int off = width / 2; off > 0; off >>= 1)
    f = join(f, {__shfl_xor_sync(0xffffffffu, f.best, off), __shfl_xor_sync(0xffffffffu, f.x, off),
                 __shfl_xor_sync(0xffffffffu, f.sum, off), __shfl_xor_sync(0xffffffffu, f.count, off), 0});
  return f;
}

struct Shared {
  Found warp[kWarps];
  Found cta[2][kMaxCluster];  // every CTA's value, written by its owner into each CTA of the cluster
  uint64_t full;
  int abort_flag;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Every thread of the cluster gets the joined value; pass counts the calls.
// A CTA writes pass n's slots after the barrier of pass n - 1, when everyone
// has read those of pass n - 2, so two sets of slots are enough.
__device__ __forceinline__ Found cluster_join(Found f, Shared* sh, int rank, int size, int& pass) {
  f = warp_join(f, 32);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh->warp[warp] = f;
  __syncthreads();
  f = warp_join(sh->warp[lane % kWarps], kWarps);
  if (size > 1) {
    Found* slots = sh->cta[pass & 1];
    if (threadIdx.x < size) {
      uint32_t remote;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(slots + rank)), "r"(threadIdx.x));
      asm volatile(
          "st.shared::cluster.u64 [%0], %1;\n\t"
          "st.shared::cluster.v2.f32 [%0 + 8], {%2, %3};\n\t"
          "st.shared::cluster.u32 [%0 + 16], %4;" ::"r"(remote),
          "l"(f.best), "f"(f.x), "f"(f.sum), "r"(f.count)
          : "memory");
    }
    cluster_sync();
    f = warp_join(slots[lane % size], size);
  } else {
    __syncthreads();
  }
  ++pass;
  return f;
}

// kGroup logits as floats from 16-byte aligned memory.
__device__ __forceinline__ void load_group(const float* p, float (&x)[kGroup]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 v = reinterpret_cast<const float4*>(p)[h];
    x[4 * h] = v.x;
    x[4 * h + 1] = v.y;
    x[4 * h + 2] = v.z;
    x[4 * h + 3] = v.w;
  }
}
__device__ __forceinline__ void load_group(const __nv_bfloat16* p, float (&x)[kGroup]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T, bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  constexpr int kPer16 = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t stage_raw[];
  __shared__ Shared sh;
  T* stage = reinterpret_cast<T*>(stage_raw);
  uint32_t rank = 0;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int size = p.cluster;
  // Waited for before the first write into another CTA: it has started.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int r = blockIdx.x / size;
  const int begin = min((int)rank * p.slice, p.V);
  const int n = min(p.slice, p.V - begin);  // this CTA's tokens [begin, begin + n)
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld_logits + begin;
  const float* noise = p.noise + r * p.ld_noise + begin;
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const bool greedy = !(temperature > 0.f) || top_k == 1 || !p.noise;

  // The slice keeps its place within 16 bytes: token i of it sits at
  // stage[shift + i]. What fills whole 16-byte units is copied in bulk, the
  // ragged ends by threads; the rest of the first and last group is -inf.
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const int groups = (shift + n + kGroup - 1) / kGroup;
  if constexpr (STAGED) {
    const int head = min(n, (kPer16 - shift) % kPer16);
    const int units = (n - head) / kPer16;
    if (threadIdx.x == 0) {
      mbar_init(&sh.full, 1);
      sh.abort_flag = 0;
      fence_mbar_init();
      mbar_arrive_expect_tx(&sh.full, units * 16);
      if (units > 0)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         smem_u32(stage + shift + head)),
                     "l"(logits + head), "r"(units * 16), "r"(smem_u32(&sh.full))
                     : "memory");
      if (!greedy) {
        const uintptr_t lo = (reinterpret_cast<uintptr_t>(noise) + 15) & ~(uintptr_t)15;
        const uintptr_t hi = reinterpret_cast<uintptr_t>(noise + n) & ~(uintptr_t)15;
        if (hi > lo)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(lo), "r"((unsigned)(hi - lo)) : "memory");
      }
    }
    const int tail = head + units * kPer16;
    for (int i = threadIdx.x; i < groups * kGroup; i += kThreads) {
      const int token = i - shift;
      if (token < 0 || token >= n)
        stage[i] = T(-INFINITY);
      else if (token < head || token >= tail)
        stage[i] = logits[token];
      else
        i += ((tail + shift - 1 - i) / kThreads) * kThreads;  // the bulk copy's part
    }
    __syncthreads();
    if (!mbar_wait_limit(&sh.full, 0, &sh.abort_flag, p.err, kWaitLimitCycles)) mbar_wait_quiet(&sh.full, 0);
  }
  // Group g holds tokens [g kGroup - shift, +kGroup) of the slice.
  auto load = [&](int g, float (&x)[kGroup]) {
    const int at = g * kGroup - shift;
    if constexpr (STAGED) {
      load_group(stage + g * kGroup, x);
    } else if (at >= 0 && at + kGroup <= n) {
      load_group(logits + at, x);
    } else {
#pragma unroll
      for (int e = 0; e < kGroup; ++e) x[e] = at + e >= 0 && at + e < n ? to_float(logits[at + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kGroup; ++e) x[e] = usable(x[e]);
  };

  // Maximum, and its lowest index.
  int pass = 0;
  float mx = -INFINITY;
  int mi = n;
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    float x[kGroup];
    load(g, x);
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (x[e] > mx) mx = x[e], mi = g * kGroup - shift + e;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const unsigned bits = __float_as_uint(mx);
  const unsigned ordered = (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  Found f = cluster_join({((unsigned long long)ordered << 32) | (0xffffffffu - (unsigned)(begin + mi)), mx, 0.f, 0, 0},
                         &sh, rank, size, pass);
  const float m = f.x;
  if (m == -INFINITY || greedy) {
    if (rank == 0 && threadIdx.x == 0) p.out[r] = m == -INFINITY ? -1 : entry_index(f.best);
    return;
  }

  // The race over all tokens, and the total weight.
  const Weight weight{m, temperature, __frcp_rn(temperature)};
  const bool whole16 = (reinterpret_cast<uintptr_t>(noise - shift) & 15) == 0;
  float best = -1.f, best_x = 0.f, total = 0.f;
  int best_i = 0;
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    const int at = g * kGroup - shift;
    float x[kGroup], e[kGroup];
    if (whole16 && at >= 0 && at + kGroup <= n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(noise + at) + h);
        e[4 * h] = v.x;
        e[4 * h + 1] = v.y;
        e[4 * h + 2] = v.z;
        e[4 * h + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) e[i] = at + i >= 0 && at + i < n ? __ldg(noise + at + i) : 1.f;
    }
    load(g, x);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const float w = weight(x[i]);
      const float ratio = __fdividef(w, e[i]);
      total += w;
      if (ratio > best && x[i] > -INFINITY) best = ratio, best_x = x[i], best_i = at + i;
    }
  }
  f = cluster_join({best >= 0.f ? entry(best, begin + best_i) : 0, best_x, total, 0, 0}, &sh, rank, size, pass);
  if (top_k > 0 || top_p < 1.f || min_p > 0.f) {
    const float mass = top_p < 1.f ? top_p * f.sum : INFINITY;
    while (true) {
      const float xj = f.x;
      const int j = entry_index(f.best);
      Found a{0, 0.f, 0.f, 0, 0};
      for (int g = threadIdx.x; g < groups; g += kThreads) {
        const int at = g * kGroup - shift;
        float x[kGroup];
        load(g, x);
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          if (x[i] >= xj && (x[i] > xj || begin + at + i < j)) {
            const float w = weight(x[i]);
            a = join(a, {entry(__fdividef(w, __ldg(noise + at + i)), begin + at + i), x[i], w, 1, 0});
          }
      }
      a = cluster_join(a, &sh, rank, size, pass);
      const bool kept = (top_k <= 0 || a.count < top_k) && a.sum < mass && weight(xj) >= min_p;
      if (kept || a.count == 0) break;
      f = a;
    }
  }
  if (rank == 0 && threadIdx.x == 0) p.out[r] = entry_index(f.best);
}

template <typename T, bool STAGED>
int launch_t(const SampleParams& p, size_t smem, cudaStream_t st) {
  if (smem > 48 * 1024 && cudaFuncSetAttribute(sample_kernel<T, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)smem) != cudaSuccess)
    return -1;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.R * p.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sample_kernel<T, STAGED>, p) != cudaSuccess) return -1;
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

template <typename T>
int launch_type(const SampleParams& p, cudaStream_t st) {
  const size_t smem = ((size_t)p.slice + 2 * kGroup) * sizeof(T);
  return smem <= kMaxStageBytes ? launch_t<T, true>(p, smem, st) : launch_t<T, false>(p, 0, st);
}

}  // namespace

int launch_sample(SampleParams p, cudaStream_t st) {
  // CTAs per row: enough that a slice is at most 16384 tokens, and with few
  // rows enough to use the SMs while a slice keeps 2048 tokens.
  p.cluster = 1;
  while (p.cluster < kMaxCluster &&
         (p.V > 16384 * p.cluster || ((long long)p.R * p.cluster < 148 && p.V > 2048 * p.cluster)))
    p.cluster *= 2;
  if ((long long)p.R * p.cluster > 0x7fffffffLL) return -2;
  p.slice = ((p.V + p.cluster - 1) / p.cluster + kGroup - 1) / kGroup * kGroup;
  return p.logits_bf16 ? launch_type<__nv_bfloat16>(p, st) : launch_type<float>(p, st);
}

}  // namespace b2a
