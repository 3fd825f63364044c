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
// shared memory, and asks for its slice of the noise in L2 at the same time if
// all of it is wanted; the passes' results are joined through the cluster's
// shared memory in a fixed order. The first race reads the noise whole, or
// only for tokens above a cut where min_p or top_k gives one; later ones only
// for the tokens ahead of the pivot.
//
// Bound by latency: with filters that of the passes (a join is 1 us, a tenth of
// it for the block to agree that no wait ran out), without them that of the
// loads (74 rows are resident, and a row's slice is asked for when its cluster
// starts). Measured on one B200 (device time, 8 draws of the inputs), 256 rows
// of 131071 bf16 logits: greedy 20 us (3.3 TB/s, half of the measured copy
// rate), unfiltered 49 us (4.1 TB/s of logits and noise), min_p 0.05 29 us,
// top_k 50 65 to 69, top_p 0.9 82 to 95, each row its own of such settings 60
// to 73; one row of 49152 fp32 logits: greedy 2.6 us, unfiltered 4.3, top_k 50
// with top_p 0.9 6.4 to 8.9.
#include "capi_internal.cuh"
#include "sample.cuh"

namespace b2a {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kGroup = 8;                      // logits a thread handles at a time
constexpr int kMaskGroups = 64 / kGroup;
constexpr int kMaxStageBytes = 200 * 1024;     // slices above this stay in global memory

// w(x) = exp(z), z = (x - m) / T rounded to fp32. The passes over all tokens
// use quick(), 2^(d log2(e) / T) in one multiplication: |z| 2^-22 off, enough
// for sums and for each thread to pick its candidate; candidates are then
// compared by CUDA's division and exponential (this file is compiled with the
// exact expf). NaN and -inf weigh 0.
struct Weight {
  float m, T, to_log2;  // to_log2: log2(e) / T
  __device__ __forceinline__ float quick(float x) const { return ex2(fmaxf((x - m) * to_log2, -150.f)); }
  __device__ __forceinline__ float operator()(float x) const { return expf(__fdiv_rn(__fsub_rn(x, m), T)); }
};

// What a pass finds, joined over threads, warps and CTAs: the entry with the
// largest score (ordered bits; 0: none), the lowest token among equals, its
// logit, and the pass's weight and count.
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kFailed = 0xffffffffu;  // score of a pass in which a wait ran out: above every logit's
struct alignas(16) Found {
  uint32_t score, token;
  float x, sum;
  int count;
};
__device__ __forceinline__ Found nothing() { return {0, kNone, 0.f, 0.f, 0}; }

__device__ __forceinline__ Found warp_join(Found f) {
  const uint32_t score = __reduce_max_sync(0xffffffffu, f.score);
  const uint32_t token = __reduce_min_sync(0xffffffffu, f.score == score ? f.token : kNone);
  const unsigned who = __ballot_sync(0xffffffffu, f.score == score && f.token == token);
  f.x = __shfl_sync(0xffffffffu, f.x, __ffs(who) - 1);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) f.sum += __shfl_xor_sync(0xffffffffu, f.sum, off);
  f.count = __reduce_add_sync(0xffffffffu, f.count);
  f.score = score;
  f.token = token;
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

// The larger of a and the group's logits (NaN ignored).
__device__ __forceinline__ float group_max(float a, const float (&x)[kGroup]) {
#pragma unroll
  for (int e = 0; e < kGroup; e += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(x[e]), "f"(x[e + 1]));
  return a;
}

// The same from 16-byte aligned memory, bf16 in pairs.
__device__ __forceinline__ float group_max(float a, const float* p) {
  float x[kGroup];
  load_group(p, x);
  return group_max(a, x);
}
__device__ __forceinline__ float group_max(float a, const __nv_bfloat16* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  uint32_t y, z;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(v.x), "r"(v.y));
  asm("max.bf16x2 %0, %1, %2;" : "=r"(z) : "r"(v.z), "r"(v.w));
  asm("max.bf16x2 %0, %0, %1;" : "+r"(y) : "r"(z));
  asm("max.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(__uint_as_float(y << 16)), "f"(__uint_as_float(y & 0xffff0000u)));
  return a;
}

// A thread's candidate in a race.
struct Candidate {
  float ratio = 0.f, x = 0.f;
  int i = -1;
  __device__ __forceinline__ void offer(float w, float e, float xi, int at) {
    const float ratio_i = __fdividef(w, e);
    if (ratio_i > ratio) ratio = ratio_i, x = xi, i = at;
  }
};

struct Shared {
  Found warp[kWarps];
  Found cta[2][kMaxCluster];  // every CTA's value, sent by its owner to each CTA of the cluster
  uint64_t arrived[2];        // counts the bytes of the values
  uint64_t full;
  int abort_flag;
};

// The cluster's CTAs as one: joins of a value from each, in turn.
struct Cluster {
  Shared* sh;
  int rank, size;
  int* err;
  long long limit;  // of a wait, in cycles
  int pass = 0;     // joins so far

  // Address of a shared variable of this CTA in CTA `to`, and a store there
  // that its barrier counts when it lands.
  static __device__ __forceinline__ uint32_t in_cta(const void* p, int to) {
    uint32_t remote;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(to));
    return remote;
  }

  // Every thread of the cluster gets the joined value. Each CTA's first warp
  // sends its value to every CTA, one hop, and each waits for its own copies:
  // no barrier of all the CTAs. A CTA sends for pass n + 2 only after it has
  // everyone's value of pass n + 1, which they sent after reading pass n's:
  // two sets of slots are enough, and after the last pass nothing is under way.
  // A score of kFailed, the CTA's own or a peer's, is what every thread of the
  // CTA gets if a wait ran out; the caller then leaves by way of leave().
  __device__ __forceinline__ Found join(Found f, bool mute = false) {
    f = warp_join(f);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh->warp[warp] = f;
    __syncthreads();
    Found* slots = sh->cta[pass & 1];
    uint64_t* bar = &sh->arrived[pass & 1];
    if (warp == 0) {
      f = warp_join(lane < kWarps ? sh->warp[lane] : nothing());
      if (lane == 0) mbar_arrive_expect_tx(bar, size * 20);
      __syncwarp();
      if (lane < size && !mute) {
        const uint32_t to = in_cta(slots + rank, lane), remote_bar = in_cta(bar, lane);
        asm volatile(
            "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%6];\n\t"
            "st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0 + 16], %5, [%6];" ::"r"(to),
            "r"(f.score), "r"(f.token), "r"(__float_as_uint(f.x)), "r"(__float_as_uint(f.sum)), "r"(f.count),
            "r"(remote_bar)
            : "memory");
      }
      __syncwarp();
    }
    const bool all_here = mbar_wait_limit(bar, (uint32_t)(pass >> 1) & 1u, &sh->abort_flag, err, limit);
    ++pass;
    if (!__syncthreads_and(all_here)) return {kFailed, kNone, 0.f, 0.f, 0};
    return warp_join(lane < size ? slots[lane] : nothing());
  }

  // Way out of a CTA that got kFailed: it sends nothing more, and its shared
  // memory stays until no peer can write to it. Every wait of the peers is
  // bounded too, so each of them gets here or has exited (which counts as
  // arriving); what the last pass still had under way is waited for, with a
  // limit, before.
  __device__ __forceinline__ void leave() {
    mbar_wait_quiet(&sh->arrived[(pass - 1) & 1], (uint32_t)((pass - 1) >> 1) & 1u, limit);
    __syncwarp();
    asm volatile(
        "barrier.cluster.arrive.release.aligned;\n\t"
        "barrier.cluster.wait.acquire.aligned;" ::
            : "memory");
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// MUTE: the cluster's last CTA sends nothing from pass p.mute_pass on, so that
// the others' waits run out (the failure path's test).
template <typename T, bool STAGED, bool MUTE>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(const SampleParams p) {
  constexpr int kPer16 = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t stage_raw[];
  __shared__ Shared sh;
  T* stage = reinterpret_cast<T*>(stage_raw);
  uint32_t rank = 0;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int size = p.cluster;
  if (threadIdx.x == 0) {
    mbar_init(&sh.full, 1);
    mbar_init(&sh.arrived[0], 1);
    mbar_init(&sh.arrived[1], 1);
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  // Waited for before the first join: every CTA has started and its barriers
  // are ready.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  grid_dep_wait();
  grid_dep_launch();
  const int r = blockIdx.x / size;
  const int begin = min((int)rank * p.slice, p.V);
  const int n = min(p.slice, p.V - begin);  // this CTA's tokens [begin, begin + n)
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld_logits + begin;
  const float* noise = p.noise + r * p.ld_noise + begin;
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;  // +inf: finite logits weigh 1
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const bool greedy = !(temperature > 0.f) || top_k == 1 || !p.noise;

  // The slice keeps its place within 16 bytes: token i of it sits at
  // stage[shift + i]. What fills whole 16-byte units is copied in bulk, the
  // ragged ends by threads; the rest of the first and last group is -inf.
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const int groups = (shift + n + kGroup - 1) / kGroup;
  bool staged = true;  // false: the slice's copy did not land in time
  if constexpr (STAGED) {
    const int head = min(n, (kPer16 - shift) % kPer16);
    const int units = (n - head) / kPer16;
    if (threadIdx.x == 0) {
      mbar_arrive_expect_tx(&sh.full, units * 16);
      if (units > 0)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         smem_u32(stage + shift + head)),
                     "l"(logits + head), "r"(units * 16), "r"(smem_u32(&sh.full))
                     : "memory");
      if (!greedy && !(min_p > 0.f) && !(top_k > 0 && top_k <= kThreads)) {  // read whole below
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
    staged = mbar_wait_limit(&sh.full, 0, &sh.abort_flag, p.err, p.wait_limit);
    if (!staged) mbar_wait_quiet(&sh.full, 0, p.wait_limit);
  }
  // Group g holds tokens [g kGroup - shift, +kGroup) of the slice, -inf outside it.
  auto load_raw = [&](int g, float (&x)[kGroup]) {
    const int at = g * kGroup - shift;
    if constexpr (STAGED) {
      load_group(stage + g * kGroup, x);
    } else if (at >= 0 && at + kGroup <= n) {
      load_group(logits + at, x);
    } else {
#pragma unroll
      for (int e = 0; e < kGroup; ++e) x[e] = at + e >= 0 && at + e < n ? to_float(logits[at + e]) : -INFINITY;
    }
  };

  Cluster cluster{&sh, (int)rank, size, p.err, p.wait_limit};
  auto join = [&](const Found& f) -> Found {
    return cluster.join(f, MUTE && (int)rank == size - 1 && cluster.pass >= p.mute_pass);
  };
  float m = -INFINITY;
  // The larger of a and group g's logits.
  auto raise = [&](float a, int g) -> float {
    if constexpr (STAGED) return group_max(a, stage + g * kGroup);
    float x[kGroup];
    load_raw(g, x);
    return group_max(a, x);
  };
  for (int g = threadIdx.x; g < groups; g += kThreads) m = raise(m, g);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const float own_max = __fadd_rn(m, 0.f);  // -0 is +0: equal logits have equal bits in the join
  const unsigned bits = __float_as_uint(own_max);
  // (The first join of every path passes it on, and with it that a copy failed.)
  const unsigned ordered = !staged ? kFailed : ((bits & 0x80000000u) ? ~bits : bits | 0x80000000u);
  // The row's answer where a wait ran out.
  auto give_up = [&] {
    if (rank == 0 && threadIdx.x == 0) p.out[r] = -1;
    cluster.leave();
  };
  // The lowest index of the maximum, -1 if that is -inf; kFailed as score if a
  // wait ran out.
  auto first_maximum = [&]() -> Found {
    Found f{ordered, kNone, own_max, 0.f, 0};
#pragma unroll 1
    for (int g = threadIdx.x; g < groups && own_max > -INFINITY && f.token == kNone; g += kThreads) {
      if (raise(-INFINITY, g) < own_max) continue;
      float x[kGroup];
      load_raw(g, x);
#pragma unroll
      for (int e = kGroup - 1; e >= 0; --e)
        if (x[e] == own_max) f.token = begin + g * kGroup - shift + e;
    }
    f = join(f);
    if (f.x == -INFINITY) f.token = kNone;
    return f;
  };
  if (greedy) {
    const Found f = first_maximum();
    if (f.score == kFailed) return give_up();
    if (rank == 0 && threadIdx.x == 0) p.out[r] = (int)f.token;
    return;
  }
  {
    const Found f = join({ordered, kNone, own_max, 0.f, 0});
    if (f.score == kFailed) return give_up();
    m = f.x;
  }
  if (m == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) p.out[r] = -1;
    return;
  }
  // A maximum of +inf: the tokens that have it weigh 1, all others 0.
  const bool infinite = m == INFINITY;
  if (infinite) m = 0.f;
  auto load = [&](int g, float (&x)[kGroup]) {
    load_raw(g, x);
    if (infinite) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e) x[e] = x[e] == INFINITY ? 0.f : -INFINITY;
    }
  };
  const Weight weight{m, temperature, 1.442695040888963f * __frcp_rn(temperature)};
  // A thread's candidate as the entry it joins with.
  auto found = [&](const Candidate& c, float sum, int count) -> Found {
    if (c.i < 0) return {0, kNone, 0.f, sum, count};
    return {__float_as_uint(fmaxf(__fdividef(weight(c.x), __ldg(noise + c.i)), 0.f)), (uint32_t)(begin + c.i), c.x, sum,
            count};
  };

  // Tokens below `cut` are not kept, whatever the race says: they weigh less
  // than min_p (lowered a little for the logarithm's error), or top_k threads
  // of this CTA alone have a logit of at least `cut`. The second bound is
  // bisected on the threads' maxima, down to an eighth of T.
  float cut = -INFINITY;
  if (min_p > 0.f && !infinite) cut = m + temperature * (__logf(min_p) - 1e-4f) - 1e-6f * fabsf(m);
  if (top_k > 0 && top_k <= kThreads && !infinite) {
    float hi = m, lo = m - 32.f * temperature;
    if (__syncthreads_count(own_max >= lo) >= top_k) {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const float mid = 0.5f * (lo + hi);
        (__syncthreads_count(own_max >= mid) >= top_k ? lo : hi) = mid;
      }
      cut = fmaxf(cut, lo);
    }
  }

  // A thread's tokens are taken in rounds of 64 (kMaskGroups groups, one bit
  // each). A slice of one round keeps its mask of tokens that may still be
  // kept, so passes after the first look only at those; a longer one looks at
  // all of them again.
  const int rounds = (groups + kThreads * kMaskGroups - 1) / (kThreads * kMaskGroups);
  auto group_of = [&](int round, int k) { return (round * kMaskGroups + k) * kThreads + (int)threadIdx.x; };
  auto logit = [&](int i) -> float {  // token i of the slice
    float x;
    if constexpr (STAGED)
      x = to_float(stage[shift + i]);
    else
      x = to_float(logits[i]);
    return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x;
  };
  // Offers the tokens in `mask` of a round to the race, four at a time (their
  // noise is requested together), and returns their weight.
  auto race = [&](Candidate& c, int round, uint64_t mask) -> float {
    float sum = 0.f;
#pragma unroll 1
    while (mask) {
      int at[4];
      float e[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int bit = __ffsll((long long)mask) - 1;
        at[h] = bit < 0 ? -1 : group_of(round, bit / kGroup) * kGroup + bit % kGroup - shift;
        mask &= mask - 1;
        e[h] = at[h] >= 0 ? __ldg(noise + at[h]) : 1.f;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float x = at[h] >= 0 ? logit(at[h]) : -INFINITY, w = weight.quick(x);
        sum += w;
        c.offer(w, e[h], x, at[h]);
      }
    }
    return sum;
  };

  // The race over all tokens that may be kept, and the total weight. Without
  // a cut the noise is read whole; with one only for the tokens above it,
  // asked for in L2 as they are found.
  const bool whole16 = (reinterpret_cast<uintptr_t>(noise - shift) & 15) == 0;
  Candidate c;
  float total = 0.f;
  uint64_t mask = ~0ull;
  if (cut > -INFINITY) {
    for (int round = 0; round < rounds; ++round) {
      mask = 0;
#pragma unroll 2
      for (int k = 0; k < kMaskGroups; ++k) {
        const int g = group_of(round, k), at = g * kGroup - shift;
        if (g >= groups) break;
        float x[kGroup];
        load(g, x);
        if (top_p < 1.f) {
#pragma unroll
          for (int i = 0; i < kGroup; ++i) total += weight.quick(x[i]);
        }
        if (group_max(-INFINITY, x) >= cut) {
          unsigned bits = 0;
#pragma unroll
          for (int i = 0; i < kGroup; ++i) bits |= (x[i] >= cut ? 1u : 0u) << i;
          mask |= (uint64_t)bits << (k * kGroup);
          asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + at + __ffs(bits) - 1));
        }
      }
      race(c, round, mask);
    }
  } else {
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
        const float w = weight.quick(x[i]);
        total += w;
        c.offer(w, e[i], x[i], at + i);
      }
    }
  }
  Found f = join(found(c, total, 0));
  if (f.score == kFailed) return give_up();
  const float mass = top_p < 1.f ? top_p * f.sum : INFINITY;
  int last = 0x7fffffff;  // tokens ahead of the pivot before: fewer every time
  while (f.score != 0 && (top_k > 0 || top_p < 1.f || weight(f.x) < min_p)) {
    const float xj = f.x;
    const int j = (int)f.token - begin;
    c = Candidate{};
    float sum = 0.f;
    int count = 0;
    for (int round = 0; round < rounds; ++round) {
      uint64_t ahead = 0;
#pragma unroll 1
      for (int k = 0; k < kMaskGroups; ++k) {
        const int g = group_of(round, k), at = g * kGroup - shift;
        if (g >= groups) break;
        if (rounds == 1 && !(mask >> (k * kGroup) & 0xffu)) continue;
        if (infinite || raise(-INFINITY, g) >= xj) {
          float x[kGroup];
          load(g, x);
          unsigned bits = 0;
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
            bits |= (x[i] > xj || (x[i] == xj && at + i < j) ? 1u : 0u) << i;
          ahead |= (uint64_t)bits << (k * kGroup);
        }
      }
      count += __popcll(ahead);
      sum += race(c, round, ahead);
      mask = ahead;
    }
    const Found a = join(found(c, sum, count));
    if (a.score == kFailed) return give_up();
    const bool kept = (top_k <= 0 || a.count < top_k) && a.sum < mass && weight(xj) >= min_p;
    if (kept || a.count == 0 || a.count >= last) break;
    last = a.count;
    f = a;
  }
  // Without a candidate (min_p above 1, say) the first token is kept all the same.
  if (f.score == 0) {
    f = first_maximum();
    if (f.score == kFailed) return give_up();
  }
  if (rank == 0 && threadIdx.x == 0) p.out[r] = (int)f.token;
}

template <typename T, bool STAGED, bool MUTE = false>
int launch_t(const SampleParams& p, size_t smem, cudaStream_t st) {
  static OncePerDevice once;
  return once.run(
      [] {
        return cudaFuncSetAttribute(sample_kernel<T, STAGED, MUTE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kMaxStageBytes) == cudaSuccess;
      },
      [&] {
        return launch_dependent(sample_kernel<T, STAGED, MUTE>, dim3((unsigned)(p.R * p.cluster)), kThreads, smem, st,
                                p.cluster, p);
      });
}

template <typename T>
int launch_type(const SampleParams& p, cudaStream_t st) {
  const size_t smem = ((size_t)p.slice + 2 * kGroup) * sizeof(T);
  return smem <= kMaxStageBytes ? launch_t<T, true>(p, smem, st) : launch_t<T, false>(p, 0, st);
}

// CTAs per row and tokens per CTA. False if the grid would be too large.
bool plan(SampleParams& p) {
  // CTAs per row: enough that a slice is at most 16384 tokens, and with few
  // rows enough to use the SMs while a slice keeps 2048 tokens.
  p.cluster = 1;
  while (p.cluster < kMaxCluster &&
         (p.V > 16384 * p.cluster || ((long long)p.R * p.cluster < 148 && p.V > 2048 * p.cluster)))
    p.cluster *= 2;
  if ((long long)p.R * p.cluster > 0x7fffffffLL) return false;
  p.slice = ((p.V + p.cluster - 1) / p.cluster + kGroup - 1) / kGroup * kGroup;
  return true;
}

}  // namespace

int launch_sample(SampleParams p, cudaStream_t st) {
  if (!plan(p)) return -2;
  return p.logits_bf16 ? launch_type<__nv_bfloat16>(p, st) : launch_type<float>(p, st);
}

int launch_sample_mute(SampleParams p, cudaStream_t st) {
  if (p.logits_bf16 || !plan(p)) return -2;
  const size_t smem = ((size_t)p.slice + 2 * kGroup) * sizeof(float);
  return smem <= kMaxStageBytes ? launch_t<float, true, true>(p, smem, st) : -2;
}

}  // namespace b2a
