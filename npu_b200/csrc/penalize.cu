// Penalties for repeated tokens, a bias and a mask on logits [R, V]. For token
// v of a row with the tokens t_0 .. t_{n-1}, of which the first m are its prompt:
//
//   seen  = v is among t_0 .. t_{n-1},  c = how often it is among t_m .. t_{n-1}
//   y = x                                 x the logit, in fp32
//   y = y > 0 ? y / r : y r               if seen
//   y = y - f c - (c > 0 ? a : 0)         f: frequency, a: presence
//   y = y + bias_v;  y = -inf             if v is not allowed
//
// each step rounded by itself in fp32, the result to the logits' type once.
//
// Bound by memory: logits read once and written once. A CTA takes a chunk of
// one row's vocabulary, requests its logits, counts the row's tokens that fall
// into the chunk in shared memory (bit 0: in the prompt, from bit 1 on: the
// count) and applies bias and mask to the registers. The few elements that a
// token names (some 1 %, but a lane in almost every warp) are then done one by
// one in a loop: with the penalties' code in line for each of a lane's elements the
// kernel took twice the instructions. The tokens are read once per chunk, from
// L2 after the first, eight requests at a time.
#include "capi_internal.cuh"
#include "penalize.cuh"

namespace b2a {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct Elements;  // 16 bytes of logits
template <>
struct Elements<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& w, int i) {
    return __uint_as_float(i & 2 ? (i & 1 ? w.w : w.z) : (i & 1 ? w.y : w.x));
  }
  static __device__ __forceinline__ void put(uint4& w, int i, float v) {
    const uint32_t u = __float_as_uint(v);
    if (i == 0) w.x = u;
    if (i == 1) w.y = u;
    if (i == 2) w.z = u;
    if (i == 3) w.w = u;
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
};
template <>
struct Elements<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& w, int i) {
    const uint32_t u = i & 4 ? (i & 2 ? w.w : w.z) : (i & 2 ? w.y : w.x);
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  }
  static __device__ __forceinline__ void put(uint4& w, int i, float v) {
    const uint32_t u = pack_bf16x2(v, v), keep = i & 1 ? 0x0000ffffu : 0xffff0000u;
    if (i >> 1 == 0) w.x = (w.x & keep) | (u & ~keep);
    if (i >> 1 == 1) w.y = (w.y & keep) | (u & ~keep);
    if (i >> 1 == 2) w.z = (w.z & keep) | (u & ~keep);
    if (i >> 1 == 3) w.w = (w.w & keep) | (u & ~keep);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                      pack_bf16x2(x[6], x[7]));
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};

// Counters of a chunk, two to a word while a row has few enough tokens.
constexpr int kNarrowTokens = 32767;
template <bool WIDE>
struct Counters {
  static constexpr int BITS = WIDE ? 32 : 16;
  static __device__ __forceinline__ void prompt(unsigned* c, int i) {
    atomicOr(c + (WIDE ? i : i >> 1), 1u << (WIDE ? 0 : 16 * (i & 1)));
  }
  static __device__ __forceinline__ void made(unsigned* c, int i) {
    atomicAdd(c + (WIDE ? i : i >> 1), 2u << (WIDE ? 0 : 16 * (i & 1)));
  }
  static __device__ __forceinline__ unsigned get(const unsigned* c, int i) {
    return WIDE ? c[i] : reinterpret_cast<const uint16_t*>(c)[i];
  }
  // Which of the N counters from number i on (a multiple of N) are not 0.
  template <int N>
  static __device__ __forceinline__ unsigned used(const unsigned* c, int i) {
    constexpr int WORDS = N * BITS / 32;
    uint32_t w[WORDS];
    if constexpr (WORDS == 2) {
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(c + i * BITS / 32);
    } else {
#pragma unroll
      for (int k = 0; k < WORDS; k += 4)
        *reinterpret_cast<uint4*>(w + k) = *reinterpret_cast<const uint4*>(c + i * BITS / 32 + k);
    }
    unsigned any = 0, m = 0;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) any |= w[k];
    if (any) {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        if constexpr (WIDE)
          m |= w[k] ? 1u << k : 0u;
        else
          m |= (w[k] & 0xffffu ? 1u << (2 * k) : 0u) | (w[k] >> 16 ? 2u << (2 * k) : 0u);
      }
    }
    return m;
  }
};

// Bits [v, v + 8) of a row's mask of `words` words (those that exist).
__device__ __forceinline__ unsigned mask_bits(const unsigned* row, int v, int words) {
  const int w = v >> 5;
  const unsigned lo = __ldg(row + w);
  const unsigned hi = (v & 31) > 24 && w + 1 < words ? __ldg(row + w + 1) : 0u;
  return __funnelshift_r(lo, hi, v & 31);
}

// N floats from p on, which lies `off` floats past a 16-byte boundary (the same for the whole CTA). Reads no further
// than the 16-byte pieces that hold them.
template <int N>
__device__ __forceinline__ void load_floats(const float* p, int off, float (&b)[N]) {
  const float4* q = reinterpret_cast<const float4*>(p - off);
  float a[N + 4];
#pragma unroll
  for (int k = 0; k < N / 4; ++k) *reinterpret_cast<float4*>(a + 4 * k) = __ldg(q + k);
  if (off == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = a[i];
    return;
  }
  *reinterpret_cast<float4*>(a + N) = __ldg(q + N / 4);
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = off == 1 ? a[i + 1] : (off == 2 ? a[i + 2] : a[i + 3]);
}

// SLOTS: 16-byte pieces of logits per thread.
template <typename T, int SLOTS, bool WIDE>
__global__ void __launch_bounds__(kThreads) penalize_kernel(const __grid_constant__ PenalizeParams p, int chunks) {
  using E = Elements<T>;
  using Count = Counters<WIDE>;
  constexpr int CHUNK = kThreads * SLOTS * E::N;
  __shared__ __align__(16) unsigned counts[CHUNK * Count::BITS / 32];
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x / chunks;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld_logits;
  T* y = static_cast<T*>(p.out) + row * p.ld_out;
  // The chunk starts on a 16-byte boundary of the row, at or before element 0.
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
  const int v0 = (int)(blockIdx.x % chunks) * CHUNK - shift;
  uint4 raw[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int v = v0 + (s * kThreads + threadIdx.x) * E::N;
    raw[s] = make_uint4(0u, 0u, 0u, 0u);
    if (v >= 0 && v + E::N <= p.V) raw[s] = *reinterpret_cast<const uint4*>(x + v);
  }
  const float rep = p.repetition ? p.repetition[row] : p.repetition_all;
  const float freq = p.frequency ? p.frequency[row] : p.frequency_all;
  const float pres = p.presence ? p.presence[row] : p.presence_all;
  int n = p.tokens ? p.L : 0;
  if (p.tokens && p.lengths) {
    const int given = p.lengths[row];
    n = min(max(given, 0), p.L);
    if (given != n && p.err && threadIdx.x == 0) atomicOr(p.err, kErrBadArgs);
  }
  const bool counted = n > 0 && (rep != 1.f || freq != 0.f || pres != 0.f);
  if (counted) {
    const int prompt = p.prompt_lengths ? p.prompt_lengths[row] : 0;
    for (int i = threadIdx.x; i < CHUNK * Count::BITS / 128; i += kThreads)
      reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
    const long long first = max(v0, 0), past = min((long long)v0 + CHUNK, (long long)p.V);
    constexpr int AHEAD = 8;
    for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < n; i0 += AHEAD * kThreads) {
      long long t[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + k * kThreads;
        t[k] = -1;
        if (i >= n) continue;
        const long long at = row * p.tokens_row + i * p.tokens_step;
        t[k] = p.tokens_64 ? __ldg(static_cast<const long long*>(p.tokens) + at)
                           : (long long)__ldg(static_cast<const int*>(p.tokens) + at);
      }
      if (i0 == (int)threadIdx.x) __syncthreads();  // the counters are 0
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (t[k] < first || t[k] >= past) continue;
        const int c = (int)(t[k] - v0);
        if (i0 + k * kThreads < prompt)
          Count::prompt(counts, c);
        else
          Count::made(counts, c);
      }
    }
    __syncthreads();
  }
  const float* bias = p.bias ? p.bias + row * p.ld_bias : nullptr;
  const int bias_off = (int)((reinterpret_cast<uintptr_t>(bias + v0) >> 2) & 3u);
  const unsigned* allowed = p.allowed ? p.allowed + row * p.ld_allowed : nullptr;
  const int words = (int)((p.V + 31LL) / 32);
  // Token v's logit x with count c.
  auto apply = [&](float x, unsigned c, int v, bool ok) -> float {
    if (c) {
      x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c > 1u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)(c >> 1))), pres);
    }
    if (bias) x = __fadd_rn(x, __ldg(bias + v));
    return ok ? x : -INFINITY;
  };
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int slot = (s * kThreads + threadIdx.x) * E::N;
    const int v = v0 + slot;
    // A piece of the bias that is not wholly in it may not be read at once.
    if (v >= 0 && v + E::N <= p.V && (!bias || (v >= 4 && v + E::N + 4 <= p.V))) {
      const unsigned bits = allowed ? mask_bits(allowed, v, words) : ~0u;
      constexpr unsigned kAll = (1u << E::N) - 1u;
      uint4 out = raw[s];
      if (bias || (bits & kAll) != kAll) {  // else the bits stay as they are (a NaN's too)
        float f[E::N];
#pragma unroll
        for (int i = 0; i < E::N; ++i) f[i] = E::get(raw[s], i);
        if (bias) {
          float b[E::N];
          load_floats(bias + v, bias_off, b);
#pragma unroll
          for (int i = 0; i < E::N; ++i) f[i] = __fadd_rn(f[i], b[i]);
        }
#pragma unroll
        for (int i = 0; i < E::N; ++i) f[i] = (bits >> i) & 1u ? f[i] : -INFINITY;
        out = E::put(f);
      }
      if (counted) {
#pragma unroll 1
        for (unsigned m = Count::template used<E::N>(counts, slot); m; m &= m - 1u) {
          const int i = __ffs(m) - 1;
          E::put(out, i, apply(E::get(raw[s], i), Count::get(counts, slot + i), v + i, (bits >> i) & 1u));
        }
      }
      if (together) {
        *reinterpret_cast<uint4*>(y + v) = out;
      } else {
        const T* values = reinterpret_cast<const T*>(&out);
#pragma unroll
        for (int i = 0; i < E::N; ++i) y[v + i] = values[i];
      }
    } else {  // the row's first and last pieces, element by element
#pragma unroll 1
      for (int i = 0; i < E::N; ++i) {
        const int w = v + i;
        if (w < 0 || w >= p.V) continue;
        const bool ok = !allowed || ((__ldg(allowed + (w >> 5)) >> (w & 31)) & 1u);
        const unsigned c = counted ? Count::get(counts, slot + i) : 0u;
        if (c || bias || !ok)
          E::store(y + w, apply(E::load(x + w), c, w, ok));
        else
          y[w] = x[w];
      }
    }
  }
}

template <typename T, int SLOTS, bool WIDE>
int launch_slots(const PenalizeParams& p, cudaStream_t st) {
  constexpr int N = Elements<T>::N, CHUNK = kThreads * SLOTS * N;
  // One more than V / CHUNK would need: a row may start up to N - 1 elements into a 16-byte piece.
  const long long chunks = ((long long)p.V + N - 1 + CHUNK - 1) / CHUNK, n = chunks * p.R;
  if (n > 0x7fffffffLL) return -2;
  return launch_dependent(penalize_kernel<T, SLOTS, WIDE>, dim3((unsigned)n), kThreads, 0, st, 0, p, (int)chunks) ==
                 cudaSuccess
             ? 0
             : -1;
}

template <typename T>
int launch_t(const PenalizeParams& p, cudaStream_t st) {
  if (p.L > kNarrowTokens) return launch_slots<T, 2, true>(p, st);
  // Few rows: small chunks, so that a row is spread over more CTAs.
  const long long pieces = (long long)p.R * ((p.V + Elements<T>::N - 1) / Elements<T>::N);
  return pieces > 148LL * 8 * kThreads ? launch_slots<T, 4, false>(p, st) : launch_slots<T, 1, false>(p, st);
}

}  // namespace

int launch_penalize(const PenalizeParams& p, cudaStream_t st) {
  return p.logits_bf16 ? launch_t<__nv_bfloat16>(p, st) : launch_t<float>(p, st);
}

}  // namespace b2a
