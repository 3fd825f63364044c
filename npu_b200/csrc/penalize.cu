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
// count) and applies everything to the registers. The tokens are read once per
// chunk, from L2 after the first.
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
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
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
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(ws[i] << 16);
      x[2 * i + 1] = __uint_as_float(ws[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                      pack_bf16x2(x[6], x[7]));
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};

// Bits [v, v + 8) of a row's mask of `words` words (those that exist).
__device__ __forceinline__ unsigned mask_bits(const unsigned* row, int v, int words) {
  const int w = v >> 5;
  const unsigned lo = __ldg(row + w);
  const unsigned hi = (v & 31) > 24 && w + 1 < words ? __ldg(row + w + 1) : 0u;
  return __funnelshift_r(lo, hi, v & 31);
}

// SLOTS: 16-byte pieces of logits per thread.
template <typename T, int SLOTS>
__global__ void __launch_bounds__(kThreads) penalize_kernel(const __grid_constant__ PenalizeParams p, int chunks) {
  using E = Elements<T>;
  constexpr int CHUNK = kThreads * SLOTS * E::N;
  __shared__ __align__(16) unsigned counts[CHUNK];
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
    for (int i = threadIdx.x; i < CHUNK / 4; i += kThreads)
      reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
    const int prompt = p.prompt_lengths ? p.prompt_lengths[row] : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const long long at = row * p.tokens_row + i * p.tokens_step;
      const long long t = p.tokens_64 ? static_cast<const long long*>(p.tokens)[at]
                                      : (long long)static_cast<const int*>(p.tokens)[at];
      const long long c = t - v0;
      if (t < 0 || t >= p.V || c < 0 || c >= CHUNK) continue;
      if (i < prompt)
        atomicOr(&counts[c], 1u);
      else
        atomicAdd(&counts[c], 2u);
    }
    __syncthreads();
  }
  const float* bias = p.bias ? p.bias + row * p.ld_bias : nullptr;
  const unsigned* allowed = p.allowed ? p.allowed + row * p.ld_allowed : nullptr;
  const int words = (int)((p.V + 31LL) / 32);
  auto apply = [&](float v, unsigned c, float b, bool ok) -> float {
    if (c) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      if (c > 1u) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)(c >> 1))), pres);
    }
    if (bias) v = __fadd_rn(v, b);
    return ok ? v : -INFINITY;
  };
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int slot = (s * kThreads + threadIdx.x) * E::N;
    const int v = v0 + slot;
    if (v >= 0 && v + E::N <= p.V) {
      unsigned c[E::N] = {};
      if (counted) {
#pragma unroll
        for (int i = 0; i < E::N; i += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(counts + slot + i);
          c[i] = w.x, c[i + 1] = w.y, c[i + 2] = w.z, c[i + 3] = w.w;
        }
      }
      const unsigned bits = allowed ? mask_bits(allowed, v, words) : ~0u;
      unsigned any = 0;
#pragma unroll
      for (int i = 0; i < E::N; ++i) any |= c[i];
      constexpr unsigned kAll = (1u << E::N) - 1u;
      if (any || bias || (bits & kAll) != kAll) {  // else the bits stay as they are (a NaN's too)
        float f[E::N];
        E::get(raw[s], f);
#pragma unroll
        for (int i = 0; i < E::N; ++i) f[i] = apply(f[i], c[i], bias ? __ldg(bias + v + i) : 0.f, (bits >> i) & 1u);
        raw[s] = E::put(f);
      }
      if (together) {
        *reinterpret_cast<uint4*>(y + v) = raw[s];
      } else {
        const T* values = reinterpret_cast<const T*>(&raw[s]);
#pragma unroll
        for (int i = 0; i < E::N; ++i) y[v + i] = values[i];
      }
    } else {  // the row's first and last piece, element by element
      for (int i = 0; i < E::N; ++i) {
        const int w = v + i;
        if (w < 0 || w >= p.V) continue;
        const bool ok = !allowed || ((__ldg(allowed + (w >> 5)) >> (w & 31)) & 1u);
        const unsigned c = counted ? counts[slot + i] : 0u;
        if (c || bias || !ok)
          E::store(y + w, apply(E::load(x + w), c, bias ? __ldg(bias + w) : 0.f, ok));
        else
          y[w] = x[w];
      }
    }
  }
}

template <typename T, int SLOTS>
int launch_slots(const PenalizeParams& p, cudaStream_t st) {
  constexpr int N = Elements<T>::N, CHUNK = kThreads * SLOTS * N;
  // One more than V / CHUNK would need: a row may start up to N - 1 elements into a 16-byte piece.
  const long long chunks = ((long long)p.V + N - 1 + CHUNK - 1) / CHUNK, n = chunks * p.R;
  if (n > 0x7fffffffLL) return -2;
  return launch_dependent(penalize_kernel<T, SLOTS>, dim3((unsigned)n), kThreads, 0, st, 0, p, (int)chunks) ==
                 cudaSuccess
             ? 0
             : -1;
}

template <typename T>
int launch_t(const PenalizeParams& p, cudaStream_t st) {
  // Few rows: small chunks, so that a row is spread over more CTAs.
  const long long pieces = (long long)p.R * ((p.V + Elements<T>::N - 1) / Elements<T>::N);
  return pieces > 148LL * 8 * kThreads ? launch_slots<T, 4>(p, st) : launch_slots<T, 1>(p, st);
}

}  // namespace

int launch_penalize(const PenalizeParams& p, cudaStream_t st) {
  return p.logits_bf16 ? launch_t<__nv_bfloat16>(p, st) : launch_t<float>(p, st);
}

}  // namespace b2a
