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
// one row's vocabulary. Bias and mask are applied to its logits in registers
// while its tokens are on their way; the tokens that fall into the chunk are
// counted in shared memory (bit 0: in the prompt, from bit 1 on: the count), and
// the first to come upon an element puts it on a list. The listed elements, some 1 %,
// are done one by one from the logits as they were and stored over the others:
// looking at every element's counter instead took most of the kernel's
// instructions (256 rows of 131071, 4096 tokens: 75 us). The tokens are read once
// per chunk, from L2 after the first, eight requests at a time.
//
// Measured on one B200 (device time): 256 rows of 131071 bf16 logits, up to 4096
// tokens each, a bias for all and a mask for each: 61 us, 2.3 TB/s (0.36 of the
// measured copy rate; without bias and mask 44, without tokens too 31): instructions,
// 60 % of the issue slots, and the round trips of a chunk one after another (settings,
// tokens, counts, listed logits). 128 rows of fp32: 37 us, 3.7 TB/s (0.57). One row of
// 49152: 3.3 us, one launch.
#include "capi_internal.cuh"
#include "penalize.cuh"

namespace b2a {

namespace {

constexpr int kThreads = 256;
constexpr int kMostRows = 65535;  // of a launch

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
  // -inf wherever the element's bit is not set.
  static __device__ __forceinline__ void keep(uint4& w, unsigned bits) {
    if (!(bits & 1u)) w.x = 0xff800000u;
    if (!(bits & 2u)) w.y = 0xff800000u;
    if (!(bits & 4u)) w.z = 0xff800000u;
    if (!(bits & 8u)) w.w = 0xff800000u;
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float round(float x) { return x; }
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
  // Bit k of four is moved to the sign of byte k; prmt with bit 3 of a selector set repeats that byte's sign.
  template <int BYTES>
  static __device__ __forceinline__ uint32_t signs(uint32_t x) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(x), "n"(BYTES));
    return r;
  }
  static __device__ __forceinline__ void keep(uint4& w, unsigned bits) {
    const uint32_t lo = (bits & 15u) * 0x10204080u, hi = ((bits >> 4) & 15u) * 0x10204080u;
    auto pick = [](uint32_t x, uint32_t m) { return (x & m) | (0xff80ff80u & ~m); };
    w.x = pick(w.x, signs<0x9988>(lo));
    w.y = pick(w.y, signs<0xbbaa>(lo));
    w.z = pick(w.z, signs<0x9988>(hi));
    w.w = pick(w.w, signs<0xbbaa>(hi));
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
};

// Counters of a chunk as wide as its logits, which take their places once the counts are known: 16 bits hold the
// counts of rows of up to kNarrowTokens tokens.
constexpr int kNarrowTokens = 32767;
template <typename Word>
__device__ __forceinline__ unsigned count_token(Word* counts, int i, bool prompt) {  // the count before
  constexpr bool NARROW = sizeof(Word) == 2;
  const int at = NARROW ? 16 * (i & 1) : 0;
  unsigned* word = reinterpret_cast<unsigned*>(counts) + (NARROW ? i >> 1 : i);
  const unsigned old = prompt ? atomicOr(word, 1u << at) : atomicAdd(word, 2u << at);
  return NARROW ? (old >> at) & 0xffffu : old;
}

// x += the floats OFF places into a.
template <int N, int OFF>
__device__ __forceinline__ void add_floats(const float (&a)[N + 4], float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fadd_rn(x[i], a[i + OFF]);
}

__device__ __forceinline__ float4 zero4() { return make_float4(0.f, 0.f, 0.f, 0.f); }

// SLOTS: 16-byte pieces of logits per thread (256 threads of 4, four CTAs an SM: at 256 rows of 131071 bf16 63 us, with
// threads or pieces twice as many 65, with six CTAs and 40 registers 82). Word: a counter.
template <typename T, int SLOTS, typename Word>
__global__ void __launch_bounds__(kThreads, 4) penalize_kernel(const __grid_constant__ PenalizeParams p) {
  using E = Elements<T>;
  constexpr int CHUNK = kThreads * SLOTS * E::N;
  static_assert(CHUNK <= 65536 && sizeof(Word) >= sizeof(T), "list entries, results in the counters' places");
  __shared__ __align__(16) Word counts[CHUNK];
  __shared__ uint16_t list[CHUNK];
  __shared__ int listed;
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.y;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld_logits;
  T* y = static_cast<T*>(p.out) + row * p.ld_out;
  // The chunk starts on a 16-byte boundary of the row, at or before element 0.
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
  const int v0 = (int)blockIdx.x * CHUNK - shift;
  if (v0 >= p.V) return;  // (the last chunk of a row that starts on a boundary)
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
  const int prompt = counted && p.prompt_lengths ? p.prompt_lengths[row] : 0;
  // The row's tokens i0, i0 + kThreads, .. less the chunk's first one: as unsigned numbers below `span` if they are in
  // the chunk.
  constexpr int AHEAD = 8;
  const int first = max(v0, 0);
  const unsigned span = (unsigned)(min((long long)v0 + CHUNK, (long long)p.V) - first);
  const long long step = p.tokens_step * (p.tokens_64 ? 8 : 4) * kThreads;  // bytes
  const char* tokens = static_cast<const char*>(p.tokens) +
                       (row * p.tokens_row + (int)threadIdx.x * p.tokens_step) * (p.tokens_64 ? 8 : 4);
  unsigned t[AHEAD];
  auto request = [&](int i0) {
    const char* at = tokens + i0 / kThreads * step;
    if (p.tokens_64) {
      uint2 w[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        w[k] = make_uint2(0u, ~0u);
        if (i0 + k * kThreads + (int)threadIdx.x < n) w[k] = *reinterpret_cast<const uint2*>(at + k * step);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) t[k] = w[k].y ? ~0u : w[k].x - (unsigned)first;
    } else {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        t[k] = ~0u;
        if (i0 + k * kThreads + (int)threadIdx.x < n)
          t[k] = *reinterpret_cast<const unsigned*>(at + k * step) - (unsigned)first;
      }
    }
  };
  if (counted) {
    request(0);
    for (int i = threadIdx.x; i < (int)(CHUNK * sizeof(Word) / 16); i += kThreads)
      reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (threadIdx.x == 0) listed = 0;
  }
  // Bias and mask: every element.
  const float* bias = p.bias ? p.bias + row * p.ld_bias : nullptr;
  const unsigned* allowed = p.allowed ? p.allowed + row * p.ld_allowed : nullptr;
  const int words = (int)((p.V + 31LL) / 32);
  // Pieces that do not lie wholly in the row (nor those of the bias that hold them) go element by element.
  auto whole = [&](int v) { return v >= (bias ? 4 : 0) && v + E::N + (bias ? 4 : 0) <= p.V; };
  auto is_allowed = [&](int v) { return !allowed || ((allowed[v >> 5] >> (v & 31)) & 1u); };
  unsigned mask[SLOTS];
  const int bias_off = (int)((reinterpret_cast<uintptr_t>(bias + v0) >> 2) & 3u);
  if (allowed) {  // every piece's words requested before the first is used
    unsigned lo[SLOTS], hi[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int v = v0 + (s * kThreads + threadIdx.x) * E::N, w = v >> 5;
      lo[s] = v >= 0 && w < words ? allowed[w] : 0u;
      hi[s] = v >= 0 && (v & 31) > 32 - E::N && w + 1 < words ? allowed[w + 1] : 0u;
    }
    if (!bias) {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        E::keep(raw[s], __funnelshift_r(lo[s], hi[s], (v0 + (int)threadIdx.x * E::N) & 31));
    } else {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) mask[s] = __funnelshift_r(lo[s], hi[s], (v0 + (int)threadIdx.x * E::N) & 31);
    }
  }
  if (bias) {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int v = v0 + (s * kThreads + threadIdx.x) * E::N;
      // The 16-byte pieces that hold these floats.
      const float4* q = reinterpret_cast<const float4*>(bias + v - bias_off);
      float a[E::N + 4], f[E::N];
#pragma unroll
      for (int k = 0; k <= E::N / 4; ++k) *reinterpret_cast<float4*>(a + 4 * k) = whole(v) ? q[k] : zero4();
      E::get(raw[s], f);
      if (bias_off < 2)
        bias_off == 0 ? add_floats<E::N, 0>(a, f) : add_floats<E::N, 1>(a, f);
      else
        bias_off == 2 ? add_floats<E::N, 2>(a, f) : add_floats<E::N, 3>(a, f);
      raw[s] = E::put(f);
      if (allowed) E::keep(raw[s], mask[s]);
    }
  }
  int named = 0;  // elements of the chunk that tokens name
  if (counted) {
    __syncthreads();  // the counters are 0
    for (int i0 = 0; i0 < n; i0 += AHEAD * kThreads) {
      if (i0 > 0) request(i0);
      // One in as many tokens as there are chunks is in this one. The few are found first and then counted in turn, so
      // that a warp runs the counting about twice and not for every k that any of its lanes has one at.
      unsigned hits = 0;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) hits |= t[k] < span ? 1u << k : 0u;
#pragma unroll 1
      for (; hits; hits &= hits - 1u) {
        const int k = __ffs(hits) - 1;
        unsigned at = t[0];
#pragma unroll
        for (int x = 1; x < AHEAD; ++x) at = k == x ? t[x] : at;
        const int c = (int)at + first - v0;
        if (count_token(counts, c, i0 + k * kThreads + (int)threadIdx.x < prompt) == 0)
          list[atomicAdd(&listed, 1)] = (uint16_t)c;
      }
    }
    __syncthreads();
    named = listed;
    for (int e = threadIdx.x; e < named; e += kThreads) {
      const int c = list[e], v = v0 + c;
      const unsigned count = (unsigned)counts[c] >> 1;
      float f = E::load(x + v);
      f = f > 0.f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
      if (count > 0) f = __fsub_rn(__fsub_rn(f, __fmul_rn(freq, (float)count)), pres);
      if (bias) f = __fadd_rn(f, bias[v]);
      if (!is_allowed(v)) f = -INFINITY;
      *reinterpret_cast<T*>(counts + c) = E::round(f);
    }
    __syncthreads();  // the logits have been read (they may be the output), the results are there
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int v = v0 + (s * kThreads + threadIdx.x) * E::N;
    if (whole(v)) {
      if (together) {
        *reinterpret_cast<uint4*>(y + v) = raw[s];
      } else {
        const T* values = reinterpret_cast<const T*>(&raw[s]);
#pragma unroll
        for (int i = 0; i < E::N; ++i) y[v + i] = values[i];
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < E::N; ++i) {
        const int w = v + i;
        if (w < 0 || w >= p.V) continue;
        T value = x[w];
        if (bias) value = E::round(__fadd_rn(E::load(x + w), bias[w]));
        if (!is_allowed(w)) value = E::round(-INFINITY);
        y[w] = value;
      }
    }
  }
  if (named > 0) {
    __syncthreads();  // after the other elements
    for (int e = threadIdx.x; e < named; e += kThreads) y[v0 + list[e]] = *reinterpret_cast<const T*>(counts + list[e]);
  }
}

template <typename T, int SLOTS, typename Word>
int launch_slots(const PenalizeParams& p, cudaStream_t st) {
  constexpr int N = Elements<T>::N, CHUNK = kThreads * SLOTS * N;
  // One more than V / CHUNK would need: a row may start up to N - 1 elements into a 16-byte piece.
  const long long chunks = ((long long)p.V + N - 1 + CHUNK - 1) / CHUNK;
  return launch_dependent(penalize_kernel<T, SLOTS, Word>, dim3((unsigned)chunks, (unsigned)p.R), kThreads, 0, st, 0,
                          p) == cudaSuccess
             ? 0
             : -1;
}

// Few rows: small chunks, so that a row is spread over more CTAs.
template <typename T, typename Word>
int launch_t(const PenalizeParams& p, cudaStream_t st) {
  constexpr int MOST = sizeof(Word) > sizeof(T) ? 2 : 4;
  const long long pieces = (long long)p.R * ((p.V + Elements<T>::N - 1) / Elements<T>::N);
  return pieces > 148LL * 8 * kThreads ? launch_slots<T, MOST, Word>(p, st) : launch_slots<T, 1, Word>(p, st);
}

}  // namespace

int launch_penalize(const PenalizeParams& all, cudaStream_t st) {
  // In pieces that a grid's second dimension holds.
  for (long long r = 0; r < all.R; r += kMostRows) {
    PenalizeParams p = all;
    const int size = p.logits_bf16 ? 2 : 4;
    p.R = (int)(all.R - r < kMostRows ? all.R - r : kMostRows);
    p.logits = static_cast<const char*>(p.logits) + r * p.ld_logits * size;
    p.out = static_cast<char*>(p.out) + r * p.ld_out * size;
    if (p.tokens) p.tokens = static_cast<const char*>(p.tokens) + r * p.tokens_row * (p.tokens_64 ? 8 : 4);
    if (p.lengths) p.lengths += r;
    if (p.prompt_lengths) p.prompt_lengths += r;
    if (p.repetition) p.repetition += r;
    if (p.frequency) p.frequency += r;
    if (p.presence) p.presence += r;
    if (p.bias) p.bias += r * p.ld_bias;
    if (p.allowed) p.allowed += r * p.ld_allowed;
    int rc;
    if (!p.logits_bf16)
      rc = launch_t<float, uint32_t>(p, st);
    else
      rc = p.L <= kNarrowTokens ? launch_t<__nv_bfloat16, uint16_t>(p, st) : launch_t<__nv_bfloat16, uint32_t>(p, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace b2a
