// k and v of a stretch of each sequence, out of the pages and into packed bf16
// rows (what attention over packed prompts reads): row n of the outputs, of
// sequence b (cu[b] <= n < cu[b + 1]), is position p = start[b] + n - cu[b],
// slot p % page of page table[b][p / page]. Rows of 8-bit pools (paged.cuh) are
// c_i s in fp32, rounded to bf16 once.
//
// Bound by memory: each row is read once and written once. A warp takes one
// token and STEPS x 256 / D of its 2 Hkv rows (k's, then v's), eight elements a
// thread, all loads before the first store.
#include <type_traits>

#include "capi_internal.cuh"
#include "gather_paged.cuh"
#include "paged.cuh"

namespace b2a {

namespace {

constexpr int kWarps = 4;  // tokens of a block

// Two e4m3 values (the low and the high byte of x) as floats: exact, by way of f16.
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t x) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)x));
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(h));
  return r;
}

__device__ __forceinline__ uint32_t scaled(uint32_t x, float s) {
  const float2 v = unpack_e4m3x2(x);
  return pack_bf16x2(v.x * s, v.y * s);
}

template <int D, int STEPS, bool E4M3>
__global__ void __launch_bounds__(32 * kWarps) gather_paged_kernel(const __grid_constant__ GatherPagedParams p) {
  using Cache = std::conditional_t<E4M3, uint8_t, __nv_bfloat16>;
  using Vec = std::conditional_t<E4M3, uint2, uint4>;  // eight elements
  constexpr int LPR = D / 8;      // lanes per row
  constexpr int ROWS = 32 / LPR;  // rows of a warp at a time
  const int lane = threadIdx.x & 31, at = 8 * (lane % LPR);
  const long long n = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);  // token
  grid_dep_wait();
  grid_dep_launch();
  if (blockIdx.x == 0 && blockIdx.y == 0 && p.err)
    for (int b = threadIdx.x; b < p.B; b += 32 * kWarps)
      if (!is_stretch(p.cu_seqlens[b], p.cu_seqlens[b + 1], p.N)) atomicOr(p.err, kErrBadArgs);
  if (n >= p.N) return;
  const int b = find_sequence(p.cu_seqlens, p.B, n);
  const int c0 = p.cu_seqlens[b], c1 = p.cu_seqlens[b + 1];
  if (n < c0 || n >= c1 || !is_stretch(c0, c1, p.N)) return;  // a row outside every sequence
  const long long pos = (long long)(p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (n - c0);
  int page_id = -1;
  unsigned slot = 0;
  if (pos >= 0 && pos < (long long)p.table_width * p.page) {
    const unsigned entry = (unsigned)(pos / (unsigned)p.page);
    slot = (unsigned)(pos - (long long)entry * p.page);
    page_id = p.block_table[b * p.table_ld + entry];
  }
  const bool in_pool = page_id >= 0 && page_id < p.n_pages;
  if (!in_pool && p.err && lane == 0) atomicOr(p.err, kErrBadArgs);

  const Cache* k = static_cast<const Cache*>(p.k_pages) + page_id * p.kps[0] + slot * p.kps[2] + at;
  const Cache* v = static_cast<const Cache*>(p.v_pages) + page_id * p.vps[0] + slot * p.vps[2] + at;
  const int j0 = (int)blockIdx.y * (STEPS * ROWS) + lane / LPR;
  Vec raw[STEPS];
  float scale[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int j = j0 + s * ROWS;
    const bool is_v = j >= p.Hkv;
    const int h = is_v ? j - p.Hkv : j;
    raw[s] = {};  // a token without a page reads as zeros
    scale[s] = 0.f;
    if (j >= 2 * p.Hkv || !in_pool) continue;
    raw[s] = __ldg(reinterpret_cast<const Vec*>(is_v ? v + h * p.vps[1] : k + h * p.kps[1]));
    if constexpr (E4M3)
      scale[s] = __ldg((is_v ? p.v_scales + page_id * p.vss[0] + h * p.vss[1]
                             : p.k_scales + page_id * p.kss[0] + h * p.kss[1]) + slot);
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int j = j0 + s * ROWS;
    if (j >= 2 * p.Hkv) continue;
    const bool is_v = j >= p.Hkv;
    __nv_bfloat16* dst = (is_v ? p.v_out : p.k_out) + (n * p.Hkv + (is_v ? j - p.Hkv : j)) * D + at;
    uint4 w;
    if constexpr (E4M3)
      w = make_uint4(scaled(raw[s].x, scale[s]), scaled(raw[s].x >> 16, scale[s]), scaled(raw[s].y, scale[s]),
                     scaled(raw[s].y >> 16, scale[s]));
    else
      w = raw[s];
    *reinterpret_cast<uint4*>(dst) = w;
  }
}

template <int D, bool E4M3>
int launch_t(const GatherPagedParams& p, cudaStream_t st) {
  constexpr int STEPS = 4, ROWS = 32 / (D / 8);
  const long long blocks = (p.N + kWarps - 1) / kWarps;
  const long long chunks = (2LL * p.Hkv + STEPS * ROWS - 1) / (STEPS * ROWS);
  if (blocks <= 0 || blocks > 0x7fffffffLL || chunks > 65535) return -2;
  return launch_dependent(gather_paged_kernel<D, STEPS, E4M3>, dim3((unsigned)blocks, (unsigned)chunks), 32 * kWarps, 0,
                          st, 0, p) == cudaSuccess
             ? 0
             : -1;
}

template <bool E4M3>
int launch_d(int D, const GatherPagedParams& p, cudaStream_t st) {
  switch (D) {
    case 64: return launch_t<64, E4M3>(p, st);
    case 128: return launch_t<128, E4M3>(p, st);
    case 256: return launch_t<256, E4M3>(p, st);
    default: return -3;
  }
}

}  // namespace

int launch_gather_paged(int D, const GatherPagedParams& p, cudaStream_t st) {
  return p.k_scales ? launch_d<true>(D, p, st) : launch_d<false>(D, p, st);
}

}  // namespace b2a
