// k and v of a stretch of each sequence, out of the pages and into packed bf16
// rows (what attention over packed prompts reads): row n of the outputs, of
// sequence b (cu[b] <= n < cu[b + 1]), is position p = start[b] + n - cu[b],
// slot p % page of page table[b][p / page]. Rows of 8-bit pools (paged.cuh) are
// c_i s in fp32, rounded to bf16 once.
//
// Bound by memory: each row is read once and written once. A warp takes up to 8
// tokens and all their 2 Hkv rows (k's, then v's): a lane looks up one token's
// sequence, position and page, and the lanes that copy a row get them by shuffle
// (looked up by each warp for one token, that was half of the instructions, and
// 80 % of the issue slots were taken). 16 bytes a load, four loads ahead of the
// first store (eight: slower, they cost registers and with them warps); 8-bit rows
// go out as 32-byte stores (42.2 us to 39.4).
//
// Measured on one B200 (device time): 32 stretches of 100 to 8192 keys, 4 heads of
// 128, pages of 64: 39.4 us from 8 bits, 5.2 TB/s (0.80 of the measured copy rate),
// 48.1 from bf16, 5.6 TB/s (0.87).
#include <type_traits>

#include "capi_internal.cuh"
#include "gather_paged.cuh"
#include "paged.cuh"

namespace b2a {

namespace {

constexpr int kWarps = 4;
constexpr int kMostTokens = 8;  // of a warp
constexpr int kSteps = 4;       // loads of a lane ahead of its stores

// Two e4m3 values (the low and the high byte of x) times s, as bf16. (To floats by way of f16: exact.)
__device__ __forceinline__ uint32_t scaled(uint32_t x, float s) {
  const float2 v = unpack_f16x2(f16_of_e4m3((uint16_t)x));
  return pack_bf16x2(v.x * s, v.y * s);
}

// The sequence that owns token n: the largest b with cu[b] <= n (0 when there is none). Each lane for itself.
__device__ __forceinline__ int find_own_sequence(const int* cu, int B, long long n) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= n)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// per_row: 2^32 / (2 Hkv), rounded up (a warp has fewer than 2^16 rows, for which that divides exactly).
template <int D, bool E4M3>
__global__ void __launch_bounds__(32 * kWarps)
    gather_paged_kernel(const __grid_constant__ GatherPagedParams p, int tokens, unsigned per_row) {
  using Cache = std::conditional_t<E4M3, uint8_t, __nv_bfloat16>;
  constexpr int N = E4M3 ? 16 : 8;  // elements of a load
  constexpr int LPR = D / N;        // lanes per row
  constexpr int ROWS = 32 / LPR;    // rows of a warp at a time
  const int lane = threadIdx.x & 31, at = N * (lane % LPR);
  const long long n0 = ((long long)blockIdx.x * kWarps + (threadIdx.x >> 5)) * tokens;  // the warp's first token
  grid_dep_wait();
  grid_dep_launch();
  if (blockIdx.x == 0 && blockIdx.y == 0 && p.err)
    for (int b = threadIdx.x; b < p.B; b += 32 * kWarps)
      if (!is_stretch(p.cu_seqlens[b], p.cu_seqlens[b + 1], p.N)) atomicOr(p.err, kErrBadArgs);
  if (n0 >= p.N) return;
  // Lane x < tokens: token n0 + x's page (-1: none, -2: a row outside every sequence) and slot.
  int my_page = -2, my_slot = 0;
  if (lane < tokens && n0 + lane < p.N) {
    const long long n = n0 + lane;
    const int b = find_own_sequence(p.cu_seqlens, p.B, n);
    const int c0 = p.cu_seqlens[b], c1 = p.cu_seqlens[b + 1];
    if (n >= c0 && n < c1 && is_stretch(c0, c1, p.N)) {
      const long long pos = (long long)(p.start_pos_arr ? p.start_pos_arr[b] : p.start_pos) + (n - c0);
      my_page = -1;
      if (pos >= 0 && pos < (long long)p.table_width * p.page) {
        const unsigned entry = (unsigned)(pos / (unsigned)p.page);
        my_slot = (int)(pos - (long long)entry * p.page);
        my_page = p.block_table[b * p.table_ld + entry];
        if (my_page < 0 || my_page >= p.n_pages) my_page = -1;
      }
      if (my_page < 0 && p.err) atomicOr(p.err, kErrBadArgs);
    }
  }
  __syncwarp();
  const int per_token = 2 * p.Hkv;
  const int rows = (int)min((long long)tokens, p.N - n0) * per_token;
  for (int r0 = (int)blockIdx.y * (kSteps * ROWS); r0 < rows; r0 += (int)gridDim.y * (kSteps * ROWS)) {
    uint4 raw[kSteps];
    float scale[kSteps];
    __nv_bfloat16* dst[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int r = r0 + s * ROWS + lane / LPR;
      const int t = (int)__umulhi((unsigned)r, per_row), j = r - t * per_token;
      const int page = __shfl_sync(0xffffffffu, my_page, t & 31), slot = __shfl_sync(0xffffffffu, my_slot, t & 31);
      const bool is_v = j >= p.Hkv;
      const int h = is_v ? j - p.Hkv : j;
      raw[s] = make_uint4(0u, 0u, 0u, 0u);  // a token without a page reads as zeros
      scale[s] = 0.f;
      dst[s] = nullptr;
      if (r >= rows || page == -2) continue;
      dst[s] = (is_v ? p.v_out : p.k_out) + ((n0 + t) * p.Hkv + h) * D + at;
      if (page < 0) continue;
      const long long* ps = is_v ? p.vps : p.kps;
      const Cache* src = static_cast<const Cache*>(is_v ? p.v_pages : p.k_pages) + page * ps[0] + h * ps[1] +
                         slot * ps[2] + at;
      raw[s] = *reinterpret_cast<const uint4*>(src);
      if constexpr (E4M3) {
        const long long* ss = is_v ? p.vss : p.kss;
        scale[s] = (is_v ? p.v_scales : p.k_scales)[page * ss[0] + h * ss[1] + slot];
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (!dst[s]) continue;
      if constexpr (E4M3) {
        const uint32_t w[4] = {raw[s].x, raw[s].y, raw[s].z, raw[s].w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[2 * i] = scaled(w[i], scale[s]);
          o[2 * i + 1] = scaled(w[i] >> 16, scale[s]);
        }
        if (p.out_v8) {  // whole 32-byte sectors
          st_global_v8(dst[s], o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]);
        } else {
          uint4* to = reinterpret_cast<uint4*>(dst[s]);
          to[0] = make_uint4(o[0], o[1], o[2], o[3]);
          to[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      } else {
        *reinterpret_cast<uint4*>(dst[s]) = raw[s];
      }
    }
  }
}

template <int D, bool E4M3>
int launch_t(const GatherPagedParams& p, cudaStream_t st) {
  constexpr int ROWS = 32 / (D / (E4M3 ? 16 : 8));
  // Few tokens are spread over more warps; one token's rows over several once a warp has no more than one.
  int tokens = kMostTokens;
  while (tokens > 1 && p.N / tokens < 148 * 16) tokens /= 2;
  const long long warps = (p.N + tokens - 1) / tokens, blocks = (warps + kWarps - 1) / kWarps;
  const long long rounds = (2LL * p.Hkv * tokens + kSteps * ROWS - 1) / (kSteps * ROWS);
  const long long split = tokens == 1 ? (rounds < 16 ? rounds : 16) : 1;
  if (blocks <= 0 || blocks > 0x7fffffffLL || 2LL * p.Hkv * tokens >= 65536) return -2;
  const unsigned per_row = (unsigned)(((1ull << 32) + 2ull * p.Hkv - 1) / (2ull * p.Hkv));
  return launch_dependent(gather_paged_kernel<D, E4M3>, dim3((unsigned)blocks, (unsigned)split), 32 * kWarps, 0, st, 0,
                          p, tokens, per_row) == cudaSuccess
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
