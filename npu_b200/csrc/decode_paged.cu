// Attention of one new token per sequence over a paged KV cache
// [n_pages, Hkv, page, D], bf16 or 8-bit (paged.cuh), sm_100a.
//
//   o_h = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q_h k_j - m),
// over keys j < seqlens[b], key j in slot j % page of page table[b][j / page];
// a sequence without keys gives 0. Query head h uses KV head h / (Hq / Hkv).
//
// Bound by HBM: every key and value of a sequence is read once for the whole
// group of query heads that shares it (8 to 16 flop per byte). One warp
// streams 64-key K / V tiles through a shared-memory ring with TMA, one copy
// per run of keys that lies in one page (box_rows, 16 to 64 keys); four warps
// take 16 keys of a tile each. Both products are computed transposed,
// S^T = K Q^T and O^T = V^T P^T, with mma.sync m16n8k16: the keys (then the
// columns of V) are its 16 rows and the query heads of a group its 8 columns,
// so a group of up to 8 heads wastes no rows and needs half the registers and
// MMAs of the other orientation (groups of 9 to 16 use two column blocks).
// P goes into the second product as two bf16 terms (its
// rounding and what the rounding left), so its relative error is 2^-16
// instead of 2^-8; the extra MMAs hide behind the loads.
//
// Work is split evenly whatever the lengths: the tiles of all (sequence, KV
// head) pairs, one after another, are cut into one equal stretch per resident
// CTA, found on the device from the lengths. A CTA walks its stretch with its
// ring running across pairs; for each
// pair a partial (m, l and O before its division) goes to the workspace, and
// a second, dependent launch joins the partials of a pair. Caches of a few
// tiles (kWholeTiles) are not cut: one CTA per pair, one launch.
//
// Measured on one B200 (device time): 128 sequences of 1024 to 32768 keys,
// 32 / 4 heads of 128, pages of 64: 411 us, 6.58 TB/s (1.01 of the measured
// copy rate); 16 of 100 to 20000, 16 / 2 gated heads of 256, pages of 48: 36 us,
// 4.9 TB/s, 4 us of it the first tile's latency and 4 the joining launch; 48 of
// 30 to 4001, 9 / 3 heads of 64, pages of 16: 13.2 us, of which those two and
// the launch are 7; one of 77 keys: 4.2 us. From an 8-bit cache: the first 218
// us, 6.4 TB/s (0.99; bound by HBM again, once two instructions a pair of values
// did what nine had; 243 to 251 after seconds of it, when the power cap holds the
// clock at 1.6 GHz), with 9 / 3 heads of 64 105 us, 5.1 TB/s (instructions), 16
// gated ones of head dim 256 28 us, 3.2 TB/s (the same latencies, half the
// bytes), groups of 16 heads 132 us where their bytes take 79 (instructions: two
// blocks of columns for each product).
//
// Slots of a page past the sequence's end may hold anything, NaN included:
// their scores are replaced by -inf and their V rows by zeros in shared
// memory before they are used.
#include "capi_internal.cuh"
#include "decode_paged.cuh"
#include "paged.cuh"

namespace b2a {

namespace {

template <int D, int NT, bool E4M3>
struct PagedCfg {
  // Blocks of 16 keys that a warp takes of a tile. 8-bit tiles come twice as
  // fast, and with two blocks a warp has two chains of instructions to run and
  // one maximum to find (128 sequences of 1024 to 32768 keys, 32 / 4 heads of
  // 128: 294 us with one block, 235 with two).
  static constexpr int KB = E4M3 ? 2 : 1;
  static constexpr int TK = 64 * KB;  // keys per tile
  static constexpr int TILE_BYTES = TK * D * (E4M3 ? 1 : 2);  // K or V tile
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int CTAS_PER_SM = decode_paged_ctas_per_sm(D, NT, E4M3);
  static constexpr int STAGES = D == 64 ? (CTAS_PER_SM == 3 ? 4 : 6) : 3;
  static constexpr int Q_ROW = D * 2 + 16;  // bytes; the 16 keep ldmatrix rows apart
  static constexpr int OFF_Q = STAGES * STAGE_BYTES;
  static constexpr int OFF_SCALES = OFF_Q + 2 * 16 * Q_ROW;  // two pairs' query heads; [STAGES][K, V][TK] fp32
  static constexpr int OFF_BAR = OFF_SCALES + (E4M3 ? STAGES * 2 * TK * 4 : 0);
  static constexpr int SMEM_BYTES = OFF_BAR + 1024 + 1024;  // barriers and m, l; alignment slack
  static constexpr int THREADS = 160;  // 4 compute warps + 1 producer warp
  static_assert(4 * 16 * D * 4 <= STAGE_BYTES, "the four warps' outputs are merged in one stage");
  static_assert((SMEM_BYTES + 1024) * CTAS_PER_SM <= 233472, "shared memory budget");
};

struct PagedBars {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t q_full[2];
  uint64_t q_empty[2];
  int abort_flag;
  float m[4][16];
  float l[4][16];
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

// Transpose of an 8x8 matrix of 16-bit elements held as fragments.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The gate of (sequence b, query head h) at columns d .. d + 3.
__device__ __forceinline__ float4 load_gate(const DecodePagedParams& p, int b, int h, int d) {
  const long long i = b * p.g_sb + h * p.g_sh + d;
  if (p.gate_bf16) {
    const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(p.gate) + i;
    if (p.vec4) {
      const uint2 v = *reinterpret_cast<const uint2*>(g);
      return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                         __uint_as_float(v.y & 0xffff0000u));
    }
    return make_float4(__bfloat162float(g[0]), __bfloat162float(g[1]), __bfloat162float(g[2]), __bfloat162float(g[3]));
  }
  const float* g = static_cast<const float*>(p.gate) + i;
  if (p.vec4) return *reinterpret_cast<const float4*>(g);
  return make_float4(g[0], g[1], g[2], g[3]);
}

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// The output at columns d .. d + 3: attention values v, gated and rounded as
// the call asks.
__device__ __forceinline__ void store_output(const DecodePagedParams& p, int b, int h, int d, float4 v, float4 gate) {
  if (p.gate)
    v = make_float4(v.x * sigmoid(gate.x), v.y * sigmoid(gate.y), v.z * sigmoid(gate.z), v.w * sigmoid(gate.w));
  const long long i = b * p.o_sb + h * p.o_sh + d;
  if (p.out_fp32) {
    float* o = static_cast<float*>(p.o) + i;
    if (p.vec4)
      *reinterpret_cast<float4*>(o) = v;
    else
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
  } else {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.o) + i;
    if (p.vec4) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    } else {
      o[0] = __float2bfloat16_rn(v.x), o[1] = __float2bfloat16_rn(v.y);
      o[2] = __float2bfloat16_rn(v.z), o[3] = __float2bfloat16_rn(v.w);
    }
  }
}

__device__ __forceinline__ float4 zero4() { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float4 axpy(float a, float4 x, float4 y) {
  return make_float4(fmaf(a, x.x, y.x), fmaf(a, x.y, y.y), fmaf(a, x.z, y.z), fmaf(a, x.w, y.w));
}
__device__ __forceinline__ float4 over(float4 x, float l) {
  const float f = l == 0.f ? 0.f : 1.f;  // a row without keys gives 0, NaN stays NaN
  const float d = l == 0.f ? 1.f : l;
  return make_float4(f * (x.x / d), f * (x.y / d), f * (x.z / d), f * (x.w / d));
}

// A length or a table's entry. SHARED: past L1 (decode_shared.cuh).
template <bool SHARED>
__device__ __forceinline__ int load_int(const int* x) {
  if constexpr (SHARED) return __ldcg(x);
  return *x;
}

// Keys of sequence b that a call attends: its length, cut to the table.
template <bool SHARED>
__device__ __forceinline__ int keys_of(const DecodePagedParams& p, int b) {
  const long long cap = (long long)p.table_width * p.page;
  const int len = load_int<SHARED>(p.seqlens + b);
  return len < 0 ? 0 : (len > cap ? (int)cap : len);
}
// Tiles of sequence b ahead of those that the call itself attends (TK: keys of a tile).
template <int TK, bool SHARED>
__device__ __forceinline__ int tiles_ahead(const DecodePagedParams& p, int b) {
  if constexpr (SHARED) return load_seq(p.seqs + b).skip / TK;
  return 0;
}
template <int TK, bool SHARED>
__device__ __forceinline__ int tiles_of(const DecodePagedParams& p, int b) {
  return max((keys_of<SHARED>(p, b) + TK - 1) / TK - tiles_ahead<TK, SHARED>(p, b), 0);
}

// The work of a pair in the units that are shared out: its tiles, and one
// more for starting and finishing it (measured at 1 us beside 0.7 us a tile
// at head dim 64, 2 beside 1.3 at 256). The extra unit follows the tiles.
__device__ __forceinline__ int units_of(int tiles) { return tiles > 0 ? tiles + 1 : 0; }

// SHARED: the units of the first 128 sequences (lane x: x, 32 + x, ..), which are
// read past L1: requested together, and kept for the two passes over them.
template <int TK, bool SHARED>
struct FirstUnits {
  __device__ __forceinline__ explicit FirstUnits(const DecodePagedParams&) {}
};
template <int TK>
struct FirstUnits<TK, true> {
  int n[4];
  __device__ __forceinline__ explicit FirstUnits(const DecodePagedParams& p) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = 32 * k + (threadIdx.x & 31);
      n[k] = b < p.B ? units_of(tiles_of<TK, true>(p, b)) : 0;
    }
  }
  __device__ __forceinline__ int at(int b0) const { return b0 < 64 ? (b0 < 32 ? n[0] : n[1]) : (b0 < 96 ? n[2] : n[3]); }
};

// All units of the call (all lanes get it). Warp-collective.
template <int TK, bool SHARED>
__device__ __forceinline__ long long total_units(const DecodePagedParams& p, const FirstUnits<TK, SHARED>& first) {
  long long n = 0;
  int b1 = 0;
  if constexpr (SHARED) {
    // 32 sequences at a time: of the longest (2^25 units each) all four would pass 32 bits.
#pragma unroll
    for (int k = 0; k < 4; ++k) n += __reduce_add_sync(0xffffffffu, first.n[k]);
    b1 = 128;
  }
#pragma unroll 4
  for (int b0 = b1; b0 < p.B; b0 += 32) {
    const int b = b0 + (threadIdx.x & 31);
    n += __reduce_add_sync(0xffffffffu, b < p.B ? units_of(tiles_of<TK, SHARED>(p, b)) : 0);
  }
  return n * p.Hkv;
}

// Units per CTA: an equal share, but no less than a few, so that the joining
// of partials stays small beside the loads.
constexpr int kMinShare = 4;
__device__ __forceinline__ long long share_of(long long total, int n_ctas) {
  const long long share = (total + n_ctas - 1) / n_ctas;
  return share < kMinShare ? kMinShare : share;
}

// A stretch of the units, pair by pair: the pairs with a tile in it.
template <int TK, bool SHARED>
struct Walk {
  long long left;  // units from this pair's first one here to the stretch's end
  int b, g;        // the pair
  int begin, t1;   // its tiles in the stretch
  int t0;          // the current one (the producer's)
  int tiles, len;  // all its tiles, its keys
  int ahead;       // tiles of the sequence before them
  // The pairs of units [from, from + count). Warp-collective. Check valid().
  __device__ __forceinline__ Walk(const DecodePagedParams& p, long long from, long long count,
                                  const FirstUnits<TK, SHARED>& first) {
    left = count;
    b = p.B;
    if (left <= 0) return;
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      int n;
      if constexpr (SHARED)
        n = b0 < 128 ? first.at(b0) : (b0 + lane < p.B ? units_of(tiles_of<TK, SHARED>(p, b0 + lane)) : 0);
      else
        n = b0 + lane < p.B ? units_of(tiles_of<TK, SHARED>(p, b0 + lane)) : 0;
      int upto = n;  // inclusive sum over the lanes
#pragma unroll
      for (int off = 1; off < 32; off *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, (long long)upto * p.Hkv > from);
      if (past) {
        const int src = __ffs(past) - 1;
        const long long before = (long long)__shfl_sync(0xffffffffu, upto - n, src) * p.Hkv;
        b = b0 + src;
        measure(p);
        const long long into = from - before;
        g = (int)(into / units_of(tiles));
        begin = (int)(into % units_of(tiles));
        break;
      }
      from -= (long long)__shfl_sync(0xffffffffu, upto, 31) * p.Hkv;
    }
    t0 = begin;
    t1 = (int)min((long long)tiles, begin + left);
    if (begin == tiles) next(p);  // only the pair's extra unit is here
  }
  __device__ __forceinline__ Walk(int b_, int g_, int len_)
      : left((len_ + TK - 1) / TK), b(b_), g(g_), begin(0), t1((len_ + TK - 1) / TK), t0(0), tiles(t1), len(len_),
        ahead(0) {}
  __device__ __forceinline__ void measure(const DecodePagedParams& p) {
    len = keys_of<SHARED>(p, b);
    ahead = tiles_ahead<TK, SHARED>(p, b);
    tiles = max((len + TK - 1) / TK - ahead, 0);
  }
  __device__ __forceinline__ bool valid() const { return left > 0; }
  __device__ __forceinline__ bool next(const DecodePagedParams& p) {
    left -= units_of(tiles) - begin;
    if (left <= 0) return false;
    t0 = begin = 0;
    if (++g == p.Hkv) {
      g = 0;
      do {
        if (++b >= p.B) {
          left = 0;
          return false;
        }
        measure(p);
      } while (tiles == 0);
    }
    t1 = (int)min((long long)tiles, left);
    return true;
  }
};

// 8-bit keys and values enter the products as f16, which holds every e4m3
// number and into which one instruction converts two (moving the bits to bf16
// and fixing the exponent took 4.5, half of the kernel's instructions). f16's range is
// too narrow for q and for P times V's scales as they are:
//   q of a head is scaled by a power of two to a largest magnitude in [1, 2):
//   what then lies below f16's normal numbers is off by 2^-25 of the largest;
//   V's scale goes into the exponent, t_j = s_j + log2 sv_j, and the running
//   maximum M is of t: w_j = 2^(t_j - M + 15) <= 2^15 weighs the e4m3 numbers of V
//   (in two f16 terms: 2^-22 of w, or 2^-40 of the largest), w_j / sv_j is P
//   for the sum. With sv_j from 2^-100 (rows of zeros) to 2^90 that is 2^115 to
//   2^-75 for the largest weight, and the sum has up to 2^31 terms: it is kept
//   times 2^-24, below 2^122, with 27 bits under the smallest of those before
//   fp32 ends (O gets the same factor when the warps' parts are merged). A weight
//   below fp32's range drops out of the sum too: 2^-24 of the largest P where
//   V's scales in a sequence differ by 2^117, less where by less.
__device__ __forceinline__ uint32_t low_f16(uint32_t w) { return f16_of_e4m3((uint16_t)w); }
__device__ __forceinline__ uint32_t high_f16(uint32_t w) { return f16_of_e4m3((uint16_t)(w >> 16)); }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
constexpr float kWeightLog2 = 15.f;               // of the largest weight of V
constexpr float kSumUnit = 5.9604644775390625e-08f;  // 2^-24

__device__ __forceinline__ int swizzle(int r, int d) { return d ^ (((r >> 1) & 3) << 3); }

// NT blocks of 8 query heads cover a group; SPLIT: the even split above; E4M3:
// 8-bit pools with a scale per key; SHARED: keys from seqs[b].skip on (with SPLIT).
template <int D, int NT, bool SPLIT, bool E4M3, bool SHARED>
__global__ void __launch_bounds__(PagedCfg<D, NT, E4M3>::THREADS, PagedCfg<D, NT, E4M3>::CTAS_PER_SM)
    decode_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ DecodePagedParams p) {
  using C = PagedCfg<D, NT, E4M3>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  PagedBars* bars = reinterpret_cast<PagedBars*>(smem + C::OFF_BAR);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // SHARED: the kernel before is the one over the shared keys, of which nothing
  // is read here; the two run side by side, and this one ends after that one
  // (end_shared), so that the joining kernel sees both. The plan and all before it
  // is acquired (decode_shared.cuh), by each thread for itself.
  if constexpr (SHARED) {
    if (ld_acquire(p.ready) != kPlanReady) grid_dep_wait();
    fence_proxy_async();
  } else {
    grid_dep_wait();
  }
  // The next kernel (the joining one when SPLIT) may take SM slots as they
  // free up.
  grid_dep_launch();
  auto end_shared = [] {
    if constexpr (SHARED) grid_dep_wait();
  };
  if (p.err && blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.B; b += C::THREADS) {
      const int len = load_int<SHARED>(p.seqlens + b);
      if (len < 0 || len > (long long)p.table_width * p.page) atomicOr(p.err, kErrBadArgs);
    }
  long long from = 0, count = 1;
  const FirstUnits<C::TK, SHARED> first(p);
  if constexpr (SPLIT) {
    const long long total = total_units<C::TK, SHARED>(p, first), share = share_of(total, p.n_ctas);
    from = blockIdx.x * share;
    count = min(share, total - from);
    if (count <= 0) {
      end_shared();
      return;
    }
  }
  using W = Walk<C::TK, SHARED>;
  auto start = [&]() -> W {
    if constexpr (SPLIT) return W(p, from, count, first);
    const int b = blockIdx.x / p.Hkv;
    return W(b, blockIdx.x % p.Hkv, keys_of<SHARED>(p, b));
  };
  W w = start();
  if (SPLIT && !w.valid()) {
    end_shared();
    return;
  }
  if (!SPLIT && w.tiles == 0) {
    for (int e = 4 * threadIdx.x; e < p.group * D; e += 4 * C::THREADS)
      store_output(p, w.b, w.g * p.group + e / D, e % D, zero4(), zero4());
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 4);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  // Rows of Q past the group stay zero.
  for (int e = threadIdx.x; e < 2 * C::Q_ROW; e += C::THREADS)
    st_shared_v4(smem_u32(smem + C::OFF_Q) + 16 * e, 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncthreads();

  const int br = p.box_rows;
  if (warp == 4) {
    // ------------------------------------------------------------ producer
    // Lane x < 2 * boxes copies one box: K boxes first, then V boxes.
    const int boxes = C::TK / br;
    const int box = lane % boxes;
    const bool is_v = lane >= boxes;
    const bool mine = lane < 2 * boxes;
    const int box_bytes = br * D * (E4M3 ? 1 : 2);
    // Every tile's page is looked up one tile ahead, across pairs too, and
    // checked when its turn comes (so that nothing waits for the lookup).
    auto has_keys = [&]() { return mine && (w.ahead + w.t0) * C::TK + box * br < w.len; };
    auto entry_of = [&]() -> int {  // table entry of this lane's box in tile w.t0
      return has_keys() ? load_int<SHARED>(p.block_table + w.b * p.table_ld +
                                           ((w.ahead + w.t0) * C::TK + box * br) / p.page)
                        : 0;
    };
    int n = 0, pairs = 0;  // tiles and pairs copied so far
    bool more = true, new_pair = true;
    int entry = entry_of();
    bool copy = has_keys();
    while (more) {
      const int slot = n % C::STAGES;
      const int g = w.g, row = ((w.ahead + w.t0) * C::TK + box * br) % p.page;
      const __nv_bfloat16* q = p.q + w.b * p.q_sb + (long long)(g * p.group + lane) * p.q_sh;
      const bool with_q = new_pair;
      ++w.t0;
      new_pair = w.t0 == w.t1;
      if (new_pair) more = w.next(p);
      const int id = entry;
      const bool now = copy;
      if (more) {
        entry = entry_of();
        copy = has_keys();
      }
      if (with_q) {
        const int qs = pairs & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->q_empty[qs], ((uint32_t)(pairs >> 1) & 1u) ^ 1u, abort_flag,
                                               p.err)))
          break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->q_full[qs], p.group * D * 2);
        __syncwarp();
        if (lane < p.group)
          bulk_load(smem + C::OFF_Q + (qs * 16 + lane) * C::Q_ROW, q, D * 2, &bars->q_full[qs]);
        ++pairs;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&bars->empty[slot], ((uint32_t)(n / C::STAGES) & 1u) ^ 1u, abort_flag,
                                             p.err)))
        break;
      uint8_t* dst = smem + slot * C::STAGE_BYTES + (is_v ? C::TILE_BYTES : 0) + box * box_bytes;
      const unsigned copies = __ballot_sync(0xffffffffu, now);
      if (lane == 0) mbar_arrive_expect_tx(&bars->full[slot], __popc(copies) * (box_bytes + (E4M3 ? 4 * br : 0)));
      __syncwarp();
      if (now) {
        const bool in_pool = id >= 0 && id < p.n_pages;
        if (!in_pool && p.err) atomicOr(p.err, kErrBadArgs);
        tma_load_5d(dst, is_v ? &tm_v : &tm_k, &bars->full[slot], 0, row, 0, g, in_pool ? id : 0);
        if constexpr (E4M3) {
          const long long page = in_pool ? id : 0;
          const float* scales = is_v ? p.v_scales + page * p.vss[0] + g * p.vss[1] + row
                                     : p.k_scales + page * p.kss[0] + g * p.kss[1] + row;
          bulk_load(smem + C::OFF_SCALES + ((slot * 2 + is_v) * C::TK + box * br) * 4, scales, 4 * br,
                    &bars->full[slot]);
        }
      }
      ++n;
    }
    if (*abort_flag && lane == 0) {
      // Let every copy still in flight land before the CTA releases smem.
      for (int i = max(0, n - C::STAGES); i < n; ++i)
        mbar_wait_quiet(&bars->full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u);
      for (int i = max(0, pairs - 2); i < pairs; ++i) mbar_wait_quiet(&bars->q_full[i & 1], (uint32_t)(i >> 1) & 1u);
    }
  } else {
    // ------------------------------------------------------------ compute warps
    const int gr = lane >> 2, tq = lane & 3;
    const float sl2 = p.scale_log2;
    const int mi = lane >> 3, mr = lane & 7;  // ldmatrix: matrix index / row in it
    // This warp's 16 keys of a tile (E4M3: and 16 of its second half) lie in one
    // box: its first row there, and the distance of the box's chunks of columns.
    constexpr int kLine = E4M3 && D == 64 ? 64 : 128;  // bytes of a row in a chunk
    auto rows_at = [&](int r) -> uint32_t {
      return (r / br) * (br * D * (E4M3 ? 1 : 2)) + (r % br) * kLine;
    };
    const uint32_t wbase = rows_at(16 * warp);
    const uint32_t chunk = br * 128;
    // 16-byte unit U of row r (0..15): the swizzle XORs the unit with the
    // row's place in its group of 8 (rows of 64 bytes: of two rows' place in
    // their group of 4).
    auto at = [&](uint32_t base, int r, int U) -> uint32_t {
      if constexpr (kLine == 64) return base + r * 64 + ((U ^ ((r >> 1) & 3)) << 4);
      return base + (U >> 3) * chunk + r * 128 + (((U & 7) ^ (r & 7)) << 4);
    };
    // A wait that ran out leaves garbage in the result and the error word set;
    // the warps still meet at every barrier below.
    int pair = 0;  // pairs done so far
    int n = 0;     // tiles taken so far
    do {
      const int n_last = n + (w.t1 - w.begin) - 1;  // the pair's last one here
      // Q^T as the B operand: column (head) gr, k in pairs 2 tq, 2 tq + 8.
      uint32_t qb[NT][D / 16][2];
      float qf[NT][2];  // E4M3: what the scores of heads 8 x + 2 tq (+ 1) are multiplied by
      const bool got = __all_sync(
          0xffffffffu, mbar_wait(&bars->q_full[pair & 1], (uint32_t)(pair >> 1) & 1u, abort_flag, p.err));
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        if constexpr (E4M3) {
          // In the order in which a word of K holds its columns: four in a row.
          const uint8_t* q = smem + C::OFF_Q + ((pair & 1) * 16 + 8 * x + gr) * C::Q_ROW + tq * 8;
          uint32_t top = 0;  // the largest magnitude, as an integer of the same order
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint2 w = *reinterpret_cast<const uint2*>(q + 32 * k);
            qb[x][k][0] = w.x;
            qb[x][k][1] = w.y;
            top = max(top, max(max(w.x & 0x7fffu, w.y & 0x7fffu), max((w.x >> 16) & 0x7fffu, (w.y >> 16) & 0x7fffu)));
          }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // 2^-e and 2^e for 2^e <= the largest < 2^(e + 1); e of a zero row or one of the smallest numbers: -126.
          const uint32_t e = max(min(top >> 7, 253u), 1u);
          const float down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t w = qb[x][k][u];
              qb[x][k][u] = pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
            }
          qf[x][0] = sl2 * __shfl_sync(0xffffffffu, up, 8 * tq);
          qf[x][1] = sl2 * __shfl_sync(0xffffffffu, up, 8 * tq + 4);
        } else {
          const uint32_t q = smem_u32(smem + C::OFF_Q) + ((pair & 1) * 16 + 8 * x + mr) * C::Q_ROW + mi * 16;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            ldsm4(q + 64 * k, qb[x][2 * k][0], qb[x][2 * k][1], qb[x][2 * k + 1][0], qb[x][2 * k + 1][1]);
        }
      }
      __syncwarp();
      if (lane == 0 && got) mbar_arrive(&bars->q_empty[pair & 1]);
      // O^T: rows 16 d + gr (+ 8) (E4M3: 16 d + 2 gr (+ 1), as V's bytes come),
      // columns (heads) 8 x + 2 tq (+ 1); this
      // thread keeps the running maximum and its part of the sum of those heads.
      float acc[NT][D / 16][4];
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[x][d][0] = acc[x][d][1] = acc[x][d][2] = acc[x][d][3] = 0.f;
        m[x][0] = m[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.f;
      }
      for (int t = w.begin; t < w.t1; ++t, ++n) {
        const int slot = n % C::STAGES;
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&bars->full[slot], (uint32_t)(n / C::STAGES) & 1u, abort_flag, p.err))) {
          n = n_last + 1;
          break;
        }
        const uint32_t stage = smem_u32(smem + slot * C::STAGE_BYTES);
        const int left = w.len - (w.ahead + t) * C::TK;  // keys from the tile's first on
        if constexpr (E4M3) {
          if (left > 16 * warp) {
            uint32_t kbase[C::KB];
            int have[C::KB];  // keys of each block that exist
#pragma unroll
            for (int i = 0; i < C::KB; ++i) {
              kbase[i] = stage + rows_at(64 * i + 16 * warp);
              have[i] = left - 64 * i - 16 * warp;
            }
            float s[C::KB][NT][4];
#pragma unroll
            for (int i = 0; i < C::KB; ++i)
#pragma unroll
              for (int x = 0; x < NT; ++x) s[i][x][0] = s[i][x][1] = s[i][x][2] = s[i][x][3] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
#pragma unroll
              for (int i = 0; i < C::KB; ++i) {
                uint32_t w4[4];
                ldsm4(at(kbase[i], 8 * (mi & 1) + mr, 2 * k + (mi >> 1)), w4[0], w4[1], w4[2], w4[3]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const uint32_t a[4] = {low_f16(w4[2 * u]), low_f16(w4[2 * u + 1]), high_f16(w4[2 * u]),
                                         high_f16(w4[2 * u + 1])};
#pragma unroll
                  for (int x = 0; x < NT; ++x) mma16816_f16(s[i][x], a, qb[x][2 * k + u][0], qb[x][2 * k + u][1]);
                }
              }
            }
            const float* scales = reinterpret_cast<const float*>(smem + C::OFF_SCALES) + slot * 2 * C::TK + 16 * warp;
            float per_sv[C::KB][2];  // kSumUnit / the scales of V's rows gr, gr + 8
#pragma unroll
            for (int i = 0; i < C::KB; ++i) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int r = gr + 8 * u;
                const float sk = scales[64 * i + r], given = scales[C::TK + 64 * i + r];
                const float sv = e4m3_scale_in_range(given), lg = __log2f(sv);
                per_sv[i][u] = r < have[i] ? __fdividef(kSumUnit, sv) : 0.f;
#pragma unroll
                for (int x = 0; x < NT; ++x) {
#pragma unroll
                  for (int c = 0; c < 2; ++c) {
                    const float tj = fmaf(s[i][x][2 * u + c] * sk, qf[x][c], lg);
                    s[i][x][2 * u + c] = r < have[i] ? tj : -INFINITY;
                  }
                }
              }
              if (have[i] < 16) {
                // V rows without a key: 0 x anything would not do (NaN).
                const int from = max(have[i], 0);
                for (int u = lane; u < (16 - from) * (D / 16); u += 32)
                  st_shared_v4(at(kbase[i] + C::TILE_BYTES, from + u / (D / 16), u % (D / 16)), 0u, 0u, 0u, 0u);
                fence_proxy_async_smem();  // before the slot's next copy
                __syncwarp();
              }
            }
            // P^T as the B operand, in two terms: the scores' fragments hold keys along gr and heads along tq, the
            // operand the reverse.
            uint32_t ph[C::KB][NT][2], pl[C::KB][NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              float a[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < C::KB; ++i) mx = fmaxf(mx, fmaxf(s[i][x][c], s[i][x][2 + c]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[x][c], mx);
                const float u = mn == -INFINITY ? 0.f : mn;
                a[c] = ex2(m[x][c] - u);
                m[x][c] = mn;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < C::KB; ++i) {
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    float& w1 = s[i][x][2 * e + c];
                    w1 = ex2(w1 - (u - kWeightLog2));
                    sum = fmaf(w1, per_sv[i][e], sum);
                  }
                }
                l[x][c] = fmaf(l[x][c], a[c], sum);
              }
              if (__any_sync(0xffffffffu, a[0] != 1.f || a[1] != 1.f)) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                  acc[x][d][0] *= a[0];
                  acc[x][d][1] *= a[1];
                  acc[x][d][2] *= a[0];
                  acc[x][d][3] *= a[1];
                }
              }
#pragma unroll
              for (int i = 0; i < C::KB; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t high = pack_f16x2(s[i][x][2 * e], s[i][x][2 * e + 1]);
                  const float2 back = unpack_f16x2(high);
                  ph[i][x][e] = transposed(high);
                  pl[i][x][e] = transposed(pack_f16x2(s[i][x][2 * e] - back.x, s[i][x][2 * e + 1] - back.y));
                }
              }
            }
#pragma unroll
            for (int i = 0; i < C::KB; ++i) {
#pragma unroll
              for (int k = 0; k < D / 32; ++k) {
                uint32_t w4[4];
                ldsm4_t(at(kbase[i] + C::TILE_BYTES, 8 * (mi >> 1) + mr, 2 * k + (mi & 1)), w4[0], w4[1], w4[2], w4[3]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  // A word has two columns of two keys; the operand wants two keys of a column.
                  const uint32_t w0 = __byte_perm(w4[u], 0, 0x3120), w1 = __byte_perm(w4[u + 2], 0, 0x3120);
                  const uint32_t a[4] = {low_f16(w0), high_f16(w0), low_f16(w1), high_f16(w1)};
#pragma unroll
                  for (int x = 0; x < NT; ++x) {
                    mma16816_f16(acc[x][2 * k + u], a, ph[i][x][0], ph[i][x][1]);
                    mma16816_f16(acc[x][2 * k + u], a, pl[i][x][0], pl[i][x][1]);
                  }
                }
              }
            }
          }
        } else {
          const uint32_t kbase = stage + wbase;
          const uint32_t vbase = kbase + C::TILE_BYTES;
          const int have = left - 16 * warp;  // keys of this warp's 16 that exist
          if (have > 0) {
            float s[NT][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t a[4];
              ldsm4(at(kbase, 8 * (mi & 1) + mr, 2 * k + (mi >> 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int x = 0; x < NT; ++x) mma16816(s[x], a, qb[x][k][0], qb[x][k][1]);
            }
            if (have < 16) {
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                if (gr >= have) s[x][0] = s[x][1] = -INFINITY;
                if (gr + 8 >= have) s[x][2] = s[x][3] = -INFINITY;
              }
              // V rows without a key: 0 x anything would not do (NaN).
              for (int u = lane; u < (16 - have) * (D / 8); u += 32)
                st_shared_v4(at(vbase, have + u / (D / 8), u % (D / 8)), 0u, 0u, 0u, 0u);
              fence_proxy_async_smem();  // before the slot's next copy
              __syncwarp();
            }
            // P^T as the B operand, in two bf16 terms: the scores' fragments
            // hold keys along gr and heads along tq, the operand the reverse.
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              float a[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float mx = fmaxf(s[x][c], s[x][2 + c]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[x][c], mx * sl2);
                const float u = mn == -INFINITY ? 0.f : mn;
                a[c] = ex2(m[x][c] - u);
                m[x][c] = mn;
                s[x][c] = ex2(fmaf(s[x][c], sl2, -u));
                s[x][2 + c] = ex2(fmaf(s[x][2 + c], sl2, -u));
                l[x][c] = fmaf(l[x][c], a[c], s[x][c] + s[x][2 + c]);
              }
              if (__any_sync(0xffffffffu, a[0] != 1.f || a[1] != 1.f)) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                  acc[x][d][0] *= a[0];
                  acc[x][d][1] *= a[1];
                  acc[x][d][2] *= a[0];
                  acc[x][d][3] *= a[1];
                }
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t high = pack_bf16x2(s[x][2 * e], s[x][2 * e + 1]);
                ph[x][e] = transposed(high);
                pl[x][e] = transposed(pack_bf16x2(s[x][2 * e] - __uint_as_float(high << 16),
                                                  s[x][2 * e + 1] - __uint_as_float(high & 0xffff0000u)));
              }
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              uint32_t a[4];
              ldsm4_t(at(vbase, 8 * (mi >> 1) + mr, 2 * d + (mi & 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                mma16816(acc[x][d], a, ph[x][0], ph[x][1]);
                mma16816(acc[x][d], a, pl[x][0], pl[x][1]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0 && n < n_last) mbar_arrive(&bars->empty[slot]);
      }
      // Merge the four warps' (m, l, O) in the last tile's stage, once all of
      // them have read it; the stage is released after that.
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const int slot = n_last % C::STAGES;
      // [4][16][D], columns swizzled by the head so that neither side's accesses
      // collide in a bank.
      float* so = reinterpret_cast<float*>(smem + slot * C::STAGE_BYTES);
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = 8 * x + 2 * tq + c;
          float lr = l[x][c];
          lr += __shfl_xor_sync(0xffffffffu, lr, 4);
          lr += __shfl_xor_sync(0xffffffffu, lr, 8);
          lr += __shfl_xor_sync(0xffffffffu, lr, 16);
          if (gr == 0) {
            bars->m[warp][r] = m[x][c];
            bars->l[warp][r] = lr;
          }
          if (r < p.group) {
            float* row = so + (warp * 16 + r) * D;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              if constexpr (E4M3) {
                *reinterpret_cast<float2*>(row + swizzle(r, 16 * d + 2 * gr)) =
                    make_float2(acc[x][d][c], acc[x][d][2 + c]);
              } else {
                row[swizzle(r, 16 * d + gr)] = acc[x][d][c];
                row[swizzle(r, 16 * d + 8 + gr)] = acc[x][d][2 + c];
              }
            }
          }
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // Thread x takes columns 4 x .. of the group's rows, 512 apart. Not
      // unrolled, and finished by the joining kernel when SPLIT: this runs
      // once per pair, and fetching more instructions from memory (which the
      // stream of keys has pushed out of L2) cost more than running them.
      const long long part = ((long long)w.b * p.Hkv + w.g + blockIdx.x) * p.group;
#pragma unroll 1
      for (int e = 4 * threadIdx.x; e < p.group * D; e += 512) {
        const int r = e / D, d = e % D;
        float M = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) M = fmaxf(M, bars->m[u][r]);
        const float Mu = (M == -INFINITY) ? 0.f : M;
        float lsum = 0.f;
        float4 osum = zero4();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          // A warp without keys here has nothing in the sum (its m is -inf).
          const float f = ex2(bars->m[u][r] - Mu);
          lsum += f * bars->l[u][r];
          osum = axpy(E4M3 ? f * kSumUnit : f, *reinterpret_cast<const float4*>(so + (u * 16 + r) * D + swizzle(r, d)), osum);
        }
        if constexpr (SPLIT) {
          *reinterpret_cast<float4*>(p.part_o + (part + r) * D + d) = osum;
          if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * (part + r)) = make_float2(M, lsum);
        } else {
          const int h = w.g * p.group + r;
          store_output(p, w.b, h, d, over(osum, lsum), p.gate ? load_gate(p, w.b, h, d) : zero4());
        }
      }
      if (SPLIT && threadIdx.x == 0) {
        int* place = p.place + 2 * ((long long)w.b * p.Hkv + w.g);
        if (w.begin == 0) place[0] = blockIdx.x;
        if (w.t1 == w.tiles) place[1] = blockIdx.x;
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 128;" ::: "memory");  // everyone has read the stage, m and l
      if (lane == 0) mbar_arrive(&bars->empty[slot]);
      ++pair;
    } while (w.next(p));
  }
  end_shared();
}

constexpr int kJoinThreads = 256;

// The partials of (sequence b, KV head g): the CTAs from the one with the pair's
// first tile to the one with its last, which the main kernel has noted (p.place):
// working it out again here from all lengths took 2 us. SHARED: the parts over
// the shared keys come after those, numbered and placed alike.
template <bool SHARED>
struct Parts {
  int own, all;       // parts
  long long row0, shared0;  // row of the head's first own and first shared part
  __device__ __forceinline__ Parts(const DecodePagedParams& p, int b, int g, int r)
      : own(0), all(0), row0(0), shared0(0) {
    const long long pair = (long long)b * p.Hkv + g;
    const int2 at = __ldcg(reinterpret_cast<const int2*>(p.place) + pair);
    if (tiles_of<64, SHARED>(p, b) > 0) {  // any size of tiles
      // (Within the CTAs there are, even if the lengths changed under the call.)
      const int c0 = max(0, min(at.x, p.n_ctas - 1));
      own = min(at.y, p.n_ctas - 1) - c0 + 1;
      row0 = (pair + c0) * p.group + r;
    }
    all = own;
    if constexpr (SHARED) {
      const SharedSeq s = load_seq(p.seqs + b);
      if (s.skip > 0) {
        const long long item = (long long)s.block * p.Hkv + g;
        const int2 of = __ldcg(reinterpret_cast<const int2*>(p.shared_place) + item);
        const int first = max(0, min(of.x, p.shared_ctas - 1));
        all += min(of.y, p.shared_ctas - 1) - first + 1;
        shared0 = (item + first) * p.block_rows + s.row + r;
      }
    }
  }
  // Part i's (m, l) and columns d .. d + 3 of O.
  __device__ __forceinline__ void load(const DecodePagedParams& p, int D, int i, int d, float2& ml, float4& o) const {
    const bool mine = !SHARED || i < own;
    const long long row = mine ? row0 + (long long)i * p.group : shared0 + (long long)(i - own) * p.block_rows;
    const float* part_ml = mine ? p.part_ml : p.shared_ml;
    const float* part_o = mine ? p.part_o : p.shared_o;
    ml = i < all ? __ldcg(reinterpret_cast<const float2*>(part_ml + 2 * row)) : make_float2(-INFINITY, 0.f);
    o = i < all ? __ldcg(reinterpret_cast<const float4*>(part_o + row * D + d)) : zero4();
  }
};

// N more parts into (m, l, o).
template <int N, bool SHARED>
__device__ __forceinline__ void join_parts(const DecodePagedParams& p, const Parts<SHARED>& parts, int D, int i0,
                                           int step, int d, float& m, float& l, float4& o) {
  float2 ml[N];
  float4 po[N];
#pragma unroll
  for (int k = 0; k < N; ++k) parts.load(p, D, i0 + k * step, d, ml[k], po[k]);
  float mn = m;
#pragma unroll
  for (int k = 0; k < N; ++k) mn = fmaxf(mn, ml[k].x);
  const float mu = mn == -INFINITY ? 0.f : mn;
  const float f0 = ex2(m - mu);
  m = mn;
  l *= f0;
  o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float f = ex2(ml[k].x - mu);
    l = fmaf(f, ml[k].y, l);
    o = axpy(f, po[k], o);
  }
}

// Joins the partials of the query heads of many sequences, which have few parts
// each: a thread takes four columns of a row and all its parts.
template <int D, bool SHARED>
__global__ void __launch_bounds__(kJoinThreads)
    decode_paged_join_rows_kernel(const __grid_constant__ DecodePagedParams p) {
  const long long x = (long long)blockIdx.x * kJoinThreads + threadIdx.x;
  const long long row = x / (D / 4);
  const int d = 4 * (int)(x % (D / 4));
  if (row >= (long long)p.B * p.Hq) return;
  const int b = (int)(row / p.Hq), h = (int)(row % p.Hq), g = h / p.group;
  grid_dep_wait();
  grid_dep_launch();
  if (SHARED && x == 0) *p.ready = 0;
  const float4 gate = p.gate ? load_gate(p, b, h, d) : zero4();
  const Parts<SHARED> parts(p, b, g, h % p.group);
  float m = -INFINITY, l = 0.f;
  float4 o = zero4();
  for (int i = 0; i < parts.all; i += 8) join_parts<8>(p, parts, D, i, 1, d, m, l, o);
  store_output(p, b, h, d, over(o, l), gate);
}

// Joins the partials of (sequence, query head) blockIdx.x. D / 4 threads read one
// part's row; the parts are dealt to such teams in turn and joined in a fixed
// order. Nothing is read before the
// wait for the main kernel: what it and the kernels before it have written (the
// lengths, by the append) is only sure to be seen after that. A dry run before
// the wait, to fetch the instructions, gained nothing (4 to 4096 sequences of
// 500 to 1500 keys, 32 / 4 heads of 128: 9.5 us to 1.77 ms without, 9.5 us to
// 1.80 ms with it).
template <int D, bool SHARED>
__global__ void __launch_bounds__(kJoinThreads) decode_paged_join_kernel(const __grid_constant__ DecodePagedParams p) {
  constexpr int TEAM = D / 4, TEAMS = kJoinThreads / TEAM;
  __shared__ float4 s_o[TEAMS][TEAM];
  __shared__ float s_m[TEAMS], s_l[TEAMS];
  const int b = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
  const int g = h / p.group, r = h % p.group;
  const int team = threadIdx.x / TEAM, d = 4 * (threadIdx.x % TEAM);
  grid_dep_wait();
  grid_dep_launch();
  if (SHARED && blockIdx.x == 0 && threadIdx.x == 0) *p.ready = 0;
  const float4 gate = p.gate && team == 0 ? load_gate(p, b, h, d) : zero4();
  const Parts<SHARED> parts(p, b, g, r);
  float m = -INFINITY, l = 0.f;
  float4 o = zero4();
  for (int i0 = team; i0 < parts.all; i0 += 4 * TEAMS) join_parts<4>(p, parts, D, i0, TEAMS, d, m, l, o);
  s_o[team][threadIdx.x % TEAM] = o;
  if (d == 0) {
    s_m[team] = m;
    s_l[team] = l;
  }
  __syncthreads();
  if (team == 0) {
    float M = -INFINITY;
#pragma unroll
    for (int u = 0; u < TEAMS; ++u) M = fmaxf(M, s_m[u]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float lsum = 0.f;
    float4 osum = zero4();
#pragma unroll
    for (int u = 0; u < TEAMS; ++u) {
      const float f = ex2(s_m[u] - Mu);
      lsum = fmaf(f, s_l[u], lsum);
      osum = axpy(f, s_o[u][threadIdx.x], osum);
    }
    store_output(p, b, h, d, over(osum, lsum), gate);
  }
}

constexpr int kWholeTiles = 8;
constexpr long long kManyRows = 1024;

// All units of a call, and the pair and tile of some of them (b2attn_diag.h). One warp.
template <int TK, bool SHARED>
__global__ void decode_paged_units_kernel(const __grid_constant__ DecodePagedParams p, const long long* units, int n,
                                          long long* out) {
  const FirstUnits<TK, SHARED> first(p);
  const long long total = total_units<TK, SHARED>(p, first);
  for (int i = 0; i < n; ++i) {
    const Walk<TK, SHARED> w(p, units[i], units[i] < 0 ? 0LL : min(1LL, total - units[i]), first);
    const bool valid = w.valid();
    if (threadIdx.x == 0) {
      out[4 * i] = total;
      out[4 * i + 1] = valid ? w.b : -1;
      out[4 * i + 2] = valid ? w.g : -1;
      out[4 * i + 3] = valid ? w.begin : -1;
    }
  }
}

template <int D, int NT, bool SPLIT, bool E4M3, bool SHARED = false>
int launch_main(const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p, long long n,
                cudaStream_t st) {
  using C = PagedCfg<D, NT, E4M3>;
  static OncePerDevice once;
  if (n > 0x7fffffffLL) return -1;
  return once.run(
      [] {
        return cudaFuncSetAttribute(decode_paged_kernel<D, NT, SPLIT, E4M3, SHARED>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::SMEM_BYTES) == cudaSuccess;
      },
      [&] {
        return launch_dependent(decode_paged_kernel<D, NT, SPLIT, E4M3, SHARED>, dim3((unsigned)n), C::THREADS,
                                C::SMEM_BYTES, st, 0, tk, tv, p);
      });
}

template <int D, bool SPLIT>
int launch_n(const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p, long long n, cudaStream_t st) {
  const bool narrow = p.group <= 8;
  if (p.k_scales)
    return narrow ? launch_main<D, 1, SPLIT, true>(tk, tv, p, n, st)
                  : launch_main<D, 2, SPLIT, true>(tk, tv, p, n, st);
  return narrow ? launch_main<D, 1, SPLIT, false>(tk, tv, p, n, st)
                : launch_main<D, 2, SPLIT, false>(tk, tv, p, n, st);
}

template <int D>
int launch_t(const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p, cudaStream_t st) {
  if (!decode_paged_splits(p.table_width, p.page))
    return launch_n<D, false>(tk, tv, p, (long long)p.B * p.Hkv, st);
  const long long heads = (long long)p.B * p.Hq;
  if (heads > 0x7fffffffLL) return -2;
  int rc;
  if (p.seqs)
    rc = p.group <= 8 ? launch_main<D, 1, true, false, true>(tk, tv, p, p.n_ctas, st)
                      : launch_main<D, 2, true, false, true>(tk, tv, p, p.n_ctas, st);
  else
    rc = launch_n<D, true>(tk, tv, p, p.n_ctas, st);
  if (rc) return rc;
  // Many rows have few parts each and need no teams (8-bit and shared forms).
  if ((p.seqs || p.k_scales) && heads >= kManyRows) {
    const auto join = p.seqs ? decode_paged_join_rows_kernel<D, true> : decode_paged_join_rows_kernel<D, false>;
    constexpr int ROWS = kJoinThreads / (D / 4);
    const dim3 grid((unsigned)((heads + ROWS - 1) / ROWS));
    return launch_dependent(join, grid, kJoinThreads, 0, st, 0, p) == cudaSuccess ? 0 : -1;
  }
  const auto join = p.seqs ? decode_paged_join_kernel<D, true> : decode_paged_join_kernel<D, false>;
  return launch_dependent(join, dim3((unsigned)heads), kJoinThreads, 0, st, 0, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

bool decode_paged_splits(int table_width, int page) { return (long long)table_width * page > 64LL * kWholeTiles; }

int decode_paged_max_ctas(int D, int group, bool e4m3, int sms) {
  return sms * decode_paged_ctas_per_sm(D, group <= 8 ? 1 : 2, e4m3);
}

int launch_decode_paged_units(const DecodePagedParams& p, int tile, const long long* units, int n, long long* out,
                              cudaStream_t st) {
  const auto kernel = p.seqs ? decode_paged_units_kernel<64, true>
                             : (tile == 64 ? decode_paged_units_kernel<64, false> : decode_paged_units_kernel<128, false>);
  kernel<<<1, 32, 0, st>>>(p, units, n, out);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int launch_decode_paged(int D, const CUtensorMap& tk, const CUtensorMap& tv, const DecodePagedParams& p,
                        cudaStream_t st) {
  switch (D) {
    case 64: return launch_t<64>(tk, tv, p, st);
    case 128: return launch_t<128>(tk, tv, p, st);
    case 256: return launch_t<256>(tk, tv, p, st);
    default: return -3;
  }
}

}  // namespace b2a
