// The shared part of single-token attention for groups of sequences whose first
// keys are the same (a system prompt, a document that many ask about), sm_100a.
//
// For query head h of sequence b in a group with prefix keys j < eff:
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  O = sum_j 2^(s_j - m) v_j,
//   s_j = scale log2(e) q_h k_j,
// left as partials which the joining kernel (decode_paged.cu) combines with
// those of the sequence's own keys. eff is the group's prefix length, cut to
// whole blocks of 64 keys; the rest counts as each sequence's own. A sequence
// shorter than eff, or alone in its group, attends all its keys by itself.
//
// One sequence's step reads every key for a handful of query heads and is bound
// by HBM; over the shared keys all sequences' heads of a KV group are rows of
// one matrix product, 4 D flop per (row, key), on the tensor cores: a row block
// is NQT tiles of 128 rows, 128 / group sequences of `group` heads each.
// Per tile S = Q K^T and O += P V with tcgen05.mma, scores double-buffered in
// TMEM (S[c & 1] of 64 keys, P over its first 32 columns), O in TMEM; K and V
// tiles of 64 keys come through rings in shared memory, one TMA copy per run of
// keys in a page and 64 columns, and feed both tiles. MMA order per tile: S(0),
// S(1), then PV(j), S(j + 2): while the softmax turns S(j) into P(j), the tensor
// core has S(j + 1) and PV(j - 1).
//
// The key blocks of all items (row block, KV head) are cut into one equal
// stretch per CTA, as in paged decode, so few rows over a long prefix fill the
// GPU too. A first, one-CTA kernel finds from the lengths which sequences take
// part, and numbers row blocks and units.
//
// Measured on one B200 (device time): 128 sequences of 16 to 2048 keys of their own
// behind 32768 shared ones, 32 / 4 heads of 128, pages of 64: 111 to 124 us a call. One
// by one, in a profile in which none overlaps another (125 in all): the plan 4.6, the
// shared keys 78.6, the own ones 31 (after the shared ones in a call too: the two
// kernels do not fit an SM together at this head dim), the join 10.3; in a call each
// starts while the one before it ends. Without the profiler each further 32768 shared
// keys cost 57 us (1.2 PFLOP/s, 0.72 of the measured bf16 burst rate, 0.86 of the
// sustained one: what the dense prefill reaches); the other 21 of the 78.6 are not
// measured apart. Tried without gain: S and P in columns of their own,
// so that S(j + 1) can go a softmax earlier (128.0 us against 127.5), two softmax
// warpgroups a tile (137: what they tell each other costs more than it hides).
// Warps: 0 TMA, 1 .. NQT MMA issue, 4 + 4 t .. softmax and partials of tile t.
#include <climits>

#include "capi_internal.cuh"
#include "decode_shared.cuh"
#include "softmax.cuh"

namespace b2a {

namespace {

constexpr int kBlock = 64;  // keys of a block

template <int D>
struct SharedCfg {
  static constexpr int NQT = D == 256 ? 1 : 2;  // tiles of a row block; TMEM has no room for two at 256
  static constexpr int KCH = D / 64;
  static constexpr int Q_CHUNK = 128 * 128;  // 128 rows x 128 B
  static constexpr int KV_CHUNK = kBlock * 128;
  static constexpr int Q_BYTES = KCH * Q_CHUNK;
  static constexpr int TILE_BYTES = KCH * KV_CHUNK;  // 64 keys of K or V
  static constexpr int KST = D == 256 ? 2 : 4;
  static constexpr int VST = D == 256 ? 3 : 4;
  static constexpr int OFF_K = NQT * Q_BYTES;
  static constexpr int OFF_V = OFF_K + KST * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_V + VST * TILE_BYTES;
  static constexpr int SMEM_BYTES = OFF_BAR + 512 + 1024;
  static constexpr int S_COL = 0;  // S[t][b] at 128 t + 64 b
  static constexpr int O_COL = 128 * NQT;
  static constexpr int TMEM_COLS = 512;
  static constexpr int THREADS = 128 + 128 * NQT;
  static_assert(O_COL + NQT * D <= TMEM_COLS, "TMEM budget");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

struct SharedBars {
  uint64_t q_full, q_free;
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  uint64_t s_full[2][2];  // [tile][buffer]
  uint64_t p_full[2][2];
  uint64_t pv_done[2][2];
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(SharedBars) <= 512, "SharedCfg::OFF_BAR");

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// ---------------------------------------------------------------- plan
constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

// Offsets of group g, and whether they are a stretch of the sequences.
__device__ __forceinline__ bool group_of(const SharedPlanParams& p, int g, int& c0, int& c1) {
  c0 = p.cu_groups ? p.cu_groups[g] : 0;
  c1 = p.cu_groups ? p.cu_groups[g + 1] : p.B;
  return c0 >= 0 && c1 >= c0 && c1 <= p.B;
}

// Inclusive sums of x and y over the warp.
__device__ __forceinline__ void warp_sums_upto(long long& x, long long& y) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const long long u = __shfl_up_sync(0xffffffffu, x, off), v = __shfl_up_sync(0xffffffffu, y, off);
    if (lane >= off) x += u, y += v;
  }
}

// Inclusive sums over the block's threads.
__device__ __forceinline__ void block_sums_upto(long long& x, long long& y, long long (*per_warp)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  warp_sums_upto(x, y);
  __syncthreads();
  if (lane == 31) per_warp[warp][0] = x, per_warp[warp][1] = y;
  __syncthreads();
  long long u = lane < kPlanWarps ? per_warp[lane][0] : 0, v = lane < kPlanWarps ? per_warp[lane][1] : 0;
  const long long own_u = u, own_v = v;
  warp_sums_upto(u, v);
  x += __shfl_sync(0xffffffffu, u - own_u, warp);
  y += __shfl_sync(0xffffffffu, v - own_v, warp);
}

// Which sequences share what, the numbers of row blocks and units, and the rows
// of each sequence. One CTA; groups and sequences are dealt to its threads. It is
// all latency, so the groups are worked out in shared memory where they fit
// (LOCAL), and atomics are few.
constexpr int kLocalGroups = 1024;

template <bool LOCAL>
__global__ void __launch_bounds__(kPlanThreads)
    decode_shared_plan_kernel(const __grid_constant__ SharedPlanParams p, int block_seqs, int tile_seqs) {
  __shared__ long long s_sum[kPlanWarps][2];
  __shared__ SharedGroup s_groups[LOCAL ? kLocalGroups : 1];
  __shared__ unsigned long long s_saved;  // keys that need not be read again
  SharedGroup* groups = LOCAL ? s_groups : p.groups;
  const int lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  const int first_len = (int)threadIdx.x < p.B ? p.seqlens[threadIdx.x] : 0;
  if (threadIdx.x == 0) s_saved = 0;
  for (int g = threadIdx.x; g < p.n_groups; g += kPlanThreads) {
    int c0, c1;
    const bool good = group_of(p, g, c0, c1);
    const int given = p.prefix_lens[g];
    const int len = given < 0 ? 0 : (given > p.cap ? (int)p.cap : given);
    if ((!good || given != len) && p.err) atomicOr(p.err, kErrBadArgs);
    SharedGroup s{};
    s.eff = good && c1 - c0 > 1 ? len / kBlock * kBlock : 0;
    s.ref = INT_MAX;
    s.first = c0;
    s.count = good ? c1 - c0 : 0;
    groups[g] = s;
  }
  __syncthreads();
  // The first sequence of a group that has all of the prefix names its pages.
  SharedSeq first_seq{};  // of this thread's first sequence
  unsigned long long saved = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int lo = 0, hi = p.n_groups - 1;  // the last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (groups[mid].first <= b)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int eff = groups[lo].eff, from = groups[lo].first, count = groups[lo].count;
    const long long len = b0 == 0 ? first_len : (b < p.B ? p.seqlens[b] : 0);
    const bool in = b < p.B && eff > 0 && b >= from && b - from < count && min(len, p.cap) >= eff;
    const int key = in ? lo : -1, before = __shfl_up_sync(0xffffffffu, key, 1);
    if (in && (lane == 0 || before != key)) atomicMin(&groups[lo].ref, b);  // one of a warp's of a group
    saved += in ? eff : 0;
    const SharedSeq s{in ? eff : 0, lo, 0, 0};
    if (b0 == 0) first_seq = s;
    if (b0 > 0 && b < p.B) p.seqs[b] = s;
  }
  __syncthreads();
  auto ref_of = [&](int g) { return LOCAL ? groups[g].ref : __ldcg(&groups[g].ref); };
  for (int g = threadIdx.x; g < p.n_groups; g += kPlanThreads)  // one of each group does read them
    if (groups[g].eff > 0 && ref_of(g) != INT_MAX) saved -= groups[g].eff;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) saved += __shfl_xor_sync(0xffffffffu, saved, off);
  if (lane == 0 && saved) atomicAdd(&s_saved, saved);
  __syncthreads();
  const bool worth = (long long)s_saved >= p.least_saved;
  long long blocks_before = 0, units_before = 0;
  for (int g0 = 0; g0 < p.n_groups; g0 += kPlanThreads) {
    const int g = g0 + threadIdx.x;
    int blocks = 0, n = 0;
    if (g < p.n_groups && worth && groups[g].eff > 0 && ref_of(g) != INT_MAX) {
      blocks = (groups[g].count + block_seqs - 1) / block_seqs;
      n = groups[g].eff / kBlock + 1;  // and one for starting and finishing an item
    }
    long long upto = blocks, units_upto = (long long)blocks * p.Hkv * n;
    const long long units = units_upto;
    block_sums_upto(upto, units_upto, s_sum);
    upto += blocks_before;
    units_upto += units_before;
    // More blocks than there is room for: offsets that overlap. Left out, and all after them.
    const bool fits = upto <= p.max_blocks;
    if (!fits && blocks > 0 && p.err) atomicOr(p.err, kErrBadArgs);
    if (g < p.n_groups) {
      groups[g].block0 = (int)(upto - blocks);
      groups[g].unit0 = units_upto - units;
      if (!fits || blocks == 0) groups[g].count = 0;
      if constexpr (LOCAL) p.groups[g] = groups[g];
    }
    // The units end where the first group that does not fit begins.
    const bool last = g == p.n_groups - 1;
    if (fits ? last : upto - blocks <= p.max_blocks) *p.total = fits ? units_upto : units_upto - units;
    if (g0 + kPlanThreads < p.n_groups) {
      __syncthreads();
      if (threadIdx.x == kPlanThreads - 1) s_sum[0][0] = upto, s_sum[0][1] = units_upto;
      __syncthreads();
      blocks_before = s_sum[0][0];
      units_before = s_sum[0][1];
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.B; b += kPlanThreads) {
    SharedSeq s = b < kPlanThreads ? first_seq : p.seqs[b];
    if (s.skip > 0) {
      const SharedGroup* g = groups + s.block;  // still the group's number
      const int i = b - g->first, at = i % block_seqs;
      if (g->count == 0)
        s = SharedSeq{0, 0, 0, 0};
      else
        s = SharedSeq{s.skip, g->block0 + i / block_seqs, at / tile_seqs * 128 + at % tile_seqs * p.group, 0};
    }
    p.seqs[b] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) st_release(p.ready, kPlanReady);  // and with it what the others wrote
}

// ---------------------------------------------------------------- the shared keys
// Units per CTA, at least: fewer CTAs leave the others' SMs to the kernel over
// each sequence's own keys (measured with 1 and 2 as well: up to 5 us slower at
// 8 to 16 sequences behind 2048 to 8192 keys, 2 us faster behind 1024).
constexpr int kMinShare = 4;

// A stretch of the units, item by item.
struct ItemWalk {
  const DecodeSharedParams& p;
  int block_seqs;
  long long left;  // units from this item's first one here to the stretch's end
  int gi;          // the group
  SharedGroup g;
  int item;        // row block * Hkv + KV head, within the group
  int begin, end;  // key blocks of the item in the stretch
  __device__ __forceinline__ int blocks() const { return (g.count + block_seqs - 1) / block_seqs; }
  __device__ __forceinline__ int units() const { return g.eff / kBlock + 1; }
  // `mine`: the lane's group of up to 32, requested before `from` was known.
  __device__ __forceinline__ ItemWalk(const DecodeSharedParams& params, int seqs, long long from, long long count,
                                      SharedGroup mine)
      : p(params), block_seqs(seqs), left(count) {
    // The last group that starts at or before the unit: 32 looked at a time, and the last 32 read whole.
    const int lane = threadIdx.x & 31;
    int lo = 0, len = p.n_groups;
    while (len > 32) {
      const int step = (len + 31) / 32;
      const bool before =
          lane * step < len && (lane == 0 || __ldcg(&p.groups[lo + lane * step].unit0) <= from);
      const int hit = 31 - __clz(__ballot_sync(0xffffffffu, before));
      len = min(step, len - hit * step);
      lo += hit * step;
    }
    if (p.n_groups > 32 && lane < len) mine = load_group(p.groups + lo + lane);
    const int hit = 31 - __clz(__ballot_sync(0xffffffffu, lane < len && (lane == 0 || mine.unit0 <= from)));
    gi = lo + hit;
    g.eff = __shfl_sync(0xffffffffu, mine.eff, hit);
    g.ref = __shfl_sync(0xffffffffu, mine.ref, hit);
    g.first = __shfl_sync(0xffffffffu, mine.first, hit);
    g.count = __shfl_sync(0xffffffffu, mine.count, hit);
    g.block0 = __shfl_sync(0xffffffffu, mine.block0, hit);
    g.unit0 = __shfl_sync(0xffffffffu, mine.unit0, hit);
    const long long into = from - g.unit0;
    item = (int)(into / units());
    begin = (int)(into % units());
    end = (int)min((long long)units() - 1, begin + left);
    if (begin == units() - 1) next();  // only the item's extra unit is here
  }
  __device__ __forceinline__ bool valid() const { return left > 0; }
  __device__ __forceinline__ bool next() {
    left -= units() - begin;
    if (left <= 0) return false;
    begin = 0;
    if (++item == blocks() * p.Hkv) {
      item = 0;
      do {
        if (++gi >= p.n_groups) {
          left = 0;
          return false;
        }
        g = load_group(p.groups + gi);
      } while (g.count == 0);
    }
    end = (int)min((long long)units() - 1, left);
    return true;
  }
  __device__ __forceinline__ int head() const { return item % p.Hkv; }
  __device__ __forceinline__ int first_seq() const { return g.first + item / p.Hkv * block_seqs; }
  __device__ __forceinline__ int seqs() const { return min(block_seqs, g.count - item / p.Hkv * block_seqs); }
  __device__ __forceinline__ long long number() const { return (long long)g.block0 * p.Hkv + item; }
};

template <int D>
__global__ void __launch_bounds__(SharedCfg<D>::THREADS, 1)
    decode_shared_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DecodeSharedParams p) {
  using C = SharedCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  SharedBars* bars = reinterpret_cast<SharedBars*>(smem + C::OFF_BAR);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int tile_seqs = 128 / p.group, block_seqs = C::NQT * tile_seqs, tile_rows = tile_seqs * p.group;
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_free, C::NQT);
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], C::NQT);
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], C::NQT);
    }
    for (int t = 0; t < C::NQT; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[t][b], 1);
        mbar_init(&bars->p_full[t][b], 4);
        mbar_init(&bars->pv_done[t][b], 1);
      }
      mbar_init(&bars->drain[t], 1);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // Rows past the tile's sequences stay zero.
  for (int e = threadIdx.x; e < C::NQT * C::Q_BYTES / 16; e += C::THREADS)
    st_shared_v4(smem_u32(smem) + 16 * e, 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  grid_dep_wait();
  grid_dep_launch();
  const SharedGroup mine = p.n_groups <= 32 && lane < p.n_groups ? load_group(p.groups + lane) : SharedGroup{};
  const long long total = __ldcg(p.total);
  const long long share = max((total + p.n_ctas - 1) / p.n_ctas, (long long)kMinShare);
  const long long from = blockIdx.x * share, count = min(share, total - from);
  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err));
  };

  if (count > 0) {
    ItemWalk w(p, block_seqs, from, count, mine);
    if (warp == 0 && w.valid()) {
      // ---------------------------------------------------------- producer
      // Lane x copies 64 columns of one run of box_rows keys of a tile. The
      // page of the next block's run is looked up one block ahead.
      const int br = p.box_rows, boxes = kBlock / br;
      const int box = lane % boxes, chunk = lane / boxes;
      const bool mine = chunk < C::KCH;
      const uint32_t at = chunk * C::KV_CHUNK + box * br * 128;
      int kn = 0, vn = 0, qn = 0;  // K and V tiles and items copied so far
      bool ok = true;
      do {
        const int* table = p.block_table + w.g.ref * p.table_ld;
        const int head = w.head();
        auto entry_of = [&](int j) -> int {
          const int e = (j * kBlock + box * br) / p.page;
          return mine && j < w.end && e < p.table_width ? table[e] : 0;
        };
        auto copy = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* full, int j, int entry) {
          if (lane == 0) mbar_arrive_expect_tx(full, C::TILE_BYTES);
          __syncwarp();
          if (mine) {
            const bool in_pool = entry >= 0 && entry < p.n_pages;
            if (!in_pool && p.err) atomicOr(p.err, kErrBadArgs);
            tma_load_5d(dst + at, map, full, 0, (j * kBlock + box * br) % p.page, chunk, head, in_pool ? entry : 0);
          }
        };
        int entry = entry_of(w.begin), last = 0;
        if (qn > 0 && !wait_all(&bars->q_free, (uint32_t)(qn - 1) & 1u)) break;
        const int tiles = w.seqs() > tile_seqs ? C::NQT : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->q_full, tiles * C::KCH * tile_rows * 128);
          for (int t = 0; t < tiles; ++t)
            for (int c = 0; c < C::KCH; ++c)
              tma_load_3d(smem + t * C::Q_BYTES + c * C::Q_CHUNK, &tm_q, &bars->q_full, 64 * c, head * p.group,
                          w.first_seq() + t * tile_seqs);
        }
        __syncwarp();
        ++qn;
        for (int j = w.begin; ok && j <= w.end; ++j) {
          if (j < w.end) {
            const int slot = kn % C::KST;
            if (!(ok = wait_all(&bars->k_empty[slot], ((uint32_t)(kn / C::KST) & 1u) ^ 1u))) break;
            copy(&tm_k, smem + C::OFF_K + slot * C::TILE_BYTES, &bars->k_full[slot], j, entry);
            ++kn;
          }
          const int next = entry_of(j + 1);
          if (j > w.begin) {
            const int slot = vn % C::VST;
            if (!(ok = wait_all(&bars->v_empty[slot], ((uint32_t)(vn / C::VST) & 1u) ^ 1u))) break;
            copy(&tm_v, smem + C::OFF_V + slot * C::TILE_BYTES, &bars->v_full[slot], j - 1, last);
            ++vn;
          }
          last = entry;
          entry = next;
        }
      } while (ok && w.next());
      if (*abort_flag && lane == 0) {
        // Let every copy still in flight land before the CTA releases smem.
        if (qn > 0) mbar_wait_quiet(&bars->q_full, (uint32_t)(qn - 1) & 1u);
        for (int i = max(0, kn - C::KST); i < kn; ++i)
          mbar_wait_quiet(&bars->k_full[i % C::KST], (uint32_t)(i / C::KST) & 1u);
        for (int i = max(0, vn - C::VST); i < vn; ++i)
          mbar_wait_quiet(&bars->v_full[i % C::VST], (uint32_t)(i / C::VST) & 1u);
      }
    } else if (warp >= 1 && warp <= C::NQT && w.valid()) {
      // ---------------------------------------------------------- MMA issue, tile t
      const int t = warp - 1;
      constexpr uint32_t IDESC_S = umma_idesc_bf16(128, kBlock, false);
      constexpr uint32_t IDESC_PV = umma_idesc_bf16(128, D, true);
      const uint64_t dQ = make_sdesc_sw128(smem_u32(smem + t * C::Q_BYTES), 16, 1024);
      const uint64_t dK = make_sdesc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
      const uint64_t dV = make_sdesc_sw128(smem_u32(smem + C::OFF_V), C::KV_CHUNK, 1024);
      const uint32_t tS = tmem + C::S_COL + 128 * t, tO = tmem + C::O_COL + D * t;
      int kn = 0, vn = 0, qn = 0;  // K and V tiles and items taken so far
      int c = 0;                   // key blocks of this tile so far
      bool ok = true;
      auto wait_k = [&](int i) { return wait_all(&bars->k_full[i % C::KST], (uint32_t)(i / C::KST) & 1u); };
      auto wait_v = [&](int i) { return wait_all(&bars->v_full[i % C::VST], (uint32_t)(i / C::VST) & 1u); };
      // S of key block j of the item: K-steps of 16 columns walk 32 bytes inside a 128-byte row, then the next chunk.
      auto issue_S = [&](int j) {
        const int slot = (kn + j) % C::KST, buf = (c + j) & 1;
        const uint64_t ka = dK + (uint64_t)((slot * C::TILE_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t qo = (uint64_t)(((k >> 2) * C::Q_CHUNK + (k & 3) * 32) >> 4);
          const uint64_t ko = (uint64_t)(((k >> 2) * C::KV_CHUNK + (k & 3) * 32) >> 4);
          umma_bf16_ss_w(tS + kBlock * buf, dQ + qo, ka + ko, IDESC_S, k > 0 ? 1u : 0u);
        }
        tc_commit_w(&bars->s_full[t][buf]);
        tc_commit_w(&bars->k_empty[slot]);
      };
      do {
        const int n = w.end - w.begin;
        if (w.seqs() > t * tile_seqs) {
          ok = wait_all(&bars->q_full, (uint32_t)qn & 1u);
          for (int j = 0; ok && j < min(n, 2); ++j) {
            if (!(ok = wait_k(kn + j))) break;
            tc_fence_after();
            issue_S(j);
          }
          if (n <= 2) tc_commit_w(&bars->q_free);  // the item's last S is issued
          for (int j = 0; ok && j < n; ++j) {
            const int buf = (c + j) & 1, slot = (vn + j) % C::VST;
            if (!(ok = wait_v(vn + j))) break;
            if (!(ok = wait_all(&bars->p_full[t][buf], (uint32_t)((c + j) >> 1) & 1u))) break;
            tc_fence_after();
            const uint64_t va = dV + (uint64_t)((slot * C::TILE_BYTES) >> 4);
#pragma unroll
            for (int s = 0; s < kBlock / 16; ++s)
              umma_bf16_ts_w(tO, tS + kBlock * buf + 8 * s, va + (uint64_t)((s * 2048) >> 4), IDESC_PV,
                             j > 0 || s > 0 ? 1u : 0u);
            tc_commit_w(&bars->pv_done[t][buf]);
            tc_commit_w(&bars->v_empty[slot]);
            if (j + 2 < n) {
              if (!(ok = wait_k(kn + j + 2))) break;
              tc_fence_after();
              issue_S(j + 2);
              if (j + 3 == n) tc_commit_w(&bars->q_free);
            }
          }
          c += n;
        } else {
          // No sequence in this tile: its shares of the tiles are given back as they land, in the order they come.
          for (int j = 0; ok && j <= n; ++j) {
            if (j < n) {
              if (!(ok = wait_k(kn + j))) break;
              if (lane == 0) mbar_arrive(&bars->k_empty[(kn + j) % C::KST]);
            }
            if (j > 0) {
              if (!(ok = wait_v(vn + j - 1))) break;
              if (lane == 0) mbar_arrive(&bars->v_empty[(vn + j - 1) % C::VST]);
            }
          }
          if (ok) ok = wait_all(&bars->q_full, (uint32_t)qn & 1u);
          if (ok && lane == 0) mbar_arrive(&bars->q_free);
        }
        kn += n;
        vn += n;
        ++qn;
      } while (ok && w.next());
      // Every MMA issued above must finish before TMEM is deallocated.
      tc_commit_w(&bars->drain[t]);
      mbar_wait_quiet(&bars->drain[t], 0);
    } else if (warp >= 4 && w.valid()) {
      // ---------------------------------------------------------- softmax and partials, tile t
      const int t = (warp - 4) >> 2, wq = warp & 3;
      const int row = wq * 32 + lane;
      const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
      const uint32_t tS = tmem + lane_off + C::S_COL + 128 * t, tO = tmem + lane_off + C::O_COL + D * t;
      const float sl2 = p.scale_log2;
      int c = 0;  // key blocks of this tile so far
      bool ok = true;
      // PV of block i is done. A parity tells a phase from its neighbours only, so a warp must neither miss one nor
      // fall two behind: with a barrier for either buffer, PV(i + 2) needs this warp's P(i + 2), which comes after its
      // wait for PV(i) (in block i + 2 at the latest).
      auto product_done = [&](int i) { return wait_all(&bars->pv_done[t][i & 1], (uint32_t)(i >> 1) & 1u); };
      do {
        if (w.seqs() <= t * tile_seqs) continue;
        const int n = w.end - w.begin;
        float m_run = -INFINITY, l_run = 0.f;
        for (int j = 0; j < n; ++j, ++c) {
          const int buf = c & 1;
          if (!(ok = wait_all(&bars->s_full[t][buf], (uint32_t)(c >> 1) & 1u))) break;
          if (c > 1 && !(ok = product_done(c - 2))) break;  // issued before S(c)
          tc_fence_after();
          uint32_t s[2][32];
          tmem_ld32(tS + kBlock * buf, s[0]);
          tmem_ld32(tS + kBlock * buf + 32, s[1]);
          tmem_wait_ld();
          float hs;
          const float a = softmax_half_tmem<0>(s, 63, sl2, m_run, tS + kBlock * buf, hs);
          l_run = fmaf(l_run, a, hs);
          if (j > 0 && __any_sync(0xffffffffu, a != 1.f)) {
            // Rare: the running maximum moved. O holds the blocks before this one once their products are done.
            if (!(ok = product_done(c - 1))) break;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
              uint32_t o[32];
              tmem_ld32(tO + 32 * x, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = f2u(u2f(o[i]) * a);
              tmem_st32(tO + 32 * x, o);
            }
          }
          // P and O are in TMEM before the MMA may read them.
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->p_full[t][buf]);
        }
        if (!ok || !(ok = product_done(c - 1))) break;
        tc_fence_after();
        const long long at = (w.number() + blockIdx.x) * (128 * C::NQT) + 128 * t + row;
        const bool used = row < tile_rows && row / p.group < w.seqs() - t * tile_seqs;
#pragma unroll 1
        for (int x = 0; x < D / 32; ++x) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * x, o);
          tmem_wait_ld();
          if (used) {
            float* dst = p.part_o + at * D + 32 * x;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              st_global_v8(dst + i, o[i], o[i + 1], o[i + 2], o[i + 3], o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
          }
        }
        if (used) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m_run, l_run);
        if (t == 0 && row == 0) {
          if (w.begin == 0) p.place[2 * w.number()] = blockIdx.x;
          if (w.end == w.units() - 1) p.place[2 * w.number() + 1] = blockIdx.x;
        }
      } while (w.next());
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int D>
int launch_t(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const DecodeSharedParams& p,
             cudaStream_t st) {
  using C = SharedCfg<D>;
  static OncePerDevice once;
  return once.run(
      [] {
        return cudaFuncSetAttribute(decode_shared_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::SMEM_BYTES) == cudaSuccess;
      },
      [&] {
        return launch_dependent(decode_shared_kernel<D>, dim3((unsigned)p.n_ctas), C::THREADS, C::SMEM_BYTES, st, 0,
                                tq, tk, tv, p);
      });
}

}  // namespace

int decode_shared_block_seqs(int D, int group) { return (D == 256 ? 1 : 2) * (128 / group); }
int decode_shared_block_rows(int D) { return D == 256 ? 128 : 256; }
int decode_shared_max_ctas(int sms) { return sms; }

int launch_decode_shared(int D, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                         const SharedPlanParams& plan, const DecodeSharedParams& p, cudaStream_t st) {
  const bool local = plan.n_groups <= kLocalGroups;
  const auto kernel = local ? decode_shared_plan_kernel<true> : decode_shared_plan_kernel<false>;
  if (launch_dependent(kernel, dim3(1), kPlanThreads, 0, st, 0, plan, decode_shared_block_seqs(D, plan.group),
                       128 / plan.group) != cudaSuccess)
    return -1;
  switch (D) {
    case 64: return launch_t<64>(tq, tk, tv, p, st);
    case 128: return launch_t<128>(tq, tk, tv, p, st);
    case 256: return launch_t<256>(tq, tk, tv, p, st);
    default: return -3;
  }
}

}  // namespace b2a
