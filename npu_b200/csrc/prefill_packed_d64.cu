// Causal GQA attention over packed sequences at head dim 64: one query tile
// of 128 rows a CTA, two CTAs an SM, and the keys shared by two softmax
// warpgroups.
//
// A tile's work per key is small at this head dim (64 MACs a score and an
// exponential), so what bounds it is how many warps there are to issue it: with
// one softmax warpgroup a CTA the two warps of a scheduler issued every third
// cycle. Here warpgroup h takes keys [64 h, 64 h + 64) of every 128-key block,
// with a score region S_h, a running maximum and sum and an output accumulator
// O_h of its own, and runs through its blocks without a word to the other. At
// the item's end the two partial results are joined as those of a split over
// the keys are: with M = max(m_0, m_1) and f_h = 2^(m_h - M),
//   o = (f_0 O_0 + f_1 O_1) / (f_0 l_0 + f_1 l_1),
// each warpgroup for 32 of the 64 columns.
//
// TMEM (256 columns): S_0, S_1 (64 each), O_0, O_1 (64 each). P_h(j) (bf16, two
// keys a column) replaces the first half of S_h(j); S_h(j+1) is issued behind
// PV_h(j) by the same thread, so it follows it in order and its barrier also
// says that O_h may be touched. The scores are read twice (maximum, then
// exponentials), 32 columns at a time: nothing is redone, and the loop stays a
// few KB of instructions, which matters more here than the second read (see
// softmax_half_packed). Kept in registers between the two, the scores spill.
//
// Measured on one B200 (device time): 32 prompts of 17 to 2048 tokens, 9 / 3
// heads, 42.2 us against 49.5 with one softmax warpgroup of 64 scores a thread
// (prefill.cu's one-tile items); 4 prompts of 4096, 129 us against 146.8 with
// its two-tile items; 3 prompts of 1 to 40, 5.9 to 6.3 us against 7.1. A
// block of 128 keys takes 1.9 us a CTA, of which MUFU is busy 1.1 (both CTAs);
// the rest is the way from P through PV and S to the next scores, 0.55 us.
//
// Warps: 0 producer, 1 and 2 UMMA issuers of the halves, 3 scheduler (work
// items as in prefill.cu), 4-7 and 8-11 softmax and epilogue.
#include "capi_internal.cuh"
#include "packed.cuh"
#include "prefill.cuh"
#include "softmax.cuh"

namespace b2a {

namespace {

struct Cfg {
  static constexpr int D = 64, BM = 128, BN = 128, HALF = 64;
  static constexpr int TILE_BYTES = 128 * D * 2;  // Q, K and V tiles
  static constexpr int STAGES = 5;
  static constexpr int OFF_KV = TILE_BYTES;
  static constexpr int OFF_BAR = OFF_KV + STAGES * TILE_BYTES;
  static constexpr int BAR_BYTES = 2560;
  static constexpr int SMEM_BYTES = OFF_BAR + BAR_BYTES + 1024;  // + alignment slack
  static constexpr int TMEM_COLS = 256;
  static constexpr int O_COL = 2 * HALF;
  static constexpr int THREADS = 384;
  // Registers a thread at launch, which the control warps then give to the
  // softmax warps.
  static constexpr int REGS = 80, REGS_LOW = 48, REGS_HIGH = 96;
  static_assert(128 * REGS_LOW + 256 * REGS_HIGH <= THREADS * REGS, "setmaxnreg split");
  static_assert(2 * THREADS * REGS <= 65536, "two CTAs an SM");
  static constexpr int CONSUMER_WARPS = 11;  // take every item from the scheduler
  static_assert(2 * SMEM_BYTES <= 232448 - 1024, "two CTAs an SM");
};

struct Bars {
  uint64_t q_full, q_free;
  uint64_t kv_full[Cfg::STAGES], kv_empty[Cfg::STAGES];
  uint64_t s_full[2];  // S_h(j) is in TMEM, and PV_h(j-1) is complete
  uint64_t p_full[2];  // P_h(j) is in TMEM and O_h at its maximum
  uint64_t o_full[2];  // the item's last PV_h is complete
  uint64_t drain[2];
  uint64_t item_full[2], item_empty[2], clc_bar;
  alignas(16) uint8_t clc_resp[16];
  int item_id[2];
  PackedBlock item_at[3];  // the ring's two, and the CTA's own
  uint32_t tmem_base;
  int abort_flag;
  float2 ml[2][Cfg::BM];  // a row's maximum and sum by each warpgroup
};
static_assert(sizeof(Bars) <= Cfg::BAR_BYTES, "barrier region");

// A CTA's work: query block `at` for query head h.
struct Item {
  int h, hk, q_row, k_row;  // first row in q, first key in k
  int rows, keys, q0, sp;   // of the sequence; the block's first row in it
  int n[2];                 // key blocks of each half; n[0] are loaded
};

__device__ __forceinline__ Item item_of(const PrefillParams& p, int lin, const PackedBlock& at) {
  Item it;
  it.h = lin % p.Hq;
  it.hk = it.h / (p.Hq / p.Hkv);
  it.q0 = at.qblk * Cfg::BM;
  it.rows = at.rows;
  it.keys = at.rows > 0 ? at.keys : 0;
  it.q_row = at.q_base + it.q0;
  it.k_row = at.k_base;
  it.sp = at.keys - at.rows;
  int end = it.keys;
  if (p.causal) end = min(end, it.sp + min(it.q0 + Cfg::BM, it.rows));
  const int halves = end <= 0 ? 0 : (end + Cfg::HALF - 1) / Cfg::HALF;
  it.n[0] = (halves + 1) / 2;
  it.n[1] = halves / 2;
  return it;
}

// All 256 softmax threads meet; true if it holds for each.
__device__ __forceinline__ bool softmax_warps_agree(bool ok) {
  int all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.and.aligned.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((int)ok)
      : "memory");
  return all != 0;
}

// 32 scores; those past column `lim` become -inf.
__device__ __forceinline__ void load_scores(uint32_t tS, int lim, uint32_t (&s)[32]) {
  tmem_ld32(tS, s);
  tmem_wait_ld();
  if (!__all_sync(0xffffffffu, lim >= 31)) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i > lim) s[i] = f2u(-INFINITY);
  }
}

__global__ void __launch_bounds__(Cfg::THREADS, 2)
    prefill_packed_d64_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PrefillParams p) {
  using C = Cfg;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + C::OFF_KV;
  Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_wait();

  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err));
  };
  // The CTA's item number n >= 1, -1 when there is none or on abort.
  PackedBlock at{};
  auto next_item = [&](int n) -> int {
    const int slot = (n - 1) & 1;
    if (!wait_all(&bars->item_full[slot], (uint32_t)((n - 1) >> 1) & 1u)) return -1;
    const int id = *reinterpret_cast<volatile int*>(&bars->item_id[slot]);
    at = bars->item_at[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->item_empty[slot]);
    return id;
  };

  if (warp == 0) {
    PackedBlocks<C::BM> blocks(p);
    at = blocks.find(blockIdx.x / p.Hq);
    if (lane == 0) {
      bars->item_at[2] = at;
      mbar_init(&bars->q_full, 1);
      mbar_init(&bars->q_free, 2);  // each issuer, after its last S of an item
      for (int s = 0; s < C::STAGES; ++s) {
        mbar_init(&bars->kv_full[s], 1);
        mbar_init(&bars->kv_empty[s], 2);
      }
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars->s_full[h], 1);
        mbar_init(&bars->p_full[h], 4);  // one arrive per softmax warp
        mbar_init(&bars->o_full[h], 1);
        mbar_init(&bars->drain[h], 1);
        mbar_init(&bars->item_full[h], 1);
        mbar_init(&bars->item_empty[h], C::CONSUMER_WARPS);
      }
      mbar_init(&bars->clc_bar, 1);
      bars->abort_flag = 0;
      fence_mbar_init();
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  // The producer's loads of item `it` from load i0 on (K_j = 2 j, V_j = 2 j + 1;
  // load g of the CTA uses slot g % STAGES in round g / STAGES).
  int ld = 0, issued = 0;
  auto load_q = [&](const Item& it) {
    mbar_arrive_expect_tx_w(&bars->q_full, C::TILE_BYTES);
    tma_load_4d_w(sQ, &tm_q, &bars->q_full, 0, it.q_row, it.h, 0);
  };
  auto load_kv = [&](const Item& it, int i) -> bool {
    const int g = ld + i, slot = g % C::STAGES;
    if (!wait_all(&bars->kv_empty[slot], ((uint32_t)(g / C::STAGES) & 1u) ^ 1u)) return false;
    mbar_arrive_expect_tx_w(&bars->kv_full[slot], C::TILE_BYTES);
    tma_load_4d_w(sKV + slot * C::TILE_BYTES, (i & 1) ? &tm_v : &tm_k, &bars->kv_full[slot], 0,
                  it.k_row + (i >> 1) * C::BN, it.hk, 0);
    issued = g + 1;
    return true;
  };
  // The first item's first tiles are requested before the block barrier.
  int first_loads = 0;
  if (warp == 0) {
    const Item it = item_of(p, blockIdx.x, at);
    if (it.n[0] > 0) {
      load_q(it);
      for (; first_loads < min(C::STAGES, 2 * it.n[0]); ++first_loads) load_kv(it, first_loads);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  at = bars->item_at[2];
  int lin = blockIdx.x;

  // Each role's code sits inside the branch that set its register budget, so
  // the compiler allocates it against that budget.
  if (warp < 4) {
  setmaxnreg_dec<C::REGS_LOW>();
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int q_rounds = 0;  // items with keys
    bool ok = true;
    for (int n = 1;; ++n) {
      const Item it = item_of(p, lin, at);
      if (it.n[0] > 0) {
        if (n > 1) {
          // Every S MMA of the previous item with keys is complete.
          if (q_rounds > 0 && !wait_all(&bars->q_free, (uint32_t)(q_rounds - 1) & 1u)) break;
          load_q(it);
        }
        ++q_rounds;
        for (int i = n == 1 ? first_loads : 0; ok && i < 2 * it.n[0]; ++i) ok = load_kv(it, i);
        if (!ok) break;
        ld += 2 * it.n[0];
      }
      lin = next_item(n);
      if (lin < 0) break;
    }
    if (*abort_flag && lane == 0) {
      // Let every copy still in flight land before the CTA releases smem.
      if (q_rounds > 0) mbar_wait_quiet(&bars->q_full, (uint32_t)(q_rounds - 1) & 1u);
      for (int g = max(0, issued - C::STAGES); g < issued; ++g)
        mbar_wait_quiet(&bars->kv_full[g % C::STAGES], (uint32_t)(g / C::STAGES) & 1u);
    }
  } else if (warp <= 2) {
    // ------------------------------------------------------------ UMMA issuers
    const int h = warp - 1;
    constexpr uint32_t IDESC_S = umma_idesc_bf16(128, C::HALF, false);
    constexpr uint32_t IDESC_PV = umma_idesc_bf16(128, C::D, true);
    const uint64_t dQ = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
    // Keys 64 h on: 64 rows of 128 bytes into the K and V tiles.
    const uint64_t dK = make_sdesc_sw128(smem_u32(sKV) + h * C::HALF * 128, 16, 1024);
    const uint64_t dV = make_sdesc_sw128(smem_u32(sKV) + h * C::HALF * 128, C::TILE_BYTES, 1024);
    const uint32_t dS = tmem + h * C::HALF, dO = tmem + C::O_COL + h * C::D;
    auto issue_S = [&](int slot) {
      const uint64_t ka = dK + (uint64_t)((slot * C::TILE_BYTES) >> 4);
#pragma unroll
      for (int k = 0; k < C::D / 16; ++k) umma_bf16_ss_w(dS, dQ + 2 * k, ka + 2 * k, IDESC_S, k > 0 ? 1u : 0u);
    };
    auto issue_PV = [&](int slot, bool acc) {
      const uint64_t va = dV + (uint64_t)((slot * C::TILE_BYTES) >> 4);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        umma_bf16_ts_w(dO, dS + 8 * s, va + (uint64_t)((s * 2048) >> 4), IDESC_PV, (acc || s > 0) ? 1u : 0u);
    };
    int G = 0, J = 0, q_rounds = 0;
    bool ok = true;
    for (int n = 1;; ++n) {
      const Item it = item_of(p, lin, at);
      const int nt = h == 0 ? it.n[0] : it.n[1];
      if (it.n[0] > 0) {
        auto slot_of = [&](int i) { return (G + i) % C::STAGES; };
        auto wait_load = [&](int i) -> bool {
          return wait_all(&bars->kv_full[slot_of(i)], (uint32_t)((G + i) / C::STAGES) & 1u);
        };
        auto next_S = [&](int j) {  // S_h(j); K_j has landed
          issue_S(slot_of(2 * j));
          tc_commit_w(&bars->s_full[h]);
          tc_commit_w(&bars->kv_empty[slot_of(2 * j)]);
          if (j + 1 == nt) tc_commit_w(&bars->q_free);
        };
        ok = wait_all(&bars->q_full, (uint32_t)q_rounds & 1u);
        ++q_rounds;
        ok = ok && (nt == 0 || wait_load(0));
        tc_fence_after();
        if (ok && nt > 0) next_S(0);
        if (ok && nt == 0) tc_commit_w(&bars->q_free);  // this half reads no Q in this item
        for (int j = 0; ok && j < nt; ++j) {
          const int vslot = slot_of(2 * j + 1);
          ok = wait_load(2 * j + 1) && (j + 1 == nt || wait_load(2 * j + 2));
          if (!ok) break;
          // The last block may reach into the next sequence's rows of V, and
          // a P of 0 does not hide a NaN there: clear this half's.
          const int from = max(it.keys - j * C::BN, h * C::HALF), to = (h + 1) * C::HALF;
          if (from < to) clear_v_rows<C::D>(smem_u32(sKV) + vslot * C::TILE_BYTES, from, to, C::TILE_BYTES);
          ok = wait_all(&bars->p_full[h], (uint32_t)(J + j) & 1u);
          if (!ok) break;
          tc_fence_after();
          issue_PV(vslot, j > 0);
          tc_commit_w(&bars->kv_empty[vslot]);
          if (j + 1 < nt)
            next_S(j + 1);
          else
            tc_commit_w(&bars->o_full[h]);
        }
        // The last block's tiles, if this half has no key in it: released once
        // they have landed (the slot is then in the round of that load).
        for (int i = 2 * nt; ok && i < 2 * it.n[0]; ++i) {
          ok = wait_load(i);
          if (ok && lane == 0) mbar_arrive(&bars->kv_empty[slot_of(i)]);
        }
        G += 2 * it.n[0];
        J += nt;
      }
      if (!ok) break;
      lin = next_item(n);
      if (lin < 0) break;
    }
    // Every MMA issued above must finish before TMEM is deallocated.
    tc_commit_w(&bars->drain[h]);
    mbar_wait_quiet(&bars->drain[h], 0);
  } else {
    // ------------------------------------------------------------ scheduler
    PackedBlocks<C::BM> blocks(p);
    for (int n = 1;; ++n) {
      if (n >= 2 && !wait_all(&bars->item_empty[n & 1], (uint32_t)((n - 2) >> 1) & 1u)) break;
      const uint32_t cpar = (uint32_t)(n - 1) & 1u;
      if (lane == 0) {
        fence_proxy_async_smem();  // the previous response was read through the generic proxy
        mbar_arrive_expect_tx(&bars->clc_bar, 16);
        clc_try_cancel(bars->clc_resp, &bars->clc_bar);
      }
      __syncwarp();
      if (!wait_all(&bars->clc_bar, cpar)) {
        // Abort: the response must still land before shared memory goes away.
        if (lane == 0) mbar_wait_quiet(&bars->clc_bar, cpar);
        break;
      }
      const int id = clc_cancelled_ctaid_x(bars->clc_resp);
      __syncwarp();
      if (id >= 0) at = blocks.find(id / p.Hq);
      if (lane == 0) {
        bars->item_id[(n - 1) & 1] = id;
        bars->item_at[(n - 1) & 1] = at;
        mbar_arrive(&bars->item_full[(n - 1) & 1]);
      }
      __syncwarp();
      if (id < 0) break;
    }
  }
  } else {
    setmaxnreg_inc<C::REGS_HIGH>();
    // ------------------------------------------------------------ softmax + epilogue
    const int h = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = lanes + h * C::HALF, tO = lanes + C::O_COL + h * C::D;
    const float sl2 = p.scale_log2;
    int J = 0;                // this half's key blocks in earlier items
    int o_rounds[2] = {0, 0};  // items in which each half had some
    for (int n = 1;; ++n) {
      const Item it = item_of(p, lin, at);
      const bool valid = it.q0 + row < it.rows;
      // The row's last visible key, counted from this half's first; rows past
      // the sequence's end, the next one's queries, see none.
      const int last =
          valid ? (p.causal ? min(it.sp + it.q0 + row, it.keys - 1) : it.keys - 1) - h * C::HALF : -C::HALF - 1;
      float m_run = -INFINITY, l_run = 0.f;
      bool ok = true;
      const int nt = h == 0 ? it.n[0] : it.n[1];
#pragma unroll 1
      for (int j = 0; j < nt; ++j) {
        const int lim = last - j * C::BN;
        ok = wait_all(&bars->s_full[h], (uint32_t)(J + j) & 1u);
        if (!ok) break;
        tc_fence_after();
        // 32-column chunks that some row of the warp sees: the others are
        // neither read nor computed (three of eight on the diagonal, and
        // warps past the sequence's end).
        const int chunks = max(min(__reduce_max_sync(0xffffffffu, lim) + 32, 64) >> 5, 0);
        uint32_t s[32];
        float mx = -INFINITY, my = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          load_scores(tS + 32 * c, lim - 32 * c, s);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            mx = fmax3(mx, u2f(s[i]), u2f(s[i + 1]));
            my = fmax3(my, u2f(s[i + 2]), u2f(s[i + 3]));
          }
        }
        // A row's maximum moves when it had none (O_h is then a sum of zeros)
        // or past the threshold.
        const float m_half = fmaxf(mx, my) * sl2;
        float a = 1.f;
        if (m_run == -INFINITY) {
          m_run = m_half;
        } else if (m_half > m_run + kRescaleThreshold) {
          a = ex2(m_run - m_half);
          m_run = m_half;
          l_run *= a;
        }
        if (j > 0 && __any_sync(0xffffffffu, a != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            tmem_ld32(tO + 32 * c, s);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = f2u(u2f(s[i]) * a);
            tmem_st32(tO + 32 * c, s);
          }
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        const float2 sc2 = make_float2(sl2, sl2), nm2 = make_float2(-m_use, -m_use);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          load_scores(tS + 32 * c, lim - 32 * c, s);
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = __ffma2_rn(make_float2(u2f(s[2 * i]), u2f(s[2 * i + 1])), sc2, nm2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            acc[i & 1] = __fadd2_rn(acc[i & 1], e);
            w[i] = pack_bf16x2(e.x, e.y);
          }
          // Over columns of S that both rounds have read.
          tmem_st16(tS + 16 * c, w);
        }
#pragma unroll 1
        for (int c = chunks; c < 2; ++c) {
          constexpr uint32_t zero[16] = {};
          tmem_st16(tS + 16 * c, zero);
        }
        const float2 sum = __fadd2_rn(acc[0], acc[1]);
        l_run += sum.x + sum.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[h]);
      }
      J += nt;
#pragma unroll
      for (int g = 0; g < 2; ++g)
        if (it.n[g] > 0) {
          ok = ok && wait_all(&bars->o_full[g], (uint32_t)o_rounds[g] & 1u);
          ++o_rounds[g];
        }
      // The halves' maxima and sums; ml is written again only after the
      // barrier at the end. On abort all leave together.
      bars->ml[h][row] = make_float2(m_run, l_run);
      if (!softmax_warps_agree(ok)) break;
      tc_fence_after();
      const float2 a = bars->ml[0][row], b = bars->ml[1][row];
      const float M = fmaxf(a.x, b.x);
      // Without a maximum the sum is 0, or NaN if scores were: shown.
      const float fa = a.x == -INFINITY ? a.y : ex2(a.x - M), fb = b.x == -INFINITY ? b.y : ex2(b.x - M);
      const float L = fa * a.y + fb * b.y;
      uint32_t o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0u;
      if (it.n[0] > 0) {
        tmem_ld32(lanes + C::O_COL + 32 * h, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = fa == 0.f ? 0u : f2u(u2f(o[i]) * fa);
      }
      if (it.n[1] > 0) {
        uint32_t o1[32];
        tmem_ld32(lanes + C::O_COL + C::D + 32 * h, o1);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (fb != 0.f) o[i] = f2u(fmaf(u2f(o1[i]), fb, u2f(o[i])));
      }
      // Both have read O_0, O_1 and ml before either goes on.
      tc_fence_before();
      lin = next_item(n);
      if (!softmax_warps_agree(lin >= 0)) lin = -1;
      if (valid) {
        store_out_chunk(p, 0, it.h, it.q_row + row, h, o, L > 0.f ? 1.f / L : 0.f);
        if (p.lse && h == 0)
          p.lse[(long long)it.h * p.Tq + it.q_row + row] =
              L > 0.f ? (M + __log2f(L)) * 0.69314718055994531f : -INFINITY;
      }
      if (lin < 0) break;
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

}  // namespace

int launch_prefill_packed_d64(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              const PrefillParams& p, cudaStream_t st) {
  static OncePerDevice once;
  const long long items = (long long)p.n_qblk * p.Hq;
  if (items <= 0 || items > 0x7fffffffLL) return -2;
  return once.run(
      [] {
        cudaFuncAttributes fa{};
        return cudaFuncSetAttribute(prefill_packed_d64_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Cfg::SMEM_BYTES) == cudaSuccess &&
               cudaFuncGetAttributes(&fa, prefill_packed_d64_kernel) == cudaSuccess && fa.numRegs >= Cfg::REGS;
      },
      [&] {
        return launch_dependent(prefill_packed_d64_kernel, dim3((unsigned)items), Cfg::THREADS, Cfg::SMEM_BYTES, st, 0,
                                tq, tk, tv, p);
      });
}

}  // namespace b2a
