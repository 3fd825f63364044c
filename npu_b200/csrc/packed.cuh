// Work items of attention over packed sequences: which query block of which
// sequence an item is, found on the device from the offsets alone (no plan,
// no workspace, no copy of the lengths to the host).
//
// The kernels are prefill_packed_d64.cu, and prefill.cu's (head dim 128) and
// prefill_d256.cu's with PACKED: a sequence's rows and keys are offsets into
// one tensor map each. Measured on one B200 (device time): prompts of 1122, 1593, 2780 and 8192 tokens, 32 / 4
// heads of 128: 590 us at first to 690 under the power limit, 1.09 to 0.93
// PFLOP/s (0.66 to 0.57 of the measured bf16 rate, as the dense kernel); chunks
// of 65 to 2501 gated tokens behind 500 cached ones, 16 / 2 heads of 256: 213 to
// 229 us, 0.78 to 0.73 PFLOP/s; 32 prompts of 17 to 2048 tokens, 9 / 3 heads of
// 64: 42.2 us, 0.33 PFLOP/s (21 % of each 128 x 128 block is padding or masked
// and most items have one to five blocks); 3 prompts of 1 to 40: 5.9 to 6.3 us,
// one launch, of which finding the block is 1.2.
#pragma once

#include <type_traits>

#include "prefill.cuh"

namespace b2a {

// Blocks are numbered heaviest first, so that the long ones do not start last:
// a block's level is its number within its sequence plus the blocks' worth of
// keys ahead of the sequence's first row, and blocks of a level are numbered
// by sequence. With S(w) = number of blocks of level >= w (a sum over the
// sequences), block i has the level w with S(w + 1) <= i < S(w), found by
// bisection, and is the (i - S(w + 1))-th of it, found with ballots.
// Warp-collective. A call takes about log2(longest / kRows) sums of B / 32
// steps each, on lengths that stay in L1.
//
// Above kPackedByPosition sequences, block i is slot i - s(b) of the last
// sequence with s(b) <= i, s(b) = cu_q[b] / kRows + b: s(b + 1) - s(b) is at
// least the sequence's number of blocks, and b is found by a search that
// narrows 32-fold a step. Offsets that decrease may hide other sequences from
// that search, and a bad pair from every block, so block b also checks pair b.
template <int kRows>
struct PackedBlocks {
  const PrefillParams& p;
  int own_n = 0, own_off = 0;  // this lane's sequence when B <= 32
  int top = 0;                 // no block has a level above this

  __device__ __forceinline__ void shape(int b, int& n, int& off) const {
    n = off = 0;
    if (b >= p.B) return;
    const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
    if (q0 < 0 || q1 < q0 || q1 > p.Tq || k0 < 0 || k1 < k0 || k1 > p.Tk) {
      if (p.err) atomicOr(p.err, kErrBadArgs);  // not a stretch of the tensors: the sequence is left out
      return;
    }
    const int rows = q1 - q0, keys = k1 - k0;
    n = (rows + kRows - 1) / kRows;
    off = max(p.causal ? keys - rows : keys, 0) / kRows;
  }
  __device__ __forceinline__ explicit PackedBlocks(const PrefillParams& params) : p(params) {
    const int lane = threadIdx.x & 31;
    if (p.B > kPackedByPosition) return;
    int most = 0;
#pragma unroll 4
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      shape(b0 + lane, own_n, own_off);
      most = max(most, own_n > 0 ? own_n + own_off : 0);
    }
    top = __reduce_max_sync(0xffffffffu, most);
  }
  __device__ __forceinline__ int count_from(int w) const {
    const int lane = threadIdx.x & 31;
    int c = 0;
#pragma unroll 4
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      int n = own_n, off = own_off;
      if (p.B > 32) shape(b0 + lane, n, off);
      c += min(max(n + off - w, 0), n);
    }
    return __reduce_add_sync(0xffffffffu, c);
  }
  // Block qblk of sequence b, empty if the sequence has no such block.
  __device__ __forceinline__ PackedBlock block(int b, int qblk) const {
    int n, off;
    shape(b, n, off);
    if (qblk < 0 || qblk >= n) return {0, 0, 0, 0, 0};
    return {p.cu_q[b], p.cu_q[b + 1] - p.cu_q[b], p.cu_k[b], p.cu_k[b + 1] - p.cu_k[b], qblk};
  }
  // Block i (every lane gets it).
  __device__ __forceinline__ PackedBlock find(int i) const {
    const int lane = threadIdx.x & 31;
    if (p.B > kPackedByPosition) {
      if (i < p.B) {
        int n, off;
        shape(i, n, off);
      }
      int lo = 0, len = p.B;
      while (len > 1) {
        const int step = (len + 31) / 32, b = lo + lane * step;
        const bool before = lane * step < len && (lane == 0 || p.cu_q[b] / kRows + b <= i);
        const int hit = 31 - __clz(__ballot_sync(0xffffffffu, before));
        len = min(step, len - hit * step);
        lo += hit * step;
      }
      return block(lo, i - (p.cu_q[lo] / kRows + lo));
    }
    int lo = 0, hi = top;  // S(hi + 1) <= i always; looking for the largest w with S(w) > i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (count_from(mid) > i)
        lo = mid;
      else
        hi = mid - 1;
    }
    int skip = i - count_from(lo + 1);
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      int n = own_n, off = own_off;
      if (p.B > 32) shape(b0 + lane, n, off);
      const bool has = lo >= off && lo < off + n;
      const unsigned m = __ballot_sync(0xffffffffu, has);
      if (skip < __popc(m)) {
        const bool it = has && __popc(m & ((1u << lane) - 1u)) == skip;
        const int src = __ffs(__ballot_sync(0xffffffffu, it)) - 1;
        const int b = b0 + src;
        return block(b, lo - __shfl_sync(0xffffffffu, off, src));
      }
      skip -= __popc(m);
    }
    return {0, 0, 0, 0, 0};
  }
};

// Stands in for PackedBlocks in kernels that do not pack.
struct NoBlocks {
  __device__ __forceinline__ explicit NoBlocks(const PrefillParams&) {}
};

}  // namespace b2a
