// What the attention kernels share: views of strided BHSD tensors, the order in
// which workgroups take blocks, and the document test that skips hidden blocks.
#pragma once

#include "attn64.h"

#include <type_traits>

namespace {

constexpr float kMinusBig = -1.0e30f;
typedef __attribute__((address_space(3))) void lds_void;

struct View {
  const bf16* p;
  int64_t sb, sh, ss;
  __device__ __forceinline__ const bf16* row(int b, int h, int s) const { return p + b * sb + h * sh + s * ss; }
};
struct MutView {
  bf16* p;
  int64_t sb, sh, ss;
  __device__ __forceinline__ bf16* row(int b, int h, int s) const { return p + b * sb + h * sh + s * ss; }
};

// Workgroup id -> (batch*head, block rank), rank-major: every head's rank-0
// block (its heaviest causal share, see the callers) is dispatched before any
// rank-1 block, and so on, so the last workgroups to start are the light ones
// and the tail stays short.  Workgroups are dispatched round-robin over the 8
// XCDs; with batch*heads a multiple of 8 all blocks of one head land on the
// same XCD, which keeps that head's K/V (forward) or Q/dO/dQ (backward) in one
// L2.
__device__ __forceinline__ void xcd_map(int id, int nblocks, int bh_total, int& bh, int& blk) {
  (void)nblocks;
  bh = id % bh_total;
  blk = id / bh_total;
}

// ============================================================================
// Skipping what document masking hides
// ============================================================================
// With segment ids a workgroup owns a block of positions (128 queries in the
// forward, the keys in the backward) and walks 64-position blocks of the other
// side.  A block none of whose ids lies between the lowest and the highest id
// of the owned block holds no visible pair, whatever the order of the ids, so
// it is neither loaded nor computed.  A block whose ids all equal the owned
// block's single id needs no per-element id compare.
// The blocks are tested 64 at a time: each wave reads its share of the ids
// (one coalesced load, a compare and a ballot per block) and the bits are
// exchanged through LDS.  That is 32 KB of ids per workgroup at 8192 positions
// against the 16 KB of K and V that every block not skipped costs.
// Measured at B2 H12 S8192 D64, documents of 1..3000 tokens: forward + backward
// 1513 -> 595 us (backward kernel 994 -> 396, forward 554 -> 232); what is left
// above the visible share of the work (about a quarter) is the uneven lengths
// of the workgroups.  Where nothing can be skipped (one document) the test costs
// 1 to 2 us per workgroup and saves the compares: B16 H12 S1024 D64 forward 87 ->
// 56, backward 188 -> 172 us; B64 H12 S256 D64 44 -> 31, 111 -> 115; B8 H6 S1024
// D128 75 -> 39, 121 -> 124; B64 H6 S256 D128 44 -> 31, 121 -> 123.  The backward
// has the test's ids loaded with its first operands (waited for on their own: 127
// at B8 H6 S1024 D128, 121 at B64 H12 S256 D64).
template <int kWaves>
struct SegScan {
  static constexpr int kPer = 64 / kWaves;  // blocks a wave tests
  using Piece = std::conditional_t<kPer == 8, uint8_t, uint16_t>;
  const int32_t* ids;  // this sequence's ids
  uint64_t* sh;        // LDS: the need and the same bits of 64 blocks (kept here: registers are short)
  int S, lo, hi;       // the owned block's id range
  int group;           // the 64 blocks that the bits describe
  bool on = true;      // off: every block is walked with the compare

  // Id range of the owned positions p0 .. p0 + 64 kOwn - 1 (those below S).
  template <int kOwn>
  __device__ __forceinline__ void init(const int32_t* seq_ids, uint64_t* lds, int seq, int p0, int lane) {
    int own[kOwn];
    fetch_own<kOwn>(own, seq_ids, lds, seq, p0, lane);
    range<kOwn>(own);
  }
  template <int kOwn>
  __device__ __forceinline__ void fetch_own(int (&own)[kOwn], const int32_t* seq_ids, uint64_t* lds, int seq, int p0,
                                            int lane) {
    ids = seq_ids;
    sh = lds;
    S = seq;
    group = -1;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) own[j] = ids[min(p0 + 64 * j + lane, S - 1)];
  }
  template <int kOwn>
  __device__ __forceinline__ void range(const int (&own)[kOwn]) {
    int a = own[0], z = a;
#pragma unroll
    for (int j = 1; j < kOwn; ++j) {
      a = min(a, own[j]);
      z = max(z, own[j]);
    }
    // Over the wave without LDS: quads, half rows, rows, then row 15 / 31 on to
    // the rows above; lane 63 ends with the whole.
#define SEG_FOLD(ctrl)                                                              \
  a = min(a, __builtin_amdgcn_update_dpp(a, a, ctrl, 0xF, 0xF, false));             \
  z = max(z, __builtin_amdgcn_update_dpp(z, z, ctrl, 0xF, 0xF, false));
    SEG_FOLD(0xB1)   // quad_perm [1, 0, 3, 2]
    SEG_FOLD(0x4E)   // quad_perm [2, 3, 0, 1]
    SEG_FOLD(0x141)  // row_half_mirror
    SEG_FOLD(0x140)  // row_mirror
    SEG_FOLD(0x142)  // row_bcast15
    SEG_FOLD(0x143)  // row_bcast31
#undef SEG_FOLD
    lo = __builtin_amdgcn_readlane(a, 63);
    hi = __builtin_amdgcn_readlane(z, 63);
  }

  // This wave's share of the ids of group g, and its bits of them into LDS.
  __device__ __forceinline__ void fetch(int (&id)[kPer], int g, int wave, int lane) const {
#pragma unroll
    for (int j = 0; j < kPer; ++j) id[j] = ids[min((64 * g + kPer * wave + j) * 64 + lane, S - 1)];
  }
  __device__ __forceinline__ void publish(const int (&id)[kPer], int g, int wave, int lane) {
    group = g;
    uint32_t n = 0, f = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int p = (64 * g + kPer * wave + j) * 64 + lane;
      const bool in = id[j] >= lo && id[j] <= hi;
      n |= __ballot(in && p < S) != 0 ? 1u << j : 0u;
      f |= __ballot(in || p >= S) == ~0ull ? 1u << j : 0u;
    }
    if (lane == 0) {
      reinterpret_cast<Piece*>(sh)[wave] = (Piece)n;
      reinterpret_cast<Piece*>(sh + 1)[wave] = (Piece)(lo == hi ? f : 0u);
    }
  }

  // (Every wave calls this the same number of times: it holds two barriers.)
  __device__ __forceinline__ void load(int g, int wave, int lane) {
    int id[kPer];
    fetch(id, g, wave, lane);
    __syncthreads();
    publish(id, g, wave, lane);
    __syncthreads();
  }

  __device__ __forceinline__ uint64_t bits(int which) const {
    const uint64_t v = sh[which];
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
  }

  // The first block at or after t (below nblk) with a visible pair, else nblk;
  // same: its ids need no compare.
  __device__ __forceinline__ int next(int t, int nblk, int wave, int lane, bool& same) {
    same = false;
    if (!on) return min(t, nblk);
    while (t < nblk) {
      if ((t >> 6) != group) load(t >> 6, wave, lane);
      const uint64_t m = bits(0) >> (t & 63);
      if (m) {
        t += __builtin_ctzll(m);
        same = bits(1) >> (t & 63) & 1;
        return min(t, nblk);
      }
      t = ((t >> 6) + 1) << 6;
    }
    return nblk;
  }
};

}  // namespace
