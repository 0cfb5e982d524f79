// Matrix products of 16-bit operands in tiles below the GEMM core's 256 x 256, for
// products that have too few of those to fill the chip:
//   C[m][n] = sum_k A(m, k) B(k, n), float32 sums.
//
// A tile is 64 MB x 64 NB, computed by four waves (2 x 2), each 32 MB x 32 NB in
// blocks of one 32x32x16 MFMA.  kGroups such sets of four waves may share a tile:
// each takes a part of K and the sums are joined through LDS, in order, which
// shortens a product that has many k and few tiles.
//
// Staging is the GEMM core's (gemm_core.h): buffer loads copy 16-byte chunks from
// global memory into LDS through a ring of three or four stages, each stage waited
// for with an exact vmcnt and one barrier; operands lie there K-major or MN-major, as they
// do in memory, so that a quarter-wave's reads meet different banks, MN-major
// fragments read with ds_read_b64_tr_b16.  A stage is
// 32 kSlabs deep.  K is any multiple of 8 (K-major) or any number (MN-major); what
// lies past K or past the operand's rows reads zeros.
#pragma once

#include "gemm_core.h"

namespace tile {

typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short lds16;
typedef __attribute__((address_space(3))) i16x8 lds16x8;
typedef __attribute__((address_space(3))) i16x4 lds16x4;

__device__ __forceinline__ f32x16 mma(i16x8 a, i16x8 b, f32x16 c, bf16) {
  return mfma32(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}
__device__ __forceinline__ f32x16 mma(i16x8 a, i16x8 b, f32x16 c, f16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// How a matrix operand of 16-bit elements lies in memory: K along the rows or the
// other way, rows with leading dimension ld, or "32-blocked": element (r, c) at
// ((c / 32) * ld + r) * 32 + c % 32, column blocks of 32 one after another, each of ld
// rows of 64 bytes.  A copy takes 1 KB: of a blocked operand 16 rows of a block, one
// run of whole lines, for which the address unit needs some 20 cycles; 64-byte pieces
// of lines (K-major rows) take it 40 to 50.
// kPairsMN: two kRowsMN matrices side by side, the second `pair` elements after the
// first, whose columns take turns in the tile in blocks of 32 (gemm::Operand's).
enum Layout { kRowsK, kRowsMN, kPairsMN, kBlockedK, kBlockedMN };

struct Operand {
  const void* p;
  int64_t ld;
  int64_t pair = 0;
};

template <int kBytes, int kStage>
__device__ __forceinline__ lds16* stage_array() {
  __shared__ __attribute__((aligned(1024))) short array[kBytes / 2];
  return (lds16*)array;
}

constexpr int wait_vm_lgkm0(int vm) { return (vm & 15) | 0x70 | ((vm >> 4) << 14); }

// Copy sources of one operand for one wave: P blocks of 1 KB a stage.  In LDS a slab
// of 32 k is K-major ([row][32 k], chunks of 8 swizzled), MN-major ([k][row],
// swizzled) or, of a kBlockedMN operand, the blocks as they are ([block][k][32 rows]).
template <int TM, Layout kLayout, int kSlabs>
struct Source {
  static constexpr int P = TM / 64 * kSlabs;
  static constexpr int kDepth = 32 * kSlabs;
  static constexpr bool kBlocked = kLayout == kBlockedK || kLayout == kBlockedMN;
  static constexpr bool kK = kLayout == kRowsK || kLayout == kBlockedK;
  const char* base;
  int64_t step;
  uint32_t off[P];
  int nvalid[P];

  static __device__ __forceinline__ int swizzle(int k) { return TM == 64 ? 4 * ((k >> 1) & 1) : 4 * (k & 3); }

  // mn0: the tile's first row, MN: the operand's rows; K range [k_begin, k_end).
  // (k_begin is a multiple of 32 and mn0 of 64: blocked stages and tiles start on a block.)
  __device__ __forceinline__ void init(Operand op, int mn0, int MN, int k_begin, int k_end, int wave, int lane) {
    if (kLayout == kPairsMN) {  // columns of one of the two matrices
      mn0 >>= 1;
      MN >>= 1;
    }
    const int r0 = kK ? mn0 : k_begin, c0 = kK ? k_begin : mn0;  // as the memory has rows and columns
    if (kBlocked) {
      base = (const char*)op.p + ((int64_t)(c0 >> 5) * op.ld + r0) * 64;
      step = 64 * (kK ? op.ld * kSlabs : (int64_t)kDepth);
    } else {
      base = (const char*)op.p + 2 * ((int64_t)r0 * op.ld + c0);
      step = 2 * (kK ? (int64_t)kDepth : kDepth * op.ld);
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int b = wave * P + j, slab = b / (TM / 16), blk = b % (TM / 16);
      int k, m;
      bool second = false;
      if (kK) {
        m = blk * 16 + (lane >> 2);
        k = 32 * slab + 8 * ((lane & 3) ^ ((m >> 2) & 3));
      } else if (!kBlocked) {
        constexpr int kChunks = TM / 8;
        const int row = blk * (512 / TM) + lane / kChunks;
        k = 32 * slab + row;
        m = 8 * ((lane % kChunks) ^ swizzle(row));
        if (kLayout == kPairsMN) {
          second = (m >> 5) & 1;
          m = 32 * (m >> 6) + (m & 31);
        }
      } else {
        k = 32 * slab + 16 * (blk & 1) + (lane >> 2);
        m = 32 * (blk >> 1) + 8 * (lane & 3);
      }
      const int r = kK ? m : k, c = kK ? k : m;
      off[j] = 2u * (uint32_t)(kBlocked ? ((int64_t)(c >> 5) * op.ld + r) * 32 + (c & 31)
                                        : (int64_t)r * op.ld + c + (second ? op.pair : 0));
      const int rem = k_end - k_begin - k;
      nvalid[j] = (mn0 + m < MN && rem > 0) ? (rem + kDepth - 1) / kDepth : 0;
    }
  }

  // Stage kt into the slabs at element `offset` of a stage array.
  __device__ __forceinline__ void issue(lds16* array, int offset, int kt, int wave) const {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base + kt * step, gemm::kRsrcRange);
#pragma unroll
    for (int j = 0; j < P; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (gemm::lds_void*)(array + (offset + (wave * P + j) * 512)), 16,
                                               kt < nvalid[j] ? off[j] : gemm::kOffZero, 0, 0, 0);
  }
};

// Fragment of rows r0 + 32 block .. + 31 at k-chunk kc (16 deep) of the slabs at
// element `offset` + kOffset of a stage array.
// kContiguous: in gemm::contiguous_row's order, so that a lane's accumulator
// elements 0 .. 15 are 16 consecutive rows.
// The lane's part of an address passes through an empty asm: the compiler finds an
// access's array through a few additions only, would make more of one sum, and takes
// an access without an array to meet every copy in flight, for which it then waits.
template <int TM, Layout kLayout, bool kContiguous, int kOffset>
__device__ __forceinline__ i16x8 frag(const lds16* array, int offset, int r0, int block, int kc, int lane) {
  typedef Source<TM, kLayout, 1> S;
  const int hl = lane >> 5;
  if (S::kK) {
    const int row = r0 + (kContiguous ? gemm::contiguous_row(lane & 31) : (lane & 31));
    const int c = 2 * (kc & 1) + hl;
    int at = offset + row * 32 + 8 * (c ^ ((row >> 2) & 3));  // (the same for row + 32)
    asm("" : "+v"(at));
    return *(const lds16x8*)(array + at + (kOffset + 1024 * block + (kc >> 1) * TM * 32));
  } else {
    // The lane supplies the address of four rows: quad q of the block's eight.
    const int cq = lane & 15, q = 4 * ((lane >> 4) & 1) + (cq & 3);
    const int quad = kContiguous ? 16 * (q & 1) + 4 * (q >> 1) : 4 * q;
    const int k = 8 * hl + (cq >> 2);
    constexpr bool kBlocks = kLayout == kBlockedMN;  // (a half-wave's reads are 256 bytes in a row there)
    constexpr int kRow = kBlocks ? 32 : TM;          // elements from one k to the next
    int at;
    if (kBlocks) {
      at = offset + r0 * 32 + k * 32 + quad;
    } else {  // (the swizzle is the same for k, k + 4 and k + 16)
      const int m = r0 + 32 * block + quad;
      at = offset + k * TM + 8 * ((m >> 3) ^ S::swizzle(k)) + 4 * ((m >> 2) & 1);
    }
    asm("" : "+v"(at));
    const lds16* const lo =
        array + at + (kOffset + (kBlocks ? 1024 * block : 0) + (kc >> 1) * TM * 32 + (kc & 1) * 16 * kRow);
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)lo);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)(lo + 4 * kRow));
    return i16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}

// A wave's block of 32 rows x 32 features of 16 bits in LDS (2 KB, of its own), on the
// way between its accumulators' layout (a lane holds a run: 16 consecutive features
// of one row) and lines (four lanes hold a row's 64 bytes, so that an access to
// global memory takes 1 KB of whole lines).  The address unit takes some 16 cycles
// for such an access, 85 for 16-byte pieces that lie 64 bytes apart from lane to
// lane and 170 where each has a line of its own: kept as runs, the result of a
// product over 768 took longer to write than to compute.  LDS serves a wave in
// order, so nothing is waited for but the data.
struct Block {
  lds16* base;
  static constexpr int kElements = 1024;
  // Chunks of 8 features are moved so that 16 lanes' accesses meet all banks once.
  static __device__ __forceinline__ int at(int row, int chunk) { return row * 32 + 8 * (chunk ^ ((row >> 2) & 3)); }
  static __device__ __forceinline__ void order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

  __device__ __forceinline__ void put_run(int lane, i16x8 low, i16x8 high) const {
    order();
    *(lds16x8*)(base + at(lane & 31, 2 * (lane >> 5))) = low;
    *(lds16x8*)(base + at(lane & 31, 2 * (lane >> 5) + 1)) = high;
    order();
  }
  __device__ __forceinline__ i16x8 get_run(int lane, int half) const {
    return *(const lds16x8*)(base + at(lane & 31, 2 * (lane >> 5) + half));
  }
  // The run as a column of the turned block: rows are features then.
  __device__ __forceinline__ void put_turned(int lane, i16x8 low, i16x8 high) const {
    order();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = 16 * (lane >> 5) + e, col = lane & 31;
      base[at(row, col >> 3) + (col & 7)] = e < 8 ? low[e & 7] : high[e & 7];
    }
    order();
  }
  // A lane's piece of turn `it` (0, 1): row and first feature.
  static __device__ __forceinline__ int line_row(int it, int lane) { return 16 * it + (lane >> 2); }
  static __device__ __forceinline__ int line_feature(int lane) { return 8 * (lane & 3); }
  __device__ __forceinline__ void put_lines(int lane, i16x8 first, i16x8 second) const {
    order();
    *(lds16x8*)(base + at(lane >> 2, lane & 3)) = first;
    *(lds16x8*)(base + at(16 + (lane >> 2), lane & 3)) = second;
    order();
  }
  __device__ __forceinline__ i16x8 get_line(int it, int lane) const {
    return *(const lds16x8*)(base + at(line_row(it, lane), lane & 3));
  }
};

// T: bf16 or f16.  MB, NB: the tile in units of 64.  LA, LB: the operands' layouts.
// kContiguous: rows of A in contiguous_row's order.
template <class T, int MB, int NB, Layout LA, Layout LB, bool kContiguous, int kSlabs = 1, int kGroups = 1,
          int kRing = 4>
struct Product {
  static constexpr int TM = 64 * MB, TN = 64 * NB, kThreads = 256 * kGroups;
  static constexpr int kStageA = TM * 32 * kSlabs, kStageB = TN * 32 * kSlabs;  // elements
  static constexpr int kStageBytes = 2 * kGroups * (kStageA + kStageB);
  static constexpr int kChunks = 2 * kSlabs, kDepth = 32 * kSlabs;
  static constexpr int kLoads = (TM + TN) / 64 * kSlabs;  // a wave's copies of a stage
  static_assert(kRing * kStageBytes <= 160 * 1024, "the ring does not fit LDS");
  static_assert(kRing == 3 || kRing == 4, "stages in flight");
  static_assert(kGroups <= 4 && (kGroups == 1 || TM * TN * 4 <= kStageBytes), "parts are joined in the stage arrays");

  // Position of a wave: its set, and within it 2 x 2.
  struct Place {
    int lane, wave, group, wm, wn;
  };
  static __device__ __forceinline__ Place place() {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    return Place{(int)threadIdx.x & 63, w & 3, w >> 2, w & 1, (w >> 1) & 1};
  }

  // After run(): a wave's blocks 0 and 1, in the first stage's memory.
  static __device__ __forceinline__ Block block(const Place& at, int which) {
    static_assert(4 * 2 * 2 * Block::kElements <= kStageBytes, "two blocks a wave");
    return Block{stage_array<kStageBytes, 0>() + (2 * at.wave + which) * Block::kElements};
  }

  struct State {
    Source<TM, LA, kSlabs> a;
    Source<TN, LB, kSlabs> b;
    Place at;
  };

  template <int S>
  static __device__ __forceinline__ void fill(const State& s, int kt) {
    lds16* const array = stage_array<kStageBytes, S>();
    const int offset = s.at.group * (kStageA + kStageB);
    s.a.issue(array, offset, kt, s.at.wave);
    s.b.issue(array, offset + kStageA, kt, s.at.wave);
  }

  template <int S>
  static __device__ __forceinline__ void read(i16x8 (&a)[MB], i16x8 (&b)[NB], const State& s, int kc) {
    const lds16* const array = stage_array<kStageBytes, S>();
    const int offset = s.at.group * (kStageA + kStageB);
#pragma unroll
    for (int i = 0; i < MB; ++i)
      a[i] = frag<TM, LA, kContiguous, 0>(array, offset, 32 * MB * s.at.wm, i, kc, s.at.lane);
#pragma unroll
    for (int i = 0; i < NB; ++i)
      b[i] = frag<TN, LB, false, kStageA>(array, offset, 32 * NB * s.at.wn, i, kc, s.at.lane);
  }

  template <int S>
  static __device__ __forceinline__ void step(f32x16 (&acc)[MB][NB], i16x8 (&a)[2][MB], i16x8 (&b)[2][NB],
                                              const State& s, int kt) {
#pragma unroll
    for (int kc = 0; kc < kChunks; ++kc) {
      const int now = kc & 1, next = now ^ 1;
      if (kc + 1 < kChunks) {
        read<S>(a[next], b[next], s, kc + 1);
      } else {
        // The next stage is there; every wave has read this one, which is refilled.
        __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((kRing - 2) * kLoads));
        wg_barrier();
        fill<S>(s, kt + kRing);
        read<(S + 1) % kRing>(a[next], b[next], s, 0);
      }
      GEMM_SCHED_FENCE();
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mma(a[now][i], b[now][j], acc[i][j], T());
      GEMM_SCHED_FENCE();
    }
  }

  // acc[i][j][e]: C of row tm0 + 32 (MB wm + i) + r(e) and column tn0 + 32 (NB wn + j) +
  // lane % 32, with r(e) = 16 (lane / 32) + e if kContiguous, else 8 (e / 4) + 4 (lane / 32)
  // + e % 4.  With kGroups > 1 only group 0's are the sums.  On return no copy into the
  // stage arrays is in flight and every wave has passed a barrier since its last read.
  static __device__ __forceinline__ void run(f32x16 (&acc)[MB][NB], Operand A, Operand B, int M, int N, int K, int tm0,
                                             int tn0, const Place& at) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass has no use for the instantiations below)
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f32x16{};
    // Whole stages a group, whole rounds of the ring.
    const int share = ((K + kGroups - 1) / kGroups + kDepth - 1) / kDepth * kDepth;
    const int begin = min(K, at.group * share), end = min(K, begin + share);
    const int nk = (share / kDepth + kRing - 1) / kRing * kRing;
    State s;
    s.at = at;
    s.a.init(A, tm0, M, begin, end, at.wave, at.lane);
    s.b.init(B, tn0, N, begin, end, at.wave, at.lane);
    fill<0>(s, 0);
    fill<1>(s, 1);
    fill<2>(s, 2);
    if constexpr (kRing == 4) fill<3>(s, 3);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((kRing - 1) * kLoads));
    wg_barrier();
    i16x8 a[2][MB], b[2][NB];
    read<0>(a[0], b[0], s, 0);
    for (int kt = 0; kt < nk; kt += kRing) {
      step<0>(acc, a, b, s, kt);
      step<1>(acc, a, b, s, kt + 1);
      step<2>(acc, a, b, s, kt + 2);
      if constexpr (kRing == 4) step<3>(acc, a, b, s, kt + 3);
    }
    GEMM_WAIT_VM0_LGKM0();
    wg_barrier();
    if constexpr (kGroups > 1) {
      typedef __attribute__((address_space(3))) f32x4 lds_f4;
      // [part][lane] of four floats: a wave's accumulators in LDS.
      auto slot = [&](lds16* array, int i, int j, int q) {
        return (lds_f4*)array + ((at.wave * MB * NB + i * NB + j) * 4 + q) * 64 + at.lane;
      };
      auto put = [&](lds16* array) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *slot(array, i, j, q) =
                  f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      };
      auto add = [&](lds16* array) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 v = *slot(array, i, j, q);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
            }
      };
      if (at.group == 1) put(stage_array<kStageBytes, 1>());
      if (kGroups > 2 && at.group == 2) put(stage_array<kStageBytes, 2>());
      if (kGroups > 3 && at.group == 3) put(stage_array<kStageBytes, 3 % kRing>());
      GPTRIG_WAIT_LGKM0();
      wg_barrier();
      if (at.group == 0) {
        add(stage_array<kStageBytes, 1>());
        if (kGroups > 2) add(stage_array<kStageBytes, 2>());
        if (kGroups > 3) add(stage_array<kStageBytes, 3 % kRing>());
      }
    }
#endif
  }
};

}  // namespace tile
