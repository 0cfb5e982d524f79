// Attention whose scores are capped by a tanh or get a bias that depends on
// distance, over causal, prefix and document masks, with heads that may share
// keys and values.  For query i and key j of one (batch, head):
//   u_ij = scale q_i . k_j
//   s_ij = c tanh(u_ij / c) - slope |i - j|     (without a cap: u_ij - slope |i - j|)
//   visible(i, j): j <= max(i, prefix - 1) and segment_i == segment_j
//   P = softmax of s over the visible j, o = P v, L_i = log2 sum_j 2^(s_ij log2 e)
//   dS = P (do v^T - delta), delta_i = o_i . do_i;  dU = dS (1 - tanh^2(u / c))
//   dv = P^T do, dk = scale dU^T q, dq = scale dU k
// Scores are taken in units of log2 e from the start, so every exponential is one
// v_exp_f32.  With w = 1 / (1 + exp(2 u / c)): tanh(u / c) = 1 - 2 w and
// 1 - tanh^2 = 4 w (1 - w); w saturates to 0 and 1 without an overflow.
// The matrix products take bf16 operands: P and dU are rounded to bf16 for them
// (half a step is 2^-8 of the value, the rounding of the results themselves); all
// else is float32.
//
// A pair that is not visible adds nothing, whatever its k, v, q or do hold.  Its P
// and dU are set to 0; but 0 x inf is not 0, so a tile that holds hidden pairs is
// searched for infinities and NaN before its rows are summed over (Dirty, below).
#pragma once

#include "attn_common.h"

namespace {

constexpr int kRows = 64;  // rows of an LDS tile

struct ScoreArgs {
  float raw;            // scale log2 e; with a cap 2 log2 e scale / cap
  float cap2;           // cap log2 e
  const float* slopes;  // [heads], nullable
  const int32_t* prefix;  // [batch], nullable
};

// The w of raw product r.
__device__ __forceinline__ float cap_w(float r, const ScoreArgs& a) {
  return __builtin_amdgcn_rcpf(1.0f + fast_exp2(r * a.raw));
}

// The larger of a lane's value and its counterpart's in the other half-wave (an
// exchange of half-waves between registers; a shuffle goes through LDS).
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// The row of accumulator element i (of 16) in the lower half of the wave; the upper half adds 4.
__host__ __device__ constexpr int acc_row(int i) { return 8 * (i >> 2) + (i & 3); }

// slope x acc_row(i), the same for every lane: kept in scalar registers.
__device__ __forceinline__ void row_bias(float (&bias)[16], float slope) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    bias[i] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, slope * (float)acc_row(i))));
}

__device__ __forceinline__ int prefix_of(const ScoreArgs& a, int b, int S) {
  return a.prefix ? min(max(a.prefix[b], 0), S) : 0;
}

// What rounding x to the bf16 `high` cut off, in 8 bits: the difference of the two as
// float32 bits, which lies in [-2^15, 2^15], over 2^8; and x again, to 16 bits.
__device__ __forceinline__ uint32_t low_bits(float x, bf16 high) {
  const int rest = (int)(__builtin_bit_cast(uint32_t, x) - __builtin_bit_cast(uint32_t, (float)high));
  return (uint32_t)min(max((rest + 128) >> 8, -128), 127) & 0xFFu;
}
__device__ __forceinline__ float with_low_bits(bf16 high, uint32_t low) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, (float)high) + (uint32_t)((int)(int8_t)low * 256));
}

// Element offset of 16-byte chunk c16 of row `row` in a tile of kRows rows: a
// tile of 128 columns is two swizzled ones of 64.
__device__ __forceinline__ int tile_at(int row, int c16) { return (c16 >> 3) * kRows * 64 + at64::swz(row, c16 & 7); }
__device__ __forceinline__ bf16x8 tile_row(const at64::lds_t* t, int row, int c16) {
  return *(const at64::lds_x8*)(t + tile_at(row, c16));
}

// Byte offsets in a tile of what a lane reads for the matrix instructions.  The
// swizzle of a row depends on it modulo 16, so these few stand for every row block,
// column block and tile, which are constants of the instructions.  (Computed where
// they were used, 25 to 45 vector operations for 32 x 32 pairs: dk and dv 112 us
// instead of 104 at B16 H12 S1024 D64 with a cap, with the loads ahead of their use; the
// two in one run, on inputs that change between launches.)
struct Lanes {
  uint32_t row[4];           // chunk 2 kc + half-wave of row lane % 32
  uint32_t low[2], high[2];  // transposed: the slots' first and second four rows, column blocks 0 and 1
  __device__ __forceinline__ void init(int lane) {
    const int hl = lane >> 5, cq = lane & 15;
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) row[kc] = 2 * at64::swz(lane & 31, 2 * kc + hl);
#pragma unroll
    for (int db = 0; db < 2; ++db) {
      const int m = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (cq & 3), r = 4 * hl + (cq >> 2);
      low[db] = 2 * (at64::swz(r, m >> 3) + (m & 4));
      high[db] = 2 * (at64::swz(r + 8, m >> 3) + (m & 4));
    }
  }
};
constexpr uint32_t kRowBytes = 128;                    // of one of a tile's halves of 64 columns
constexpr uint32_t kColumns64 = kRows * kRowBytes;     // from one of them to the next
typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ const at64::lds_t* byte_at(const at64::lds_t* t, uint32_t offset) {
  return (const at64::lds_t*)((const lds_char*)t + offset);
}
// Operand kc of 32 rows; at: byte offset of the first, a multiple of 16 rows.
__device__ __forceinline__ bf16x8 row_operand(const at64::lds_t* t, const Lanes& l, uint32_t at, int kc) {
  return *(const at64::lds_x8*)byte_at(t, (l.row[kc & 3] + at) + (kc >> 2) * kColumns64);
}
// Transposed operand of columns 32 db .. +31 and 16 rows, in accumulator order.
__device__ __forceinline__ bf16x8 column_operand(const at64::lds_t* t, const Lanes& l, uint32_t at, int c, int db) {
  const uint32_t constant = (db >> 1) * kColumns64 + 16 * c * kRowBytes;
  const bf16x4 lo = at64::read_tr(byte_at(t, (l.low[db & 1] + at) + constant));
  const bf16x4 hi = at64::read_tr(byte_at(t, (l.high[db & 1] + at) + constant));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// 16 bytes a lane, or 4, global -> LDS: lane l's land at lds + 16 l (4 l).
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, at64::lds_t* lds, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)lds, 16, offset, 0, 0, 0);
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, void* lds, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)lds, 4, offset, 0, 0, 0);
}

// One tile of 64 rows x D columns, global -> LDS by the DMA path.  Wave w of
// kWaves fills its 1 KB blocks of 8 rows each; rows at or past S and columns at or
// past `dim` read as zeros.
template <int D, int kWaves = 4>
struct Fill {
  static constexpr int NB = D / 8 / kWaves;
  int off[NB];
  int stride;  // bytes a row
  __device__ __forceinline__ void init(int64_t row_stride, int dim, int wave, int lane) {
    stride = (int)row_stride * 2;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int blk = NB * wave + j;
      const int row = 8 * (blk & 7) + (lane >> 3);
      const int t = (row >> 1) & 7;
      const int c = 8 * (blk >> 3) + ((lane & 7) ^ (((t & 1) << 2) | (t >> 1)));
      off[j] = 8 * c < dim ? row * stride + 16 * c : INT32_MIN;  // (past every buffer)
    }
  }
  __device__ __forceinline__ void operator()(__amdgpu_buffer_rsrc_t rs, at64::lds_t* tile, int row0, int wave) const {
#pragma unroll
    for (int j = 0; j < NB; ++j) dma16(rs, tile + (NB * wave + j) * 512, off[j] + row0 * stride);
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t slice(const bf16* base, int S, int64_t row_stride, int dim) {
  return make_rsrc(base, (uint32_t)(((int64_t)(S - 1) * row_stride + dim) * 2));
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// What the ids of a tile's 64 rows mean for one wave's own 32 positions, where the
// document test of the whole workgroup could not tell: per half of the tile
// whether any pair may be visible, and whether ids have to be compared for it.
struct WaveIds {
  int lo, hi;  // the wave's own ids (each in both half-waves)
  __device__ __forceinline__ void init(int own) {
    lo = hi = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor(lo, o));
      hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
  }
  // Bits 0 and 1: the halves with a visible pair; docs: those whose ids have to be compared.
  __device__ __forceinline__ int look(const int* ids, int lane, int& docs) const {
    const int id = ids[lane];
    const uint64_t within = __ballot(id >= lo && id <= hi);
    const uint32_t in0 = (uint32_t)within, in1 = (uint32_t)(within >> 32);
    docs = (lo != hi || in0 != ~0u ? 1 : 0) | (lo != hi || in1 != ~0u ? 2 : 0);
    return (in0 ? 1 : 0) | (in1 ? 2 : 0);
  }
};

// Rows of an LDS tile that hold an infinity or NaN, for tiles with hidden pairs
// (at the causal border and where documents meet): each of the 4 waves searches 16
// rows, four lanes a row, and one barrier shares what they found.  Where there
// is such a row, the caller records which of its own results it reaches, and
// clear() puts zeros in the place of its infinities and NaN; nothing else of a
// kernel knows of it.
// (One 1 KB read and two operations a word per wave, on two tiles of a workgroup.)
template <int D>
struct Dirty {
  uint64_t* found;  // LDS, [4]: bit l of wave w's word: row 16 w + l / 4

  __device__ __forceinline__ bool find(const at64::lds_t* tile, int wave, int lane) const {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = u16x2{};
    if (wave < 4)  // (a workgroup of 8 waves leaves it to 4)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const u32x4 w = __builtin_bit_cast(u32x4, tile_row(tile, 16 * wave + (lane >> 2), (lane & 3) + 4 * j));
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[e] & 0x7FFF7FFFu));
    }
    const uint64_t mine = __ballot(top[0] >= 0x7F80u || top[1] >= 0x7F80u);
    if (lane == 0 && wave < 4) found[wave] = mine;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((found[0] | found[1] | found[2] | found[3]) != 0);
  }
  __device__ __forceinline__ bool row(int r) const { return (found[r >> 4] >> 4 * (r & 15) & 15) != 0; }
  // (Every wave has recorded what it needs of the tile by the first barrier.)
  __device__ __forceinline__ void clear(at64::lds_t* tile, int wave, int lane) const {
    __syncthreads();
    const int r = 16 * wave + (lane >> 2);
    if (wave < 4 && row(r))
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        at64::lds_x8* const at = (at64::lds_x8*)(tile + tile_at(r, (lane & 3) + 4 * j));
        bf16x8 v = *at;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fabsf((float)v[e]) < INFINITY ? v[e] : (bf16)0.f;
        *at = v;
      }
    __syncthreads();
  }
};

// acc[db] += (columns of a tile, 32 rows)^T x, x the wave's 32 x 32 operand in
// accumulator order (16 rows of this lane's column as bf16).  The tile's operands are
// loaded ahead, so that their way from LDS is behind other work.
template <int DB>
struct Columns {
  bf16x8 v[2][DB];
  __device__ __forceinline__ void load(const at64::lds_t* t, const Lanes& l, uint32_t at) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < DB; ++db) v[c][db] = column_operand(t, l, at, c, db);
  }
  __device__ __forceinline__ void product(f32x16 (&acc)[DB], const bf16x8 (&x)[2]) const {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = mfma32(v[c][db], x[c], acc[db]);
  }
};

// c + the sum of x, two values an instruction.
__device__ __forceinline__ float sum_of(const bf16x8 (&x)[2], float c) {
  const bf16x2 ones = {(bf16)1.0f, (bf16)1.0f};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[i >> 2][2 * (i & 3)], x[i >> 2][2 * (i & 3) + 1]}, ones, c, false);
  return c;
}

// ---------------------------------------------------------------------------
// Host side: what every entry point checks, and the choice of a kernel
// ---------------------------------------------------------------------------
struct ScoredCall {
  const void* p[9];
  int64_t st[27];
  ScoreArgs args;
  int dim;
  bool cap;

  View view(int i) const { return {(const bf16*)p[i], st[3 * i], st[3 * i + 1], st[3 * i + 2]}; }
  MutView out(int i) const { return {(bf16*)const_cast<void*>(p[i]), st[3 * i], st[3 * i + 1], st[3 * i + 2]}; }

  // kv: bit i set where tensor i has kv_heads heads (for its default strides).
  int init(const void* const* tensors, int n, uint32_t kv, int batch, int heads, int kv_heads, int seq, int head_dim,
           const int64_t* strides, float softmax_scale, float score_cap, const float* slopes, const int32_t* prefix) {
    for (int i = 0; i < n; ++i) {
      if (!tensors[i]) return GPTRIG_E_NULL;
      if ((uintptr_t)tensors[i] & 15) return GPTRIG_E_SHAPE;
      p[i] = tensors[i];
    }
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq <= 0 || head_dim <= 0 || head_dim % 8)
      return GPTRIG_E_SHAPE;
    if (head_dim > 128) return GPTRIG_E_UNSUPPORTED;
    // 2^22 workgroups of up to 512 threads (a launch has fewer than 2^32 threads).
    if ((long long)batch * heads * (((long long)seq + 63) / 64) > 1 << 22) return GPTRIG_E_SHAPE;
    if (!(softmax_scale > 0.f) || !(softmax_scale <= 3.0e38f)) return GPTRIG_E_SHAPE;
    if (!(score_cap >= 0.f) || score_cap > 1000.f) return GPTRIG_E_SHAPE;
    dim = head_dim;
    for (int i = 0; i < n; ++i) {
      const int64_t hn = kv >> i & 1 ? kv_heads : heads;
      const int64_t plain[3] = {hn * seq * head_dim, (int64_t)seq * head_dim, head_dim};
      for (int j = 0; j < 3; ++j) {
        const int64_t s = strides ? strides[3 * i + j] : plain[j];
        if (s < 0 || (s & 7)) return GPTRIG_E_SHAPE;
        st[3 * i + j] = s;
      }
      // A (batch, head) slice is addressed by 32-bit byte offsets, a tile past its end included.
      if (((long long)seq + 64) * st[3 * i + 2] * 2 >= (1ll << 31)) return GPTRIG_E_SHAPE;
    }
    cap = score_cap > 0.f;
    args.raw = softmax_scale * GPTRIG_LOG2E;
    args.cap2 = score_cap * GPTRIG_LOG2E;
    if (cap) {
      args.raw = 2.0f * GPTRIG_LOG2E * (softmax_scale / score_cap);
      if (!(args.raw > 0.f && args.raw <= 3.0e38f)) return GPTRIG_E_SHAPE;
    }
    args.slopes = slopes;
    args.prefix = prefix;
    return GPTRIG_OK;
  }
};

// Whether workgroups own 64 rows instead of 128, two waves to every 32 of them
// (each with one half of every tile): where there are few workgroups for the CUs'
// slots, of uneven length at that, since it halves the longest.  us with 128 / 64
// rows, 12 heads, capped, in brackets the workgroups of 128.  Rows of the forward and
// of dq, forward and backward: D64 B4 S1024 (384) 29 / 23 and 84 / 81, B4 S2048 (768) 63
// / 54 and 168 / 160, B8 S2048 (1536) 94 / 97 and 277 / 290, B2 S8192 documents (1536)
// 157 / 163 and 366 / 390; D128 B4 S1024 35 / 32, B4 S2048 83 / 83, B8 S2048 142 / 156.
// Keys of the backward: D64 B4 S1024 83 / 79, B4 S2048 166 / 160, B8 S2048 290 / 305;
// D128 B1 S1024 (96) 69 / 63, B2 S1024 (192) 75 / 71, B4 S1024 102 / 119, B4 S2048 263 /
// 312.
inline bool split_rows(long long batch_heads, int seq, int dim, bool keys) {
  const int most = dim <= 64 ? 1024 : keys ? 192 : 768;
  return batch_heads * ceil_div(seq, 128) <= most;
}

// Rows of a workgroup of the forward and of dq, keys of one of dk and dv, and the
// parts that the heads of a group are divided into for the latter: the fewest that
// divide it and give kWant workgroups (they are of uneven length, so several a CU;
// each part's sums are written and read once more).  us of a backward with kWant
// 256 / 512 / 1024, 16 query heads on 4: D128 B4 S2048 391 / 331 / 375, B2 S2048 224 /
// 191 / 194, B4 S2048 documents 474 / 363 / 344; D64 B4 S2048 274 / 242 / 252, B8 S2048
// 382 / 382 / 387.
constexpr long long kWant = 512;
struct Blocks {
  bool row_split, key_split;
  int rows, keys, parts;  // rows and keys of a block
  Blocks(int batch, int heads, int kv_heads, int seq, int dim) {
    const int G = heads / kv_heads;
    const long long blocks = (long long)batch * kv_heads * ceil_div(seq, 128);
    parts = G;
    for (int p = 1; p < G; ++p)
      if (G % p == 0 && blocks * p >= kWant) {
        parts = p;
        break;
      }
    row_split = split_rows((long long)batch * heads, seq, dim, false);
    key_split = split_rows((long long)batch * kv_heads * parts, seq, dim, true);
    rows = row_split ? 64 : 128;
    keys = key_split ? 64 : 128;
  }
};

// Which block a workgroup has: by a plan (see scored_plan_kernel) that lists
// batch x blocks, the longest first, each for all its heads; or by rank, the last
// block first where `last_first` (longest first, without a prefix or documents).
__device__ __forceinline__ void block_of(const int* plan, int id, int blocks, int batch, int heads, bool last_first,
                                         int& bh, int& block) {
  if (plan) {
    const int item = min(max(plan[id / heads], 0), batch * blocks - 1);
    bh = item / blocks * heads + id % heads;
    block = item % blocks;
  } else {
    xcd_map(id, blocks, batch * heads, bh, block);
    if (last_first) block = blocks - 1 - block;
  }
}

// CALL(head dim of the kernel, cap, bias, segment ids) for a call c.
#define SCORED_BIAS_SEG(CALL, c, D, CAP, seg)                                                          \
  do {                                                                                                 \
    if (c.args.slopes && seg) { CALL(D, CAP, true, true); }                                            \
    else if (c.args.slopes) { CALL(D, CAP, true, false); }                                             \
    else if (seg) { CALL(D, CAP, false, true); }                                                       \
    else { CALL(D, CAP, false, false); }                                                               \
  } while (0)
#define SCORED_DISPATCH(CALL, c, seg)                                                                  \
  do {                                                                                                 \
    if (c.dim <= 64 && c.cap) SCORED_BIAS_SEG(CALL, c, 64, true, seg);                                 \
    else if (c.dim <= 64) SCORED_BIAS_SEG(CALL, c, 64, false, seg);                                    \
    else if (c.cap) SCORED_BIAS_SEG(CALL, c, 128, true, seg);                                          \
    else SCORED_BIAS_SEG(CALL, c, 128, false, seg);                                                    \
  } while (0)

}  // namespace
