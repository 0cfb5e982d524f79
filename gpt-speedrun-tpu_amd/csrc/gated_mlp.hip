// Gated feed-forward block on the GEMM core.
//
//   [g | u] = x W,  W [d][2f]      h = act(g) u      y = h V,  V [f][d_out]
//   dh = dy V^T     dg = dh u act'(g)     du = dh act(g)
//   dx = [dg | du] W^T     dW = x^T [dg | du]     dV = h^T dy
//   act(g) = g s(g) (silu, s the logistic function) or gelu(g), tanh form
//
// Every product is bound by the matrix cores: 6 n d f operations forward and 12
// n d f backward (d_out = d), against a few bytes for each of n (d + f).  What
// stands beside the products is therefore kept inside them:
//   - gate and up columns of W take turns in a tile in blocks of 32 (a paired
//     operand of the core), so a lane holds g and u of the same 16 features of one
//     token and makes h of them;
//   - the product dy V^T reads g and u in its epilogue and writes dg and du.
// Roundings: h, dg and du to bfloat16, in which the next product takes them, g and u
// to 11 bits where the backward is to find them (h itself comes from the unrounded
// ones).  Everything else is float32.
//
// The weight gradients cut the tokens into slices where the tiles alone do not
// fill the chip; each slice writes its float32 sums to the workspace and a small
// pass adds them in order, so the result does not depend on timing.
//
// Measured, 65536 tokens, d 768, f 2048 (a large library product reaches 1000 to 1200
// TFLOP/s): x W with what is kept 472 us (873 TFLOP/s; 0.8 GB written), h V 208 (991),
// dy V^T 399 (517; 1.1 GB read and written), dx 374 (1103), both weights' gradients 622
// (994) and 26 for their parts.
#include "tile_core.h"

namespace {

using tile::f16;
using tile::f16x8;
using tile::i16x8;

using gemm::BM;
using gemm::BN;
using gemm::Operand;

enum { kSilu = 0, kGelu = 1 };

// The activation and its derivative.
template <int kAct>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (kAct == kGelu) return gelu_f(x);
  return x * __builtin_amdgcn_rcpf(1.0f + fast_exp2(-GPTRIG_LOG2E * x));
}
template <int kAct>
__device__ __forceinline__ void act_both(float x, float& a, float& slope) {
  if constexpr (kAct == kGelu) {
    a = gelu_f(x);
    slope = gelu_grad_f(x);
  } else {
    const float s = __builtin_amdgcn_rcpf(1.0f + fast_exp2(-GPTRIG_LOG2E * x));
    a = x * s;
    slope = s * __builtin_fmaf(x, 1.0f - s, 1.0f);
  }
}

// What the backward finds of g and u: float16 [n][2f], each run of 16 features (the
// last may be shorter) scaled by a power of two that brings its largest to 2^14 ..
// 2^15, and those powers, a byte each, [2][runs][n].  11 bits where bfloat16 has 8,
// in the same space: with bfloat16 the gradients of x and W were 1.76 times as far
// off as their own rounding alone, which is 1.41 times now.  (What is 2^-39 of its
// run's largest or less is lost: float16 ends at 2^-25.)
__host__ __device__ inline int runs_of(int f) { return (f + 15) / 16; }

struct Kept {
  f16* values;
  uint8_t* powers;

  // Of the lane's token and of its run in block `block` of 32 features from f0 (a
  // multiple of 64) on.
  static __device__ __forceinline__ uint32_t power_at(int block, int f0, int first, int n, int f, int lane) {
    const bool inside = f0 + 32 * block + 16 * (lane >> 5) < f && first + (lane & 31) < n;
    return inside ? (lane >> 5) * (uint32_t)n + (lane & 31) : gemm::kOffZero;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t power_rows(int half, int block, int f0, int first, int n, int f) const {
    return make_rsrc(powers + ((int64_t)half * runs_of(f) + (f0 >> 4) + 2 * block) * n + first, gemm::kRsrcRange);
  }
  __device__ __forceinline__ void put_power(int half, int block, int power, int f0, int first, int n, int f,
                                            int lane) const {
    __builtin_amdgcn_raw_buffer_store_b8((uint8_t)power, power_rows(half, block, f0, first, n, f),
                                         power_at(block, f0, first, n, f, lane), 0, 0);
  }
  __device__ __forceinline__ int get_power(int half, int block, int f0, int first, int n, int f, int lane) const {
    return __builtin_amdgcn_raw_buffer_load_b8(power_rows(half, block, f0, first, n, f),
                                               power_at(block, f0, first, n, f, lane), 0, 0);
  }
};

// The float32 exponent field of a run's largest value, and the factor that goes with it.
// The lowest power is 15, whose factor 2^126 and its reciprocal are both normal numbers: a
// run whose largest is below 2^-112 stays below 2^14.  Infinities and NaN stay what they are
// at any power and do not count.
__device__ __forceinline__ int power_of(const float (&v)[16]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]));
  if (most == __builtin_inff()) {
    most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]) == __builtin_inff() ? 0.f : fabsf(v[i]));
  }
  return max(15, __builtin_bit_cast(int, most) >> 23);
}
__device__ __forceinline__ float scale_down(int power) { return __builtin_bit_cast(float, (268 - power) << 23); }
// Its reciprocal.  (Of a power that is not there, and reads 0, any number: its values are zeros.)
__device__ __forceinline__ float scale_up(int power) { return __builtin_bit_cast(float, (uint32_t)(power - 14) << 23); }

// A wave's 32 rows of 64 features of 16 bits in LDS, on the way between its
// accumulators' layout (runs of 16 features of a row) and lines: eight lanes hold 128
// bytes of a row.  (tile::Block's reasons; here the rows lie in row-major matrices,
// where 64 features make a whole line.)  The memory is beside the stage ring, which
// fills for the next tile meanwhile.
__shared__ __attribute__((aligned(1024))) short g_band[8 * 2048];

// A thread's lane, worked out anew: what a tile's end derives from it does not wait in
// registers through the main loop.
__device__ __forceinline__ int fresh_lane() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid & 63;
}

struct Band {
  int lane, offset;
  static __device__ __forceinline__ void order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
  // (An opaque sum, see tile::frag; volatile, or all of them would wait in registers
  // through the main loop.)
  __device__ __forceinline__ tile::lds16x8* slot(int row, int chunk) const {
    int at = offset + row * 64 + 8 * (chunk ^ ((row >> 1) & 7));
    asm volatile("" : "+v"(at));
    return (tile::lds16x8*)((tile::lds16*)g_band + at);
  }
  __device__ __forceinline__ void put_run(int block, i16x8 low, i16x8 high) const {
    *slot(lane & 31, 4 * block + 2 * (lane >> 5)) = low;
    *slot(lane & 31, 4 * block + 2 * (lane >> 5) + 1) = high;
  }
  __device__ __forceinline__ i16x8 get_run(int block, int half) const {
    return *slot(lane & 31, 4 * block + 2 * (lane >> 5) + half);
  }
  // Offsets of the lane's pieces of rows 8 it .. from a uniform place (first row, first
  // feature) of a matrix, as many as there are; past them one that reads zeros and
  // writes nothing.
  __device__ __forceinline__ uint32_t line(int it, uint32_t ld, int rows, int features) const {
    const int row = 8 * it + (lane >> 3);
    return row < rows && 8 * (lane & 7) < features ? 2 * (row * ld + 8 * (lane & 7)) : gemm::kOffZero;
  }
  // (All of the offset in the vector register: with a part in a scalar one the compiler
  // let the store's first data register be written anew before the last lanes of every
  // 16 had been read, here on gfx950.)
  __device__ __forceinline__ void store(void* place, uint32_t ld, int rows, int features) const {
    order();
    const __amdgpu_buffer_rsrc_t r = make_rsrc(place, gemm::kRsrcRange);
#pragma unroll
    for (int it = 0; it < 4; ++it)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, *slot(8 * it + (lane >> 3), lane & 7)), r,
                                             line(it, ld, rows, features), 0, 0);
    order();
  }
  __device__ __forceinline__ void fetch(i16x8 (&v)[4], const void* place, uint32_t ld, int rows, int features) const {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(place, gemm::kRsrcRange);
#pragma unroll
    for (int it = 0; it < 4; ++it)
      v[it] = __builtin_bit_cast(
          i16x8, __builtin_amdgcn_raw_buffer_load_b128(r, line(it, ld, rows, features), 0, 0));
  }
  __device__ __forceinline__ void put_lines(const i16x8 (&v)[4]) const {
    order();
#pragma unroll
    for (int it = 0; it < 4; ++it) *slot(8 * it + (lane >> 3), lane & 7) = v[it];
    order();
  }
};

__device__ __forceinline__ i16x8 bf16_run(const float* v) { return __builtin_bit_cast(i16x8, pack8(v)); }
__device__ __forceinline__ i16x8 f16_run(const float* v, float scale) {
  f16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (f16)(v[i] * scale);
  return __builtin_bit_cast(i16x8, r);
}

struct UpArgs {
  Kept kept;
  bf16* h;  // [n][f]
  int n, k, f, group;
};

template <int kAct, bool kKeep>
__global__ void __launch_bounds__(gemm::THREADS) gated_up_kernel(Operand W, Operand X, UpArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int ntiles = ((2 * a.f + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  auto coords = [&](int t, int& tm, int& tn) { gemm::tile_coords(t, 2 * a.f, a.n, tm, tn, a.group); };
  auto pre = [](int, int) {};
  auto epi = [&](f32x16(&acc)[4][2], int tm, int tn) {
    const int f0 = tm * (BM / 2) + 64 * wm;
    if (f0 >= a.f) return;  // (uniform; no barrier below)
    const int lane = fresh_lane();
    const Band band{lane, wave * 2048};
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int first = tn * BN + 64 * wn + 32 * nb;
      Band::order();
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = act_f<kAct>(acc[2 * p][nb][i]) * acc[2 * p + 1][nb][i];
        band.put_run(p, bf16_run(h), bf16_run(h + 8));
      }
      band.store(a.h + (int64_t)first * a.f + f0, a.f, a.n - first, a.f - f0);
      if constexpr (kKeep) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // gate, up
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = acc[2 * p + half][nb][i];
            const int power = power_of(v);
            const float scale = scale_down(power);
            band.put_run(p, f16_run(v, scale), f16_run(v + 8, scale));
            a.kept.put_power(half, p, power, f0, first, a.n, a.f, lane);
          }
          band.store(a.kept.values + (int64_t)first * 2 * a.f + (int64_t)half * a.f + f0, 2 * a.f, a.n - first, a.f - f0);
        }
      }
    }
  };
  gemm::persistent<false, true, true, true>(W, X, 2 * a.f, a.n, a.k, ntiles, coords, pre, epi);
}

struct DownBwdArgs {
  Kept kept;
  bf16* d_gate_up;  // [n][2f], rows ld apart
  int ld, n, k, f, group;
};

template <int kAct>
__global__ void __launch_bounds__(gemm::THREADS) gated_down_bwd_kernel(Operand V, Operand DY, DownBwdArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int ntiles = ((a.f + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  auto coords = [&](int t, int& tm, int& tn) { gemm::tile_coords(t, a.f, a.n, tm, tn, a.group); };
  auto pre = [](int, int) {};
  auto epi = [&](f32x16(&acc)[4][2], int tm, int tn) {
    const int lane = threadIdx.x & 63;
    const Band band{lane, wave * 2048};
    // 32 tokens x 64 features at a time, the next ones asked for before the stores.
    i16x8 lines[2][4];
    int powers[2][2];
    auto fetch = [&](int step) {
      const int f0 = tm * BM + 128 * wm + 64 * (step & 1), first = tn * BN + 64 * wn + 32 * (step >> 1);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        band.fetch(lines[half], a.kept.values + (int64_t)first * 2 * a.f + (int64_t)half * a.f + f0, 2 * a.f,
                   a.n - first, a.f - f0);
#pragma unroll
        for (int p = 0; p < 2; ++p) powers[half][p] = a.kept.get_power(half, p, f0, first, a.n, a.f, lane);
      }
    };
    fetch(0);
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const int f0 = tm * BM + 128 * wm + 64 * (step & 1), first = tn * BN + 64 * wn + 32 * (step >> 1);
      const int nb = step >> 1;
      i16x8 g[2][2];
      band.put_lines(lines[0]);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) g[p][h] = band.get_run(p, h);
      band.put_lines(lines[1]);
      GEMM_SCHED_FENCE();
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float scale_g = scale_up(powers[0][p]), scale_u = scale_up(powers[1][p]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // dg takes u's place in the band, du that of g in registers.
          tile::lds16x8* const at = band.slot(lane & 31, 4 * p + 2 * (lane >> 5) + h);
          const f16x8 gates = __builtin_bit_cast(f16x8, g[p][h]), ups = __builtin_bit_cast(f16x8, *at);
          float vg[8], vu[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float dh = acc[2 * (step & 1) + p][nb][8 * h + i];
            float value, slope;
            act_both<kAct>((float)gates[i] * scale_g, value, slope);
            vg[i] = dh * ((float)ups[i] * scale_u) * slope;
            vu[i] = dh * value;
          }
          *at = bf16_run(vg);
          g[p][h] = bf16_run(vu);
          GEMM_SCHED_FENCE();  // (the eights one after another: together they pass the registers)
        }
      }
      if (step < 3) fetch(step + 1);
      bf16* const place = a.d_gate_up + (int64_t)first * a.ld + f0;
      band.store(place, a.ld, a.n - first, a.f - f0);
#pragma unroll
      for (int p = 0; p < 2; ++p) band.put_run(p, g[p][0], g[p][1]);
      band.store(place + a.f, a.ld, a.n - first, a.f - f0);
    }
  };
  gemm::persistent<true, true, true>(V, DY, a.f, a.n, a.k, ntiles, coords, pre, epi);
}

// ---- few tokens ----
//
// The same three products in tiles of 64 tokens, where those of 256 x 256 would leave
// most of the chip idle.  Four sets of waves share a tile's K and add their parts
// through LDS: a workgroup's time is that of its loads, one after the other.

// A workgroup's tile.  kByTokens: those of one token tile follow one another on one
// XCD, whose L2 then reads the tokens once (h V and dx of 8192 tokens 39 -> 33 and 79
// -> 68 us); else they are dealt out to the XCDs in turn, which spreads the weights
// (x W of 1024 tokens 20 against 26 us).
template <bool kByTokens>
__device__ __forceinline__ void few_tile(int features, int tile_m, int& tm, int& tn) {
  const int across = (features + tile_m - 1) / tile_m;
  const int pid = kByTokens ? gemm::xcd_swizzle(blockIdx.x, gridDim.x) : blockIdx.x;
  tm = pid % across;
  tn = pid / across;
}

// A lane's run of 16 features of a row.
__device__ __forceinline__ void store_run(bf16* row, int feature, int features, const float* v) {
  if (feature < features) *reinterpret_cast<bf16x8*>(row + feature) = pack8(v);
  if (feature + 8 < features) *reinterpret_cast<bf16x8*>(row + feature + 8) = pack8(v + 8);
}

template <int kAct>
__global__ void __launch_bounds__(1024) gated_up_few_kernel(tile::Operand W, tile::Operand X, UpArgs a) {
  typedef tile::Product<bf16, 2, 1, tile::kPairsMN, tile::kRowsK, true, 1, 4, 3> P;
  const auto at = P::place();
  int tm, tn;
  few_tile<false>(2 * a.f, P::TM, tm, tn);
  f32x16 acc[2][1];
  P::run(acc, W, X, 2 * a.f, a.n, a.k, tm * P::TM, tn * P::TN, at);
  if (at.group) return;
  const int lane = at.lane, first = tn * P::TN + 32 * at.wn, token = first + (lane & 31);
  const int f0 = tm * (P::TM / 2) + 32 * at.wm, feature = f0 + 16 * (lane >> 5);
  float g[16], u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    g[i] = acc[0][0][i];
    u[i] = acc[1][0][i];
  }
  if (a.kept.values) {
    // (Powers are laid out by blocks of 64 features.)
    const int block = (f0 >> 5) & 1;
    const int power_g = power_of(g), power_u = power_of(u);
    a.kept.put_power(0, block, power_g, f0 & ~63, first, a.n, a.f, lane);
    a.kept.put_power(1, block, power_u, f0 & ~63, first, a.n, a.f, lane);
    if (token < a.n) {
      short* const row = (short*)a.kept.values + (int64_t)token * 2 * a.f + feature;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (feature + 8 * e < a.f) {
          *(i16x8*)(row + 8 * e) = f16_run(g + 8 * e, scale_down(power_g));
          *(i16x8*)(row + a.f + 8 * e) = f16_run(u + 8 * e, scale_down(power_u));
        }
    }
  }
  if (token >= a.n) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (feature + 8 * e >= a.f) continue;
    float h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = act_f<kAct>(g[8 * e + i]) * u[8 * e + i];
    *reinterpret_cast<bf16x8*>(a.h + (int64_t)token * a.f + feature + 8 * e) = pack8(h);
  }
}

template <int kAct>
__global__ void __launch_bounds__(1024) gated_down_bwd_few_kernel(tile::Operand V, tile::Operand DY, DownBwdArgs a) {
  typedef tile::Product<bf16, 1, 1, tile::kRowsK, tile::kRowsK, true, 1, 4> P;
  const auto at = P::place();
  int tm, tn;
  few_tile<false>(a.f, P::TM, tm, tn);
  f32x16 acc[1][1];
  P::run(acc, V, DY, a.f, a.n, a.k, tm * P::TM, tn * P::TN, at);
  if (at.group) return;
  const int lane = at.lane, first = tn * P::TN + 32 * at.wn, token = first + (lane & 31);
  const int f0 = tm * P::TM + 32 * at.wm, feature = f0 + 16 * (lane >> 5), block = (f0 >> 5) & 1;
  const float scale_g = scale_up(a.kept.get_power(0, block, f0 & ~63, first, a.n, a.f, lane));
  const float scale_u = scale_up(a.kept.get_power(1, block, f0 & ~63, first, a.n, a.f, lane));
  if (token >= a.n) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (feature + 8 * e >= a.f) continue;
    const int64_t own = (int64_t)token * 2 * a.f + feature + 8 * e;
    const f16x8 g = *(const f16x8*)(a.kept.values + own), u = *(const f16x8*)(a.kept.values + own + a.f);
    float dg[8], du[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float dh = acc[0][0][8 * e + i];
      float value, slope;
      act_both<kAct>((float)g[i] * scale_g, value, slope);
      dg[i] = dh * ((float)u[i] * scale_u) * slope;
      du[i] = dh * value;
    }
    bf16* const to = a.d_gate_up + (int64_t)token * a.ld + feature + 8 * e;
    *reinterpret_cast<bf16x8*>(to) = pack8(dg);
    *reinterpret_cast<bf16x8*>(to + a.f) = pack8(du);
  }
}

// y [n][m] = x [n][k] w, w [k][m] (kRowsMN) or [m][k] (kRowsK), in tiles of 64 T x 64 T.
template <tile::Layout kW, int T, int kGroups>
__global__ void __launch_bounds__(256 * kGroups, kGroups == 1 ? 2 : 1)
    gated_linear_few_kernel(tile::Operand W, tile::Operand X, bf16* y, int n, int k, int m) {
  typedef tile::Product<bf16, T, T, kW, tile::kRowsK, true, 1, kGroups> P;
  const auto at = P::place();
  int tm, tn;
  few_tile<true>(m, P::TM, tm, tn);
  f32x16 acc[T][T];
  P::run(acc, W, X, m, n, k, tm * P::TM, tn * P::TN, at);
  if (at.group) return;
#pragma unroll
  for (int nb = 0; nb < T; ++nb) {
    const int token = tn * P::TN + 32 * (T * at.wn + nb) + (at.lane & 31);
    if (token >= n) continue;
#pragma unroll
    for (int mb = 0; mb < T; ++mb) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = acc[mb][nb][i];
      store_run(y + (int64_t)token * m, tm * P::TM + 32 * (T * at.wm + mb) + 16 * (at.lane >> 5), m, v);
    }
  }
}

// ---- weight gradients ----

struct GradItem {
  const bf16 *x, *dy;  // [n][rows], [n][cols]
  int64_t ldx, lddy;
  bf16* dw;      // [rows][cols]
  float* parts;  // [split][rows][cols]
  int rows, cols;
  int first;  // the item's first workgroup
};
struct GradItems {
  GradItem item[2];
  int count, n, split;
};

__global__ void __launch_bounds__(gemm::THREADS) gated_weight_grad_kernel(GradItems g) {
  const int which = g.count > 1 && (int)blockIdx.x >= g.item[1].first;
  const GradItem w = g.item[which];
  const int total = (which + 1 < g.count ? g.item[1].first : (int)gridDim.x) - w.first;
  int tm, tn, split;
  gemm::split_tile_coords((int)blockIdx.x - w.first, total, w.rows, w.cols, tm, tn, split);
  const int slice = ((g.n + g.split - 1) / g.split + gemm::BK - 1) / gemm::BK * gemm::BK;
  const int begin = min(g.n, split * slice), end = min(g.n, begin + slice);
  f32x16 acc[4][2];
  gemm::mainloop_pp<false, false>(acc, Operand{w.x, w.ldx}, Operand{w.dy, w.lddy}, w.rows, w.cols, begin, end, tm * BM,
                                  tn * BN);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hl = lane >> 5, l32 = lane & 31, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int col = tn * BN + 64 * wn + 32 * nb + l32;
    if (col >= w.cols) continue;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
      const int row0 = tm * BM + 128 * wm + 32 * mb + 4 * hl;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = row0 + 8 * (i >> 2) + (i & 3);
        if (row >= w.rows) continue;
        const int64_t at = (int64_t)row * w.cols + col;
        if (g.split == 1)
          w.dw[at] = (bf16)acc[mb][nb][i];
        else
          w.parts[(int64_t)split * w.rows * w.cols + at] = acc[mb][nb][i];
      }
    }
  }
}

__global__ void __launch_bounds__(256) gated_add_parts_kernel(GradItems g) {
  const GradItem w = g.item[blockIdx.y];
  const int64_t size = (int64_t)w.rows * w.cols;
  for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < size; i += 4ll * 256 * gridDim.x) {
    f32x4 sum = *reinterpret_cast<const f32x4*>(w.parts + i);
    for (int s = 1; s < g.split; ++s) sum += *reinterpret_cast<const f32x4*>(w.parts + s * size + i);
    bf16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (bf16)sum[j];
    *reinterpret_cast<bf16x4*>(w.dw + i) = o;
  }
}

int tiles_of(int rows, int cols) { return ceil_div(rows, BM) * ceil_div(cols, BN); }

// Slices of the tokens for both weight gradients: rounds of CUs, each of a
// slice's stages and, in stages, about 20 for the tile's write (and 10 more for
// its share of the pass that adds the parts).
int grad_split(int tiles, int n) {
  const int cus = gemm::device_cus(), stages = ceil_div(n, gemm::BK);
  int best = 1;
  double best_cost = 1e300;
  for (int s = 1; s <= 32 && s <= stages; ++s) {
    const double cost = (double)ceil_div((int64_t)tiles * s, cus) * (((ceil_div(stages, s) + 3) & ~3) + (s > 1 ? 30 : 20));
    if (cost < best_cost * 0.999) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

struct Bwd {
  size_t d_gate_up, parts_w, parts_v, total;  // bytes
  int ld;  // of d_gate_up: rows of whole lines (dx of 5001 x 1000, f 2664: 123 -> 113 us)
  int split;
};

Bwd plan_bwd(int n, int d, int f, int d_out) {
  Bwd b{};
  b.split = grad_split(tiles_of(d, 2 * f) + tiles_of(f, d_out), n);
  b.ld = (2 * f + 63) & ~63;
  b.d_gate_up = round_up((size_t)n * b.ld * 2);
  if (b.split > 1) {
    b.parts_w = round_up((size_t)b.split * d * 2 * f * 4);
    b.parts_v = round_up((size_t)b.split * f * d_out * 4);
  }
  b.total = b.d_gate_up + b.parts_w + b.parts_v;
  return b;
}

Kept kept_at(void* p, int n, int f) {
  return Kept{(f16*)p, p ? (uint8_t*)p + (size_t)n * 2 * f * 2 : nullptr};
}

constexpr int kMostWidth = 1 << 20;
constexpr int64_t kMostStride = 1 << 22;  // a tile's rows stay within the core's 32-bit byte offsets

int check_sizes(int n, int d, int f, int d_out) {
  if (n < 0 || n > 0x7fffff00 || d <= 0 || f <= 0 || d_out <= 0 || d % 8 || f % 8 || d_out % 8) return GPTRIG_E_SHAPE;
  if (d > kMostWidth || 2 * (int64_t)f > kMostWidth || d_out > kMostWidth) return GPTRIG_E_SHAPE;
  const int64_t widest = d > 2 * f ? (d > d_out ? d : d_out) : (2 * f > d_out ? 2 * f : d_out);
  if ((int64_t)ceil_div(n, BN) * ceil_div(widest, BM) >= 0x7fffffff) return GPTRIG_E_SHAPE;
  return GPTRIG_OK;
}

bool rows_ok(const void* p, int64_t ld, int width) {
  return ld >= width && ld % 8 == 0 && ld <= kMostStride && ((uintptr_t)p & 15) == 0;
}

// Tiles of 256 x 256 from which a product takes them.  Measured at d 768, f 2048 (us, by
// tokens, their number behind; the large tiles against 64 tokens with four sets of
// waves, against 128 x 128):
//   x W      1024 (64) 26 / 20, 2048 (128) 28 / 37
//   dy V^T   1024 (32) 33 / 18, 2048 (64) 33 / 33, 4096 (128) 36 / 63
//   h V      1 (3) 42 / 7 / 16, 1024 (12) 44 / 12 / 18, 2048 (24) 45 / 21 / 19,
//            4096 (48) 46 / 33 / 20, 8192 (96) 53 / 65 / 33, 16384 (192) 63 / 129 / 63
//   dx       1 77 / 12 / 28, 1024 82 / 21 / 31, 8192 91 / 130 / 68, 16384 114 / 264 / 127
// That is one pair of widths: the rule knows the number of tiles, not the depth K, and
// elsewhere the better form may be another (dx of 5001 x 1000 with K 5328, 80 tiles: 111
// in 128 x 128, 82 in large tiles cut along K with their parts added after).
constexpr int kPairTiles = 68;                   // x W and dy V^T, against 64 tokens
constexpr int kLinearTiles = 150, kLinearFew = 18;  // h V and dx, against 128 x 128; those against 64 x 64

unsigned persistent_grid(int tiles) {
  const int cus = gemm::device_cus();
  return (unsigned)(tiles < cus ? tiles : cus);
}

int tile_group(int m_tiles) { return m_tiles <= 16 ? m_tiles : gemm::kGroupM; }

// Whether the product of m features over n tokens with g and u at its end goes to the tiles of 64 tokens.
bool few(int n, int m) { return tiles_of(m, n) < kPairTiles; }

unsigned few_grid(int m, int tile_m, int n, int tile_n = 64) { return (unsigned)(ceil_div(m, tile_m) * ceil_div(n, tile_n)); }

template <tile::Layout kW>
void launch_linear_few(const tile::Operand& W, const tile::Operand& X, void* y, int n, int k, int m, bool wide,
                       hipStream_t s) {
  if (wide)
    gated_linear_few_kernel<kW, 2, 1><<<few_grid(m, 128, n, 128), 256, 0, s>>>(W, X, (bf16*)y, n, k, m);
  else
    gated_linear_few_kernel<kW, 1, 4><<<few_grid(m, 64, n), 1024, 0, s>>>(W, X, (bf16*)y, n, k, m);
}

int linear(const void* x, int64_t ldx, const void* w, int64_t ldw, bool w_kmajor, void* y, int n, int k, int m,
           hipStream_t s) {
  const int tiles = tiles_of(m, n);
  if (tiles >= kLinearTiles) return gptrig_linear(x, ldx, w, ldw, w_kmajor, nullptr, y, m, n, k, m, s);
  const tile::Operand W{w, ldw}, X{x, ldx};
  if (w_kmajor)
    launch_linear_few<tile::kRowsK>(W, X, y, n, k, m, tiles >= kLinearFew, s);
  else
    launch_linear_few<tile::kRowsMN>(W, X, y, n, k, m, tiles >= kLinearFew, s);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

template <int kAct>
void launch_up(const Operand& W, const Operand& X, const UpArgs& a, hipStream_t s) {
  if (few(a.n, 2 * a.f)) {
    const tile::Operand w{W.p, W.ld, W.pair}, x{X.p, X.ld};
    gated_up_few_kernel<kAct><<<few_grid(2 * a.f, 128, a.n), 1024, 0, s>>>(w, x, a);
    return;
  }
  const unsigned grid = persistent_grid(tiles_of(2 * a.f, a.n));
  if (a.kept.values)
    gated_up_kernel<kAct, true><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
  else
    gated_up_kernel<kAct, false><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
}

template <int kAct>
void launch_down_bwd(const Operand& V, const Operand& DY, const DownBwdArgs& a, hipStream_t s) {
  if (few(a.n, a.f))
    gated_down_bwd_few_kernel<kAct><<<few_grid(a.f, 64, a.n), 1024, 0, s>>>({V.p, V.ld}, {DY.p, DY.ld}, a);
  else
    gated_down_bwd_kernel<kAct><<<persistent_grid(tiles_of(a.f, a.n)), gemm::THREADS, 0, s>>>(V, DY, a);
}

}  // namespace

extern "C" {

int gptrig_gated_mlp_fwd(const void* x, int64_t ldx, const void* gate_up_w, int64_t ldw, const void* down_w,
                         int64_t ldv, int activation, void* kept, void* h, void* y, int n, int d, int f, int d_out,
                         void* stream) {
  if (!x || !gate_up_w || !down_w || !h || !y) return GPTRIG_E_NULL;
  if (activation != kSilu && activation != kGelu) return GPTRIG_E_UNSUPPORTED;
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK) return GPTRIG_E_SHAPE;
  if (!rows_ok(x, ldx, d) || !rows_ok(gate_up_w, ldw, 2 * f) || !rows_ok(down_w, ldv, d_out)) return GPTRIG_E_SHAPE;
  if (((uintptr_t)kept | (uintptr_t)h | (uintptr_t)y) & 15) return GPTRIG_E_SHAPE;
  if (n == 0) return GPTRIG_OK;
  const hipStream_t s = (hipStream_t)stream;
  const Operand W{(const bf16*)gate_up_w, ldw, 0, f}, X{(const bf16*)x, ldx};
  const UpArgs a{kept_at(kept, n, f), (bf16*)h, n, d, f, tile_group(ceil_div(2 * f, BM))};
  if (activation == kSilu)
    launch_up<kSilu>(W, X, a, s);
  else
    launch_up<kGelu>(W, X, a, s);
  GPTRIG_CHECK_LAUNCH();
  return linear(h, f, down_w, ldv, false, y, n, f, d_out, s);
}

size_t gptrig_gated_mlp_kept_bytes(int n, int f) {
  if (check_sizes(n, 8, f, 8) != GPTRIG_OK) return 0;
  return (size_t)n * 2 * f * 2 + (size_t)n * 2 * runs_of(f);
}

size_t gptrig_gated_mlp_bwd_workspace_bytes(int n, int d, int f, int d_out) {
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK || n == 0) return 0;
  return plan_bwd(n, d, f, d_out).total;
}

int gptrig_gated_mlp_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* gate_up_w, int64_t ldw,
                         const void* down_w, int64_t ldv, int activation, const void* kept, const void* h, void* dx,
                         void* d_gate_up_w, void* d_down_w, int n, int d, int f, int d_out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (!dy || !x || !gate_up_w || !down_w || !kept || !h || !workspace) return GPTRIG_E_NULL;
  if (activation != kSilu && activation != kGelu) return GPTRIG_E_UNSUPPORTED;
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK || n == 0) return GPTRIG_E_SHAPE;
  if (!rows_ok(x, ldx, d) || !rows_ok(dy, lddy, d_out) || !rows_ok(gate_up_w, ldw, 2 * f) ||
      !rows_ok(down_w, ldv, d_out))
    return GPTRIG_E_SHAPE;
  if (((uintptr_t)kept | (uintptr_t)h | (uintptr_t)dx | (uintptr_t)d_gate_up_w | (uintptr_t)d_down_w |
       (uintptr_t)workspace) & 15)
    return GPTRIG_E_SHAPE;
  const Bwd b = plan_bwd(n, d, f, d_out);
  if (workspace_bytes < b.total) return GPTRIG_E_WORKSPACE;
  const hipStream_t s = (hipStream_t)stream;
  bf16* const dgu = (bf16*)workspace;
  if (dx || d_gate_up_w) {
    const Operand V{(const bf16*)down_w, ldv}, DY{(const bf16*)dy, lddy};
    const DownBwdArgs a{kept_at(const_cast<void*>(kept), n, f), dgu, b.ld, n, d_out, f, tile_group(ceil_div(f, BM))};
    if (activation == kSilu)
      launch_down_bwd<kSilu>(V, DY, a, s);
    else
      launch_down_bwd<kGelu>(V, DY, a, s);
    GPTRIG_CHECK_LAUNCH();
  }
  if (dx) {
    const int status = linear(dgu, b.ld, gate_up_w, ldw, true, dx, n, 2 * f, d, s);
    if (status != GPTRIG_OK) return status;
  }
  GradItems g{};
  g.n = n;
  g.split = b.split;
  int first = 0;
  if (d_gate_up_w) {
    g.item[g.count++] = GradItem{(const bf16*)x, dgu, ldx, b.ld, (bf16*)d_gate_up_w,
                                 (float*)((char*)workspace + b.d_gate_up), d, 2 * f, first};
    first += tiles_of(d, 2 * f) * b.split;
  }
  if (d_down_w) {
    g.item[g.count++] = GradItem{(const bf16*)h, (const bf16*)dy, f, lddy, (bf16*)d_down_w,
                                 (float*)((char*)workspace + b.d_gate_up + b.parts_w), f, d_out, first};
    first += tiles_of(f, d_out) * b.split;
  }
  if (g.count) {
    gated_weight_grad_kernel<<<first, gemm::THREADS, 0, s>>>(g);
    GPTRIG_CHECK_LAUNCH();
    if (b.split > 1) {
      gated_add_parts_kernel<<<dim3(512, g.count), 256, 0, s>>>(g);
      GPTRIG_CHECK_LAUNCH();
    }
  }
  return GPTRIG_OK;
}

}  // extern "C"
