// Orthogonalised updates by Newton-Schulz products (as the Muon optimiser uses them).
//
// For a matrix u [rows][cols], with m the shorter and n the longer side and X [m][n]
// the matrix u / (|u| + eps) (|u| the root of its squares' sum) or its transpose:
//   steps times   A = X X^T,   B = b A + c A A,   X <- a X + B X
// and the result X, transposed back, in bfloat16.  It drives the singular values
// towards 1 and leaves the directions as they are.
//
// Bound: the matrix cores.  A step has 6 m m n operations less the symmetric halves:
// A and A A are symmetric, and only their tiles on and below the diagonal are
// computed, each written twice (3 m m n + m m m instead of 4 m m n + 2 m m m).
//
// What is held in fewer than 32 bits.  The products take float16 operands (11 bits;
// every value here is below 2 in size, the normalised X's around (m n)^-1/2, and
// what float16 flushes near 2^-25 is far below the sums' own rounding) and add in
// float32.  X itself is held in two float16, the operand `hi` and the rest `lo`,
// scaled by 2^11 so that it keeps its bits: 22 bits, or 2^-36 where that is more (values
// below 2^-14).  That is what the result needs:
// an error of X in the directions of small singular values grows by a each step (485
// times in five), but only through the term a X, which is computed from all 22 bits;
// in B X the rounding of X meets B, which is small in those directions, and the
// rounding of B multiplies what is there.  The diagonals of A and B stay in float32
// and out of the products (A = D + O: A A = D D + D O + O D + O O; a X + B X = (a +
// diag B) X + the rest): the more alike the singular values, the more of A and B lies
// there.  In simulations, of 1 to 2000 rows and of spectra from flat to falling by
// 10^6, the result is then off by 1.0 to 1.2 times the rounding to bfloat16 alone (1.6
// for some of five rows); with the diagonals in float16 by 1.0 to 2.8 times, with X in
// one float16 by up to 24, in one bfloat16 by up to 200.
//
// One launch does a product for every matrix of a list (48 matrices of a model of 12
// layers fill the chip where one would not); matrices of one shape are a group, laid
// out at a stride, and the groups' table travels as a kernel argument.
//
// Measured, 48 matrices of 768 rows (85M float32) and five steps: the norms 81 us (4.2
// TB/s), the load 116 (680 MB, what the norms read in part from the last cache), a gram
// product 100 (12 of 18 tiles, 870 TFLOP/s with what they hold twice), a square 52, an
// update 213 (130 GFLOP, 613 TFLOP/s: 112 us for the product alone, the rest for X's 680
// MB in and out at its end).
#include "tile_core.h"

namespace {

using tile::f16;
using tile::f16x8;
using tile::i16x8;

constexpr int kMostGroups = 16;   // shapes of a launch
constexpr int kMostTensors = 64;  // tensors of a launch
constexpr int kPart = 16384;      // elements of a partial sum of squares
constexpr float kLow = 2048.0f;   // scale of X's lower part
constexpr int64_t kMostBytes = 2ll << 30;  // workspace of a launch, where a matrix alone does not need more

struct Group {
  int m, n;      // the shorter and the longer side
  int tall;      // the tensors have more rows than columns: X is the transpose
  int count;     // matrices
  int parts;     // partial sums of squares a matrix
  int sum0;      // the first one's index
  int64_t x0;    // first element in hi and lo
  int64_t a0;    // in A and B
  int64_t d0;    // in their diagonals
  // Columns of X and of A with their padding: whole blocks of 32.
  __host__ __device__ int ldx() const { return (n + 31) & ~31; }
  __host__ __device__ int lda() const { return (m + 31) & ~31; }
};

// X, A and B lie 32-blocked with m rows (tile_core.h): element (r, c).
__device__ __forceinline__ int64_t blocked(int m, int r, int c) { return ((int64_t)(c >> 5) * m + r) * 32 + (c & 31); }

struct Tensor {
  const void* in;
  bf16* out;
  int group, first;  // its matrices are first, first + 1, ... of the group
};

struct Args {
  Group g[kMostGroups];
  Tensor t[kMostTensors];
  int first[kMostGroups + 1];  // each group's first workgroup of this launch, and the end in the others
  int groups, tensors;
  double* sums;
  f16 *hi, *hi_next, *lo, *A, *B;
  float *diag_a, *diag_b;  // of A, and a more than of B; A and B themselves have zeros there
  float a, b, c, eps;
};

// Workgroup -> group, and its index within it.  kSpread: each XCD takes a
// contiguous share of every group, so that tiles that read the same rows meet in
// one L2 and no XCD gets the matrices with the longest rows (the gram products of a
// model's 48 matrices: 163 us with a contiguous share of the whole launch).
template <bool kSpread>
__device__ __forceinline__ int find_group(const Args& s, int pid, int& local) {
  // (All of s.first in one load: a search would wait for each of its own.)
  int g = 0;
#pragma unroll
  for (int i = 1; i < kMostGroups; ++i) g += pid >= s.first[i];
  local = pid - s.first[g];
  if (kSpread) local = gemm::xcd_swizzle(local, s.first[g + 1] - s.first[g]);
  return g;
}

__device__ __forceinline__ const Tensor& find_tensor(const Args& s, int group, int matrix) {
  int at = 0;
  for (int i = 0; i < s.tensors; ++i)
    if (s.t[i].group == group && s.t[i].first <= matrix) at = i;  // (ascending within a group)
  return s.t[at];
}

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((shared[0] + shared[1]) + shared[2]) + shared[3];
}

// A float32 that stays one: without it the compiler may round a product or a sum to
// float16 from its exact value where the float16 is stored and from its float32 value
// where the rest is taken from it, and in one of some thousand the two differ by a
// step.
__device__ __forceinline__ float settled(float x) {
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ f16x8 to_f16(const float* v) {
  f16x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (f16)v[e];
  return r;
}

// Four consecutive elements of a row, as many as there are.
template <typename T>
__device__ __forceinline__ f32x4 load_four(const T* from, int left, bool whole) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  f32x4 v{};
  if (whole && left >= 4) {
    const T4 x = *reinterpret_cast<const T4*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)x[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) v[e] = (float)from[e];
  }
  return v;
}

// Sums of squares in 64 bits: no overflow for any float32, whatever the scale.
template <typename T>
__global__ void __launch_bounds__(256) ortho_norm_kernel(Args s) {
  __shared__ double shared[4];
  int local;
  const int gi = find_group<false>(s, blockIdx.x, local);
  const Group& g = s.g[gi];
  const int matrix = local / g.parts, part = local % g.parts;
  const Tensor& t = find_tensor(s, gi, matrix);
  const int64_t size = (int64_t)g.m * g.n;
  const T* in = (const T*)t.in + (matrix - t.first) * size;
  const int64_t begin = (int64_t)part * kPart, end = begin + kPart < size ? begin + kPart : size;
  const bool whole = (uintptr_t)(in + begin) % (4 * sizeof(T)) == 0;
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = begin + 4 * threadIdx.x; i < end; i += 4 * 256) {
    const f32x4 v = load_four(in + i, end - i < 4 ? (int)(end - i) : 4, whole);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_fma((double)v[e], (double)v[e], sum);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) s.sums[g.sum0 + (int64_t)matrix * g.parts + part] = sum;
}

// X of a matrix, 64 x 64 of it a workgroup: normalised, turned where the matrix is
// tall, cut in two float16, with zeros up to the row length.
template <typename T>
__global__ void __launch_bounds__(256) ortho_load_kernel(Args s) {
  __shared__ double shared[4];
  __shared__ float turned[64][65];
  int local;
  const int gi = find_group<false>(s, blockIdx.x, local);
  const Group& g = s.g[gi];
  const int ld = g.ldx();
  const int across = (ld + 63) / 64, down = (g.m + 63) / 64;
  const int matrix = local / (across * down), at = local % (across * down);
  const int i0 = at / across * 64, j0 = at % across * 64;
  const Tensor& t = find_tensor(s, gi, matrix);
  const int64_t size = (int64_t)g.m * g.n;
  const T* in = (const T*)t.in + (matrix - t.first) * size;
  const int quad = 4 * (threadIdx.x & 15), line = threadIdx.x >> 4;  // of 64 elements, of 16 lines four times
  // Rows of four elements are aligned where the row length and the tensor are.
  const bool whole = (g.tall ? g.m : g.n) % 4 == 0 && (uintptr_t)in % (4 * sizeof(T)) == 0;
  f32x4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = 16 * k + line;
    const int row = (g.tall ? j0 : i0) + r, col = (g.tall ? i0 : j0) + quad;  // of the tensor
    const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n;
    v[k] = row < rows ? load_four(in + (int64_t)row * cols + col, cols - col, whole) : f32x4{};
  }
  double sum = 0.0;
  for (int i = threadIdx.x; i < g.parts; i += 256) sum += s.sums[g.sum0 + (int64_t)matrix * g.parts + i];
  sum = block_sum(sum, shared);
  // (In 64 bits: the norm of large float32, and the inverse of a small one, are none.)
  const double scale = 1.0 / (sqrt(sum) + (double)s.eps);
  if (g.tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) turned[16 * k + line][quad + e] = v[k][e];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = turned[quad + e][16 * k + line];
  }
  typedef f16 f16x4 __attribute__((ext_vector_type(4)));
  const int64_t x0 = g.x0 + (int64_t)matrix * g.m * ld;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = i0 + 16 * k + line, j = j0 + quad;
    if (i >= g.m || j >= ld) continue;
    f16x4 high, low;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = settled((float)((double)v[k][e] * scale));
      high[e] = (f16)x;
      low[e] = (f16)((x - (float)high[e]) * kLow);
    }
    *(f16x4*)(s.hi + x0 + blocked(g.m, i, j)) = high;
    *(f16x4*)(s.lo + x0 + blocked(g.m, i, j)) = low;
  }
}

// Tiles of a product: 64 MB features x 64 NB rows.
struct Wide {
  static constexpr int MB = 4, NB = 2, kSlabs = 1, kRing = 3;
};
struct Narrow {
  static constexpr int MB = 1, NB = 1, kSlabs = 2, kRing = 4;
};

// The tiles of a symmetric result with features at or before a row, `down` rows of
// tiles: a tile is 1 or 2 rows of tiles wide, row ti of them has ti / kWide + 1.
template <class Shape>
__host__ __device__ inline int triangle_tiles(int down) {
  constexpr int kWide = Shape::MB / Shape::NB;
  const int pairs = down / kWide;
  return kWide * pairs * (pairs + 1) / 2 + (down % kWide) * (pairs + 1);
}
template <class Shape>
__device__ __forceinline__ void triangle(int t, int& ti, int& tj) {
  constexpr int kWide = Shape::MB / Shape::NB;
  static_assert(kWide == 1 || kWide == 2, "see above");
  // p: the last number of whole (pairs of) rows with at most t tiles.
  int p = (int)((__builtin_sqrtf(1.0f + (8.0f / kWide) * t) - 1.0f) * 0.5f);
  while (kWide * p * (p + 1) / 2 > t) --p;
  while (kWide * (p + 1) * (p + 2) / 2 <= t) ++p;
  const int rest = t - kWide * p * (p + 1) / 2;
  ti = kWide * p + rest / (p + 1);
  tj = rest % (p + 1);
}

enum { kGram = 0, kSquare = 1, kUpdate = 2, kLast = 3 };

// One product of a step for every matrix.  The tile is computed as [feature][row]:
// the lane holds 16 consecutive features of a row of the result.
template <int kKind, class Shape>
__global__ void __launch_bounds__(256, 2) ortho_product_kernel(Args s) {
  constexpr bool kSymmetric = kKind == kGram || kKind == kSquare;
  constexpr int MB = Shape::MB, NB = Shape::NB;
  typedef tile::Product<f16, MB, NB, kSymmetric ? tile::kBlockedK : tile::kBlockedMN, tile::kBlockedK, true,
                        Shape::kSlabs, 1, Shape::kRing>
      P;
  int local;
  // Every other product walks the matrices backwards: it begins with those that the
  // one before ended with and that the caches still hold.
  const int gi = find_group<true>(s, kSymmetric ? blockIdx.x : gridDim.x - 1 - blockIdx.x, local);
  const Group& g = s.g[gi];
  const int m = g.m, lda = g.lda(), ldx = g.ldx();
  const int down = (m + P::TN - 1) / P::TN;
  int matrix, ti, tj;
  if (kSymmetric) {
    const int tiles = triangle_tiles<Shape>(down);
    matrix = local / tiles;
    triangle<Shape>(local % tiles, ti, tj);
  } else {
    const int tiles = down * ((ldx + P::TM - 1) / P::TM);
    matrix = local / tiles;
    const int at = local % tiles;
    ti = at % down;
    tj = at / down;
  }
  const f16* const hi = s.hi + g.x0 + (int64_t)matrix * m * ldx;
  f16* const A = s.A + g.a0 + (int64_t)matrix * m * lda;
  f16* const B = s.B + g.a0 + (int64_t)matrix * m * lda;
  const auto at = P::place();
  f32x16 acc[MB][NB];
  if constexpr (kKind == kGram)
    P::run(acc, {hi, m}, {hi, m}, m, m, ldx, tj * P::TM, ti * P::TN, at);
  else if constexpr (kKind == kSquare)
    P::run(acc, {A, m}, {A, m}, m, m, m, tj * P::TM, ti * P::TN, at);
  else
    P::run(acc, {hi, m}, {B, m}, ldx, m, m, tj * P::TM, ti * P::TN, at);
  // A symmetric result: where the wave's features lie against the tile's rows, in
  // rows of tiles.  What lies past them is another tile's mirror image.
  const int past = kSymmetric ? tj * (MB / NB) + at.wm * MB / (2 * NB) - ti : 0;
  if (kSymmetric && past > 0) return;
  const int lane = at.lane, ld = kSymmetric ? lda : ldx;
  const tile::Block block = P::block(at, 0), block_low = P::block(at, 1);
  f16* const lo = s.lo + (hi - s.hi);
  float* const diag_a = s.diag_a + g.d0 + (int64_t)matrix * lda;
  float* const diag_b = s.diag_b + g.d0 + (int64_t)matrix * lda;
  bf16* out = nullptr;
  if constexpr (kKind == kLast) {
    const Tensor& t = find_tensor(s, gi, matrix);
    out = t.out + (int64_t)(matrix - t.first) * m * g.n;
  }
  // A block's two lines of the lane, in 16 bits: `to` its place in a blocked matrix.
  auto store = [&](const tile::Block& b, f16* to, int rows) {
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const i16x8 v = b.get_line(it, lane);
      if (tile::Block::line_row(it, lane) < rows) *(i16x8*)(to + 512 * it + 8 * lane) = v;
    }
  };
  const int row_first = ti * P::TN + 32 * NB * at.wn, f_first = tj * P::TM + 32 * MB * at.wm;
  // What the blocks hold already, asked for some blocks ahead and so ahead of the
  // stores between: behind those, a block's loads would cost a trip to memory each.
  constexpr int kBlocks = MB * NB, kAhead = kBlocks < 4 ? kBlocks : 4;
  i16x8 old[kAhead][2], rest[kAhead][2];
  auto fetch = [&](int b) {
    const f16* const from = kSymmetric ? A : hi;
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      // (Of the last row and block again where there are none: results of those are not kept.)
      const int row = min(row_first + 32 * (b / MB) + tile::Block::line_row(it, lane), m - 1);
      const int64_t own = blocked(m, row, min(f_first + 32 * (b % MB), ld - 32) + tile::Block::line_feature(lane));
      old[b % kAhead][it] = *(const i16x8*)(from + own);
      if constexpr (!kSymmetric) rest[b % kAhead][it] = *(const i16x8*)(lo + own);
    }
  };
  if constexpr (kKind != kGram) {
#pragma unroll
    for (int b = 0; b < kAhead; ++b) fetch(b);
  }
  // The diagonals at the lane's rows, and (of A) at the wave's features: a feature a lane.
  float at_row[NB], at_feature[(MB + 1) / 2];
  if constexpr (kKind != kGram) {
    const float* const from = kKind == kSquare ? diag_a : diag_b;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) at_row[nb] = from[min(row_first + 32 * nb + (lane & 31), lda - 1)];
  }
  if constexpr (kKind == kSquare) {
#pragma unroll
    for (int k = 0; k < (MB + 1) / 2; ++k) at_feature[k] = diag_a[min(f_first + 64 * k + lane, lda - 1)];
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row0 = row_first + 32 * nb;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int b = nb * MB + mb, j0 = f_first + 32 * mb;
      const bool inside = row0 < m && j0 < ld;  // (uniform)
      const int64_t own = blocked(m, row0, j0);
      if constexpr (kKind != kGram) block.put_lines(lane, old[b % kAhead][0], old[b % kAhead][1]);
      if constexpr (!kSymmetric) block_low.put_lines(lane, rest[b % kAhead][0], rest[b % kAhead][1]);
      if constexpr (kKind != kGram)
        if (b + kAhead < kBlocks) fetch(b + kAhead);
      if (!inside) continue;
      float v[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f16x8 x{}, x_low{};
        if constexpr (kKind != kGram) x = __builtin_bit_cast(f16x8, block.get_run(lane, h));
        if constexpr (!kSymmetric) x_low = __builtin_bit_cast(f16x8, block_low.get_run(lane, h));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float& r = v[8 * h + e];
          r = acc[mb][nb][8 * h + e];
          if constexpr (kKind == kSquare) {
            // b A + c A A off the diagonal, A = D + O: (b + c (D_i + D_j)) O + c O O.
            const float other = __shfl(at_feature[mb / 2], 32 * (mb & 1) + 16 * (lane >> 5) + 8 * h + e);
            r = __builtin_fmaf(__builtin_fmaf(s.c, at_row[nb] + other, s.b), (float)x[e], s.c * r);
          }
          if constexpr (!kSymmetric)
            r = settled(__builtin_fmaf(at_row[nb], __builtin_fmaf((float)x_low[e], 1.0f / kLow, (float)x[e]), r));
        }
      }
      if (kSymmetric && row0 == j0) {
        // The diagonal leaves in float32: of A as it is, of B as b D + c (D D + O O) + a.
        // (Rows past the last are written too, zeros of A: what lies there is read.)
        float own_diag = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e == (lane & 31) - 16 * (lane >> 5)) {
            own_diag = v[e];
            v[e] = 0.f;
          }
        if (((lane & 31) >> 4) == (lane >> 5)) {
          if constexpr (kKind == kGram)
            diag_a[row0 + (lane & 31)] = own_diag;
          else
            diag_b[row0 + (lane & 31)] =
                __builtin_fmaf(at_row[nb], __builtin_fmaf(s.c, at_row[nb], s.b), own_diag) + s.a;
        }
      }
      const int rows = m - row0;
      if constexpr (kKind != kLast) {
        f16* const result = kKind == kGram ? A : kKind == kSquare ? B : s.hi_next + (hi - s.hi);
        const i16x8 low = __builtin_bit_cast(i16x8, to_f16(v)), high = __builtin_bit_cast(i16x8, to_f16(v + 8));
        block.put_run(lane, low, high);
        store(block, result + own, rows);
        if constexpr (kKind == kUpdate) {  // (the lines that this lane has read)
          const f16x8 l = __builtin_bit_cast(f16x8, low), u = __builtin_bit_cast(f16x8, high);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = (v[e] - (float)(e < 8 ? l[e & 7] : u[e & 7])) * kLow;
          block_low.put_run(lane, __builtin_bit_cast(i16x8, to_f16(v)), __builtin_bit_cast(i16x8, to_f16(v + 8)));
          store(block_low, lo + own, rows);
        }
        // The mirrored tile, in which rows past the last are the rows' ends: zeros.  (Those
        // lanes have v of operands that read zeros, but of another row's elements of A.)
        if (kSymmetric && past < 0) {
          const bool there = row0 + (lane & 31) < m;
          block.put_turned(lane, there ? low : i16x8{}, there ? high : i16x8{});
          store(block, result + blocked(m, j0, row0), m - j0);
        }
      } else {
        // Rows of the result, or of its transpose.
        const i16x8 low = __builtin_bit_cast(i16x8, pack8(v)), high = __builtin_bit_cast(i16x8, pack8(v + 8));
        if (g.tall)
          block.put_turned(lane, low, high);
        else
          block.put_run(lane, low, high);
        const int across = g.tall ? m : g.n, lines = g.tall ? g.n - j0 : rows;
        const int first = (g.tall ? row0 : j0) + tile::Block::line_feature(lane);
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const i16x8 x = block.get_line(it, lane);
          const int line = tile::Block::line_row(it, lane);
          if (line >= lines) continue;
          short* const to = (short*)out + (int64_t)((g.tall ? j0 : row0) + line) * across + first;
          if (across % 8 == 0 && first < across) {
            *(i16x8*)to = x;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (first + e < across) to[e] = x[e];
          }
        }
      }
    }
  }
}

// ---- host side ----

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

struct Sizes {
  int64_t x = 0, a = 0, d = 0, sums = 0;  // elements of hi (and lo, hi_next), of A (and B), a diagonal, of the sums
  size_t bytes() const {
    return 3 * round_up((size_t)x * 2) + 2 * round_up((size_t)a * 2) + 2 * round_up((size_t)d * 4) +
           round_up((size_t)sums * 8);
  }
};

Group group_of(const gptrig_matrices& t) {
  Group g{};
  g.tall = t.rows > t.cols;
  g.m = g.tall ? t.cols : t.rows;
  g.n = g.tall ? t.rows : t.cols;
  g.parts = ceil_div((int64_t)g.m * g.n, kPart);
  return g;
}

Sizes size_of(const Group& g, int64_t count) {
  Sizes s;
  s.x = count * g.m * g.ldx();
  s.a = count * g.m * g.lda();
  s.d = count * g.lda();
  s.sums = count * g.parts;
  return s;
}

// Walks a list in launches' worth: at most kMostTensors tensors of kMostGroups shapes
// and kMostBytes of workspace each; a tensor's matrices may be spread over several.
struct Walk {
  const gptrig_matrices* list;
  int count;
  int at = 0;          // the tensor that is next
  int64_t inside = 0;  // and its matrices that are done

  // The next launch's table and sizes; false at the end.
  bool next(Args& s, Sizes& total, size_t item) {
    s.groups = s.tensors = 0;
    total = Sizes{};
    while (at < count && s.tensors < kMostTensors) {
      const gptrig_matrices& t = list[at];
      const Group shape = group_of(t);
      if (t.count == 0 || shape.m == 0) {
        ++at;
        continue;
      }
      int gi = 0;
      while (gi < s.groups && (s.g[gi].m != shape.m || s.g[gi].n != shape.n || s.g[gi].tall != shape.tall)) ++gi;
      if (gi == kMostGroups) break;
      const Sizes one = size_of(shape, 1);
      const int64_t left = kMostBytes - (int64_t)total.bytes();
      int64_t take = left / (6 * one.x + 4 * one.a + 8 * one.d + 8 * one.sums);
      if (take <= 0) {
        if (s.tensors) break;
        take = 1;
      }
      if (take > t.count - inside) take = t.count - inside;
      if (take > 65536) take = 65536;
      if (gi == s.groups) {
        // Longest rows first: their workgroups take longest in the gram products.
        for (gi = s.groups++; gi > 0 && s.g[gi - 1].n < shape.n; --gi) s.g[gi] = s.g[gi - 1];
        s.g[gi] = shape;
        for (int i = 0; i < s.tensors; ++i) s.t[i].group += s.t[i].group >= gi;
      }
      Group& g = s.g[gi];
      const int64_t size = (int64_t)t.rows * t.cols;
      s.t[s.tensors++] =
          Tensor{(const char*)t.in + inside * size * item, (bf16*)t.out + inside * size, gi, g.count};
      g.count += (int)take;
      const Sizes more = size_of(shape, take);
      total.x += more.x;
      total.a += more.a;
      total.d += more.d;
      total.sums += more.sums;
      inside += take;
      if (inside < t.count) break;
      inside = 0;
      ++at;
    }
    Sizes from;
    for (int i = 0; i < s.groups; ++i) {
      Group& g = s.g[i];
      g.x0 = from.x;
      g.a0 = from.a;
      g.d0 = from.d;
      g.sum0 = (int)from.sums;
      const Sizes more = size_of(g, g.count);
      from.x += more.x;
      from.a += more.a;
      from.d += more.d;
      from.sums += more.sums;
    }
    return s.groups > 0;
  }
};

int check_list(const gptrig_matrices* list, int count) {
  if (count < 0) return GPTRIG_E_SHAPE;
  if (count && !list) return GPTRIG_E_NULL;
  for (int i = 0; i < count; ++i) {
    const gptrig_matrices& t = list[i];
    if (t.count < 0 || t.rows < 0 || t.cols < 0 || t.rows > 65536 || t.cols > 65536) return GPTRIG_E_SHAPE;
  }
  return GPTRIG_OK;
}

// Workgroups of a launch, `each` a matrix of a group; fills s.first.  (At most some
// millions: kMostTensors of 65536 matrices, or what kMostBytes or one matrix hold.)
template <class F>
int64_t count_groups(Args& s, F each) {
  int64_t total = 0;
  for (int i = 0; i < s.groups; ++i) {
    s.first[i] = (int)total;
    total += each(s.g[i]) * s.g[i].count;
  }
  for (int i = s.groups; i <= kMostGroups; ++i) s.first[i] = (int)total;
  return total;
}

template <int kKind, class Shape>
int64_t count_tiles(Args& s) {
  return count_groups(s, [](const Group& g) -> int64_t {
    const int64_t down = ceil_div(g.m, 64 * Shape::NB);
    return kKind == kGram || kKind == kSquare ? triangle_tiles<Shape>(down)
                                              : down * ceil_div(g.ldx(), 64 * Shape::MB);
  });
}

template <int kKind>
int product(Args& s, hipStream_t stream) {
  // The wide tile needs fewer reads an operation; the narrow one fills the chip with fewer matrices.
  const int64_t wide = count_tiles<kKind, Wide>(s);
  if (wide >= gemm::device_cus()) {
    ortho_product_kernel<kKind, Wide><<<(unsigned)wide, 256, 0, stream>>>(s);
  } else {
    const int64_t narrow = count_tiles<kKind, Narrow>(s);
    ortho_product_kernel<kKind, Narrow><<<(unsigned)narrow, 256, 0, stream>>>(s);
  }
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

}  // namespace

extern "C" {

size_t gptrig_orthogonalize_workspace_bytes(const gptrig_matrices* list, int count) {
  if (check_list(list, count) != GPTRIG_OK) return 0;
  Walk walk{list, count};
  Args s;
  Sizes total;
  size_t most = 0;
  while (walk.next(s, total, 2)) most = total.bytes() > most ? total.bytes() : most;
  return most;
}

int gptrig_orthogonalize(const gptrig_matrices* list, int count, int type, int steps, float a, float b, float c,
                         float eps, void* workspace, size_t workspace_bytes, void* stream) {
  const int checked = check_list(list, count);
  if (checked != GPTRIG_OK) return checked;
  if (type != GPTRIG_TYPE_BF16 && type != GPTRIG_TYPE_F32) return GPTRIG_E_DTYPE;
  if (steps < 1 || !(eps >= 0.f)) return GPTRIG_E_SHAPE;
  const size_t item = type == GPTRIG_TYPE_F32 ? 4 : 2;
  for (int i = 0; i < count; ++i) {
    if (list[i].count == 0 || list[i].rows == 0 || list[i].cols == 0) continue;
    if (!list[i].in || !list[i].out) return GPTRIG_E_NULL;
    if ((uintptr_t)list[i].in % item || (uintptr_t)list[i].out % 16) return GPTRIG_E_SHAPE;
  }
  const size_t need = gptrig_orthogonalize_workspace_bytes(list, count);
  if (need && !workspace) return GPTRIG_E_NULL;
  if ((uintptr_t)workspace % 16) return GPTRIG_E_SHAPE;
  if (workspace_bytes < need) return GPTRIG_E_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  Walk walk{list, count};
  Args s;
  s.a = a;
  s.b = b;
  s.c = c;
  s.eps = eps;
  Sizes total;
  while (walk.next(s, total, item)) {
    const size_t x = round_up((size_t)total.x * 2), sq = round_up((size_t)total.a * 2);
    char* at = (char*)workspace;
    s.hi = (f16*)at;
    s.hi_next = (f16*)(at + x);
    s.lo = (f16*)(at + 2 * x);
    s.A = (f16*)(at + 3 * x);
    s.B = (f16*)(at + 3 * x + sq);
    const size_t diag = round_up((size_t)total.d * 4);
    s.diag_a = (float*)(at + 3 * x + 2 * sq);
    s.diag_b = (float*)(at + 3 * x + 2 * sq + diag);
    s.sums = (double*)(at + 3 * x + 2 * sq + 2 * diag);
    int64_t grid = count_groups(s, [](const Group& g) -> int64_t { return g.parts; });
    if (type == GPTRIG_TYPE_F32)
      ortho_norm_kernel<float><<<(unsigned)grid, 256, 0, st>>>(s);
    else
      ortho_norm_kernel<bf16><<<(unsigned)grid, 256, 0, st>>>(s);
    GPTRIG_CHECK_LAUNCH();
    grid = count_groups(s, [](const Group& g) -> int64_t {
      return (int64_t)ceil_div(g.ldx(), 64) * ceil_div(g.m, 64);
    });
    if (type == GPTRIG_TYPE_F32)
      ortho_load_kernel<float><<<(unsigned)grid, 256, 0, st>>>(s);
    else
      ortho_load_kernel<bf16><<<(unsigned)grid, 256, 0, st>>>(s);
    GPTRIG_CHECK_LAUNCH();
    for (int step = 0; step < steps; ++step) {
      int status = product<kGram>(s, st);
      if (status == GPTRIG_OK) status = product<kSquare>(s, st);
      if (status == GPTRIG_OK) status = step + 1 < steps ? product<kUpdate>(s, st) : product<kLast>(s, st);
      if (status != GPTRIG_OK) return status;
      f16* const last = s.hi;
      s.hi = s.hi_next;
      s.hi_next = last;
    }
  }
  return GPTRIG_OK;
}

}  // extern "C"
