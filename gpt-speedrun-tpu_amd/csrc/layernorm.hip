// Layer normalisation over the last dimension, forward and backward:
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
//   y  = h scale + bias
//   g  = dy scale;  dx = r (g - mean(g) - h mean(g h))
//   dscale = sum over rows of dy h;  dbias = sum over rows of dy
// Everything between the loads and the stores is float32 (the mean first, then
// the squares of the differences from it), so each output is rounded once, to
// its own type.  Rows of any width, row stride and alignment: a row is read in
// 16-byte pieces wherever it starts (the loads need no alignment here), its last
// few values one by one.
#include "common.h"

#include <algorithm>

namespace {

enum { kBf16 = GPTRIG_TYPE_BF16, kF32 = GPTRIG_TYPE_F32 };

// N values of type T from a place of any alignment.
template <typename T, int N>
struct __attribute__((packed)) Piece {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_piece(float (&out)[N], const T* __restrict__ row, int at, int d) {
  if (at + N <= d) {
    const Piece<T, N> p = *reinterpret_cast<const Piece<T, N>*>(row + at);
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = (float)p.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = at + j < d ? (float)row[at + j] : 0.f;
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_piece(T* __restrict__ row, const float (&v)[N], int at, int d) {
  if (at + N <= d) {
    Piece<T, N> p;
#pragma unroll
    for (int j = 0; j < N; ++j) p.v[j] = (T)v[j];
    *reinterpret_cast<Piece<T, N>*>(row + at) = p;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j < d) row[at + j] = (T)v[j];
  }
}

// Sum over the L lanes that share a row; every one of them gets it.  L = 256 (a
// whole workgroup) goes through red[4], which the caller keeps apart from the
// previous sum's.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0] + red[1] + red[2] + red[3];
  }
  return v;
}

// A lane's C pieces of a row held by L lanes, without a branch: the row's last
// piece ends with the row, so where the width is no multiple of V it repeats some
// columns of the piece before (skip of them; V for a lane past the row's end).
// Sums leave those out; stores write the same values to them twice.
template <typename T, int V, int L, int C, bool kEven>
struct Row {
  int at[C], skip[C];
  __device__ __forceinline__ void init(int lane, int d) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int first = V * (lane + L * c);
      at[c] = min(first, d - V);
      skip[c] = min(first - at[c], V);
    }
  }
  // 1 for a column that piece c owns, else 0.
  __device__ __forceinline__ bool owns(int c, int j) const { return kEven ? skip[c] == 0 : j >= skip[c]; }
  __device__ __forceinline__ bool some(int c) const { return skip[c] < V; }
};
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> piece(const T* row, int at) {
  return *reinterpret_cast<const Piece<T, V>*>(row + at);
}

// ---------------------------------------------------------------------------
// Forward: L lanes hold a row, C pieces of V = 16 bytes each, so x is read once.
// Bound by HBM: 65536 x 768 bf16 (201 MB in and out) on inputs that change between
// launches 38 us, 5.3 TB/s, the rate of a large copy.
// ---------------------------------------------------------------------------
template <typename T, typename P, int L, int C, bool kEven>
__global__ void __launch_bounds__(256) layernorm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                            const P* __restrict__ scale, const P* __restrict__ bias,
                                                            T* __restrict__ y, float* __restrict__ mean,
                                                            float* __restrict__ rstd, int64_t rows, int d, float eps) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][4];
  const int lane = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= rows) return;  // (with L = 256 the whole workgroup)
  const T* xr = x + row * ldx;
  Row<T, V, L, C, kEven> my;
  my.init(lane, d);
  Piece<T, V> raw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) raw[c] = piece<T, V>(xr, my.at[c]);
  float v[C][V];
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[c][j] = (float)raw[c].v[j];
      sum += my.owns(c, j) ? v[c][j] : 0.f;
    }
  const float mu = row_sum<L>(sum, red[0]) / (float)d;
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[c][j] -= mu;
      sq += my.owns(c, j) ? v[c][j] * v[c][j] : 0.f;
    }
  const float r = rsqrtf(row_sum<L>(sq, red[1]) / (float)d + eps);
  if (lane == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!my.some(c)) continue;
    const Piece<P, V> s = piece<P, V>(scale, my.at[c]);
    Piece<P, V> b;
    if (bias) b = piece<P, V>(bias, my.at[c]);
    Piece<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = (T)fmaf(v[c][j] * r, (float)s.v[j], bias ? (float)b.v[j] : 0.f);
    *reinterpret_cast<Piece<T, V>*>(y + row * d + my.at[c]) = o;
  }
}

// Rows of more than 1024 pieces (bf16 from 8193 columns on, float32 from 4097: a
// workgroup of 4 pieces a lane, though 8 of float32 would be no more values than 4 of
// bf16): three passes over the row, the later two from the caches.
template <typename T, typename P>
__global__ void __launch_bounds__(256) layernorm_fwd_wide_kernel(const T* __restrict__ x, int64_t ldx,
                                                                 const P* __restrict__ scale,
                                                                 const P* __restrict__ bias, T* __restrict__ y,
                                                                 float* __restrict__ mean, float* __restrict__ rstd,
                                                                 int d, float eps) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][4];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  float v[V];
  float sum = 0.f;
  for (int64_t at = V * threadIdx.x; at < d; at += V * 256) {
    load_piece<T, V>(v, xr, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j) sum += v[j];
  }
  const float mu = row_sum<256>(sum, red[0]) / (float)d;
  float sq = 0.f;
  for (int64_t at = V * threadIdx.x; at < d; at += V * 256) {
    load_piece<T, V>(v, xr, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (at + j < d) sq += (v[j] - mu) * (v[j] - mu);
  }
  const float r = rsqrtf(row_sum<256>(sq, red[1]) / (float)d + eps);
  if (threadIdx.x == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
  for (int64_t at = V * threadIdx.x; at < d; at += V * 256) {
    float s[V], b[V];
    load_piece<T, V>(v, xr, (int)at, d);
    load_piece<P, V>(s, scale, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = 0.f;
    if (bias) load_piece<P, V>(b, bias, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = fmaf((v[j] - mu) * r, s[j], b[j]);
    store_piece<T, V>(y + row * d, s, (int)at, d);
  }
}

// ---------------------------------------------------------------------------
// Backward.  A workgroup walks rows with the same columns in the same lanes, so
// the column sums of dy h and dy stay in registers; they are joined over the
// workgroup in LDS at the end and leave as one partial row, and
// layernorm_columns_kernel adds the partial rows in a fixed order (no atomics:
// the gradients are the same on every run).
// ---------------------------------------------------------------------------
// The next row's pieces are on their way while this row is summed.  Bound by HBM:
// 65536 x 768 bf16 (302 MB), as above, 54 us, 5.6 TB/s (without the row ahead 88 us);
// the columns kernel 4 us.
template <typename T, typename P, int L, int C, bool kEven>
__global__ void __launch_bounds__(256)
    layernorm_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                         const P* __restrict__ scale, const float* __restrict__ mean, const float* __restrict__ rstd,
                         T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int d) {
  constexpr int V = 16 / sizeof(T), G = 256 / L;  // G rows at a time
  __shared__ float red[2][2][4];
  __shared__ float join[G > 1 ? G : 1][G > 1 ? L * V : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  Row<T, V, L, C, kEven> my;
  my.init(lane, d);
  float ds[C][V], db[C][V], s[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Piece<P, V> p = piece<P, V>(scale, my.at[c]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[c][j] = (float)p.v[j];
      ds[c][j] = db[c][j] = 0.f;
    }
  }
  const float inv_d = 1.f / (float)d;
  const int64_t step = (int64_t)gridDim.x * G;
  Piece<T, V> gp[C], xp[C];
  float mu = 0.f, r = 0.f;
  auto load = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      gp[c] = piece<T, V>(dy + row * lddy, my.at[c]);
      xp[c] = piece<T, V>(x + row * ldx, my.at[c]);
    }
    mu = mean[row];
    r = rstd[row];
  };
  int turn = 0;
  int64_t row = (int64_t)blockIdx.x * G + group;
  if (row < rows) load(row);
  for (; row < rows; row += step, turn ^= 1) {
    float g[C][V], h[C][V];
    float a = 0.f, b = 0.f;
    const float my_r = r;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[c][j] = ((float)xp[c].v[j] - mu) * r;
        const float u = (float)gp[c].v[j], own = my.owns(c, j) ? u : 0.f;
        db[c][j] += own;
        ds[c][j] = fmaf(own, h[c][j], ds[c][j]);
        g[c][j] = u * s[c][j];
        a = fmaf(own, s[c][j], a);
        b = fmaf(my.owns(c, j) ? g[c][j] : 0.f, h[c][j], b);
      }
    load(row + step < rows ? row + step : row);
    if (dx) {
      a = row_sum<L>(a, red[turn][0]) * inv_d;
      b = row_sum<L>(b, red[turn][1]) * inv_d;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (!my.some(c)) continue;
        Piece<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = (T)(my_r * (g[c][j] - a - h[c][j] * b));
        *reinterpret_cast<Piece<T, V>*>(dx + row * d + my.at[c]) = o;
      }
    }
  }
  if (!partial) return;
  float* const out = partial + (size_t)blockIdx.x * 2 * d;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if constexpr (G > 1) {
        // (By the columns that a piece owns: those it repeats are the piece's before.)
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) join[group][V * lane + j] = which ? db[c][j] : ds[c][j];
        __syncthreads();
        for (int i = threadIdx.x; i < L * V; i += 256) {
          float t = 0.f;
#pragma unroll
          for (int k = 0; k < G; ++k) t += join[k][i];
          const int first = V * (i / V + L * c), at = min(first, d - V), col = at + i % V;
          if (col >= first) out[(size_t)which * d + col] = t;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (my.owns(c, j)) out[(size_t)which * d + my.at[c] + j] = which ? db[c][j] : ds[c][j];
      }
    }
}

// Wide rows: dx with two passes over each row ...
template <typename T, typename P>
__global__ void __launch_bounds__(256)
    layernorm_bwd_wide_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                              const P* __restrict__ scale, const float* __restrict__ mean,
                              const float* __restrict__ rstd, T* __restrict__ dx, int d) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][4];
  const int64_t row = blockIdx.x;
  const T* gr = dy + row * lddy;
  const T* xr = x + row * ldx;
  const float mu = mean[row], r = rstd[row];
  float g[V], h[V], s[V];
  float a = 0.f, b = 0.f;
  for (int64_t at = V * threadIdx.x; at < d; at += V * 256) {
    load_piece<T, V>(g, gr, (int)at, d);
    load_piece<T, V>(h, xr, (int)at, d);
    load_piece<P, V>(s, scale, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float t = g[j] * s[j];
      a += t;
      b = fmaf(t, (h[j] - mu) * r, b);
    }
  }
  a = row_sum<256>(a, red[0]) / (float)d;
  b = row_sum<256>(b, red[1]) / (float)d;
  for (int64_t at = V * threadIdx.x; at < d; at += V * 256) {
    load_piece<T, V>(g, gr, (int)at, d);
    load_piece<T, V>(h, xr, (int)at, d);
    load_piece<P, V>(s, scale, (int)at, d);
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = r * (g[j] * s[j] - a - (h[j] - mu) * r * b);
    store_piece<T, V>(dx + row * d, g, (int)at, d);
  }
}

// ... and the column sums over blocks of rows: blockIdx.x the columns (V a
// thread), blockIdx.y the block of rows.
template <typename T>
__global__ void __launch_bounds__(256)
    layernorm_bwd_wide_columns_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                      float* __restrict__ partial, int64_t rows, int d) {
  constexpr int V = 16 / sizeof(T);
  const int64_t at = (int64_t)V * (blockIdx.x * 256 + threadIdx.x);
  if (at >= d) return;
  float ds[V], db[V], g[V], h[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ds[j] = db[j] = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    load_piece<T, V>(g, dy + row * lddy, (int)at, d);
    load_piece<T, V>(h, x + row * ldx, (int)at, d);
    const float mu = mean[row], r = rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ds[j] = fmaf(g[j], (h[j] - mu) * r, ds[j]);
      db[j] += g[j];
    }
  }
  float* const out = partial + (size_t)blockIdx.y * 2 * d;
  store_piece<float, V>(out, ds, (int)at, d);
  store_piece<float, V>(out + d, db, (int)at, d);
}

// dscale and dbias from the partial rows: 16 columns of one of the two by 16
// slices of the partial rows per workgroup.
template <typename P>
__global__ void __launch_bounds__(256) layernorm_columns_kernel(const float* __restrict__ partial, int parts, int d,
                                                                P* __restrict__ dscale, P* __restrict__ dbias) {
  __shared__ float red[16][17];
  P* const out = blockIdx.y ? dbias : dscale;
  if (!out) return;
  const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + lane;
  float s = 0.f;
  if (col < d) {
    const float* p = partial + (size_t)blockIdx.y * d + col;
#pragma unroll 8
    for (int i = slice; i < parts; i += 16) s += p[(size_t)i * 2 * d];
  }
  red[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && col < d) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][lane];
    out[col] = (P)s;
  }
}

// Lanes a row and pieces a lane for pieces of V values: 32 lanes of up to 4
// pieces, then 64, then a workgroup of up to 4; {0, 0} for wider rows, and for rows
// of less than a piece.  (Width 768 bf16, forward: 3 pieces of 32 lanes 38 us, 2 of
// 64, a quarter of which are idle, 43; the backward 54 with either.)
// Never fewer than 32 lanes, so most of them idle on rows of a few pieces.  TB/s of
// forward / backward at 2^25 values in a loop on the same inputs (part of them in the
// last cache): bf16 16 columns 0.6 / 0.5, 64 2.3 / 2.0, 128 3.9 / 3.6, 256 to 2048 5.6 to
// 6.1 / 4.6 to 5.6, 4096 5.5 / 4.7, 8192 5.2 / 3.6, wider (bytes that the backward's
// second reading adds not counted) 3.5 / 2.1; float32 64 3.4 / 3.4, 256 to 4096 5.2 to 5.9
// / 4.6 to 5.2, 8192 3.6 / 2.6.
struct Shape {
  int lanes, pieces;
};
Shape row_shape(int d, int v) {
  const int pieces = ceil_div(d, v);
  if (d < v) return {0, 0};
  if (pieces <= 128) return {32, ceil_div(pieces, 32)};
  if (pieces <= 256) return {64, ceil_div(pieces, 64)};
  if (pieces <= 1024) return {256, ceil_div(pieces, 256)};
  return {0, 0};
}

// Partial rows at most: two workgroups a CU.  Backward and columns of 65536 x 768 with
// 256 / 512 / 1024: 59 / 58 / 65 us (other counts were timed at this width only).
constexpr int kParts = 512;

int parts_of(int64_t rows, int d, int v) {
  const Shape s = row_shape(d, v);
  const int64_t groups = s.lanes ? (rows + 256 / s.lanes - 1) / (256 / s.lanes) : rows;
  return (int)(groups < 1 ? 1 : groups < kParts ? groups : kParts);
}

#define LN_SHAPES(CALL)                                                                             \
  switch (sh.lanes * 8 + sh.pieces) {                                                               \
    case 32 * 8 + 1: CALL(32, 1); break;                                                            \
    case 32 * 8 + 2: CALL(32, 2); break;                                                            \
    case 32 * 8 + 3: CALL(32, 3); break;                                                            \
    case 32 * 8 + 4: CALL(32, 4); break;                                                            \
    case 64 * 8 + 3: CALL(64, 3); break;                                                            \
    case 64 * 8 + 4: CALL(64, 4); break;                                                            \
    case 256 * 8 + 2: CALL(256, 2); break;                                                          \
    case 256 * 8 + 3: CALL(256, 3); break;                                                          \
    case 256 * 8 + 4: CALL(256, 4); break;                                                          \
  }

// Workgroups of a launch at most (it has fewer than 2^32 threads a dimension).
constexpr int64_t kGrid = 1 << 22;

template <typename T, typename P>
void launch_fwd(const void* x, int64_t ldx, const void* scale, const void* bias, void* y, float* mean, float* rstd,
                int64_t rows, int d, float eps, hipStream_t st) {
  const Shape sh = row_shape(d, 16 / sizeof(T));
  const int64_t most = kGrid * (sh.lanes ? 256 / sh.lanes : 1);
  if (rows > most) {
    launch_fwd<T, P>(x, ldx, scale, bias, y, mean, rstd, most, d, eps, st);
    launch_fwd<T, P>((const T*)x + most * ldx, ldx, scale, bias, (T*)y + most * d, mean ? mean + most : nullptr,
                     rstd ? rstd + most : nullptr, rows - most, d, eps, st);
    return;
  }
  if (!sh.lanes) {
    layernorm_fwd_wide_kernel<T, P><<<(unsigned)rows, 256, 0, st>>>((const T*)x, ldx, (const P*)scale, (const P*)bias,
                                                                    (T*)y, mean, rstd, d, eps);
    return;
  }
  const unsigned grid = (unsigned)((rows + 256 / sh.lanes - 1) / (256 / sh.lanes));
  const bool even = d % (16 / sizeof(T)) == 0;
#define LN_FWD_(L, C, EVEN)                                                                                       \
  layernorm_fwd_kernel<T, P, L, C, EVEN><<<grid, 256, 0, st>>>((const T*)x, ldx, (const P*)scale, (const P*)bias,  \
                                                               (T*)y, mean, rstd, rows, d, eps)
#define LN_FWD(L, C) if (even) LN_FWD_(L, C, true); else LN_FWD_(L, C, false)
  LN_SHAPES(LN_FWD)
#undef LN_FWD
#undef LN_FWD_
}

template <typename T, typename P>
void launch_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* scale, const float* mean,
                const float* rstd, void* dx, void* dscale, void* dbias, float* partial, int64_t rows, int d,
                hipStream_t st) {
  const Shape sh = row_shape(d, 16 / sizeof(T));
  const int parts = parts_of(rows, d, 16 / sizeof(T));
  const bool even = d % (16 / sizeof(T)) == 0;
  if (!dscale && !dbias) partial = nullptr;
  if (rows > 0) {
    if (sh.lanes) {
#define LN_BWD_(L, C, EVEN)                                                                                           \
  layernorm_bwd_kernel<T, P, L, C, EVEN>                                                                              \
      <<<partial ? (unsigned)parts : (unsigned)std::min((rows + 256 / L - 1) / (256 / L), kGrid), 256, 0, st>>>(      \
          (const T*)dy, lddy, (const T*)x, ldx, (const P*)scale, mean, rstd, (T*)dx, partial, rows, d)
#define LN_BWD(L, C) if (even) LN_BWD_(L, C, true); else LN_BWD_(L, C, false)
      LN_SHAPES(LN_BWD)
#undef LN_BWD
#undef LN_BWD_
    } else {
      for (int64_t at = 0; dx && at < rows; at += kGrid)
        layernorm_bwd_wide_kernel<T, P><<<(unsigned)std::min(rows - at, kGrid), 256, 0, st>>>(
            (const T*)dy + at * lddy, lddy, (const T*)x + at * ldx, ldx, (const P*)scale, mean + at, rstd + at,
            (T*)dx + at * d, d);
      if (partial)
        layernorm_bwd_wide_columns_kernel<T>
            <<<dim3(ceil_div(d, 256 * (16 / sizeof(T))), parts), 256, 0, st>>>((const T*)dy, lddy, (const T*)x, ldx, mean,
                                                                              rstd, partial, rows, d);
    }
  }
  if (partial)
    layernorm_columns_kernel<P><<<dim3(ceil_div(d, 16), 2), 256, 0, st>>>(partial, rows > 0 ? parts : 0, d, (P*)dscale,
                                                                          (P*)dbias);
}

bool type_ok(int t) { return t == kBf16 || t == kF32; }
bool aligned(const void* p, int type) { return ((uintptr_t)p & (type == kBf16 ? 1 : 3)) == 0; }

}  // namespace

extern "C" {

int gptrig_layernorm_fwd(const void* x, int64_t ldx, int x_type, const void* scale, const void* bias, int param_type,
                         void* y, float* mean, float* rstd, int64_t rows, int d, float eps, void* stream) {
  if (!x || !scale || !y || (mean == nullptr) != (rstd == nullptr)) return GPTRIG_E_NULL;
  if (!type_ok(x_type) || !type_ok(param_type)) return GPTRIG_E_DTYPE;
  if (rows < 0 || rows > INT32_MAX || d <= 0 || d > (1 << 30) || ldx < 0 || !(eps >= 0.f)) return GPTRIG_E_SHAPE;
  if (!aligned(x, x_type) || !aligned(y, x_type) || !aligned(scale, param_type) || !aligned(bias, param_type))
    return GPTRIG_E_SHAPE;
  if (rows == 0) return GPTRIG_OK;
  hipStream_t s = (hipStream_t)stream;
  if (x_type == kBf16 && param_type == kBf16)
    launch_fwd<bf16, bf16>(x, ldx, scale, bias, y, mean, rstd, rows, d, eps, s);
  else if (x_type == kBf16)
    launch_fwd<bf16, float>(x, ldx, scale, bias, y, mean, rstd, rows, d, eps, s);
  else if (param_type == kBf16)
    launch_fwd<float, bf16>(x, ldx, scale, bias, y, mean, rstd, rows, d, eps, s);
  else
    launch_fwd<float, float>(x, ldx, scale, bias, y, mean, rstd, rows, d, eps, s);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

size_t gptrig_layernorm_bwd_workspace_bytes(int64_t rows, int d, int x_type) {
  if (rows < 0 || d <= 0 || !type_ok(x_type)) return 0;
  return (size_t)parts_of(rows, d, x_type == kBf16 ? 8 : 4) * 2 * d * sizeof(float);
}

int gptrig_layernorm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int x_type, const void* scale,
                         int param_type, const float* mean, const float* rstd, void* dx, void* dscale, void* dbias,
                         void* workspace, size_t workspace_bytes, int64_t rows, int d, void* stream) {
  if (!dy || !x || !scale || !mean || !rstd) return GPTRIG_E_NULL;
  if (!type_ok(x_type) || !type_ok(param_type)) return GPTRIG_E_DTYPE;
  if (rows < 0 || rows > INT32_MAX || d <= 0 || d > (1 << 30) || ldx < 0 || lddy < 0) return GPTRIG_E_SHAPE;
  if (!aligned(dy, x_type) || !aligned(x, x_type) || !aligned(dx, x_type) || !aligned(scale, param_type) ||
      !aligned(dscale, param_type) || !aligned(dbias, param_type) || ((uintptr_t)workspace & 15))
    return GPTRIG_E_SHAPE;
  if (dscale || dbias) {
    if (!workspace) return GPTRIG_E_NULL;
    if (workspace_bytes < gptrig_layernorm_bwd_workspace_bytes(rows, d, x_type)) return GPTRIG_E_WORKSPACE;
  } else if (!dx || rows == 0) {
    return GPTRIG_OK;
  }
  hipStream_t s = (hipStream_t)stream;
  float* const ws = (float*)workspace;
  if (x_type == kBf16 && param_type == kBf16)
    launch_bwd<bf16, bf16>(dy, lddy, x, ldx, scale, mean, rstd, dx, dscale, dbias, ws, rows, d, s);
  else if (x_type == kBf16)
    launch_bwd<bf16, float>(dy, lddy, x, ldx, scale, mean, rstd, dx, dscale, dbias, ws, rows, d, s);
  else if (param_type == kBf16)
    launch_bwd<float, bf16>(dy, lddy, x, ldx, scale, mean, rstd, dx, dscale, dbias, ws, rows, d, s);
  else
    launch_bwd<float, float>(dy, lddy, x, ldx, scale, mean, rstd, dx, dscale, dbias, ws, rows, d, s);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

}  // extern "C"
