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
//     token and writes h, and for the backward g and u, straight from its
//     accumulators;
//   - the product dy V^T reads g and u in its epilogue and writes dg and du.
// Roundings to bfloat16: h, dg and du, which the next product takes in that type,
// and g and u where the backward is to find them (h itself comes from the
// unrounded ones).  Everything else is float32.
//
// The weight gradients cut the tokens into slices where the tiles alone do not
// fill the chip; each slice writes its float32 sums to the workspace and a small
// pass adds them in order, so the result does not depend on timing.
#include "gemm_core.h"

namespace {

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

struct UpArgs {
  bf16* gate_up;  // [n][2f], NULL: not kept
  bf16* h;        // [n][f]
  int n, k, f, group;
};

// The lane's 16 consecutive features of a token, 8 at a time.
__device__ __forceinline__ void store_run(bf16* dst, const float (&v)[16], int left) {
  if (left > 0) *reinterpret_cast<bf16x8*>(dst) = pack8(v);
  if (left > 8) *reinterpret_cast<bf16x8*>(dst + 8) = pack8(v + 8);
}

template <int kAct, bool kKeep>
__global__ void __launch_bounds__(gemm::THREADS) gated_up_kernel(Operand W, Operand X, UpArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hl = lane >> 5, l32 = lane & 31, wm = wave & 1, wn = wave >> 1;
  const int ntiles = ((2 * a.f + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  auto coords = [&](int t, int& tm, int& tn) { gemm::tile_coords(t, 2 * a.f, a.n, tm, tn, a.group); };
  auto pre = [](int, int) {};
  auto epi = [&](f32x16(&acc)[4][2], int tm, int tn) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int token = tn * BN + 64 * wn + 32 * nb + l32;
      if (token >= a.n) continue;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int feature = tm * (BM / 2) + 64 * wm + 32 * p + 16 * hl;
        const int left = a.f - feature;  // a multiple of 8
        float g[16], u[16], h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          g[i] = acc[2 * p][nb][i];
          u[i] = acc[2 * p + 1][nb][i];
          h[i] = act_f<kAct>(g[i]) * u[i];
        }
        store_run(a.h + (int64_t)token * a.f + feature, h, left);
        if constexpr (kKeep) {
          bf16* const row = a.gate_up + (int64_t)token * 2 * a.f + feature;
          store_run(row, g, left);
          store_run(row + a.f, u, left);
        }
      }
    }
  };
  gemm::persistent<false, true, true, true>(W, X, 2 * a.f, a.n, a.k, ntiles, coords, pre, epi);
}

struct DownBwdArgs {
  const bf16* gate_up;  // [n][2f]
  bf16* d_gate_up;      // [n][2f]
  int n, k, f, group;
};

template <int kAct>
__global__ void __launch_bounds__(gemm::THREADS) gated_down_bwd_kernel(Operand V, Operand DY, DownBwdArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hl = lane >> 5, l32 = lane & 31, wm = wave & 1, wn = wave >> 1;
  const int ntiles = ((a.f + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  auto coords = [&](int t, int& tm, int& tn) { gemm::tile_coords(t, a.f, a.n, tm, tn, a.group); };
  auto pre = [](int, int) {};
  auto epi = [&](f32x16(&acc)[4][2], int tm, int tn) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int token = tn * BN + 64 * wn + 32 * nb + l32;
      if (token >= a.n) continue;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        const int feature = tm * BM + 128 * wm + 32 * mb + 16 * hl;
        const int left = a.f - feature;
        const int64_t at = (int64_t)token * 2 * a.f + feature;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (left <= 8 * half) continue;
          const bf16x8 g = *reinterpret_cast<const bf16x8*>(a.gate_up + at + 8 * half);
          const bf16x8 u = *reinterpret_cast<const bf16x8*>(a.gate_up + at + a.f + 8 * half);
          float dg[8], du[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float dh = acc[mb][nb][8 * half + i];
            float value, slope;
            act_both<kAct>((float)g[i], value, slope);
            dg[i] = dh * (float)u[i] * slope;
            du[i] = dh * value;
          }
          *reinterpret_cast<bf16x8*>(a.d_gate_up + at + 8 * half) = pack8(dg);
          *reinterpret_cast<bf16x8*>(a.d_gate_up + at + a.f + 8 * half) = pack8(du);
        }
      }
    }
  };
  gemm::persistent<true, true, true>(V, DY, a.f, a.n, a.k, ntiles, coords, pre, epi);
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
  int split;
};

Bwd plan_bwd(int n, int d, int f, int d_out) {
  Bwd b{};
  b.split = grad_split(tiles_of(d, 2 * f) + tiles_of(f, d_out), n);
  b.d_gate_up = round_up((size_t)n * 2 * f * 2);
  if (b.split > 1) {
    b.parts_w = round_up((size_t)b.split * d * 2 * f * 4);
    b.parts_v = round_up((size_t)b.split * f * d_out * 4);
  }
  b.total = b.d_gate_up + b.parts_w + b.parts_v;
  return b;
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

unsigned persistent_grid(int tiles) {
  const int cus = gemm::device_cus();
  return (unsigned)(tiles < cus ? tiles : cus);
}

int tile_group(int m_tiles) { return m_tiles <= 16 ? m_tiles : gemm::kGroupM; }

}  // namespace

extern "C" {

int gptrig_gated_mlp_fwd(const void* x, int64_t ldx, const void* gate_up_w, int64_t ldw, const void* down_w,
                         int64_t ldv, int activation, void* gate_up, void* h, void* y, int n, int d, int f, int d_out,
                         void* stream) {
  if (!x || !gate_up_w || !down_w || !h || !y) return GPTRIG_E_NULL;
  if (activation != kSilu && activation != kGelu) return GPTRIG_E_UNSUPPORTED;
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK) return GPTRIG_E_SHAPE;
  if (!rows_ok(x, ldx, d) || !rows_ok(gate_up_w, ldw, 2 * f) || !rows_ok(down_w, ldv, d_out)) return GPTRIG_E_SHAPE;
  if (((uintptr_t)gate_up | (uintptr_t)h | (uintptr_t)y) & 15) return GPTRIG_E_SHAPE;
  if (n == 0) return GPTRIG_OK;
  const hipStream_t s = (hipStream_t)stream;
  const Operand W{(const bf16*)gate_up_w, ldw, 0, f}, X{(const bf16*)x, ldx};
  const UpArgs a{(bf16*)gate_up, (bf16*)h, n, d, f, tile_group(ceil_div(2 * f, BM))};
  const unsigned grid = persistent_grid(tiles_of(2 * f, n));
  if (activation == kSilu && gate_up)
    gated_up_kernel<kSilu, true><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
  else if (activation == kSilu)
    gated_up_kernel<kSilu, false><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
  else if (gate_up)
    gated_up_kernel<kGelu, true><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
  else
    gated_up_kernel<kGelu, false><<<grid, gemm::THREADS, 0, s>>>(W, X, a);
  GPTRIG_CHECK_LAUNCH();
  return gptrig_linear(h, f, down_w, ldv, 0, nullptr, y, d_out, n, f, d_out, stream);
}

size_t gptrig_gated_mlp_bwd_workspace_bytes(int n, int d, int f, int d_out) {
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK || n == 0) return 0;
  return plan_bwd(n, d, f, d_out).total;
}

int gptrig_gated_mlp_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* gate_up_w, int64_t ldw,
                         const void* down_w, int64_t ldv, int activation, const void* gate_up, const void* h, void* dx,
                         void* d_gate_up_w, void* d_down_w, int n, int d, int f, int d_out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (!dy || !x || !gate_up_w || !down_w || !gate_up || !h || !workspace) return GPTRIG_E_NULL;
  if (activation != kSilu && activation != kGelu) return GPTRIG_E_UNSUPPORTED;
  if (check_sizes(n, d, f, d_out) != GPTRIG_OK || n == 0) return GPTRIG_E_SHAPE;
  if (!rows_ok(x, ldx, d) || !rows_ok(dy, lddy, d_out) || !rows_ok(gate_up_w, ldw, 2 * f) ||
      !rows_ok(down_w, ldv, d_out))
    return GPTRIG_E_SHAPE;
  if (((uintptr_t)gate_up | (uintptr_t)h | (uintptr_t)dx | (uintptr_t)d_gate_up_w | (uintptr_t)d_down_w |
       (uintptr_t)workspace) & 15)
    return GPTRIG_E_SHAPE;
  const Bwd b = plan_bwd(n, d, f, d_out);
  if (workspace_bytes < b.total) return GPTRIG_E_WORKSPACE;
  const hipStream_t s = (hipStream_t)stream;
  bf16* const dgu = (bf16*)workspace;
  if (dx || d_gate_up_w) {
    const Operand V{(const bf16*)down_w, ldv}, DY{(const bf16*)dy, lddy};
    const DownBwdArgs a{(const bf16*)gate_up, dgu, n, d_out, f, tile_group(ceil_div(f, BM))};
    const unsigned grid = persistent_grid(tiles_of(f, n));
    if (activation == kSilu)
      gated_down_bwd_kernel<kSilu><<<grid, gemm::THREADS, 0, s>>>(V, DY, a);
    else
      gated_down_bwd_kernel<kGelu><<<grid, gemm::THREADS, 0, s>>>(V, DY, a);
    GPTRIG_CHECK_LAUNCH();
  }
  if (dx) {
    const int status = gptrig_linear(dgu, 2 * (int64_t)f, gate_up_w, ldw, 1, nullptr, dx, d, n, 2 * f, d, stream);
    if (status != GPTRIG_OK) return status;
  }
  GradItems g{};
  g.n = n;
  g.split = b.split;
  int first = 0;
  if (d_gate_up_w) {
    g.item[g.count++] = GradItem{(const bf16*)x, dgu, ldx, 2 * (int64_t)f, (bf16*)d_gate_up_w,
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
