// Backward of the attention of scored_attention.h, in two passes that each own
// what they sum, so no atomics: results do not depend on the order of anything.
//   dq: a workgroup owns 128 queries of one head, like the forward, and walks the
//     keys; it also leaves delta_i = o_i . do_i for the other pass.
//   dk, dv: a workgroup owns 128 keys of one kv head and walks the queries of
//     every head of its group.
// Both compute the scores and dP anew (3 and 4 products of the pair matrix
// instead of 5 in one pass), which costs less than carrying dq across
// workgroups through float32 atomics.
//
// A visible infinity or NaN in a tile that also holds hidden pairs makes the rows
// of dq, or of dk and dv, that it reaches NaN throughout.
#include "scored_attention.h"

namespace {

constexpr int kOwn = 128;  // queries or keys of a workgroup: 4 waves x 32

template <int D, bool kCap, bool kBias, bool kSeg>
__global__ void __launch_bounds__(256, 2)
    scored_dq_kernel(View Q, View K, View V, View O, View dO, const float* __restrict__ lse2,
                     const int32_t* __restrict__ seg, float* __restrict__ delta, MutView dQ, ScoreArgs a, int B, int H,
                     int Hk, int S, int dim, float scale) {
  constexpr int KC = D / 16, DB = D / 32;
  __shared__ __attribute__((aligned(16))) bf16 fk0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fk1[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv1[kRows * D];
  __shared__ uint64_t dirty_s[4], scan_s[2];

  const int nq = (S + kOwn - 1) / kOwn;
  int bh, qb;
  xcd_map(blockIdx.x, nq, B * H, bh, qb);
  qb = nq - 1 - qb;
  const int b = bh / H, h = bh % H, hk = h / (H / Hk);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int q0 = qb * kOwn, qw0 = q0 + 32 * wave, my_q = qw0 + l32;
  const int last_prefix = __builtin_amdgcn_readfirstlane(prefix_of(a, b, S)) - 1;
  const int my_last = min(max(my_q, last_prefix), S - 1);
  const int all_see = max(qw0, last_prefix);
  const int wave_last = max(qw0 + 31, last_prefix);
  const int ntiles = max(min(q0 + kOwn, S) - 1, last_prefix) / kRows + 1;
  const float slope2 = kBias ? a.slopes[h] * GPTRIG_LOG2E : 0.f;

  bf16x8 qreg[KC], greg[KC];
  float my_delta = 0.f;
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int c = 16 * kc + 8 * hl;
    const bool ok = my_q < S && c < dim;
    qreg[kc] = ok ? *reinterpret_cast<const bf16x8*>(Q.row(b, h, my_q) + c) : bf16x8{};
    greg[kc] = ok ? *reinterpret_cast<const bf16x8*>(dO.row(b, h, my_q) + c) : bf16x8{};
    const bf16x8 o = ok ? *reinterpret_cast<const bf16x8*>(O.row(b, h, my_q) + c) : bf16x8{};
#pragma unroll
    for (int j = 0; j < 8; ++j) my_delta = fmaf((float)o[j], (float)greg[kc][j], my_delta);
  }
  my_delta += __shfl_xor(my_delta, 32);
  const size_t my_row = (size_t)bh * S + my_q;
  const float my_lse = my_q < S ? lse2[my_row] : 0.f;
  if (my_q < S && hl == 0) delta[my_row] = my_delta;
  const int seg_q = (kSeg && my_q < S) ? seg[(size_t)b * S + my_q] : 0;
  SegScan<4> scan;
  if constexpr (kSeg) scan.template init<kOwn / 64>(seg + (size_t)b * S, scan_s, S, q0, lane);

  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
  bool spoilt = false;

  const __amdgpu_buffer_rsrc_t k_rs = slice(K.row(b, hk, 0), S, K.ss, dim);
  const __amdgpu_buffer_rsrc_t v_rs = slice(V.row(b, hk, 0), S, V.ss, dim);
  Fill<D> kf, vf;
  kf.init(K.ss, dim, wave, lane);
  vf.init(V.ss, dim, wave, lane);

  auto half = [&](const at64::lds_t* kt, const at64::lds_t* vt, int kv0, int sb,
                  bool same) __attribute__((always_inline)) {
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      s = mfma32(tile_row(kt, 32 * sb + l32, 2 * kc + hl), qreg[kc], s);
      dp = mfma32(tile_row(vt, 32 * sb + l32, 2 * kc + hl), greg[kc], dp);
    }
    const int kh0 = kv0 + 32 * sb;
    const float x = (float)(my_q - kh0 - 4 * hl);
    const bool both_ways = kBias && kh0 + 31 > qw0 && last_prefix > qw0;
    const float b0 = -slope2 * x - my_lse;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float w, t = base_score<kCap>(s[i], a, w);
      if constexpr (kBias) {
        if (both_ways) t = fmaf(-slope2, fabsf(x - (float)acc_row(i)), t) - my_lse;
        else t += fmaf(slope2, (float)acc_row(i), b0);
      } else {
        t -= my_lse;
      }
      float ds = fast_exp2(t) * (dp[i] - my_delta);
      if constexpr (kCap) ds *= fmaf(-w, w, w);  // (1 - tanh^2) / 4
      s[i] = ds;
    }
    if (kh0 + 31 > all_see || kh0 + 32 > S || (kSeg && !same)) {
      const int lim = my_last - kh0 - 4 * hl;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        bool vis = acc_row(i) <= lim;
        if (kSeg && !same) vis = vis && seg[(size_t)b * S + min(kh0 + 4 * hl + acc_row(i), S - 1)] == seg_q;
        s[i] = vis ? s[i] : 0.f;
      }
    }
    bf16x8 ds8[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) ds8[i >> 3][i & 7] = (bf16)s[i];
    product<DB>(acc, kt, 32 * sb, ds8, lane);
  };

  auto clean = [&](at64::lds_t* kt, int kv0, bool same) {
    const Dirty<D> dirty{dirty_s};
    if (!dirty.find(kt, wave, lane)) return;
#pragma unroll 1
    for (int r = 0; r < kRows; ++r) {
      if (!__builtin_amdgcn_readfirstlane(dirty.row(r))) continue;
      bool vis = kv0 + r <= my_last;
      if (kSeg && !same) vis = vis && seg[(size_t)b * S + min(kv0 + r, S - 1)] == seg_q;
      spoilt |= vis;
    }
    dirty.clear(kt, wave, lane);
  };

  auto tile = [&](at64::lds_t* kt, const at64::lds_t* vt, at64::lds_t* nkt, at64::lds_t* nvt, int it, int nx,
                  bool same) __attribute__((always_inline)) {
    const int kv0 = it * kRows;
    if (nx < ntiles) {
      kf(k_rs, nkt, nx * kRows, wave);
      vf(v_rs, nvt, nx * kRows, wave);
    }
    if (kv0 + kRows - 1 > max(q0, last_prefix) || (kSeg && !same)) clean(kt, kv0, same);
    if (kv0 <= wave_last) half(kt, vt, kv0, 0, same);
    __builtin_amdgcn_sched_barrier(0);  // keep the halves' live ranges apart
    if (kv0 + 32 <= wave_last) half(kt, vt, kv0, 1, same);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next tile has landed
    __syncthreads();
  };

  at64::lds_t* const k0s = gemm::lds_cast(fk0);
  at64::lds_t* const k1s = gemm::lds_cast(fk1);
  at64::lds_t* const v0s = gemm::lds_cast(fv0);
  at64::lds_t* const v1s = gemm::lds_cast(fv1);
  auto next = [&](int t, bool& same) {
    if constexpr (kSeg) return scan.next(t, ntiles, wave, lane, same);
    same = true;
    return t;
  };
  bool same = true, same_n = true;
  int it = next(0, same);
  kf(k_rs, k0s, it * kRows, wave);
  vf(v_rs, v0s, it * kRows, wave);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  while (true) {
    int nx = next(it + 1, same_n);
    tile(k0s, v0s, k1s, v1s, it, nx, same);
    if (nx >= ntiles) break;
    it = nx;
    nx = next(it + 1, same);
    tile(k1s, v1s, k0s, v0s, it, nx, same_n);
    if (nx >= ntiles) break;
    it = nx;
  }

  if (my_q < S) {
    const float f = spoilt ? __builtin_nanf("") : kCap ? 4.0f * scale : scale;
    bf16* row = dQ.row(b, h, my_q);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d0 = 32 * db + 8 * r + 4 * hl;
        if (d0 >= dim) continue;
        bf16x4 v;
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = (bf16)(acc[db][4 * r + t] * f);
        *reinterpret_cast<bf16x4*>(row + d0) = v;
      }
  }
}

// dk and dv.  Each wave computes S = Q K^T and dP = do V^T with a lane holding one
// key, whose k and v stay in registers as operands, and sums dv^T += do^T P and
// dk^T += Q^T dU over the queries.
template <int D, bool kCap, bool kBias, bool kSeg>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1)
    scored_dkv_kernel(View Q, View K, View V, View dO, const float* __restrict__ lse2,
                      const float* __restrict__ delta, const int32_t* __restrict__ seg, MutView dK, MutView dV,
                      ScoreArgs a, int B, int H, int Hk, int S, int dim, float scale) {
  constexpr int KC = D / 16, DB = D / 32;
  __shared__ __attribute__((aligned(16))) bf16 fq0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fq1[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fg0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fg1[kRows * D];
  __shared__ __attribute__((aligned(16))) float ls0[kRows], ls1[kRows], dl0[kRows], dl1[kRows];
  __shared__ __attribute__((aligned(16))) int sg0[kRows], sg1[kRows];
  __shared__ uint64_t dirty_s[4], scan_s[2];

  const int nkv = (S + kOwn - 1) / kOwn, G = H / Hk;
  int bh, kb;
  xcd_map(blockIdx.x, nkv, B * Hk, bh, kb);
  const int b = bh / Hk, hk = bh % Hk;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int k0 = kb * kOwn, kw0 = k0 + 32 * wave, my_k = kw0 + l32;
  const int last_prefix = __builtin_amdgcn_readfirstlane(prefix_of(a, b, S)) - 1;

  bf16x8 kfr[KC], vfr[KC];
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int c = 16 * kc + 8 * hl;
    const bool ok = my_k < S && c < dim;
    kfr[kc] = ok ? *reinterpret_cast<const bf16x8*>(K.row(b, hk, my_k) + c) : bf16x8{};
    vfr[kc] = ok ? *reinterpret_cast<const bf16x8*>(V.row(b, hk, my_k) + c) : bf16x8{};
  }
  const int seg_k = (kSeg && my_k < S) ? seg[(size_t)b * S + my_k] : 0;
  SegScan<4> scan;
  if constexpr (kSeg) scan.template init<kOwn / 64>(seg + (size_t)b * S, scan_s, S, k0, lane);

  f32x16 dv_acc[DB], dk_acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    dv_acc[db] = f32x16{};
    dk_acc[db] = f32x16{};
  }
  bool spoilt = false;

  Fill<D> qf, gf;
  qf.init(Q.ss, dim, wave, lane);
  gf.init(dO.ss, dim, wave, lane);
  // Rows of head h: past the last one lse and delta read as zeros like q and do.
  auto fill = [&](at64::lds_t* qt, at64::lds_t* gt, float* ls, float* dl, int* sg, int h, int qq0) {
    qf(slice(Q.row(b, h, 0), S, Q.ss, dim), qt, qq0, wave);
    gf(slice(dO.row(b, h, 0), S, dO.ss, dim), gt, qq0, wave);
    const size_t row = ((size_t)b * H + h) * S;
    if (wave == 0)
      dma4(make_rsrc(lse2 + row, (uint32_t)S * 4u), ls, (qq0 + lane) * 4);
    if (wave == 1)
      dma4(make_rsrc(delta + row, (uint32_t)S * 4u), dl, (qq0 + lane) * 4);
    if (kSeg && wave == 2)
      dma4(make_rsrc(seg + (size_t)b * S, (uint32_t)S * 4u), sg, (qq0 + lane) * 4);
  };

  // 32 queries qq0 + 32 qs .. of the tile.
  auto half = [&](const at64::lds_t* qt, const at64::lds_t* gt, const float* ls, const float* dl, const int* sg,
                  int qq0, int qs, float slope2, bool same) __attribute__((always_inline)) {
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      s = mfma32(tile_row(qt, 32 * qs + l32, 2 * kc + hl), kfr[kc], s);
      dp = mfma32(tile_row(gt, 32 * qs + l32, 2 * kc + hl), vfr[kc], dp);
    }
    const int qh0 = qq0 + 32 * qs;
    const float x = (float)(qh0 + 4 * hl - my_k);  // the distance of element 0
    const bool both_ways = kBias && kw0 + 31 > qh0 && last_prefix > qh0;
    const float b0 = -slope2 * x;
    float p[16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + 32 * qs + 8 * r + 4 * hl);
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(dl + 32 * qs + 8 * r + 4 * hl);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = 4 * r + t;
        float w, u = base_score<kCap>(s[i], a, w);
        if constexpr (kBias) {
          if (both_ways) u = fmaf(-slope2, fabsf(x + (float)acc_row(i)), u);
          else u += fmaf(-slope2, (float)acc_row(i), b0);
        }
        p[i] = fast_exp2(u - l4[t]);
        float ds = p[i] * (dp[i] - d4[t]);
        if constexpr (kCap) ds *= fmaf(-w, w, w);  // (1 - tanh^2) / 4
        s[i] = ds;
      }
    }
    if (kw0 + 31 > max(qh0, last_prefix) || qh0 + 32 > S || (kSeg && !same)) {
      // Query qh0 + 4 hl + c sees my_k from c = first on, all of them inside the prefix.
      const int first = my_k <= last_prefix ? -64 : my_k - qh0 - 4 * hl, end = S - qh0 - 4 * hl;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        bool vis = acc_row(i) >= first && acc_row(i) < end;
        if (kSeg && !same) vis = vis && sg[32 * qs + 4 * hl + acc_row(i)] == seg_k;
        p[i] = vis ? p[i] : 0.f;
        s[i] = vis ? s[i] : 0.f;
      }
    }
    bf16x8 p8[2], ds8[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p8[i >> 3][i & 7] = (bf16)p[i];
      ds8[i >> 3][i & 7] = (bf16)s[i];
    }
    product<DB>(dv_acc, gt, 32 * qs, p8, lane);
    product<DB>(dk_acc, qt, 32 * qs, ds8, lane);
  };

  auto clean = [&](at64::lds_t* t, const int* sg, int qq0, bool same) {
    const Dirty<D> dirty{dirty_s};
    if (dirty.find(t, wave, lane)) {
#pragma unroll 1
      for (int r = 0; r < kRows; ++r) {
        if (!__builtin_amdgcn_readfirstlane(dirty.row(r))) continue;
        bool vis = my_k <= max(qq0 + r, last_prefix);
        if (kSeg && !same) vis = vis && sg[r] == seg_k;
        spoilt |= vis;
      }
      dirty.clear(t, wave, lane);
    }
  };

  auto tile = [&](at64::lds_t* qt, at64::lds_t* gt, const float* ls, const float* dl, const int* sg, int qb, float slope2,
                  bool same) __attribute__((always_inline)) {
    const int qq0 = qb * kRows;
    if (k0 + kOwn - 1 > max(qq0, last_prefix) || (kSeg && !same)) {
      clean(qt, sg, qq0, same);
      __syncthreads();  // (the second search reuses the first one's words)
      clean(gt, sg, qq0, same);
    }
    const bool here = kw0 < S;
    if (here && kw0 <= max(qq0 + 31, last_prefix)) half(qt, gt, ls, dl, sg, qq0, 0, slope2, same);
    __builtin_amdgcn_sched_barrier(0);  // keep the halves' live ranges apart
    if (here && kw0 <= max(qq0 + 63, last_prefix)) half(qt, gt, ls, dl, sg, qq0, 1, slope2, same);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next tile has landed
    __syncthreads();
  };

  at64::lds_t* const q0s = gemm::lds_cast(fq0);
  at64::lds_t* const q1s = gemm::lds_cast(fq1);
  at64::lds_t* const g0s = gemm::lds_cast(fg0);
  at64::lds_t* const g1s = gemm::lds_cast(fg1);
  const int nqb = (S + kRows - 1) / kRows, start = k0 <= last_prefix ? 0 : k0 / kRows;
  // The tiles of one head after another; g: the head in its group.
  auto next = [&](int t, int& g, bool& same) {
    if constexpr (kSeg) {
      t = scan.next(t, nqb, wave, lane, same);
      if (t >= nqb) {
        ++g;
        t = scan.next(start, nqb, wave, lane, same);
      }
    } else {
      same = true;
      if (t >= nqb) {
        ++g;
        t = start;
      }
    }
    return t;
  };
  auto slope_of = [&](int g) { return kBias ? a.slopes[hk * G + g] * GPTRIG_LOG2E : 0.f; };
  int g = 0, gn = 0;
  bool same = true, same_n = true;
  int qb = next(start, g, same), nx;
  gn = g;
  fill(q0s, g0s, ls0, dl0, sg0, hk * G + g, qb * kRows);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  while (true) {  // (The workgroup's own positions hold visible pairs: every head has a first tile.)
    nx = next(qb + 1, gn, same_n);
    if (gn < G) fill(q1s, g1s, ls1, dl1, sg1, hk * G + gn, nx * kRows);
    tile(q0s, g0s, ls0, dl0, sg0, qb, slope_of(g), same);
    if (gn >= G) break;
    qb = nx, g = gn;
    nx = next(qb + 1, gn, same);
    if (gn < G) fill(q0s, g0s, ls0, dl0, sg0, hk * G + gn, nx * kRows);
    tile(q1s, g1s, ls1, dl1, sg1, qb, slope_of(g), same_n);
    if (gn >= G) break;
    qb = nx, g = gn;
  }

  if (my_k < S) {
    const float bad = spoilt ? __builtin_nanf("") : 1.0f;
    const float f = bad * (kCap ? 4.0f * scale : scale);
    bf16* krow = dK.row(b, hk, my_k);
    bf16* vrow = dV.row(b, hk, my_k);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d0 = 32 * db + 8 * r + 4 * hl;
        if (d0 >= dim) continue;
        bf16x4 k4, v4;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          k4[t] = (bf16)(dk_acc[db][4 * r + t] * f);
          v4[t] = (bf16)(dv_acc[db][4 * r + t] * bad);
        }
        *reinterpret_cast<bf16x4*>(krow + d0) = k4;
        *reinterpret_cast<bf16x4*>(vrow + d0) = v4;
      }
  }
}

}  // namespace

extern "C" {

size_t gptrig_scored_attn_bwd_workspace_bytes(int batch, int heads, int kv_heads, int seq, int head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || seq <= 0 || head_dim <= 0) return 0;
  return (size_t)batch * heads * seq * sizeof(float);
}

int gptrig_scored_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout,
                           const float* lse2, const int32_t* segment_ids, const int32_t* prefix_lengths,
                           const float* distance_slopes, void* dq, void* dk, void* dv, void* workspace,
                           size_t workspace_bytes, int batch, int heads, int kv_heads, int seq, int head_dim,
                           const int64_t* strides, float softmax_scale, float score_cap, void* stream) {
  ScoredCall c;
  if (!lse2 || !workspace) return GPTRIG_E_NULL;
  const void* tensors[8] = {q, k, v, o, dout, dq, dk, dv};
  const int status = c.init(tensors, 8, 0b11000110u, batch, heads, kv_heads, seq, head_dim, strides, softmax_scale,
                            score_cap, distance_slopes, prefix_lengths);
  if (status != GPTRIG_OK) return status;
  if (workspace_bytes < gptrig_scored_attn_bwd_workspace_bytes(batch, heads, kv_heads, seq, head_dim))
    return GPTRIG_E_WORKSPACE;
  if ((uintptr_t)workspace & 15) return GPTRIG_E_SHAPE;
  const long long grid = (long long)batch * heads * ceil_div(seq, kOwn);
  if (grid > INT32_MAX) return GPTRIG_E_SHAPE;
  const unsigned kv_grid = (unsigned)((long long)batch * kv_heads * ceil_div(seq, kOwn));
  hipStream_t s = (hipStream_t)stream;
  const View Q = c.view(0), K = c.view(1), V = c.view(2), O = c.view(3), dO = c.view(4);
  const MutView dQ = c.out(5), dK = c.out(6), dV = c.out(7);
  float* const delta = (float*)workspace;
#define SCORED_BWD(D, CAP, BIAS, SEG)                                                                              \
  scored_dq_kernel<D, CAP, BIAS, SEG><<<(unsigned)grid, 256, 0, s>>>(Q, K, V, O, dO, lse2, segment_ids, delta, dQ,   \
                                                                     c.args, batch, heads, kv_heads, seq, head_dim,  \
                                                                     softmax_scale);                                 \
  scored_dkv_kernel<D, CAP, BIAS, SEG><<<kv_grid, 256, 0, s>>>(Q, K, V, dO, lse2, delta, segment_ids, dK, dV, c.args, \
                                                               batch, heads, kv_heads, seq, head_dim, softmax_scale)
  SCORED_DISPATCH(SCORED_BWD, c, segment_ids != nullptr);
#undef SCORED_BWD
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

}  // extern "C"
