// Backward of the attention of scored_attention.h, in two passes that each own
// what they sum, so no atomics: results do not depend on the order of anything.
//   dq: a workgroup owns 128 queries of one head, like the forward, and walks the
//     keys; it also leaves delta_i = o_i . do_i for the other pass, of o and o_low,
//     which holds what the rounding of o to bf16 cut off: delta is subtracted from
//     dP values of its own size, so a rounded o would add half as much to the error
//     of dq and dk as the rounding of dU does (0.9 and 1.7 in 1000 of dq's norm).
//   dk, dv: a workgroup owns 128 keys of one kv head and walks the queries of
//     every head of its group.
// Both compute the scores and dP anew: 3 and 4 products of the pair matrix instead
// of 5 in one pass that adds dq up in float32 atomics.  The causal attention of
// attention.hip is such a pass: plain scores, B16 H12 S1024 D64 148 us against 136 for
// the two here, B4 H16 S2048 D128 495 against 293, of other bits on every run.
//
// Bound by the issue of vector and matrix instructions, which overlap little at two
// waves a SIMD.  In a loop of passes on the same inputs, B16 H12 S1024 D64, cap 30: dq
// 75 us (of a CU's busy time 70% vector, 24% matrix instructions), dk and dv 93 us (56%,
// 25%; all of them 79%).  B4 H16/4 S2048 D128, cap and bias: 140 us (57%, 34%) and 174
// us (43%, 34%; all of them 67%), and 14 for the join.
//
// A visible infinity or NaN in a tile that also holds hidden pairs makes the rows
// of dq, or of dk and dv, that it reaches NaN throughout.
#include "scored_attention.h"

namespace {

constexpr int kOwn = 128;  // queries or keys of a workgroup: 4 waves x 32

// A wave's accumulators in LDS, in the room of one tile, and back.
template <int DB>
__device__ __forceinline__ void put(float* at, const f32x16 (&acc)[DB], int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) at[(16 * db + i) * 64 + lane] = acc[db][i];
}
template <int DB>
__device__ __forceinline__ void add(f32x16 (&acc)[DB], const float* at, int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] += at[(16 * db + i) * 64 + lane];
}

// The dq pass leaves two numbers a query for the other pass: the constant of its
// exponents, cap log2 e - L_i (with a bias less slope (i mod 64), the part of the
// bias that is the query's own in its tile), and -delta_i.
//
// At D = 64 without a bias the loop fits the 168 registers of three waves a SIMD, with
// kt's transposed operands loaded only after the vector work: B16 H12 S1024, cap 30, 89
// us against 104 with the loads ahead of it at two waves (the two in one run, on inputs
// that change between launches).  With a bias, two waves and the loads ahead.
template <int D, bool kCap, bool kBias, bool kSeg, int kSplit>
__global__ void __launch_bounds__(256, D == 64 && !kBias ? 3 : 2)
    scored_dq_kernel(View Q, View K, View V, View O, View dO, const uint8_t* __restrict__ o_low,
                     const float* __restrict__ lse2, const int32_t* __restrict__ seg, const int* __restrict__ plan,
                     float* __restrict__ shifts, float* __restrict__ minus_delta, MutView dQ, ScoreArgs a, int B, int H, int Hk, int S, int dim, float scale) {
  constexpr int KC = D / 16, DB = D / 32;
  __shared__ __attribute__((aligned(16))) bf16 fk0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fk1[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv1[kRows * D];
  __shared__ __attribute__((aligned(16))) int sg0[kRows], sg1[kRows];
  __shared__ uint64_t dirty_s[4], scan_s[2];

  constexpr int kMine = kOwn / kSplit;
  const int nq = (S + kMine - 1) / kMine;
  int bh, qb;
  block_of(plan, blockIdx.x, nq, B, H, true, bh, qb);
  const int b = bh / H, h = bh % H, hk = h / (H / Hk);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int own = wave % (4 / kSplit), part = wave / (4 / kSplit);  // (as in the forward)
  const int q0 = qb * kMine, qw0 = q0 + 32 * own, my_q = qw0 + l32;
  const int last_prefix = __builtin_amdgcn_readfirstlane(prefix_of(a, b, S)) - 1;
  const int my_last = min(max(my_q, last_prefix), S - 1);
  const int wave_last = max(qw0 + 31, last_prefix);
  const int ntiles = max(min(q0 + kMine, S) - 1, last_prefix) / kRows + 1;
  const float slope2 = kBias ? a.slopes[h] * GPTRIG_LOG2E : 0.f;
  float bias[16], raw = a.raw, twice = -2.0f * a.cap2;
  if constexpr (kBias) {
    row_bias(bias, slope2);
    asm("" : "+v"(raw), "+v"(twice));
  }

  bf16x8 qreg[KC], greg[KC];
  const size_t my_row = (size_t)bh * S + my_q;
  float delta = 0.f;
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int c = 16 * kc + 8 * hl;
    const bool ok = my_q < S && c < dim;
    qreg[kc] = ok ? *reinterpret_cast<const bf16x8*>(Q.row(b, h, my_q) + c) : bf16x8{};
    greg[kc] = ok ? *reinterpret_cast<const bf16x8*>(dO.row(b, h, my_q) + c) : bf16x8{};
    const bf16x8 o = ok ? *reinterpret_cast<const bf16x8*>(O.row(b, h, my_q) + c) : bf16x8{};
    const uint2 low = ok ? *reinterpret_cast<const uint2*>(o_low + my_row * dim + c) : uint2{};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      delta = fmaf(with_low_bits(o[j], (j < 4 ? low.x : low.y) >> (8 * (j & 3))), (float)greg[kc][j], delta);
  }
  delta += __shfl_xor(delta, 32);
  const float shift = my_q < S ? (kCap ? a.cap2 : 0.f) - lse2[my_row] : 0.f;
  if (my_q < S && hl == 0 && part == 0) {
    shifts[my_row] = kBias ? fmaf(-slope2, (float)(my_q & (kRows - 1)), shift) : shift;
    minus_delta[my_row] = -delta;
  }
  const int seg_q = kSeg ? seg[(size_t)b * S + min(my_q, S - 1)] : 0;
  WaveIds ids;
  SegScan<4> scan;
  if constexpr (kSeg) {
    ids.init(seg_q);
    scan.template init<kMine / 64>(seg + (size_t)b * S, scan_s, S, q0, lane);
  }

  Lanes lanes;
  lanes.init(lane);
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
  bool spoilt = false;

  const __amdgpu_buffer_rsrc_t k_rs = slice(K.row(b, hk, 0), S, K.ss, dim);
  const __amdgpu_buffer_rsrc_t v_rs = slice(V.row(b, hk, 0), S, V.ss, dim);
  Fill<D> kf, vf;
  kf.init(K.ss, dim, wave, lane);
  vf.init(V.ss, dim, wave, lane);
  auto fill = [&](at64::lds_t* kt, at64::lds_t* vt, int* sg, int kv0) {
    kf(k_rs, kt, kv0, wave);
    vf(v_rs, vt, kv0, wave);
    if (kSeg && wave == 2) dma4(make_rsrc(seg + (size_t)b * S, (uint32_t)S * 4u), sg, (kv0 + lane) * 4);
  };

  auto half = [&](const at64::lds_t* kt, const at64::lds_t* vt, const int* sg, int kv0, int sb,
                  int docs) __attribute__((always_inline)) {
    const uint32_t at = 32 * kRowBytes * sb;
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int k0 = 0; k0 < KC; k0 += 4) {
      bf16x8 kr[4], vr[4];
#pragma unroll
      for (int kc = 0; kc < 4; ++kc) {
        kr[kc] = row_operand(kt, lanes, at, k0 + kc);
        vr[kc] = row_operand(vt, lanes, at, k0 + kc);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kc = 0; kc < 4; ++kc) {
        s = mfma32(kr[kc], qreg[k0 + kc], s);
        dp = mfma32(vr[kc], greg[k0 + kc], dp);
      }
    }
    constexpr bool kAhead = D == 64 && kBias;  // (elsewhere registers are short)
    Columns<DB> kcol;
    if (kAhead) kcol.load(kt, lanes, at);
    __builtin_amdgcn_sched_barrier(0);
    const int kh0 = kv0 + 32 * sb;
    const float x = (float)(my_q - kh0 - 4 * hl);
    const float off = kBias ? fmaf(-slope2, x, shift) : shift;
    float w[kCap ? 16 : 1];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (kCap) {
        w[i] = cap_w(s[i], a);
        s[i] = kBias ? fmaf(twice, w[i], bias[i]) + off : fmaf(twice, w[i], off);
      } else {
        s[i] = kBias ? fmaf(s[i], raw, bias[i]) + off : fmaf(s[i], raw, off);
      }
    }
    const bool after = kh0 + 31 > qw0;
    if constexpr (kBias) {  // (as in the forward)
      if (kh0 > qw0 + 31) {
        const float twice_off = 2.0f * slope2 * x;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fmaf(-2.0f, bias[i], s[i] + twice_off);
      } else if (after && last_prefix > qw0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fmaf(-2.0f * slope2, fmaxf((float)acc_row(i) - x, 0.f), s[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = fast_exp2(s[i]) * (dp[i] - delta);
      if constexpr (kCap) s[i] *= fmaf(-w[i], w[i], w[i]);  // (1 - tanh^2) / 4
    }
    if ((after && kh0 + 31 > last_prefix) || kh0 + 32 > S || (kSeg && docs)) {
      const int lim = my_last - kh0 - 4 * hl;
      if (kSeg && docs) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const i32x4 id = *reinterpret_cast<const i32x4*>(sg + 32 * sb + 8 * r + 4 * hl);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            s[4 * r + t] = acc_row(4 * r + t) <= lim && id[t] == seg_q ? s[4 * r + t] : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = acc_row(i) <= lim ? s[i] : 0.f;
      }
    }
    bf16x8 ds8[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) ds8[i >> 3][i & 7] = (bf16)s[i];
    __builtin_amdgcn_sched_barrier(0);
    if (!kAhead) kcol.load(kt, lanes, at);
    kcol.product(acc, ds8);
  };

  auto clean = [&](at64::lds_t* kt, const int* sg, int kv0, bool same) {
    const Dirty<D> dirty{dirty_s};
    if (!dirty.find(kt, wave, lane)) return;
#pragma unroll 1
    for (int r = 0; r < kRows; ++r) {
      if (!__builtin_amdgcn_readfirstlane(dirty.row(r))) continue;
      bool vis = kv0 + r <= my_last;
      if (kSeg && !same) vis = vis && sg[r] == seg_q;
      spoilt |= vis;
    }
    dirty.clear(kt, wave, lane);
  };

  auto tile = [&](at64::lds_t* kt, const at64::lds_t* vt, const int* sg, at64::lds_t* nkt, at64::lds_t* nvt, int* nsg,
                  int it, int nx, bool same) __attribute__((always_inline)) {
    const int kv0 = it * kRows;
    int sb = 0, end = 0, docs = 0;
    if (it < ntiles) {
      if (nx < ntiles) fill(nkt, nvt, nsg, nx * kRows);
      if (kv0 + kRows - 1 > max(q0, last_prefix) || (kSeg && !same)) clean(kt, sg, kv0, same);
      end = kv0 > wave_last ? 0 : kv0 + 32 > wave_last ? 1 : 2;
      if (kSeg && !same) {
        const int in = ids.look(sg, lane, docs);
        sb = in & 1 ? 0 : 1;
        end = min(end, in & 2 ? 2 : in);
      }
      if (kSplit == 2) {
        sb = max(sb, part);
        end = min(end, part + 1);
      }
    }
#pragma unroll 1
    for (; sb < end; ++sb) half(kt, vt, sg, kv0, sb, docs >> sb & 1);
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
  fill(k0s, v0s, sg0, it * kRows);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  while (it < ntiles) {
    const int nx = next(it + 1, same_n);
    tile(k0s, v0s, sg0, k1s, v1s, sg1, it, nx, same);
    it = next(nx + 1, same);
    tile(k1s, v1s, sg1, k0s, v0s, sg0, nx, it, same_n);
  }

  if constexpr (kSplit == 2) {
    float* const at = reinterpret_cast<float*>(own ? fv0 : fk0);
    if (part) put<DB>(at, acc, lane);
    __syncthreads();
    if (part) return;
    add<DB>(acc, at, lane);
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
//
// kSplit waves share 32 keys, each with its half of every tile.  At D = 128 the sums
// of a wave are 128 registers: with k and v in registers too there is room for one
// wave a SIMD, which waits for every product; so where there are enough of them 8
// waves own 128 keys, two waves a SIMD, and k and v are in LDS (B4 H16/4 S2048 capped
// and biased, forward and backward: 535 us with one wave a SIMD, 497 with two, when
// this was chosen; 451 with the later steps).
template <int D, bool kCap, bool kBias, bool kSeg, int kSplit, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, D == 64 || kWaves == 8 ? 2 : 1)
    scored_dkv_kernel(View Q, View K, View V, View dO, const float* __restrict__ shifts,
                      const float* __restrict__ minus_delta, const int32_t* __restrict__ seg,
                      const int* __restrict__ plan, MutView dK, MutView dV, float* __restrict__ partial, int parts, ScoreArgs a, int B, int H, int Hk, int S, int dim,
                      float scale) {
  constexpr int KC = D / 16, DB = D / 32, kGroups = kWaves / kSplit, kMine = 32 * kGroups;
  constexpr bool kKeysInLds = kWaves == 8;
  __shared__ __attribute__((aligned(16))) bf16 fk[kKeysInLds ? kMine * D : 8];
  __shared__ __attribute__((aligned(16))) bf16 fv[kKeysInLds ? kMine * D : 8];
  __shared__ __attribute__((aligned(16))) bf16 fq0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fq1[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fg0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fg1[kRows * D];
  __shared__ __attribute__((aligned(16))) float ls0[kRows], ls1[kRows], dl0[kRows], dl1[kRows];
  __shared__ __attribute__((aligned(16))) int sg0[kRows], sg1[kRows];
  __shared__ uint64_t dirty_s[4], scan_s[2];

  // parts workgroups share the heads of a group where there are few keys to own.
  const int nkv = (S + kMine - 1) / kMine, G = H / Hk / parts;
  int bh, kb;
  block_of(plan, blockIdx.x, nkv, B, Hk * parts, false, bh, kb);
  const int b = bh / parts / Hk, hk = bh / parts % Hk, h0 = hk * (H / Hk) + bh % parts * G;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int group = wave % kGroups, part = wave / kGroups;
  const int k0 = kb * kMine, kw0 = k0 + 32 * group, my_k = kw0 + l32;
  const int last_prefix = __builtin_amdgcn_readfirstlane(prefix_of(a, b, S)) - 1;

  // The keys' operands: in registers, or as tiles of 64 keys in LDS.
  at64::lds_t* const ks = gemm::lds_cast(fk);
  at64::lds_t* const vs = gemm::lds_cast(fv);
  bf16x8 kfr[KC], vfr[KC];
  if constexpr (kKeysInLds) {
    Fill<D, kWaves> kf, vf;
    kf.init(K.ss, dim, wave, lane);
    vf.init(V.ss, dim, wave, lane);
#pragma unroll
    for (int i = 0; i < kMine / kRows; ++i) {  // (waited for with the first queries)
      kf(slice(K.row(b, hk, 0), S, K.ss, dim), ks + i * kRows * D, k0 + i * kRows, wave);
      vf(slice(V.row(b, hk, 0), S, V.ss, dim), vs + i * kRows * D, k0 + i * kRows, wave);
    }
  } else {
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const int c = 16 * kc + 8 * hl;
      const bool ok = my_k < S && c < dim;
      kfr[kc] = ok ? *reinterpret_cast<const bf16x8*>(K.row(b, hk, my_k) + c) : bf16x8{};
      vfr[kc] = ok ? *reinterpret_cast<const bf16x8*>(V.row(b, hk, my_k) + c) : bf16x8{};
    }
  }
  // (Byte offset of the wave's keys in LDS.)
  const uint32_t key_at = (32 * group / kRows) * kRows * D * 2 + (32 * group % kRows) * kRowBytes;
  const int seg_k = kSeg ? seg[(size_t)b * S + min(my_k, S - 1)] : 0;
  WaveIds ids;
  SegScan<kWaves> scan;
  if constexpr (kSeg) {
    ids.init(seg_k);
    scan.template init<kMine / 64>(seg + (size_t)b * S, scan_s, S, k0, lane);
  }

  Lanes lanes;
  lanes.init(lane);
  f32x16 dv_acc[DB], dk_acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    dv_acc[db] = f32x16{};
    dk_acc[db] = f32x16{};
  }
  bool spoilt = false;

  Fill<D, kWaves> qf, gf;
  qf.init(Q.ss, dim, wave, lane);
  gf.init(dO.ss, dim, wave, lane);
  // The rows of one head at a time: past the last everything reads as zeros.
  __amdgpu_buffer_rsrc_t q_rs, g_rs, l_rs, d_rs;
  auto of_head = [&](int g) {
    const int h = h0 + min(g, G - 1);
    q_rs = slice(Q.row(b, h, 0), S, Q.ss, dim);
    g_rs = slice(dO.row(b, h, 0), S, dO.ss, dim);
    const size_t row = ((size_t)b * H + h) * S;
    l_rs = make_rsrc(shifts + row, (uint32_t)S * 4u);
    d_rs = make_rsrc(minus_delta + row, (uint32_t)S * 4u);
  };
  auto fill = [&](at64::lds_t* qt, at64::lds_t* gt, float* ls, float* dl, int* sg, int qq0) {
    qf(q_rs, qt, qq0, wave);
    gf(g_rs, gt, qq0, wave);
    if (wave == 0) dma4(l_rs, ls, (qq0 + lane) * 4);
    if (wave == 1) dma4(d_rs, dl, (qq0 + lane) * 4);
    if (kSeg && wave == 2) dma4(make_rsrc(seg + (size_t)b * S, (uint32_t)S * 4u), sg, (qq0 + lane) * 4);
  };

  // 32 queries qq0 + 32 qs .. of the tile.
  float raw = a.raw, twice = -2.0f * a.cap2;
  auto half = [&](const at64::lds_t* qt, const at64::lds_t* gt, const float* ls, const float* dl, const int* sg,
                  int qq0, int qs, float slope2, int docs) __attribute__((always_inline)) {
    const int own = 32 * qs + 4 * hl;  // row of element 0
    f32x16 s = f32x16{}, dp;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(dl + own + 8 * r);
#pragma unroll
      for (int t = 0; t < 4; ++t) dp[4 * r + t] = d4[t];
    }
    const uint32_t at = 32 * kRowBytes * qs;
    constexpr int kStep = kKeysInLds ? 2 : 4;  // operands in flight
#pragma unroll
    for (int k0 = 0; k0 < KC; k0 += kStep) {
      bf16x8 qr[kStep], gr[kStep], kr[kStep], vr[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        qr[i] = row_operand(qt, lanes, at, k0 + i);
        kr[i] = kKeysInLds ? row_operand(ks, lanes, key_at, k0 + i) : kfr[k0 + i];
        gr[i] = row_operand(gt, lanes, at, k0 + i);
        vr[i] = kKeysInLds ? row_operand(vs, lanes, key_at, k0 + i) : vfr[k0 + i];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        s = mfma32(qr[i], kr[i], s);
        dp = mfma32(gr[i], vr[i], dp);
      }
    }
    Columns<DB> gc, qc;
    if (kWaves == 4) gc.load(gt, lanes, at);
    f32x4 l16[4];
    if (kWaves == 4)
#pragma unroll
      for (int r = 0; r < 4; ++r) l16[r] = *reinterpret_cast<const f32x4*>(ls + own + 8 * r);
    __builtin_amdgcn_sched_barrier(0);
    const int qh0 = qq0 + 32 * qs;
    const float off = -slope2 * (float)(qq0 - my_k);
    const bool after = kw0 + 31 > qh0;  // some key comes after some query
    const bool masked = (after && kw0 + 31 > last_prefix) || qh0 + 32 > S || (kSeg && docs);
    bf16x8 p8[2], ds8[2];
    // kAll: every key comes after every query and all are visible, so the distance
    // counts the other way; kBorder: the pairs are looked at one by one.
    auto middle = [&](auto border, auto all) __attribute__((always_inline)) {
      constexpr bool kBorder = decltype(border)::value, kAll = decltype(all)::value;
      const float ahead = kAll ? 2.0f * slope2 * (float)(qh0 + 4 * hl - my_k) : 0.f;
      // Query own + c sees my_k from c = first on, all of them inside the prefix.
      const int first = my_k <= last_prefix ? -64 : my_k - qh0 - 4 * hl, end = S - qh0 - 4 * hl;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 l4 = kWaves == 4 ? l16[r] : *reinterpret_cast<const f32x4*>(ls + own + 8 * r);
        const i32x4 id = kBorder && kSeg ? *reinterpret_cast<const i32x4*>(sg + own + 8 * r) : i32x4{};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int i = 4 * r + t, c = acc_row(i);
          float e, w = 0.f;
          if constexpr (kCap) {
            w = cap_w(s[i], a);
            e = fmaf(twice, w, l4[t]);
          } else {
            e = fmaf(s[i], raw, l4[t]);
          }
          if constexpr (kBias) e += off;
          if constexpr (kAll) e += fmaf(2.0f * slope2, (float)c, ahead);
          if constexpr (kBias && kBorder)  // keys after their query, where a prefix shows them
            e = fmaf(-2.0f * slope2, fmaxf((float)(my_k - qh0 - 4 * hl - c), 0.f), e);
          float p = fast_exp2(e), ds = p * dp[i];
          if constexpr (kCap) ds *= fmaf(-w, w, w);  // (1 - tanh^2) / 4
          if constexpr (kBorder) {
            bool vis = c >= first && c < end;
            if (kSeg) vis = vis && (!docs || id[t] == seg_k);
            p = vis ? p : 0.f;
            ds = vis ? ds : 0.f;
          }
          p8[i >> 3][i & 7] = (bf16)p;
          ds8[i >> 3][i & 7] = (bf16)ds;
        }
      }
    };
    if (masked || (kBias && after && qh0 + 31 >= kw0)) middle(std::true_type{}, std::false_type{});
    else if (kBias && after) middle(std::false_type{}, std::bool_constant<kBias>{});
    else middle(std::false_type{}, std::false_type{});
    __builtin_amdgcn_sched_barrier(0);
    if (kWaves == 8) gc.load(gt, lanes, at);
    else qc.load(qt, lanes, at);
    gc.product(dv_acc, p8);
    if (kWaves == 8) qc.load(qt, lanes, at);
    qc.product(dk_acc, ds8);
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

  auto tile = [&](at64::lds_t* qt, at64::lds_t* gt, const float* ls, const float* dl, const int* sg, int qb, int g,
                  float slope2, bool same) __attribute__((always_inline)) {
    const int qq0 = qb * kRows;
    int qs = 0, end = 0, docs = 0;
    if (g < G) {
      if (k0 + kMine - 1 > max(qq0, last_prefix) || (kSeg && !same)) {
        clean(qt, sg, qq0, same);
        __syncthreads();  // (the second search reuses the first one's words)
        clean(gt, sg, qq0, same);
      }
      qs = kw0 <= max(qq0 + 31, last_prefix) ? 0 : kw0 <= qq0 + 63 ? 1 : 2;
      end = kw0 < S ? 2 : 0;
      if (kSeg && !same) {
        const int in = ids.look(sg, lane, docs);
        qs = max(qs, in & 1 ? 0 : 1);
        end = min(end, in & 2 ? 2 : in);
      }
      if (kSplit == 2) {
        qs = max(qs, part);
        end = min(end, part + 1);
      }
    }
#pragma unroll 1
    for (; qs < end; ++qs) half(qt, gt, ls, dl, sg, qq0, qs, slope2, docs >> qs & 1);
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
  int g = 0;
  bool same = true, same_n = true;
  int qb = next(start, g, same);
  auto slope_of = [&](int g) { return kBias ? a.slopes[h0 + min(g, G - 1)] * GPTRIG_LOG2E : 0.f; };
  of_head(g);
  float slope = slope_of(g);
  fill(q0s, g0s, ls0, dl0, sg0, qb * kRows);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  while (g < G) {  // (The workgroup's own positions hold visible pairs: every head has a first tile.)
    int gn = g;
    const int nx = next(qb + 1, gn, same_n);
    float slope_n = slope;
    if (gn != g) {
      of_head(gn);
      slope_n = slope_of(gn);
    }
    if (gn < G) fill(q1s, g1s, ls1, dl1, sg1, nx * kRows);
    tile(q0s, g0s, ls0, dl0, sg0, qb, g, slope, same);
    g = gn;
    qb = next(nx + 1, g, same);
    slope = slope_n;
    if (g != gn) {
      of_head(g);
      slope = slope_of(g);
    }
    if (g < G) fill(q0s, g0s, ls0, dl0, sg0, qb * kRows);
    tile(q1s, g1s, ls1, dl1, sg1, nx, gn, slope_n, same_n);
  }

  if constexpr (kSplit == 2) {
    // (Each group's sums take a tile's room, dk's and dv's one after the other.)
    float* const at = reinterpret_cast<float*>(group == 0 ? fq0 : group == 1 ? fq1 : group == 2 ? fg0 : fg1);
    if (part) put<DB>(at, dk_acc, lane);
    __syncthreads();
    if (!part) add<DB>(dk_acc, at, lane);
    __syncthreads();
    if (part) put<DB>(at, dv_acc, lane);
    __syncthreads();
    if (part) return;
    add<DB>(dv_acc, at, lane);
  }
  if (my_k < S) {
    const float bad = spoilt ? __builtin_nanf("") : 1.0f;
    const float f = bad * (kCap ? 4.0f * scale : scale);
    if (parts > 1) {
      const size_t rows = (size_t)B * Hk * parts * S, row = (size_t)bh * S + my_k;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d0 = 32 * db + 8 * r + 4 * hl;
          if (d0 >= dim) continue;
          f32x4 k4, v4;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            k4[t] = dk_acc[db][4 * r + t] * f;
            v4[t] = dv_acc[db][4 * r + t] * bad;
          }
          *reinterpret_cast<f32x4*>(partial + row * dim + d0) = k4;
          *reinterpret_cast<f32x4*>(partial + (rows + row) * dim + d0) = v4;
        }
      return;
    }
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

// dk and dv from the parts' sums: a thread adds 8 columns of one row of either, the parts in order.
__global__ void __launch_bounds__(256) scored_join_kernel(const float* __restrict__ partial, int parts, MutView dK,
                                                          MutView dV, int B, int Hk, int S, int dim) {
  const int per = dim / 8;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)B * Hk * S;
  const bool values = t >= rows * per;
  const int64_t u = values ? t - rows * per : t;
  if (u >= rows * per) return;
  const int64_t row = u / per;
  const int c = 8 * (int)(u % per), s = (int)(row % S), bh = (int)(row / S);
  f32x4 lo = f32x4{}, hi = f32x4{};
  for (int p = 0; p < parts; ++p) {
    const float* at = partial + ((values ? rows * parts : 0) + ((int64_t)bh * parts + p) * S + s) * dim + c;
    lo += *reinterpret_cast<const f32x4*>(at);
    hi += *reinterpret_cast<const f32x4*>(at + 4);
  }
  const bf16x8 o = {(bf16)lo[0], (bf16)lo[1], (bf16)lo[2], (bf16)lo[3],
                    (bf16)hi[0], (bf16)hi[1], (bf16)hi[2], (bf16)hi[3]};
  *reinterpret_cast<bf16x8*>((values ? dV : dK).row(bh / Hk, bh % Hk, s) + c) = o;
}

size_t row_numbers_bytes(int batch, int heads, int seq) {
  return ((size_t)batch * heads * seq * sizeof(float) + 255) & ~(size_t)255;
}

}  // namespace

extern "C" {

size_t gptrig_scored_attn_bwd_workspace_bytes(int batch, int heads, int kv_heads, int seq, int head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq <= 0 || head_dim <= 0) return 0;
  const int parts = Blocks(batch, heads, kv_heads, seq, head_dim).parts;
  const size_t sums = parts > 1 ? (size_t)2 * batch * kv_heads * parts * seq * head_dim * sizeof(float) : 0;
  return 2 * row_numbers_bytes(batch, heads, seq) + sums;
}

int gptrig_scored_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout,
                           const void* o_low, const float* lse2, const int32_t* segment_ids, const int32_t* prefix_lengths,
                           const float* distance_slopes, const void* plan, void* dq, void* dk, void* dv, void* workspace,
                           size_t workspace_bytes, int batch, int heads, int kv_heads, int seq, int head_dim,
                           const int64_t* strides, float softmax_scale, float score_cap, void* stream) {
  ScoredCall c;
  if (!lse2 || !o_low || !workspace) return GPTRIG_E_NULL;
  const void* tensors[8] = {q, k, v, o, dout, dq, dk, dv};
  const int status = c.init(tensors, 8, 0b11000110u, batch, heads, kv_heads, seq, head_dim, strides, softmax_scale,
                            score_cap, distance_slopes, prefix_lengths);
  if (status != GPTRIG_OK) return status;
  if (workspace_bytes < gptrig_scored_attn_bwd_workspace_bytes(batch, heads, kv_heads, seq, head_dim))
    return GPTRIG_E_WORKSPACE;
  if (((uintptr_t)workspace | (uintptr_t)o_low | (uintptr_t)plan) & 15) return GPTRIG_E_SHAPE;
  const Blocks blocks(batch, heads, kv_heads, seq, head_dim);
  const bool split = blocks.row_split, kv_split = blocks.key_split;
  const int parts = blocks.parts, row_blocks = ceil_div(seq, blocks.rows);
  const unsigned grid = (unsigned)(batch * heads * row_blocks);
  const unsigned kv_grid = (unsigned)(batch * kv_heads * parts * ceil_div(seq, blocks.keys));
  if (!gptrig_scored_attn_plan_bytes(batch, heads, kv_heads, seq, head_dim)) plan = nullptr;
  const int* const row_plan = (const int*)plan;
  const int* const key_plan = plan ? row_plan + batch * row_blocks : nullptr;
  hipStream_t s = (hipStream_t)stream;
  const View Q = c.view(0), K = c.view(1), V = c.view(2), O = c.view(3), dO = c.view(4);
  const MutView dQ = c.out(5), dK = c.out(6), dV = c.out(7);
  float* const shifts = (float*)workspace;
  float* const minus_delta = shifts + row_numbers_bytes(batch, heads, seq) / sizeof(float);
  float* const partial = minus_delta + row_numbers_bytes(batch, heads, seq) / sizeof(float);
#define SCORED_DQ(D, CAP, BIAS, SEG, SPLIT)                                                                          \
  scored_dq_kernel<D, CAP, BIAS, SEG, SPLIT><<<grid, 256, 0, s>>>(                                         \
      Q, K, V, O, dO, (const uint8_t*)o_low, lse2, segment_ids, row_plan, shifts, minus_delta, dQ, c.args, batch, heads, \
      kv_heads, seq, head_dim, softmax_scale)
#define SCORED_DKV(D, CAP, BIAS, SEG, SPLIT, WAVES)                                                                  \
  scored_dkv_kernel<D, CAP, BIAS, SEG, SPLIT, WAVES><<<kv_grid, 64 * WAVES, 0, s>>>(                                 \
      Q, K, V, dO, shifts, minus_delta, segment_ids, key_plan, dK, dV, partial, parts, c.args, batch, heads, kv_heads, seq,    \
      head_dim, softmax_scale)
#define SCORED_BWD(D, CAP, BIAS, SEG)                                           \
  if (split) SCORED_DQ(D, CAP, BIAS, SEG, 2);                                   \
  else SCORED_DQ(D, CAP, BIAS, SEG, 1);                                         \
  if (kv_split) SCORED_DKV(D, CAP, BIAS, SEG, 2, 4);                            \
  else SCORED_DKV(D, CAP, BIAS, SEG, (D == 64 ? 1 : 2), (D == 64 ? 4 : 8))
  SCORED_DISPATCH(SCORED_BWD, c, segment_ids != nullptr);
#undef SCORED_BWD
#undef SCORED_DKV
#undef SCORED_DQ
  if (parts > 1) {
    const long long threads = 2ll * batch * kv_heads * seq * (head_dim / 8);  // (of fewer than kWant blocks)
    scored_join_kernel<<<ceil_div(threads, 256), 256, 0, s>>>(partial, parts, dK, dV, batch, kv_heads, seq, head_dim);
  }
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

}  // extern "C"
