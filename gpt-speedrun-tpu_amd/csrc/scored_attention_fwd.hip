// Forward of the attention of scored_attention.h.  A workgroup owns 128 queries
// of one head (4 waves x 32) and walks the tiles of 64 keys that any of them can
// see.  Each wave computes S^T = K Q^T, so a lane holds one query and 16 of 32
// keys: the softmax is lane-local but for one exchange between the half-waves,
// and P^T is already the operand of o^T = V^T P^T.
//
// Bound by vector operations, not by the products: a pair of the capped score costs
// two exponentials, a reciprocal and six or seven others against 4 D operations of the matrix
// cores.  Times of the kernel alone, in a loop of passes on the same inputs: B16 H12
// S1024 D64, cap 30: 63 us, of a CU's busy time 76% vector and 19% matrix
// instructions, and 18% of the time without work at the start and the end (four waves a
// SIMD instead of three take as long); B4 H16/4 S2048 D128, cap and bias: 123 us (65%
// and 24%; two waves a SIMD).  At D = 64 three workgroups share a CU (168 registers).
#include "scored_attention.h"

namespace {

constexpr int kQueries = 128;  // of a workgroup; kSplit 2: 64

// With a prefix or documents the blocks of a call are of very uneven length, and
// long ones that start last keep a few CUs busy alone: so their order is planned,
// the longest first, in a launch of its own.  Blocks of the same 1/512 of the longest
// possible are in any order; nothing but the time depends on it.
constexpr int kPlanItems = 2048, kPlanBuckets = 512;
struct Plan {
  int blocks[2], size[2];  // rows (0) and keys (1): blocks of a sequence, positions of one
};
// Workgroup 0 orders the blocks of rows, workgroup 1 those of keys: their lengths in
// tiles, counted from the lowest and highest id of each tile where there are
// documents, sorted by counting.
__global__ void __launch_bounds__(1024) scored_plan_kernel(const int32_t* __restrict__ seg,
                                                           const int32_t* __restrict__ prefix, int* __restrict__ plan,
                                                           Plan sizes, int B, int S) {
  __shared__ int lowest[kPlanItems], highest[kPlanItems], length[kPlanItems], count[kPlanBuckets];
  const int which = blockIdx.x, tid = threadIdx.x;
  const int tiles = (S + kRows - 1) / kRows, blocks = sizes.blocks[which], size = sizes.size[which];
  const int items = B * blocks;
  if (which) plan += B * sizes.blocks[0];
  for (int i = tid; i < kPlanBuckets; i += 1024) count[i] = 0;
  const int l16 = tid & 15;  // 16 lanes a tile, and then a block
  if (seg)
    for (int i = tid >> 4; i < B * tiles; i += 64) {
      const int32_t* const ids = seg + (size_t)(i / tiles) * S;
      int id[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) id[j] = ids[min(i % tiles * kRows + 16 * j + l16, S - 1)];
      int lo = min(min(id[0], id[1]), min(id[2], id[3])), hi = max(max(id[0], id[1]), max(id[2], id[3]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
      }
      if (l16 == 0) {
        lowest[i] = lo;
        highest[i] = hi;
      }
    }
  __syncthreads();
  for (int i = tid >> 4; i < items; i += 64) {
    const int b = i / blocks, at = i % blocks * size, own = at / kRows, after = min(at + size, S);
    const int p = prefix ? min(max(prefix[b], 0), S) : 0;
    const int from = which == 0 || at < p ? 0 : own;
    const int to = which ? tiles : (max(after, p) + kRows - 1) / kRows;
    int n = to - from;
    if (seg) {
      const int* const lo = lowest + b * tiles;
      const int* const hi = highest + b * tiles;
      const int last = (after - 1) / kRows, low = min(lo[own], lo[last]), high = max(hi[own], hi[last]);
      n = 0;
#pragma unroll 4
      for (int t = from + l16; t < to; t += 16) n += lo[t] <= high && hi[t] >= low;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) n += __shfl_xor(n, o);
    }
    if (l16 == 0) {
      length[i] = (int)((long long)(tiles - n) * (kPlanBuckets - 1) / tiles);
      atomicAdd(&count[length[i]], 1);
    }
  }
  __syncthreads();
  if (tid < 64) {  // the first place of each bucket
    int sum = 0;
    for (int i = 0; i < kPlanBuckets / 64; ++i) sum += count[tid * (kPlanBuckets / 64) + i];
    int place = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(place, o);
      if (tid >= o) place += below;
    }
    place -= sum;
    for (int i = 0; i < kPlanBuckets / 64; ++i) {
      const int n = count[tid * (kPlanBuckets / 64) + i];
      count[tid * (kPlanBuckets / 64) + i] = place;
      place += n;
    }
  }
  __syncthreads();
  for (int i = tid; i < items; i += 1024) plan[atomicAdd(&count[length[i]], 1)] = i;
}

template <int D, bool kCap, bool kBias, bool kSeg, int kSplit>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2)
    scored_fwd_kernel(View Q, View K, View V, MutView O, uint8_t* __restrict__ o_low, float* __restrict__ lse2,
                      const int32_t* __restrict__ seg, const int* __restrict__ plan, ScoreArgs a, int B, int H, int Hk,
                      int S, int dim) {
  constexpr int KC = D / 16, DB = D / 32;
  // Without a bias s stays the raw product or, with a cap, its w: the softmax scales it.
  constexpr bool kRaw = !kCap && !kBias, kW = kCap && !kBias;
  constexpr float kHidden = kW ? INFINITY : -INFINITY;  // (a score falls with w)
  __shared__ __attribute__((aligned(16))) bf16 fk0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fk1[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv0[kRows * D];
  __shared__ __attribute__((aligned(16))) bf16 fv1[kRows * D];
  __shared__ __attribute__((aligned(16))) int sg0[kRows], sg1[kRows];

  constexpr int kMine = kQueries / kSplit;
  const int nq = (S + kMine - 1) / kMine;
  int bh, qb;
  block_of(plan, blockIdx.x, nq, B, H, true, bh, qb);
  const int b = bh / H, h = bh % H, hk = h / (H / Hk);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  // Two waves share 32 queries where kSplit is 2, each with one half of every tile.
  const int own = wave % (4 / kSplit), part = wave / (4 / kSplit);
  const int q0 = qb * kMine, qw0 = q0 + 32 * own, my_q = qw0 + l32;
  const int last_prefix = __builtin_amdgcn_readfirstlane(prefix_of(a, b, S)) - 1;
  const int my_last = min(max(my_q, last_prefix), S - 1);  // the last key this lane's query may see
  const int wave_last = max(qw0 + 31, last_prefix);
  const int ntiles = max(min(q0 + kMine, S) - 1, last_prefix) / kRows + 1;
  const float slope2 = kBias ? a.slopes[h] * GPTRIG_LOG2E : 0.f;

  float bias[16];  // of a key acc_row(i) after element 0's
  // (An instruction reads one scalar register: the bias's, so the factors are vectors.)
  float raw = a.raw, twice = -2.0f * a.cap2;
  if constexpr (kBias) {
    row_bias(bias, slope2);
    asm("" : "+v"(raw), "+v"(twice));
  }

  bf16x8 qreg[KC];
#pragma unroll
  for (int kc = 0; kc < KC; ++kc)
    qreg[kc] = my_q < S && 16 * kc + 8 * hl < dim
                   ? *reinterpret_cast<const bf16x8*>(Q.row(b, h, my_q) + 16 * kc + 8 * hl) : bf16x8{};
  const int seg_q = kSeg ? seg[(size_t)b * S + min(my_q, S - 1)] : 0;
  WaveIds ids;
  __shared__ uint64_t scan_s[2];
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
  float m_run = kMinusBig, l_run = 0.f, r_run = 0.f;  // r: the sum of the rounded P

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

  // One half of a tile, keys kh0 .. kh0 + 31.  docs: ids have to be compared.
  auto half = [&](const at64::lds_t* kt, const at64::lds_t* vt, const int* sg, int kv0, int sb,
                  int docs) __attribute__((always_inline)) {
    const uint32_t at = 32 * kRowBytes * sb;
    bf16x8 kr[KC];
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) kr[kc] = row_operand(kt, lanes, at, kc);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 s = f32x16{};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) s = mfma32(kr[kc], qreg[kc], s);
    Columns<DB> vc;
    vc.load(vt, lanes, at);
    __builtin_amdgcn_sched_barrier(0);
    const int kh0 = kv0 + 32 * sb;
    // Scores less `off`, which is the same for all of a lane's keys: what a score
    // has in common with the others of its query costs no operation here.
    float off = kCap ? a.cap2 : 0.f;
    if constexpr (!kRaw) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (kCap) {
          const float w = cap_w(s[i], a);
          s[i] = kBias ? fmaf(twice, w, bias[i]) : w;
        } else {
          s[i] = fmaf(s[i], raw, bias[i]);
        }
      }
      if constexpr (kBias) off = fmaf(-slope2, (float)(my_q - kh0 - 4 * hl), off);  // element 0's
    }
    const bool after = kh0 + 31 > qw0;  // some key comes after some query
    if constexpr (kBias) {
      // The distance of such a pair counts the other way.
      if (kh0 > qw0 + 31) {  // all of them
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fmaf(-2.0f, bias[i], s[i]);
        off = fmaf(2.0f * slope2, (float)(my_q - kh0 - 4 * hl), off);
      } else if (after && last_prefix > qw0) {
        const float x = (float)(my_q - kh0 - 4 * hl);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fmaf(-2.0f * slope2, fmaxf((float)acc_row(i) - x, 0.f), s[i]);
      }
    }
    if ((after && kh0 + 31 > last_prefix) || kh0 + 32 > S || (kSeg && docs)) {
      const int lim = my_last - kh0 - 4 * hl;
      if (kSeg && docs) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const i32x4 id = *reinterpret_cast<const i32x4*>(sg + 32 * sb + 8 * r + 4 * hl);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            s[4 * r + t] = acc_row(4 * r + t) <= lim && id[t] == seg_q ? s[4 * r + t] : kHidden;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = acc_row(i) <= lim ? s[i] : kHidden;
      }
    }
    float m_tile = kHidden;
#pragma unroll
    for (int i = 0; i < 16; ++i) m_tile = kW ? fminf(m_tile, s[i]) : fmaxf(m_tile, s[i]);
    if constexpr (kRaw) m_tile *= a.raw;  // (raw > 0)
    if constexpr (kW) m_tile *= twice;
    m_tile += off;  // (with a bias each half-wave has its own)
    m_tile = max_halves(m_tile);
    // (With a cap a fixed reference would do, at 1% less time; but the largest P of a
    // row is then no power of two, and its rounding adds a fifth to the error of o and,
    // through delta, 4 to 13% to that of dq and dk.)
    // The running maximum moves only when a row's maximum exceeds it by more
    // than 8 (log2): P stays below 2^8 and most halves rescale nothing.
    const bool grow = m_tile > m_run + 8.0f;
    const float m_new = grow ? m_tile : m_run;
    if (__ballot(grow)) {
      const float alpha = fast_exp2(m_run - m_new);
      l_run *= alpha;
      r_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
    }
    m_run = m_new;
    const float shift = off - m_new;
    bf16x8 pb[2];
    float lsum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = fast_exp2(kRaw ? fmaf(s[i], a.raw, shift) : kW ? fmaf(s[i], twice, shift) : s[i] + shift);
      lsum += p;
      pb[i >> 3][i & 7] = (bf16)p;
    }
    l_run += lsum;
    r_run = sum_of(pb, r_run);
    vc.product(acc, pb);
  };

  // Infinities and NaN of visible v rows in tiles that clear() changed: a bit per
  // accumulator element, for +inf and for -inf (both: NaN).
  __shared__ uint64_t dirty_s[4];
  uint64_t plus = 0, minus = 0;
  auto clean = [&](at64::lds_t* vt, const int* sg, int kv0, bool same) {
    const Dirty<D> dirty{dirty_s};
    if (!dirty.find(vt, wave, lane)) return;
#pragma unroll 1
    for (int r = 0; r < kRows; ++r) {
      if (!__builtin_amdgcn_readfirstlane(dirty.row(r))) continue;
      bool vis = kv0 + r <= my_last;
      if (kSeg && !same) vis = vis && sg[r] == seg_q;
#pragma unroll 1
      for (int e = 0; e < 16 * DB; ++e) {
        const int col = 32 * (e >> 4) + acc_row(e & 15) + 4 * hl;
        const float v = (float)*(vt + tile_at(r, col >> 3) + (col & 7));
        if (vis && !(v < INFINITY)) plus |= 1ull << e;    // (+inf or NaN)
        if (vis && !(v > -INFINITY)) minus |= 1ull << e;
      }
    }
    dirty.clear(vt, wave, lane);
  };

  // Tile `it` from (kt, vt, sg), the next one, nx, on its way to (nkt, nvt, nsg).
  // The halves and the two tiles of the loop below stand in loops without other
  // exits: acc then has one place (conditional copies of it cost a quarter of the
  // vector instructions and spilled).
  auto tile = [&](const at64::lds_t* kt, at64::lds_t* vt, const int* sg, at64::lds_t* nkt, at64::lds_t* nvt, int* nsg,
                  int it, int nx, bool same) __attribute__((always_inline)) {
    const int kv0 = it * kRows;
    int sb = 0, end = 0, docs = 0;
    if (it < ntiles) {
      if (nx < ntiles) fill(nkt, nvt, nsg, nx * kRows);
      if (kv0 + kRows - 1 > max(q0, last_prefix) || (kSeg && !same)) clean(vt, sg, kv0, same);
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
  while (it < ntiles) {  // (A workgroup's own positions hold visible pairs: there is a first tile.)
    const int nx = next(it + 1, same_n);
    tile(k0s, v0s, sg0, k1s, v1s, sg1, it, nx, same);
    it = next(nx + 1, same);
    tile(k1s, v1s, sg1, k0s, v0s, sg0, nx, it, same_n);
  }

  if constexpr (kSplit == 2) {  // the second half's sums join the first's
    __shared__ float ml[2][3][64];
    float* const at = reinterpret_cast<float*>(own ? fv0 : fk0);  // a tile's room is an accumulator's
    if (part) {
      ml[own][0][lane] = m_run;
      ml[own][1][lane] = l_run;
      ml[own][2][lane] = r_run;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) at[(16 * db + i) * 64 + lane] = acc[db][i];
    }
    __syncthreads();
    if (part) return;
    const float m1 = ml[own][0][lane], m = fmaxf(m_run, m1);
    const float f0 = fast_exp2(m_run - m), f1 = fast_exp2(m1 - m);
    m_run = m;
    l_run = l_run * f0 + ml[own][1][lane] * f1;
    r_run = r_run * f0 + ml[own][2][lane] * f1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = acc[db][i] * f0 + at[(16 * db + i) * 64 + lane] * f1;
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32), r_tot = r_run + __shfl_xor(r_run, 32);
  if (__ballot((plus | minus) != 0)) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool p = plus >> (16 * db + i) & 1, m = minus >> (16 * db + i) & 1;
        if (p || m) acc[db][i] += p && m ? __builtin_nanf("") : p ? INFINITY : -INFINITY;
      }
  }
  if (my_q < S) {
    // Over the sum of the P that the product took: their roundings weigh against each
    // other instead of scaling o (of few visible keys one rounding is all of it).
    const float inv = 1.0f / r_tot;
    bf16* orow = O.row(b, h, my_q);
    uint8_t* const low_row = o_low ? o_low + (((size_t)b * H + h) * S + my_q) * dim : nullptr;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d0 = 32 * db + 8 * r + 4 * hl;
        if (d0 >= dim) continue;
        bf16x4 o4;
        uint32_t low = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float x = acc[db][4 * r + t] * inv;
          o4[t] = (bf16)x;
          low |= low_bits(x, o4[t]) << (8 * t);
        }
        *reinterpret_cast<bf16x4*>(orow + d0) = o4;
        if (low_row) *reinterpret_cast<uint32_t*>(low_row + d0) = low;
      }
    if (hl == 0 && lse2) lse2[((size_t)b * H + h) * S + my_q] = m_run + __log2f(l_tot);
  }
}

}  // namespace

extern "C" {

size_t gptrig_scored_attn_plan_bytes(int batch, int heads, int kv_heads, int seq, int head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq <= 0 || head_dim <= 0) return 0;
  const Blocks k(batch, heads, kv_heads, seq, head_dim);
  const long long rows = (long long)batch * ceil_div(seq, k.rows), keys = (long long)batch * ceil_div(seq, k.keys);
  // (Where every workgroup starts at once their order matters little.)  The plan costs 4
  // to 8 us a call.  us forward and backward with / without, H12 D64 biased: documents
  // of 1500 B1 S8192 403 / 421, B2 493 / 572; of 700 B8 S4096 674 / 773; of 200 B16 S1024
  // 251 / 247; prefixes B2 S2000 169 / 180, B4 247 / 290.
  if ((long long)batch * ceil_div(seq, kRows) > kPlanItems || rows * heads <= 512) return 0;
  return (size_t)(rows + keys) * sizeof(int);
}

int gptrig_scored_attn_plan(const int32_t* segment_ids, const int32_t* prefix_lengths, void* plan, size_t plan_bytes,
                            int batch, int heads, int kv_heads, int seq, int head_dim, void* stream) {
  const size_t need = gptrig_scored_attn_plan_bytes(batch, heads, kv_heads, seq, head_dim);
  if (!need) return GPTRIG_E_SHAPE;
  if (!plan) return GPTRIG_E_NULL;
  if (plan_bytes < need) return GPTRIG_E_WORKSPACE;
  if ((uintptr_t)plan & 15) return GPTRIG_E_SHAPE;
  const Blocks k(batch, heads, kv_heads, seq, head_dim);
  const Plan sizes = {{ceil_div(seq, k.rows), ceil_div(seq, k.keys)}, {k.rows, k.keys}};
  scored_plan_kernel<<<2, 1024, 0, (hipStream_t)stream>>>(segment_ids, prefix_lengths, (int*)plan, sizes, batch, seq);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

int gptrig_scored_attn_fwd(const void* q, const void* k, const void* v, const int32_t* segment_ids,
                           const int32_t* prefix_lengths, const float* distance_slopes, const void* plan,
                           void* o, void* o_low, float* lse2, int batch, int heads, int kv_heads, int seq, int head_dim,
                           const int64_t* strides, float softmax_scale, float score_cap, void* stream) {
  ScoredCall c;
  if (((uintptr_t)o_low | (uintptr_t)plan) & 15) return GPTRIG_E_SHAPE;
  const void* tensors[4] = {q, k, v, o};
  const int status = c.init(tensors, 4, 0b0110u, batch, heads, kv_heads, seq, head_dim, strides, softmax_scale,
                            score_cap, distance_slopes, prefix_lengths);
  if (status != GPTRIG_OK) return status;
  hipStream_t s = (hipStream_t)stream;
  const View Q = c.view(0), K = c.view(1), V = c.view(2);
  const MutView O = c.out(3);
  const Blocks blocks(batch, heads, kv_heads, seq, head_dim);
  if (!gptrig_scored_attn_plan_bytes(batch, heads, kv_heads, seq, head_dim)) plan = nullptr;
  const unsigned grid = (unsigned)(batch * heads * ceil_div(seq, blocks.rows));
#define SCORED_FWD_(D, CAP, BIAS, SEG, SPLIT)                                                                       \
  scored_fwd_kernel<D, CAP, BIAS, SEG, SPLIT><<<grid, 256, 0, s>>>(Q, K, V, O, (uint8_t*)o_low, lse2, segment_ids,  \
                                                                   (const int*)plan, c.args, batch, heads, kv_heads, seq, head_dim)
#define SCORED_FWD(D, CAP, BIAS, SEG)            \
  if (blocks.row_split) SCORED_FWD_(D, CAP, BIAS, SEG, 2); \
  else SCORED_FWD_(D, CAP, BIAS, SEG, 1)
  SCORED_DISPATCH(SCORED_FWD, c, segment_ids != nullptr);
#undef SCORED_FWD
#undef SCORED_FWD_
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

}  // extern "C"
