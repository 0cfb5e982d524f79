// One AdamW step over a list of tensors, each with memory of its own.  Per
// element, in float32 with the scalars rounded from double:
//   g = grad clip;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p -= lr lr_mult ((m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps) + decay p)
// with {lr_mult, eps, decay} from the tensor's row of hparams.  Moments are
// float32 or 8 bits.
//
// 8-bit moments: e4m3 codes with a float32 scale per 256 consecutive values of a
// tensor (the last block may be shorter); a value is code x scale, scale = the
// block's largest finite magnitude / 448.  The step itself uses the new moments
// before they are rounded; only what is kept for the next step is.
// With three mantissa bits a moving average that is rounded to nearest stands
// still: v's decay of 1 - b2 = 5% a step is less than half of the 6 to 12%
// between neighbouring codes, so v could grow but not shrink.  Each magnitude y =
// |value| / scale is therefore rounded down after adding a random share u of its
// step, which is right on average:
//   code = step floor(y / step + u),  step = 2^(max(floor(log2 y), -6) - 3)
// A v above zero keeps at least the smallest code, 2^-9: a v of zero beside a
// momentum that is not would divide by eps alone.  A value that is infinite or NaN
// becomes the NaN code and stays out of the scale, so it spoils no neighbour.
// Blocks of m whose largest magnitude is below 2^-100 are kept as zeros, and blocks of
// v from 2^-117 down (v is a square; a scale below that is no normal float32).  So that
// no step divides by eps alone, a v of such a block with a momentum counts as 2^-117
// in the next step, and a new v of 0 as 2^-149: the most that was cut off.
// Every product, sum and quotient up to a code is rounded to float32 on its own (no
// fused ones): a value close to a tie goes to either of two codes 12% apart, so the
// last bit decides a few codes of a million, and anyone who computes the formula in
// float32 gets the same ones.
// u comes from 32 bits h(seed, tensor, i), m's from the low half, v's from the
// high one, (half + 0.5) / 2^16.  h is a multiply and shift mixer over the
// fractional bits of the golden ratio, sqrt 2 and sqrt 3:
//   mix(x): x ^= x >> 16; x *= R2; x ^= x >> 15; x *= R3; x ^= x >> 16
//   h = mix(i PHI + mix(mix(seed) + tensor PHI) + (i >> 32) R3)
// A captured graph replays the same scalars, so a seed among them would give every
// replay the same u: an element would then stand still or decay for good, as without
// any.  There the seed is read from device memory.
#include "common.h"

#include <math.h>
#include <stdlib.h>

#include <algorithm>

namespace {

constexpr uint32_t kPhi = 0x9E3779B9u, kR2 = 0x6A09E667u, kR3 = 0xBB67AE85u;
constexpr int kMost = 48;      // tensors a launch: their table travels as a kernel argument of 3.5 KB
constexpr int kBlock = 256;    // values a scale
constexpr int kUnroll = 4;     // blocks a wave has in flight (2: the same time, 8: 2% more, 12% with 8 bits)
constexpr int kChunk = 4 * kUnroll * kBlock;  // values a workgroup
constexpr float kTinyM = 0x1p-100f, kTinyV = 0x1p-117f;

struct Item {
  float* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  bf16* shadow;
  int64_t n;
  int first;  // the tensor's first workgroup
  int index;  // its place in the caller's list
};
struct Items {
  Item item[kMost];
  int count;
};
struct Scalars {
  float lr, b1, omb1, b2, omb2, ibc1, ibc2;  // ibc: 1 / (1 - beta^step)
  uint32_t seed;  // mix(seed)
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= kR2;
  x ^= x >> 15;
  x *= kR3;
  return x ^ (x >> 16);
}

// Four values from a place aligned as one of them; kWhole: all four exist.
template <typename T>
struct __attribute__((packed)) Four {
  T v[4];
};
template <bool kWhole, typename T>
__device__ __forceinline__ void load4(float (&out)[4], const T* __restrict__ at, int left) {
  if (kWhole || left >= 4) {
    const Four<T> f = *reinterpret_cast<const Four<T>*>(at);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = (float)f.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = j < left ? (float)at[j] : 0.f;
  }
}
template <bool kWhole, typename T>
__device__ __forceinline__ void store4(T* __restrict__ at, const float (&v)[4], int left) {
  if (kWhole || left >= 4) {
    Four<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = (T)v[j];
    *reinterpret_cast<Four<T>*>(at) = f;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) at[j] = (T)v[j];
  }
}

struct __attribute__((packed)) Codes {
  uint32_t v;
};
template <bool kWhole>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* __restrict__ at, int left) {
  if (kWhole || left >= 4) return reinterpret_cast<const Codes*>(at)->v;
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) c |= j < left ? (uint32_t)at[j] << (8 * j) : 0u;
  return c;
}
template <bool kWhole>
__device__ __forceinline__ void store_codes(uint8_t* __restrict__ at, uint32_t c, int left) {
  if (kWhole || left >= 4) {
    reinterpret_cast<Codes*>(at)->v = c;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) at[j] = (uint8_t)(c >> (8 * j));
}
__device__ __forceinline__ void decode(float (&out)[4], uint32_t c, float scale) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  out[0] = a[0] * scale;
  out[1] = a[1] * scale;
  out[2] = b[0] * scale;
  out[3] = b[1] * scale;
}

// The largest of the wave's values (none negative or NaN), without LDS.
__device__ __forceinline__ float largest(float v) {
#define FOLD(ctrl)                                                                                                \
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), \
                                                                     ctrl, 0xF, 0xF, false)));
  FOLD(0xB1)   // quads, then half rows, rows, and row 15 / 31 on to the rows above
  FOLD(0x4E)
  FOLD(0x141)
  FOLD(0x140)
  FOLD(0x142)
  FOLD(0x143)
#undef FOLD
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// The codes of a lane's four values of a block that the wave holds, and the
// block's scale.  shift: where the random half-words are.
template <bool kFloor>
__device__ __forceinline__ uint32_t encode(const float (&x)[4], const uint32_t (&bits)[4], int shift, float& scale) {
#pragma clang fp contract(off)
  float top = 0.f;
  bool finite[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    finite[j] = fabsf(x[j]) <= 3.402823466e38f;
    top = finite[j] ? fmaxf(top, fabsf(x[j])) : top;
  }
  top = largest(top);
  const bool none = top < (kFloor ? kTinyV : kTinyM);
  scale = none ? 0.f : top * (1.0f / 448.0f);
  const float inv = none ? 0.f : 1.0f / scale;
  float code[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // |x| / scale, correctly rounded (for a v below 2^-100 to the last bit or two).
    const float q = fabsf(x[j]) * inv, y = fminf(fmaf(fmaf(-q, scale, fabsf(x[j])), inv, q), 448.0f);
    uint32_t step = __builtin_bit_cast(uint32_t, y) & 0x7F800000u;
    step = (step < 0x3C800000u ? 0x3C800000u : step) - 0x01800000u;  // at least 2^-6, over 8
    const float u = fmaf((float)((bits[j] >> shift) & 0xFFFFu), 0x1p-16f, 0x1p-17f);
    float c = floorf(fmaf(y, __builtin_bit_cast(float, 0x7F000000u - step), u)) * __builtin_bit_cast(float, step);
    if (kFloor) c = y > 0.f ? fmaxf(c, 0x1p-9f) : c;
    c = finite[j] ? c : __builtin_nanf("");
    code[j] = kFloor ? c : copysignf(c, x[j]);
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(code[0], code[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(code[2], code[3], w, true);
  return (uint32_t)w;
}

// One chunk of a tensor.  Bound by HBM: 229M parameters with float32 moments and
// gradients (6.4 GB) 1200 us, 5.4 TB/s, the rate of a large copy.  8-bit moments
// (3.7 GB) 685 us, 5.4 TB/s, with about 100 vector operations an element (the hash
// 10, each encoding 20), a little less than the time of their 16 bytes.  So the square
// root and the reciprocal of the step are the instructions of one unit in the last
// place, the root of a small v taken of 2^24 times it (the instruction does not take
// denormals).
template <typename G, bool k8, bool kWhole>
__device__ __forceinline__ void update_chunk(const Item& it, const Scalars& k, float lr, float eps, float decay,
                                             float clip, int64_t base) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = it.n;
  float* const p = it.p;
  const G* const g = (const G*)it.g;
  float pv[kUnroll][4], gv[kUnroll][4], mv[kUnroll][4], vv[kUnroll][4];
  uint32_t mc[kUnroll], vc[kUnroll];
  float ms[kUnroll], vs[kUnroll];
  auto block_of = [&](int u) { return base + (wave + 4 * u) * kBlock; };
  auto left_of = [&](int64_t at) { return kWhole ? 4 : (int)(n - at < 4 ? (n - at < 0 ? 0 : n - at) : 4); };
  // Every load of the chunk before the first use.
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t block = block_of(u), at = block + 4 * lane;
    const int left = left_of(at);
    load4<kWhole, float>(pv[u], p + at, left);
    load4<kWhole, G>(gv[u], g + at, left);
    if constexpr (k8) {
      mc[u] = load_codes<kWhole>((const uint8_t*)it.m + at, left);
      vc[u] = load_codes<kWhole>((const uint8_t*)it.v + at, left);
      ms[u] = kWhole || block < n ? it.ms[block / kBlock] : 0.f;
      vs[u] = kWhole || block < n ? it.vs[block / kBlock] : 0.f;
    } else {
      load4<kWhole, float>(mv[u], (const float*)it.m + at, left);
      load4<kWhole, float>(vv[u], (const float*)it.v + at, left);
    }
  }
  const uint32_t key = k8 ? mix(k.seed + (uint32_t)it.index * kPhi) + (uint32_t)(base >> 32) * kR3 : 0u;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t block = block_of(u), at = block + 4 * lane;
    if (!kWhole && block >= n) break;  // (the whole wave)
    const int left = left_of(at);
    if constexpr (k8) {
      decode(mv[u], mc[u], ms[u]);
      decode(vv[u], vc[u], vs[u]);
      if (vs[u] == 0.f)  // (the whole wave)
#pragma unroll
        for (int j = 0; j < 4; ++j) vv[u][j] = vv[u][j] == 0.f && mv[u][j] != 0.f ? kTinyV : vv[u][j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = gv[u][j] * clip;
      const float m = k.b1 * mv[u][j] + k.omb1 * gj;
      const float v = k.b2 * vv[u][j] + k.omb2 * gj * gj;
      const float vhat = (k8 && v == 0.f ? 0x1p-149f : v) * k.ibc2;
      const bool small = vhat < 1.0f;
      const float root = __builtin_amdgcn_sqrtf(vhat * (small ? 0x1p24f : 1.0f));
      const float step = (m * k.ibc1) * __builtin_amdgcn_rcpf(fmaf(root, small ? 0x1p-12f : 1.0f, eps));
      pv[u][j] = fmaf(-lr, fmaf(decay, pv[u][j], step), pv[u][j]);
      // (Past the tensor's end m and v are 0 unless clip is infinite or NaN.)
      mv[u][j] = kWhole || j < left ? m : 0.f;
      vv[u][j] = kWhole || j < left ? v : 0.f;
    }
    store4<kWhole, float>(p + at, pv[u], left);
    if (it.shadow) store4<kWhole, bf16>(it.shadow + at, pv[u], left);
    if constexpr (k8) {
      uint32_t bits[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bits[j] = mix((uint32_t)(at + j) * kPhi + key);  // (a chunk crosses no 2^32)
      const uint32_t m8 = encode<false>(mv[u], bits, 0, ms[u]);
      const uint32_t v8 = encode<true>(vv[u], bits, 16, vs[u]);
      store_codes<kWhole>((uint8_t*)it.m + at, m8, left);
      store_codes<kWhole>((uint8_t*)it.v + at, v8, left);
      if (lane == 0) {
        it.ms[block / kBlock] = ms[u];
        it.vs[block / kBlock] = vs[u];
      }
    } else {
      store4<kWhole, float>((float*)it.m + at, mv[u], left);
      store4<kWhole, float>((float*)it.v + at, vv[u], left);
    }
  }
}

template <typename G, bool k8>
__global__ void __launch_bounds__(256) adamw_tensors_kernel(Items items, Scalars k, const float* __restrict__ hparams,
                                                            const float* __restrict__ clip_scale,
                                                            const int64_t* __restrict__ seed) {
  if (k8 && seed) k.seed = mix((uint32_t)*seed);
  // The tensor of this workgroup: the last whose first workgroup is not after it.
  int lo = 0, hi = items.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int)blockIdx.x >= items.item[mid].first) lo = mid;
    else hi = mid - 1;
  }
  const Item& it = items.item[lo];
  const int64_t base = (int64_t)((int)blockIdx.x - it.first) * kChunk;
  const float lr = k.lr * hparams[3 * it.index], eps = hparams[3 * it.index + 1], decay = hparams[3 * it.index + 2];
  const float clip = clip_scale ? *clip_scale : 1.0f;
  if (base + kChunk <= it.n) update_chunk<G, k8, true>(it, k, lr, eps, decay, clip, base);
  else update_chunk<G, k8, false>(it, k, lr, eps, decay, clip, base);
}

// GPTRIG_E_OVERLAP where an array that the step writes shares memory with another of its arrays.
int check_written(const gptrig_adamw_tensor* tensors, int count, bool k8, size_t grad_bytes) {
  struct Range {
    uintptr_t from, to;
    bool written;
  };
  Range few[7 * 64];
  Range* const r = count <= 64 ? few : (Range*)malloc(sizeof(Range) * 7 * (size_t)count);
  if (!r) return GPTRIG_E_WORKSPACE;
  int n = 0;
  for (int i = 0; i < count; ++i) {
    const gptrig_adamw_tensor& t = tensors[i];
    if (t.n == 0) continue;
    const size_t size = (size_t)t.n, scales = (size_t)((t.n + kBlock - 1) / kBlock) * 4;
    auto put = [&](const void* p, size_t bytes, bool written = true) {
      if (p) r[n++] = {(uintptr_t)p, (uintptr_t)p + bytes, written};
    };
    put(t.grad, grad_bytes * size, false);
    put(t.param, 4 * size);
    put(t.m, (k8 ? 1 : 4) * size);
    put(t.v, (k8 ? 1 : 4) * size);
    put(t.shadow, 2 * size);
    if (k8) {
      put(t.m_scale, scales);
      put(t.v_scale, scales);
    }
  }
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.from < b.from; });
  int status = GPTRIG_OK;
  uintptr_t end = 0, written_end = 0;
  for (int i = 0; i < n; ++i) {
    if (r[i].from < (r[i].written ? end : written_end)) status = GPTRIG_E_OVERLAP;
    end = std::max(end, r[i].to);
    if (r[i].written) written_end = std::max(written_end, r[i].to);
  }
  if (r != few) free(r);
  return status;
}

// seed_at: the seed in device memory, or null for `seed`.
int update(const gptrig_adamw_tensor* tensors, int count, int grad_type, int state_bits, const float* tensor_hparams,
           double lr, double beta1, double beta2, int step, const float* clip_scale, uint32_t seed,
           const int64_t* seed_at, void* stream) {
  if (count < 0 || step <= 0 || !(beta1 >= 0. && beta1 < 1.) || !(beta2 >= 0. && beta2 < 1.)) return GPTRIG_E_SHAPE;
  if (grad_type != GPTRIG_TYPE_BF16 && grad_type != GPTRIG_TYPE_F32) return GPTRIG_E_DTYPE;
  if (state_bits != 8 && state_bits != 32) return GPTRIG_E_UNSUPPORTED;
  if (count == 0) return GPTRIG_OK;
  if (!tensors || !tensor_hparams) return GPTRIG_E_NULL;
  const bool k8 = state_bits == 8;
  for (int i = 0; i < count; ++i) {
    const gptrig_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.n > ((int64_t)1 << 35)) return GPTRIG_E_SHAPE;
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.m || !t.v || (k8 && (!t.m_scale || !t.v_scale))) return GPTRIG_E_NULL;
    const uintptr_t words = (uintptr_t)t.param | (uintptr_t)t.m_scale | (uintptr_t)t.v_scale |
                            (k8 ? 0 : (uintptr_t)t.m | (uintptr_t)t.v);
    if ((words & 3) || ((uintptr_t)t.grad & (grad_type == GPTRIG_TYPE_F32 ? 3 : 1)) || ((uintptr_t)t.shadow & 1))
      return GPTRIG_E_SHAPE;
  }
  const int written = check_written(tensors, count, k8, grad_type == GPTRIG_TYPE_F32 ? 4 : 2);
  if (written != GPTRIG_OK) return written;
  Scalars k;
  k.lr = (float)lr;
  k.b1 = (float)beta1;
  k.omb1 = (float)(1.0 - beta1);
  k.b2 = (float)beta2;
  k.omb2 = (float)(1.0 - beta2);
  k.ibc1 = (float)(1.0 / (1.0 - pow(beta1, (double)step)));
  k.ibc2 = (float)(1.0 / (1.0 - pow(beta2, (double)step)));
  k.seed = mix(seed);
  hipStream_t s = (hipStream_t)stream;
  int i = 0;
  while (i < count) {
    Items items;
    int64_t blocks = 0;
    items.count = 0;
    for (; i < count && items.count < kMost; ++i) {
      const gptrig_adamw_tensor& t = tensors[i];
      if (t.n == 0) continue;
      const int64_t more = (t.n + kChunk - 1) / kChunk;
      if (blocks + more >= 1 << 24) break;  // (2^32 threads; a tensor of 2^35 values, 2^23 chunks, always fits)
      items.item[items.count++] = {t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, (bf16*)t.shadow, t.n, (int)blocks, i};
      blocks += more;
    }
    if (blocks == 0) continue;
    const unsigned grid = (unsigned)blocks;
    if (grad_type == GPTRIG_TYPE_F32) {
      if (k8) adamw_tensors_kernel<float, true><<<grid, 256, 0, s>>>(items, k, tensor_hparams, clip_scale, seed_at);
      else adamw_tensors_kernel<float, false><<<grid, 256, 0, s>>>(items, k, tensor_hparams, clip_scale, seed_at);
    } else {
      if (k8) adamw_tensors_kernel<bf16, true><<<grid, 256, 0, s>>>(items, k, tensor_hparams, clip_scale, seed_at);
      else adamw_tensors_kernel<bf16, false><<<grid, 256, 0, s>>>(items, k, tensor_hparams, clip_scale, seed_at);
    }
    GPTRIG_CHECK_LAUNCH();
  }
  return GPTRIG_OK;
}

}  // namespace

extern "C" {

int gptrig_adamw_tensors(const gptrig_adamw_tensor* tensors, int count, int grad_type, int state_bits,
                         const float* tensor_hparams, double lr, double beta1, double beta2, int step,
                         const float* clip_scale, uint32_t seed, void* stream) {
  return update(tensors, count, grad_type, state_bits, tensor_hparams, lr, beta1, beta2, step, clip_scale, seed, nullptr,
                stream);
}

int gptrig_adamw_tensors_device_seed(const gptrig_adamw_tensor* tensors, int count, int grad_type, int state_bits,
                                     const float* tensor_hparams, double lr, double beta1, double beta2, int step,
                                     const float* clip_scale, const int64_t* seed, void* stream) {
  if (!seed) return GPTRIG_E_NULL;
  if ((uintptr_t)seed & 7) return GPTRIG_E_SHAPE;
  return update(tensors, count, grad_type, state_bits, tensor_hparams, lr, beta1, beta2, step, clip_scale, 0, seed,
                stream);
}

}  // extern "C"
