// Token embedding with a scale, and its gradient by sorted tokens.
//
//   forward   y[i] = scale * table[t_i], a row of zeros where t_i is outside [0, vocab)
//   backward  dtable[v] = scale * sum over i with t_i = v, ascending, of dy[i]
//
// Both move rows and compute next to nothing: HBM bounds them, or the launches
// where there are few tokens.  Measured, 65536 tokens of 768 columns: bfloat16 rows of
// a float32 table of 50304 38 us (3.9 TB/s with each row of the table that is named
// read once), the sums of the gradient 64 us (255 MB, 4.0 TB/s; a large copy 5.1), the
// four launches of its sort 22 us, the join 9.
//
// The gradient adds each row's terms in a fixed order, so that a call gives the
// same bits every time, which atomics do not:
//   1. (token, position) pairs are sorted by token, stably, by a radix sort of 8
//      bits a pass: a histogram of each block's digits, then a scatter in which
//      every block finds its bins' places from all histograms.  Up to kOneBlock
//      tokens one workgroup does all passes.  Tokens outside the vocabulary get
//      the key `vocab` and end up last.
//   2. The sorted pairs are cut into chunks of equal length, whatever rows they
//      belong to, so that a token that takes a tenth of the batch does not hold
//      up one workgroup.  A wave adds a chunk's rows, 256 columns of them, in
//      float32; rows that lie inside the chunk are written, of a row that crosses
//      its start or its end the part goes to the workspace (at most two a chunk).
//      The same launch writes zeros to the rows that no token names.
//   3. Rows that cross chunks are joined from their parts, in order.  The launch before
//      lists them; the list's order changes nothing.
#include <algorithm>

#include "common.h"

namespace {

constexpr int kDigits = 256;      // bins of a pass
// Most tokens that one workgroup sorts, in LDS: 22 us for 8191 of them against 23 in
// four launches, which cost the host more besides.
constexpr int kOneBlock = 8192;
constexpr int kMostBlocks = 256;  // most workgroups of a pass
constexpr int kSlab = 256;        // columns of a row that a wave holds: four a lane

struct Sort {
  const void* tokens;
  int wide;  // tokens are int64
  int vocab;
  int n;
  int seg;  // positions of a block
  int blocks;
  int* crossing;  // a number that the sort leaves 0
};

template <bool kWide>
__device__ __forceinline__ int token_key(const void* tokens, int64_t i, int vocab) {
  const int64_t t = kWide ? static_cast<const int64_t*>(tokens)[i] : static_cast<const int32_t*>(tokens)[i];
  return t >= 0 && t < vocab ? (int)t : vocab;
}

__device__ __forceinline__ int load_key(const Sort& s, const int* keys, int i) {
  if (keys) return keys[i];
  return s.wide ? token_key<true>(s.tokens, i, s.vocab) : token_key<false>(s.tokens, i, s.vocab);
}

// counts[block][digit] of the digit at `shift`; keys NULL: the tokens themselves.
__global__ void __launch_bounds__(1024) radix_histogram_kernel(Sort s, const int* __restrict__ keys,
                                                              int* __restrict__ counts, int shift) {
  __shared__ int bins[kDigits];
  if (threadIdx.x < kDigits) bins[threadIdx.x] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * s.seg;
  const int end = (int)min((int64_t)s.n, begin + s.seg);
  for (int i = (int)begin + (int)threadIdx.x; i < end; i += 1024)
    atomicAdd(&bins[(load_key(s, keys, i) >> shift) & (kDigits - 1)], 1);
  __syncthreads();
  if (threadIdx.x < kDigits) counts[blockIdx.x * kDigits + threadIdx.x] = bins[threadIdx.x];
}

// Where a lane's key goes: place[digit] is where the wave's next key of that digit
// does.  The lanes of one digit find each other by eight ballots, and their order is
// the lanes' order.
__device__ __forceinline__ int take_place(int* place, int digit, bool valid, int lane) {
  uint64_t same = __ballot(valid);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1);
    same &= (digit >> b) & 1 ? set : ~set;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1));
  int at = 0;
  if (valid) at = place[digit] + rank;
  // (Every lane has read its place before the last of each digit moves it on;
  // the fences order the lanes' accesses for the compiler and cost nothing.)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (valid && (same >> lane) == 1) place[digit] = at + 1;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return at;
}

// place[wave][digit] from the number of the wave's keys to where they begin.
template <int kWaves>
__device__ __forceinline__ void begin_places(int (*place)[kDigits], const int* bases, int tid) {
  if (tid >= kDigits) return;
  int at = bases[tid];
  for (int w = 0; w < kWaves; ++w) {
    const int c = place[w][tid];
    place[w][tid] = at;
    at += c;
  }
}

// One block's stable scatter of positions [begin, end) by the digit at `shift`.
// Each wave owns a contiguous share of them.
template <int kWaves>
__device__ void scatter_block(const Sort& s, const int* keys, const int* positions, int* keys_out, int* positions_out,
                              int shift, int begin, int end, int (*place)[kDigits], int* bases) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int share = ((end - begin + kWaves * 64 - 1) / (kWaves * 64)) * 64;
  const int from = min(end, begin + wave * share), to = min(end, from + share);
  for (int i = tid; i < kWaves * kDigits; i += 64 * kWaves) (&place[0][0])[i] = 0;
  __syncthreads();
  for (int i = from + lane; i < to; i += 64) atomicAdd(&place[wave][(load_key(s, keys, i) >> shift) & (kDigits - 1)], 1);
  __syncthreads();
  begin_places<kWaves>(place, bases, tid);
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    const bool valid = i < to;
    const int key = valid ? load_key(s, keys, i) : 0;
    const int digit = (key >> shift) & (kDigits - 1);
    const int at = take_place(place[wave], digit, valid, lane);
    if (valid) {
      keys_out[at] = key;
      positions_out[at] = positions ? positions[i] : i;
    }
  }
}

// Exclusive prefix sums of totals[0 .. 255] in LDS by the first 256 threads.
__device__ void exclusive_scan(int* totals, int tid) {
  for (int step = 1; step < kDigits; step <<= 1) {
    int add = 0;
    if (tid < kDigits && tid >= step) add = totals[tid - step];
    __syncthreads();
    if (tid < kDigits) totals[tid] += add;
    __syncthreads();
  }
  int before = 0;
  if (tid > 0 && tid < kDigits) before = totals[tid - 1];
  __syncthreads();
  if (tid < kDigits) totals[tid] = before;
  __syncthreads();
}

__global__ void __launch_bounds__(1024)
    radix_scatter_kernel(Sort s, const int* __restrict__ keys, const int* __restrict__ positions,
                         const int* __restrict__ counts, int* __restrict__ keys_out, int* __restrict__ positions_out,
                         int shift) {
  __shared__ int place[16][kDigits];
  __shared__ int bases[kDigits], before[kDigits];
  const int tid = threadIdx.x, digit = tid & (kDigits - 1);
  if (tid < kDigits) bases[tid] = before[tid] = 0;
  if (blockIdx.x == 0 && tid == 0) *s.crossing = 0;
  __syncthreads();
  // Four threads a digit share the blocks.
  int mine = 0, total = 0;
#pragma unroll 8
  for (int b = tid / kDigits; b < s.blocks; b += 4) {
    const int c = counts[b * kDigits + digit];
    total += c;
    mine += b < (int)blockIdx.x ? c : 0;
  }
  atomicAdd(&bases[digit], total);
  atomicAdd(&before[digit], mine);
  __syncthreads();
  exclusive_scan(bases, tid);
  if (tid < kDigits) bases[tid] += before[tid];
  const int64_t begin = (int64_t)blockIdx.x * s.seg;
  scatter_block<16>(s, keys, positions, keys_out, positions_out, shift, (int)begin,
                    (int)min((int64_t)s.n, begin + s.seg), place, bases);
}

// All passes of a short sort.  The pairs stay in LDS, where a pass puts them in a new
// order without the address unit's 170 cycles for 64 places (in memory: 34 us for 8191
// pairs, 22 now); a lane holds the eight it is to place.
__global__ void __launch_bounds__(1024) radix_one_block_kernel(Sort s, int* keys_out, int* positions_out, int passes) {
  constexpr int kWaves = 16, kHeld = kOneBlock / (64 * kWaves);
  __shared__ int place[kWaves][kDigits];
  __shared__ int bases[kDigits];
  __shared__ int keys[kOneBlock], positions[kOneBlock];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = wave * 64 * kHeld + lane;
  if (tid == 0) *s.crossing = 0;
  int key[kHeld], position[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    position[j] = first + 64 * j;
    key[j] = load_key(s, nullptr, min(position[j], s.n - 1));
  }
  for (int p = 0; p < passes; ++p) {
    auto digit = [&](int j) { return (key[j] >> (8 * p)) & (kDigits - 1); };
    for (int i = tid; i < kWaves * kDigits; i += 64 * kWaves) (&place[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (first + 64 * j < s.n) atomicAdd(&place[wave][digit(j)], 1);
    __syncthreads();
    if (tid < kDigits) {
      int total = 0;
      for (int w = 0; w < kWaves; ++w) total += place[w][tid];
      bases[tid] = total;
    }
    __syncthreads();
    exclusive_scan(bases, tid);
    begin_places<kWaves>(place, bases, tid);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const bool valid = first + 64 * j < s.n;
      const int at = take_place(place[wave], digit(j), valid, lane);
      if (valid) {
        keys[at] = key[j];
        positions[at] = position[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (first + 64 * j < s.n) {
        key[j] = keys[first + 64 * j];
        position[j] = positions[first + 64 * j];
      }
  }
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (first + 64 * j < s.n) {
      keys_out[first + 64 * j] = key[j];
      positions_out[first + 64 * j] = position[j];
    }
}

// ---- rows ----

// Four columns of a row: consecutive ones in one access, or (rows without
// alignment) 64 apart.
template <typename T, bool kVec>
__device__ __forceinline__ f32x4 load_columns(const T* row, int column, int lane, int d) {
  f32x4 v{};
  if constexpr (kVec) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int c = column + 4 * lane;
    if (c < d) {
      const T4 x = *reinterpret_cast<const T4*>(row + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (float)x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column + 64 * j + lane;
      if (c < d) v[j] = (float)row[c];
    }
  }
  return v;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_columns(T* row, f32x4 v, int column, int lane, int d) {
  if constexpr (kVec) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int c = column + 4 * lane;
    if (c < d) {
      T4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (T)v[j];
      *reinterpret_cast<T4*>(row + c) = x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column + 64 * j + lane;
      if (c < d) row[c] = (T)v[j];
    }
  }
}

template <typename TT, typename OT, bool kVec>
__global__ void __launch_bounds__(256)
    embedding_rows_kernel(const void* __restrict__ tokens, int wide, const TT* __restrict__ table, int64_t ldt,
                          OT* __restrict__ y, int64_t n, int d, int vocab, float scale) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  auto key_of = [&](int64_t at) {
    return wide ? token_key<true>(tokens, min(at, n - 1), vocab) : token_key<false>(tokens, min(at, n - 1), vocab);
  };
  for (int ahead = key_of(i); i < n; i += waves) {
    const int key = __builtin_amdgcn_readfirstlane(ahead);
    ahead = key_of(i + waves);
    const TT* row = table + (int64_t)key * ldt;
    OT* out = y + i * d;
    // Four slabs in flight: a wave's rows wait for each other otherwise.
    for (int column = 0; column < d; column += 4 * kSlab) {
      f32x4 v[4]{};
      if (key < vocab) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = load_columns<TT, kVec>(row, column + k * kSlab, lane, d);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] *= scale;
        store_columns<OT, kVec>(out, v[k], column + k * kSlab, lane, d);
      }
    }
  }
}

struct Reduce {
  const int* keys;       // sorted
  const int* positions;  // of each key, ascending within a key
  float* parts;          // [chunks][2][d]: of a row that began before the chunk, of one that goes on after it
  int* crossing;         // the number of rows that cross chunks, then the chunks where they begin (in any order)
  int n, d, vocab, chunk, chunks, slabs;
  float scale;
};

// A wave adds the rows of one chunk, kSlab columns of them.
template <typename GT, typename OT, bool kVec>
__device__ __forceinline__ void add_chunk(const Reduce& r, const GT* __restrict__ dy, int64_t lddy,
                                          OT* __restrict__ dtable, int chunk, int column, int lane) {
  const int64_t begin = (int64_t)chunk * r.chunk;
  const int count = (int)min((int64_t)r.chunk, r.n - begin);
  // Lane l holds the chunk's l-th pair (a chunk has at most 64).
  const int key = lane < count ? r.keys[begin + lane] : r.vocab;
  const int position = lane < count ? r.positions[begin + lane] : 0;
  const int last_before = begin > 0 ? r.keys[begin - 1] : -1;
  const int first_after = begin + count < r.n ? r.keys[begin + count] : r.vocab;
  int current = __builtin_amdgcn_readfirstlane(key);
  bool head = current == last_before;
  float* const parts = r.parts + (int64_t)chunk * 2 * r.d;
  f32x4 sum{};
  auto flush = [&](int row, bool from_before, bool goes_on) {
    if (row >= r.vocab) return;
    if (from_before || goes_on) {
      store_columns<float, kVec>(parts + (from_before ? 0 : r.d), sum, column, lane, r.d);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] *= r.scale;
      store_columns<OT, kVec>(dtable + (int64_t)row * r.d, sum, column, lane, r.d);
    }
  };
  constexpr int kAhead = 8;  // rows in flight
  for (int e0 = 0; e0 < count; e0 += kAhead) {
    f32x4 rows[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int at = e0 + e < count ? e0 + e : count - 1;
      const int p = __builtin_amdgcn_readlane(position, at);
      rows[e] = load_columns<GT, kVec>(dy + (int64_t)p * lddy, column, lane, r.d);
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (e0 + e < count) {
        const int k = __builtin_amdgcn_readlane(key, e0 + e);
        if (k != current) {
          flush(current, head, false);
          current = k;
          head = false;
          sum = f32x4{};
        }
        sum += rows[e];
      }
    }
  }
  const bool goes_on = current == first_after && current < r.vocab;
  flush(current, head, goes_on);
  if (goes_on && !head && column == 0 && lane == 0) r.crossing[1 + atomicAdd(r.crossing, 1)] = chunk;
}

// First index of the sorted keys that is at least k.
__device__ __forceinline__ int key_bound(const int* keys, int high, int k) {
  int low = 0;
  while (low < high) {
    const int mid = low + ((high - low) >> 1);
    if (keys[mid] < k) low = mid + 1;
    else high = mid;
  }
  return low;
}

constexpr int kZeroRows = 16;  // rows a wave looks at for those without a token

template <typename GT, typename OT, bool kVec>
__global__ void __launch_bounds__(256) embedding_reduce_kernel(Reduce r, const GT* __restrict__ dy, int64_t lddy,
                                                               OT* __restrict__ dtable, int64_t add_waves,
                                                               int64_t zero_waves) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); w < add_waves + zero_waves; w += waves) {
    if (w < add_waves) {
      add_chunk<GT, OT, kVec>(r, dy, lddy, dtable, (int)(w / r.slabs), (int)(w % r.slabs) * kSlab, lane);
      continue;
    }
    const int64_t first = (w - add_waves) * kZeroRows;
    const int row = (int)min(first + (lane & (kZeroRows - 1)), (int64_t)r.vocab - 1);
    const int at = key_bound(r.keys, r.n, row);
    const bool absent = at >= r.n || r.keys[at] != row;
    uint64_t rows = __ballot(absent && lane < kZeroRows && first + lane < r.vocab);
    while (rows) {  // uniform
      const int which = __builtin_ctzll(rows);
      rows &= rows - 1;
      OT* out = dtable + (first + which) * r.d;
      for (int column = 0; column < r.d; column += kSlab) store_columns<OT, kVec>(out, f32x4{}, column, lane, r.d);
    }
  }
}

constexpr int kJoin = 8;  // waves that join a row's parts

// Rows that cross chunks: a workgroup for each (and each slab of it) adds its parts,
// each wave those of every eighth chunk, the waves' sums in order.
template <typename OT, bool kVec>
__global__ void __launch_bounds__(64 * kJoin) embedding_join_kernel(Reduce r, OT* __restrict__ dtable) {
  __shared__ f32x4 sums[kJoin][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t items = (int64_t)*r.crossing * r.slabs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int chunk = r.crossing[1 + item / r.slabs], column = (int)(item % r.slabs) * kSlab;
    const int64_t end = ((int64_t)chunk + 1) * r.chunk;
    const int key = r.keys[end - 1];
    // The chunk where it ends: the last that begins with it, looked for 64 at a time.
    int last = chunk;
    for (uint64_t more = ~0ull; more == ~0ull;) {
      const int64_t at = ((int64_t)last + 1 + lane) * r.chunk;
      more = __ballot(at < r.n && r.keys[min(at, (int64_t)r.n - 1)] == key);
      last += more == ~0ull ? 64 : __builtin_ctzll(~more);
    }
    f32x4 sum{};
    if (wave == 0) sum = load_columns<float, kVec>(r.parts + ((int64_t)chunk * 2 + 1) * r.d, column, lane, r.d);
    int c = chunk + 1 + wave;
    constexpr int kAhead = 8;  // parts in flight
    for (; c + (kAhead - 1) * kJoin <= last; c += kAhead * kJoin) {
      f32x4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        v[j] = load_columns<float, kVec>(r.parts + (int64_t)(c + kJoin * j) * 2 * r.d, column, lane, r.d);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) sum += v[j];
    }
    for (; c <= last; c += kJoin) sum += load_columns<float, kVec>(r.parts + (int64_t)c * 2 * r.d, column, lane, r.d);
    __syncthreads();  // (the last item's sums are read)
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kJoin; ++w) sum += sums[w][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] *= r.scale;
      store_columns<OT, kVec>(dtable + (int64_t)key * r.d, sum, column, lane, r.d);
    }
  }
}

// ---- host side ----

struct Plan {
  int passes, seg, blocks, chunk, chunks, slabs;
  size_t pairs, counts, crossing, parts, total;  // bytes: one int array, the histograms, ...; all of it
};

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

Plan make_plan(int n, int d, int vocab) {
  Plan p{};
  int bits = 0;
  while (bits < 31 && (vocab >> bits) != 0) ++bits;  // (the key `vocab` is one of them)
  p.passes = std::max(1, (bits + 7) / 8);
  p.seg = std::max(2048, ceil_div(ceil_div(n, kMostBlocks), 2048) * 2048);
  p.blocks = n <= kOneBlock ? 1 : ceil_div(n, p.seg);
  // Pairs a chunk: enough waves for the chip where there are few, fewer parts where there are many.
  p.chunk = 4;
  while (p.chunk < 32 && n / (2 * p.chunk) >= 2048) p.chunk *= 2;
  p.chunks = ceil_div(n, p.chunk);
  p.slabs = ceil_div(d, kSlab);
  p.pairs = round_up((size_t)n * 4);
  p.counts = round_up((size_t)p.blocks * kDigits * 4);
  p.crossing = round_up(((size_t)p.chunks + 1) * 4);
  p.parts = round_up((size_t)p.chunks * 2 * d * 4);
  p.total = 4 * p.pairs + p.counts + p.crossing + p.parts;
  return p;
}

bool known(int type) { return type == GPTRIG_TYPE_BF16 || type == GPTRIG_TYPE_F32; }
size_t size_of(int type) { return type == GPTRIG_TYPE_F32 ? 4 : 2; }

// Whether rows of four-element accesses are aligned.
bool aligned(const void* p, int64_t ld, int type) { return ld % 4 == 0 && (uintptr_t)p % (4 * size_of(type)) == 0; }

constexpr int64_t kMostGrid = 1 << 20;  // workgroups a launch; more work is looped over

constexpr unsigned kJoinGrid = 1024;    // of the join, which learns on the GPU how much there is
constexpr unsigned kRowsGrid = 2048;    // of the lookup: eight a CU, which is all that a CU holds

unsigned grid_of(int64_t items, int per_block) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(kMostGrid, (items + per_block - 1) / per_block));
}

template <typename TT, typename OT>
void launch_rows(bool vec, const void* tokens, int wide, const void* table, int64_t ldt, void* y, int64_t n, int d,
                 int vocab, float scale, hipStream_t s) {
  const unsigned grid = std::min(grid_of(n, 4), kRowsGrid);
  if (vec)
    embedding_rows_kernel<TT, OT, true><<<grid, 256, 0, s>>>(tokens, wide, (const TT*)table, ldt, (OT*)y, n, d, vocab, scale);
  else
    embedding_rows_kernel<TT, OT, false><<<grid, 256, 0, s>>>(tokens, wide, (const TT*)table, ldt, (OT*)y, n, d, vocab, scale);
}

template <typename GT, typename OT, bool kVec>
int launch_reduce_as(const Reduce& r, const void* dy, int64_t lddy, void* dtable, hipStream_t s) {
  const int64_t add = (int64_t)r.chunks * r.slabs, zero = ((int64_t)r.vocab + kZeroRows - 1) / kZeroRows;
  embedding_reduce_kernel<GT, OT, kVec><<<grid_of(add + zero, 4), 256, 0, s>>>(r, (const GT*)dy, lddy, (OT*)dtable, add,
                                                                              zero);
  GPTRIG_CHECK_LAUNCH();
  if (!add) return GPTRIG_OK;
  embedding_join_kernel<OT, kVec><<<std::min(grid_of(add, 1), kJoinGrid), 64 * kJoin, 0, s>>>(r, (OT*)dtable);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

template <typename GT, typename OT>
int launch_reduce(bool vec, const Reduce& r, const void* dy, int64_t lddy, void* dtable, hipStream_t s) {
  return vec ? launch_reduce_as<GT, OT, true>(r, dy, lddy, dtable, s)
             : launch_reduce_as<GT, OT, false>(r, dy, lddy, dtable, s);
}

int check_sizes(int64_t n, int d, int vocab) {
  return n < 0 || n >= (1ll << 31) - 65536 || d <= 0 || d > 1 << 24 || vocab <= 0 || vocab == 0x7fffffff
             ? GPTRIG_E_SHAPE
             : GPTRIG_OK;
}

}  // namespace

extern "C" {

int gptrig_scaled_embedding_fwd(const void* tokens, int tokens_are_int64, const void* table, int64_t ldt,
                                int table_type, void* y, int y_type, int64_t n, int d, int vocab, float scale,
                                void* stream) {
  if (!tokens || !table || !y) return GPTRIG_E_NULL;
  if (!known(table_type) || !known(y_type)) return GPTRIG_E_DTYPE;
  if (check_sizes(n, d, vocab) != GPTRIG_OK || ldt < 0) return GPTRIG_E_SHAPE;
  if ((uintptr_t)tokens % (tokens_are_int64 ? 8 : 4) || (uintptr_t)table % size_of(table_type) ||
      (uintptr_t)y % size_of(y_type))
    return GPTRIG_E_SHAPE;
  if (n == 0) return GPTRIG_OK;
  const bool vec = d % 4 == 0 && aligned(table, ldt, table_type) && aligned(y, d, y_type);
  const hipStream_t s = (hipStream_t)stream;
  if (table_type == GPTRIG_TYPE_F32 && y_type == GPTRIG_TYPE_F32)
    launch_rows<float, float>(vec, tokens, tokens_are_int64, table, ldt, y, n, d, vocab, scale, s);
  else if (table_type == GPTRIG_TYPE_F32)
    launch_rows<float, bf16>(vec, tokens, tokens_are_int64, table, ldt, y, n, d, vocab, scale, s);
  else if (y_type == GPTRIG_TYPE_F32)
    launch_rows<bf16, float>(vec, tokens, tokens_are_int64, table, ldt, y, n, d, vocab, scale, s);
  else
    launch_rows<bf16, bf16>(vec, tokens, tokens_are_int64, table, ldt, y, n, d, vocab, scale, s);
  GPTRIG_CHECK_LAUNCH();
  return GPTRIG_OK;
}

size_t gptrig_scaled_embedding_bwd_workspace_bytes(int64_t n, int d, int vocab) {
  if (check_sizes(n, d, vocab) != GPTRIG_OK || n == 0) return 0;
  return make_plan((int)n, d, vocab).total;
}

int gptrig_scaled_embedding_bwd(const void* tokens, int tokens_are_int64, const void* dy, int64_t lddy, int dy_type,
                                void* dtable, int table_type, int64_t n, int d, int vocab, float scale,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (!dtable || (n > 0 && (!tokens || !dy))) return GPTRIG_E_NULL;
  if (!known(table_type) || !known(dy_type)) return GPTRIG_E_DTYPE;
  if (check_sizes(n, d, vocab) != GPTRIG_OK || lddy < 0) return GPTRIG_E_SHAPE;
  if ((uintptr_t)tokens % (tokens_are_int64 ? 8 : 4) || (uintptr_t)dy % size_of(dy_type) ||
      (uintptr_t)dtable % size_of(table_type) || (uintptr_t)workspace % 16)
    return GPTRIG_E_SHAPE;
  const hipStream_t s = (hipStream_t)stream;
  Plan p{};
  int* keys = nullptr;
  int* positions = nullptr;
  int* crossing = nullptr;
  float* parts = nullptr;
  if (n > 0) {
    p = make_plan((int)n, d, vocab);
    if (!workspace) return GPTRIG_E_NULL;
    if (workspace_bytes < p.total) return GPTRIG_E_WORKSPACE;
    char* at = (char*)workspace;
    int* const keys_a = (int*)at;
    int* const positions_a = (int*)(at + p.pairs);
    int* const keys_b = (int*)(at + 2 * p.pairs);
    int* const positions_b = (int*)(at + 3 * p.pairs);
    int* const counts = (int*)(at + 4 * p.pairs);
    crossing = (int*)(at + 4 * p.pairs + p.counts);
    parts = (float*)(at + 4 * p.pairs + p.counts + p.crossing);
    const Sort sort{tokens, tokens_are_int64, vocab, (int)n, p.seg, p.blocks, crossing};
    if (p.blocks == 1) {
      radix_one_block_kernel<<<1, 1024, 0, s>>>(sort, keys_b, positions_b, p.passes);
      GPTRIG_CHECK_LAUNCH();
      keys = keys_b;
      positions = positions_b;
    } else {
      for (int pass = 0; pass < p.passes; ++pass) {
        int* const keys_to = pass & 1 ? keys_a : keys_b;
        int* const positions_to = pass & 1 ? positions_a : positions_b;
        radix_histogram_kernel<<<p.blocks, 1024, 0, s>>>(sort, keys, counts, 8 * pass);
        GPTRIG_CHECK_LAUNCH();
        radix_scatter_kernel<<<p.blocks, 1024, 0, s>>>(sort, keys, positions, counts, keys_to, positions_to, 8 * pass);
        GPTRIG_CHECK_LAUNCH();
        keys = keys_to;
        positions = positions_to;
      }
    }
  }
  const Reduce r{keys, positions, parts, crossing, (int)n, d, vocab, std::max(1, p.chunk), p.chunks, ceil_div(d, kSlab), scale};
  const bool vec = d % 4 == 0 && (n == 0 || aligned(dy, lddy, dy_type)) && aligned(dtable, d, table_type);
  if (dy_type == GPTRIG_TYPE_F32 && table_type == GPTRIG_TYPE_F32)
    return launch_reduce<float, float>(vec, r, dy, lddy, dtable, s);
  if (dy_type == GPTRIG_TYPE_F32) return launch_reduce<float, bf16>(vec, r, dy, lddy, dtable, s);
  if (table_type == GPTRIG_TYPE_F32) return launch_reduce<bf16, float>(vec, r, dy, lddy, dtable, s);
  return launch_reduce<bf16, bf16>(vec, r, dy, lddy, dtable, s);
}

}  // extern "C"
