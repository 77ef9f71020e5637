// Gradient of an embedding lookup, each row's sum taken in the order of the tokens: no atomic additions, the same bits every time.
//   1. order:  the rows sorted by key (stable).  Up to kOneTile rows one kernel counts, for every row, the rows before it; up to kPackedRows it does so in
//      tiles, and a second one finds each row's place in all tiles; more rows take radix passes of up to 10 bits (count, scan, scatter).
//      (8200 rows: one tile of all 14.6 us; stable passes of one block in its shared memory 31.5; radix passes 29.)
//   2. reduce: the sorted rows in chunks of 8 or 16, a group of threads each, whatever the words' frequencies are; a sum that begins and
//      ends in a chunk goes to its row of the gradient, one that crosses an end leaves its part in the workspace.
//   3. join:   the parts of a sum, in order.
// Where the gradient is written whole, its rows are cleared by further blocks of the sorting kernels: these wait on latency, the clearing on memory.
// Bound by the bytes of dy and of the gradient's rows: 65536 rows of 1024 in fp32 into 250054 words 225 us (floor 200: dy, the gradient); by
// themselves the kernels take 248, most of the difference is their starts.  Sums in 32 bits, one rounding at the end.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include "b200_ptx.cuh"
#include "bounds_check.cuh"
#include "launch.cuh"
#include "tuning_api.h"

namespace b200 {

namespace {

constexpr int kRowBits = 14, kPackedRows = 1 << kRowBits;      // rows whose number fits beside a key into 32 bits
constexpr int kOneTile = 2048, kMergeTile = 256;               // rows ranked in one go; of a tile where tiles are merged
constexpr int kRankEach = 2, kRankRows = 16 * kRankEach;       // rows of a group of 16 threads, and of a block
constexpr int kMergeRows = 64;                                 // rows of a block that merges, 4 threads to each
constexpr int kTile = 1024;                                    // rows of a block of a radix pass
constexpr int kDigitBits = 10;                                 // at most

struct Keys {
  const int64_t* tokens;
  const int64_t* positions;
  int rows, vocab, keys;
  long pad;
  __device__ __forceinline__ int of(int64_t t, int64_t p) const {            // `keys`: the row has none
    if (t == pad || t < 0 || t >= vocab) return keys;
    if (!positions) return static_cast<int>(t);
    return p < 0 ? 0 : p >= keys ? keys - 1 : static_cast<int>(p);
  }
  // keys of rows r, r + step, ...: all asked for before the first is looked at
  template <int kN> __device__ __forceinline__ void of(int r, int step, int end, int (&key)[kN]) const {
    int64_t t[kN], p[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      t[j] = r + j * step < end ? tokens[r + j * step] : -1;
      p[j] = positions && r + j * step < end ? positions[r + j * step] : 0;
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) key[j] = of(t[j], p[j]);
  }
};

// parts [at, to) of `of` of the memory to clear, by the blocks from `first` on, 16 KB each: short blocks write at 7.2 TB/s, 6 to an SM that go through it
// all at 5.9 (1 GB)
struct Clear {
  uint4* p;
  long n;
  int first, at, to, of;
  __device__ __forceinline__ bool mine() const { return static_cast<int>(blockIdx.x) >= first; }
  __device__ __forceinline__ void run() const {
    const long begin = n * at / of + static_cast<long>(blockIdx.x - first) * 1024, end = n * to / of;
#pragma unroll 4
    for (int j = threadIdx.x; j < 1024; j += blockDim.x)
      if (begin + j < end) p[begin + j] = make_uint4(0, 0, 0, 0);
  }
  // the next kernel's share, behind its own blocks: the blocks in all
  int next(int blocks, int parts) {
    first = blocks;
    at = to;
    to += parts;
    return blocks + static_cast<int>((n * to / of - n * at / of + 1023) / 1024);
  }
};

// Every row's place in its tile: the number of rows of the tile before it, 16 threads to the same rows, each over every 16th group of 4.  Key and row
// make one number of 32 bits, so that equal keys are in the order of their rows.  Whole: there is one tile, and the places are the rows' own.
template <bool kWhole>
__global__ void __launch_bounds__(256) tile_rank_kernel(const Keys k, int tile, uint32_t* __restrict__ tiles, int* __restrict__ order,
                                                        int* __restrict__ sorted, int* __restrict__ joins, const Clear clear) {
  let_next_start();
  if (clear.mine()) { clear.run(); return; }
  __shared__ __align__(16) uint32_t all[kWhole ? kOneTile : kMergeTile];
  const int base = static_cast<int>(blockIdx.x) * kRankRows / tile * tile, count = min(tile, k.rows - base), padded = (count + 63) & ~63;
  if (blockIdx.x == 0 && threadIdx.x < 2) joins[threadIdx.x] = 0;
  constexpr int kLoads = (kWhole ? kOneTile : kMergeTile) / 256;
  int key[kLoads];
  k.of(base + threadIdx.x, 256, base + count, key);
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int at = threadIdx.x + j * 256;
    if (at < padded) all[at] = at < count ? static_cast<uint32_t>(key[j]) << kRowBits | static_cast<uint32_t>(base + at) : 0xFFFFFFFFu;
  }
  __syncthreads();
  const int lane16 = threadIdx.x & 15, first = static_cast<int>(blockIdx.x) * kRankRows - base + (threadIdx.x >> 4) * kRankEach;
  uint32_t mine[kRankEach];
  int before[kRankEach] = {};
#pragma unroll
  for (int j = 0; j < kRankEach; ++j) mine[j] = first + j < padded ? all[first + j] : 0xFFFFFFFFu;
#pragma unroll 4
  for (int i = lane16; i < padded / 4; i += 16) {
    const uint4 u = reinterpret_cast<const uint4*>(all)[i];
#pragma unroll
    for (int j = 0; j < kRankEach; ++j) before[j] += (u.x < mine[j]) + (u.y < mine[j]) + (u.z < mine[j]) + (u.w < mine[j]);
  }
#pragma unroll
  for (int j = 0; j < kRankEach; ++j) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) before[j] += __shfl_xor_sync(0xffffffffu, before[j], o);
    if (lane16 == 0 && first + j < count) {
      if constexpr (kWhole) {
        order[before[j]] = first + j;
        sorted[before[j]] = static_cast<int>(mine[j] >> kRowBits);
      } else {
        tiles[base + before[j]] = mine[j];
      }
    }
  }
}

// A row's place among all: in every sorted tile the rows before it, by bisection (4 threads to a row, every fourth tile each).  `tiles` is written while this
// kernel is already there, so it is not __restrict__: loads of what never changes may be moved in front of the wait.
__global__ void __launch_bounds__(256) merge_rank_kernel(const uint32_t* tiles, int rows, int* order, int* sorted, const Clear clear) {
  let_next_start();
  if (clear.mine()) { clear.run(); return; }
  wait_for_previous();
  extern __shared__ __align__(16) uint32_t tile_of[];
  const int count = (rows + kMergeTile - 1) / kMergeTile;
#pragma unroll 8
  for (int i = threadIdx.x; i < count * kMergeTile; i += 256) tile_of[i] = i < rows ? tiles[i] : 0xFFFFFFFFu;
  __syncthreads();
  const int at = blockIdx.x * kMergeRows + (threadIdx.x >> 2);
  if (at >= rows) return;
  const uint32_t mine = tile_of[at];
  int place = 0;
#pragma unroll 4
  for (int t = threadIdx.x & 3; t < count; t += 4) {
    const uint32_t* const tile = tile_of + t * kMergeTile;
    int before = 0;
#pragma unroll
    for (int step = kMergeTile / 2; step > 0; step >>= 1) before += tile[before + step - 1] < mine ? step : 0;
    place += before + (tile[before] < mine);
  }
  const uint32_t group = 0xFu << (threadIdx.x & 28);
  place += __shfl_xor_sync(group, place, 1);
  place += __shfl_xor_sync(group, place, 2);
  if ((threadIdx.x & 3) == 0) {
    order[place] = static_cast<int>(mine & (kPackedRows - 1));
    sorted[place] = static_cast<int>(mine >> kRowBits);
  }
}

// Lanes with the same digit among those with one (d >= 0), a vote for each bit: a match of whole words takes several times as long.
__device__ __forceinline__ uint32_t same_digit(int d, int bits) {
  uint32_t same = __ballot_sync(0xffffffffu, d >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool one = (d >> b) & 1;
    const uint32_t m = __ballot_sync(0xffffffffu, one);
    same &= one ? m : ~m;
  }
  return same;
}

// ---- radix passes ----------------------------------------------------------------------------------------------------------
struct Pass {
  const int* key;           // null: the first pass, keys from the tokens
  const int* row;
  int* key_out;
  int* row_out;
  int* counts;              // [bins][tiles]
  int shift, digit, bins, tiles;
};

template <int kN> __device__ __forceinline__ void keys_at(const Keys& k, const Pass& p, int i, int step, int end, int (&key)[kN]) {
  if (!p.key) { k.of(i, step, end, key); return; }
#pragma unroll
  for (int j = 0; j < kN; ++j) key[j] = i + j * step < end ? p.key[i + j * step] : 0;
}

__global__ void __launch_bounds__(256) radix_count_kernel(const Keys k, const Pass p, int* __restrict__ joins, const Clear clear) {
  let_next_start();
  if (clear.mine()) { clear.run(); return; }
  wait_for_previous();
  if (blockIdx.x == 0 && threadIdx.x < 2) joins[threadIdx.x] = 0;
  __shared__ int bins[1 << kDigitBits];
  for (int b = threadIdx.x; b < p.bins; b += 256) bins[b] = 0;
  __syncthreads();
  const int begin = blockIdx.x * kTile + threadIdx.x;
  int key[kTile / 256];
  keys_at(k, p, begin, 256, k.rows, key);
#pragma unroll
  for (int j = 0; j < kTile / 256; ++j)
    if (begin + j * 256 < k.rows) atomicAdd(&bins[(key[j] >> p.shift) & (p.bins - 1)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins; b += 256) p.counts[static_cast<long>(b) * p.tiles + blockIdx.x] = bins[b];
}

// counts -> their exclusive sums, one block
__global__ void __launch_bounds__(1024) radix_scan_kernel(int* counts, int n) {
  let_next_start();
  wait_for_previous();
  __shared__ int warps[32];
  __shared__ int carry;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (t == 0) carry = 0;
  __syncthreads();
  constexpr int kEach = 32;                                     // one wait for 32768 counts
  for (int base = 0; base < n; base += 1024 * kEach) {
    int v[kEach], sum = 0;
#pragma unroll
    for (int j = 0; j < kEach; j += 4) {                        // (where n is no multiple of 4, what is behind it counts for nothing)
      const int i = base + t * kEach + j;
      const int4 u = i < n ? *reinterpret_cast<const int4*>(counts + i) : make_int4(0, 0, 0, 0);
      v[j] = u.x; v[j + 1] = u.y; v[j + 2] = u.z; v[j + 3] = u.w;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) sum += v[j];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += u; }
    if (lane == 31) warps[warp] = before;
    __syncthreads();
    if (warp == 0) {
      int w = warps[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += u; }
      warps[lane] = w;
    }
    __syncthreads();
    int at = carry + before - sum + (warp ? warps[warp - 1] : 0);
#pragma unroll
    for (int j = 0; j < kEach; j += 4) {
      const int i = base + t * kEach + j;
      const int4 u = make_int4(at, at + v[j], at + v[j] + v[j + 1], at + v[j] + v[j + 1] + v[j + 2]);
      if (i < n) *reinterpret_cast<int4*>(counts + i) = u;
      at = u.w + v[j + 3];
    }
    __syncthreads();
    if (t == 1023) carry = at;
    __syncthreads();
  }
}

// A warp has kTile / 8 rows one after another: it counts its digits, the warps' counts are summed in order, then rows go to their places.
__global__ void __launch_bounds__(256) radix_scatter_kernel(const Keys k, const Pass p, const Clear clear) {
  let_next_start();
  if (clear.mine()) { clear.run(); return; }
  wait_for_previous();
  extern __shared__ int at[];                                   // [8][bins]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < 8 * p.bins; b += 256) at[b] = 0;
  __syncthreads();
  const int begin = blockIdx.x * kTile + warp * (kTile / 8), end = min(k.rows, begin + kTile / 8);
  int* const mine = at + warp * p.bins;
  const uint32_t below = (1u << lane) - 1;
  constexpr int kRounds = kTile / 256;
  int key[kRounds], row[kRounds];
  keys_at(k, p, begin + lane, 32, k.rows, key);
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    const int i = begin + j * 32 + lane;
    row[j] = p.row && i < end ? p.row[i] : i;
  }
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    const int i = begin + j * 32 + lane, d = i < end ? (key[j] >> p.shift) & (p.bins - 1) : -1;
    const uint32_t same = same_digit(d, p.digit);
    if (d >= 0 && (same & below) == 0) mine[d] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins; b += 256) {
    int sum = p.counts[static_cast<long>(b) * p.tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < 8; ++w) { const int n = at[w * p.bins + b]; at[w * p.bins + b] = sum; sum += n; }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    const int i = begin + j * 32 + lane, d = i < end ? (key[j] >> p.shift) & (p.bins - 1) : -1;
    const uint32_t same = same_digit(d, p.digit);
    const int place = d >= 0 ? mine[d] + __popc(same & below) : 0;
    __syncwarp();
    if (d >= 0) {
      p.key_out[place] = key[j];
      p.row_out[place] = row[j];
      if ((same & below) == 0) mine[d] += __popc(same);
    }
    __syncwarp();
  }
}

// ---- sums ------------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <typename T, int kN> struct alignas(sizeof(T) * kN) Pack { T v[kN]; };

struct Sum {
  const int* order;
  const int* sorted;
  const void* dy;
  void* grad;
  float* parts;             // [chunks][2][width]: of a sum that began before the chunk, of one that goes on behind it
  int* joins;               // chunks in which a sum begins that goes on behind them: numbers of those that end in the next and of the others; both lists
  int rows, keys, width, chunk, chunks;
  float scale, p;
  unsigned long long seed, stream_id;
  const unsigned long long* seed_dev;
};

// One addition an element and call: the gradient does not depend on an order, and nothing waits for what was there.
template <typename T, int kN, bool kAdd>
__device__ __forceinline__ void to_grad(const Sum& s, int key, int col, const float (&acc)[kN]) {
  const long at = static_cast<long>(key) * s.width + col;
  if constexpr (kAdd) {
    float* g = static_cast<float*>(s.grad) + at;
    if constexpr (kN % 4 == 0) {
#pragma unroll
      for (int j = 0; j < kN; j += 4)
        asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(g + j), "f"(acc[j] * s.scale), "f"(acc[j + 1] * s.scale),
                     "f"(acc[j + 2] * s.scale), "f"(acc[j + 3] * s.scale) : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(g + j), "f"(acc[j] * s.scale) : "memory");
    }
  } else {
    Pack<T, kN> o;
#pragma unroll
    for (int j = 0; j < kN; ++j) o.v[j] = from_f<T>(acc[j] * s.scale);
    *reinterpret_cast<Pack<T, kN>*>(static_cast<T*>(s.grad) + at) = o;
  }
}

template <int kBytes> __device__ __forceinline__ void copy_vector(void* to, const void* from) {
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else if constexpr (kBytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

// blockDim = (column vectors, chunks of this block), whole warps to a chunk; a lane has the key and the row of one of its sorted rows.  Every thread
// copies its columns of all the chunk's rows to shared memory (kCopy) before it adds up the first: 64 KB a block on their way, and three blocks
// to an SM, whatever the words' frequencies are.
template <typename T, int kN, bool kDrop, bool kAdd>
__global__ void __launch_bounds__(256, 3) reduce_kernel(const Sum s) {
  constexpr int kBytes = sizeof(T) * kN;
  constexpr bool kCopy = kBytes >= 8;
  extern __shared__ __align__(16) unsigned char held[];         // [chunk][256] vectors
  const int c = blockIdx.x * blockDim.y + threadIdx.y, lane = threadIdx.x & 31, thread = threadIdx.y * blockDim.x + threadIdx.x;
  let_next_start();
  wait_for_previous();
  if (c >= s.chunks) return;
  const int begin = c * s.chunk, count = min(s.rows - begin, s.chunk);
  const DropRng rng(s.seed + ((kDrop && s.seed_dev) ? *s.seed_dev : 0ull), s.stream_id, s.p);
  const int my_key = lane < count ? s.sorted[begin + lane] : s.keys, my_row = lane < count ? s.order[begin + lane] : 0;
  const int before = begin > 0 ? s.sorted[begin - 1] : -1, after = begin + count < s.rows ? s.sorted[begin + count] : -1;
  const int first = __shfl_sync(0xffffffffu, my_key, 0);
  const int with_key = __popc(__ballot_sync(0xffffffffu, my_key < s.keys));       // rows without a key come last
  if (with_key == 0) return;
  for (int base = 0; base < s.width; base += blockDim.x * kN) {
    const int col = base + threadIdx.x * kN;
    const bool in = col < s.width;
    const T* const dy = static_cast<const T*>(s.dy) + col;
    if constexpr (kCopy) {
#pragma unroll 4
      for (int j = 0; j < with_key; ++j) {
        const int row = __shfl_sync(0xffffffffu, my_row, j);
        if (in) copy_vector<kBytes>(held + (j * 256 + thread) * kBytes, dy + static_cast<long>(row) * s.width);
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    }
    float acc[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) acc[j] = 0.f;
    const auto flush = [&](int key, bool began_before, bool goes_on) {
      if (!in) return;
      if (began_before || goes_on) {
        float* part = s.parts + (static_cast<long>(c) * 2 + (began_before ? 0 : 1)) * s.width + col;
        if constexpr (kN % 4 == 0) {
#pragma unroll
          for (int j = 0; j < kN; j += 4) *reinterpret_cast<float4*>(part + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < kN; ++j) part[j] = acc[j];
        }
      } else {
        to_grad<T, kN, kAdd>(s, key, col, acc);
      }
    };
    int key = first;
    bool began_before = key == before;
#pragma unroll 1
    for (int j = 0; j < with_key; ++j) {
      const int of = __shfl_sync(0xffffffffu, my_key, j), row = __shfl_sync(0xffffffffu, my_row, j);
      if (of != key) {
        flush(key, began_before, false);
        key = of;
        began_before = false;
#pragma unroll
        for (int q = 0; q < kN; ++q) acc[q] = 0.f;
      }
      if (in) {
        Pack<T, kN> v;
        if constexpr (kCopy) v = *reinterpret_cast<const Pack<T, kN>*>(held + (j * 256 + thread) * kBytes);
        else v = *reinterpret_cast<const Pack<T, kN>*>(dy + static_cast<long>(row) * s.width);
#pragma unroll
        for (int q = 0; q < kN; ++q) {
          float f = to_f<T>(v.v[q]);
          if constexpr (kDrop) {
            const unsigned long long at = static_cast<unsigned long long>(row) * s.width + col;
            bool keep;
            if constexpr (kN % 4 == 0) keep = rng.keep(rng.word((at >> 2) + q / 4), q % 4);
            else keep = rng.keep(rng.word((at + q) >> 2), static_cast<int>((at + q) & 3));
            f = keep ? f * rng.scale : 0.f;
          }
          acc[q] += f;
        }
      }
    }
    const bool goes_on = with_key == s.chunk && key == after;
    flush(key, began_before, goes_on);
    if (base == 0 && threadIdx.x == 0 && goes_on && !began_before) {
      const int at = begin + 2 * s.chunk;                       // behind the next chunk
      const bool is_long = at < s.rows && s.sorted[at - 1] == key && s.sorted[at] == key;
      s.joins[2 + (is_long ? s.chunks : 0) + atomicAdd(s.joins + is_long, 1)] = c;
    }
  }
}

// The sums that begin in a chunk and go on behind it.  Most end in the next chunk: two parts, a warp of the first half of the blocks to each sum.  The others
// take a block of the second half and a share of the columns each, the parts in 8 runs one after another, the runs in order; their end is found by 32 looks at a time.  (The list's order does not
// matter: every sum is joined by itself.)
template <typename T, int kN, bool kAdd>
__global__ void __launch_bounds__(256) join_kernel(const Sum s) {
  constexpr int kRuns = 8, kCols = 32;
  __shared__ float runs[kRuns][kCols * kN];
  const int x = threadIdx.x & 31, run = threadIdx.x >> 5, half = gridDim.x / 2;
  const bool first_half = static_cast<int>(blockIdx.x) < half;
  wait_for_previous();
  const int sums = first_half ? s.joins[0] : 0, long_sums = first_half ? 0 : s.joins[1];
  for (int i = (blockIdx.y * half + blockIdx.x) * kRuns + run; i < sums; i += half * gridDim.y * kRuns) {
    const int c = s.joins[2 + i], key = s.sorted[(c + 1) * s.chunk];
    const float* const first = s.parts + (static_cast<long>(c) * 2 + 1) * s.width;
    const float* const second = s.parts + static_cast<long>(c + 1) * 2 * s.width;
#pragma unroll 4
    for (int col = x * kN; col < s.width; col += 32 * kN) {
      float acc[kN];
      if constexpr (kN % 4 == 0) {
#pragma unroll
        for (int j = 0; j < kN; j += 4) {
          const float4 a = *reinterpret_cast<const float4*>(first + col + j), b = *reinterpret_cast<const float4*>(second + col + j);
          acc[j] = a.x + b.x; acc[j + 1] = a.y + b.y; acc[j + 2] = a.z + b.z; acc[j + 3] = a.w + b.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) acc[j] = first[col + j] + second[col + j];
      }
      to_grad<T, kN, kAdd>(s, key, col, acc);
    }
  }
  if (first_half) return;
  for (int i = static_cast<int>(blockIdx.x) - half; i < long_sums; i += half) {
    const int c = s.joins[2 + s.chunks + i], key = s.sorted[(c + 1) * s.chunk];
    int lo = (c + 1) * s.chunk, hi = s.rows;                    // the first place behind the sum's last is in [lo, hi]
    while (lo < hi) {
      const int step = (hi - lo + 31) / 32, at = lo + x * step;
      const bool same = at < hi && s.sorted[at] == key;
      const int n = __popc(__ballot_sync(0xffffffffu, same));   // looks that still see the key
      if (n == 0) break;
      const int next = lo + n * step;
      lo = lo + (n - 1) * step + 1;
      hi = min(hi, next);
    }
    const int n = (lo - 1) / s.chunk - c;                       // parts in the chunks behind this one
    const int from = static_cast<int>(static_cast<long>(n + 1) * run / kRuns), to = static_cast<int>(static_cast<long>(n + 1) * (run + 1) / kRuns);
    for (int base = blockIdx.y * kCols * kN; base < s.width; base += gridDim.y * kCols * kN) {
      const int col = base + x * kN;
      float acc[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) acc[j] = 0.f;
      if (col < s.width) {
#pragma unroll 8
        for (int q = from; q < to; ++q) {
          const float* part = s.parts + (static_cast<long>(c + q) * 2 + (q == 0 ? 1 : 0)) * s.width + col;
          if constexpr (kN % 4 == 0) {
#pragma unroll
            for (int j = 0; j < kN; j += 4) {
              const float4 v = *reinterpret_cast<const float4*>(part + j);
              acc[j] += v.x; acc[j + 1] += v.y; acc[j + 2] += v.z; acc[j + 3] += v.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < kN; ++j) acc[j] += part[j];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kN; ++j) runs[run][x * kN + j] = acc[j];
      __syncthreads();
      if (run == 0 && col < s.width) {
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          acc[j] = 0.f;
#pragma unroll
          for (int r = 0; r < kRuns; ++r) acc[j] += runs[r][x * kN + j];
        }
        to_grad<T, kN, kAdd>(s, key, col, acc);
      }
      __syncthreads();
    }
  }
}

// out[r] = table[token] * scale
template <typename T, int kN>
__global__ void __launch_bounds__(256) rows_kernel(const int64_t* __restrict__ tokens, const T* __restrict__ table, T* __restrict__ out, int rows,
                                                   int vocab, int width, float scale) {
  for (int r = blockIdx.x * blockDim.y + threadIdx.y; r < rows; r += gridDim.x * blockDim.y) {
    int64_t t = tokens[r];
    if (t < 0 || t >= vocab) { NMTG_BOUNDS_HIT(); t = 0; }
    for (int col = threadIdx.x * kN; col < width; col += blockDim.x * kN) {
      Pack<T, kN> v = *reinterpret_cast<const Pack<T, kN>*>(table + t * width + col);
#pragma unroll
      for (int j = 0; j < kN; ++j) v.v[j] = from_f<T>(to_f<T>(v.v[j]) * scale);
      *reinterpret_cast<Pack<T, kN>*>(out + static_cast<long>(r) * width + col) = v;
    }
  }
}

const char* problem(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
long up16(long n) { return (n + 15) & ~15L; }

// Rows of a chunk (at most 32, a lane to each): enough chunks for every SM where there are few rows, fewer parts to join where there are many
constexpr int kMostChunk = 16;
int chunk_of(int rows) { return rows < 4096 ? 8 : kMostChunk; }
int key_bits(int keys) {           // of numbers up to `keys`
  int b = 1;
  while (b < 31 && (1L << b) <= keys) ++b;
  return b;
}

// dim3(threads over the columns, rows or chunks of a block)
dim3 shape(int width, int n) {
  int x = 32;
  while (x < 256 && x * n < width) x *= 2;
  return dim3(x, 256 / x);
}

template <typename T, int kN, bool kDrop, bool kAdd>
const char* sums(const Sum& s, cudaStream_t stream) {
  const dim3 block = shape(s.width, kN);
  const int vector = sizeof(T) * kN, smem = vector >= 8 ? s.chunk * 256 * vector : 0;
  cudaError_t e = cudaFuncSetAttribute(reduce_kernel<T, kN, kDrop, kAdd>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostChunk * 256 * 16);
  if (e != cudaSuccess) return problem(e);
  const char* err = launch_behind(true, reduce_kernel<T, kN, kDrop, kAdd>, dim3((s.chunks + block.y - 1) / block.y), block, smem, stream, s);
  if (err || s.chunks < 2) return err;
  const int cols = (s.width + 32 * kN - 1) / (32 * kN), across = cols < 8 ? cols : 8, want = (s.chunks + 7) / 8, most = 16 * num_sms() / across;
  return launch_behind(true, join_kernel<T, kN, kAdd>, dim3(2 * (want < most ? want : most), across), dim3(256), 0, stream, s);
}

template <typename T, int kN, bool kAdd>
const char* sums_drop(const Sum& s, cudaStream_t stream) {
  return s.p > 0.f ? sums<T, kN, true, kAdd>(s, stream) : sums<T, kN, false, kAdd>(s, stream);
}

// Elements of a vector: 16 bytes, 4 elements of a 16-bit type, or one (34056 rows of 300 in bf16: 50 us with the lookup, one by one 90)
template <typename T>
const char* sums_type(const Sum& s, bool add, cudaStream_t stream) {
  constexpr int kN = 16 / sizeof(T);
  const bool on = aligned(s.dy) && aligned(s.grad);
  if (on && s.width % kN == 0) return add ? sums_drop<T, kN, true>(s, stream) : sums_drop<T, kN, false>(s, stream);
  if constexpr (kN > 4)
    if (on && s.width % 4 == 0) return add ? sums_drop<T, 4, true>(s, stream) : sums_drop<T, 4, false>(s, stream);
  return add ? sums_drop<T, 1, true>(s, stream) : sums_drop<T, 1, false>(s, stream);
}

template <typename T, int kN>
const char* gather_by(const int64_t* tokens, const void* table, void* out, int rows, int vocab, int width, float scale, cudaStream_t stream) {
  const dim3 block = shape(width, kN);
  const int blocks = (rows + static_cast<int>(block.y) - 1) / static_cast<int>(block.y), most = 32 * num_sms();
  const int grid = blocks < most ? blocks : most;
  rows_kernel<T, kN><<<grid, block, 0, stream>>>(tokens, static_cast<const T*>(table), static_cast<T*>(out), rows, vocab, width, scale);
  return problem(cudaGetLastError());
}
template <typename T>
const char* gather(const int64_t* tokens, const void* table, void* out, int rows, int vocab, int width, float scale, cudaStream_t stream) {
  constexpr int kN = 16 / sizeof(T);
  const bool on = aligned(table) && aligned(out);
  if (on && width % kN == 0) return gather_by<T, kN>(tokens, table, out, rows, vocab, width, scale, stream);
  if (on && width % 4 == 0) return gather_by<T, 4>(tokens, table, out, rows, vocab, width, scale, stream);
  return gather_by<T, 1>(tokens, table, out, rows, vocab, width, scale, stream);
}

}  // namespace
}  // namespace b200

using namespace b200;

long nmtg_embed_grad_workspace(int rows, int keys, int width) {
  const long n = rows, chunks = (n + chunk_of(rows) - 1) / chunk_of(rows), tiles = (n + kTile - 1) / kTile;
  return 4 * up16(4 * n) + up16(4 * tiles << kDigitBits) + up16(4 * (2 * chunks + 2)) + up16(8 * chunks * width);
}

const char* nmtg_embed_grad(const NmtgEmbedGrad* d) {
  cudaStream_t stream = d->stream;
  const int size = d->dtype == 0 ? 4 : 2;
  const long bytes = d->accumulate ? 0 : static_cast<long>(d->keys) * d->width * size;
  if (bytes > 0 && !aligned(d->grad)) return "embedding gradient: not on a 16-byte boundary";
  if (d->rows <= 0 || d->keys <= 0 || d->width <= 0) return bytes > 0 ? problem(cudaMemsetAsync(d->grad, 0, bytes, stream)) : nullptr;
  const int n = d->rows, bits = key_bits(d->keys);
  Keys k = {d->tokens, d->positions, n, d->vocab, d->keys, d->pad};
  char* at = static_cast<char*>(d->workspace);
  const auto take = [&](long b) { char* here = at; at += up16(b); return reinterpret_cast<int*>(here); };
  int *key[2], *row[2];
  for (int i = 0; i < 2; ++i) { key[i] = take(4L * n); row[i] = take(4L * n); }
  const int tiles = (n + kTile - 1) / kTile;
  int* counts = take(4L * tiles << kDigitBits);
  const int chunk = chunk_of(n), chunks = (n + chunk - 1) / chunk;
  int* joins = take(4L * (2 * chunks + 2));
  // whole vectors are cleared beside the sort, the last bytes by themselves
  Clear clear = {static_cast<uint4*>(d->accumulate ? nullptr : d->grad), bytes / 16, 0, 0, 0, 1};
  if (bytes % 16) {
    const cudaError_t e = cudaMemsetAsync(static_cast<char*>(d->grad) + bytes / 16 * 16, 0, bytes % 16, stream);
    if (e != cudaSuccess) return cudaGetErrorString(e);
  }
  int last = 0;
  cudaError_t e;
  const int blocks = (n + kRankRows - 1) / kRankRows;
  if (n <= kOneTile && bits + kRowBits <= 32) {
    const int grid = clear.next(blocks, 1);
    tile_rank_kernel<true><<<grid, 256, 0, stream>>>(k, kOneTile, nullptr, row[0], key[0], joins, clear);
    if ((e = cudaGetLastError()) != cudaSuccess) return cudaGetErrorString(e);
  } else if (n <= kPackedRows && bits + kRowBits <= 32) {
    const int smem = (n + kMergeTile - 1) / kMergeTile * kMergeTile * 4;
    if ((e = cudaFuncSetAttribute(merge_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPackedRows * 4)) != cudaSuccess)
      return cudaGetErrorString(e);
    uint32_t* const tiles = reinterpret_cast<uint32_t*>(key[1]);
    clear.of = 4;
    int grid = clear.next(blocks, 3);
    tile_rank_kernel<false><<<grid, 256, 0, stream>>>(k, kMergeTile, tiles, nullptr, nullptr, joins, clear);
    if ((e = cudaGetLastError()) != cudaSuccess) return cudaGetErrorString(e);
    grid = clear.next((n + kMergeRows - 1) / kMergeRows, 1);
    if (const char* err = launch_behind(true, merge_rank_kernel, grid, 256, smem, stream, tiles, n, row[0], key[0], clear)) return err;
  } else {
    const int passes = (bits + kDigitBits - 1) / kDigitBits, digit = (bits + passes - 1) / passes;
    const size_t smem = 8 * sizeof(int) << digit;
    clear.of = 2 * passes;               // none beside the scan: its loads would wait behind the writes (4 us without them, 31 with a fifth of 1 GB)
    for (int i = 0; i < passes; ++i) {
      Pass p = {i ? key[(i - 1) & 1] : nullptr, i ? row[(i - 1) & 1] : nullptr, key[i & 1], row[i & 1], counts, i * digit, digit, 1 << digit, tiles};
      int grid = clear.next(tiles, 1);
      const char* err = launch_behind(i > 0, radix_count_kernel, grid, 256, 0, stream, k, p, joins, clear);
      if (err) return err;
      if ((err = launch_behind(true, radix_scan_kernel, 1, 1024, 0, stream, counts, tiles << digit))) return err;
      grid = clear.next(tiles, 1);
      if ((err = launch_behind(true, radix_scatter_kernel, grid, 256, smem, stream, k, p, clear))) return err;
      last = i & 1;
    }
  }
  float* const parts = reinterpret_cast<float*>(take(8L * chunks * d->width));
  const Sum s = {row[last], key[last], d->dy, d->grad, parts, joins, n, d->keys, d->width, chunk, chunks, d->scale, d->p, d->seed, d->stream_id, d->seed_dev};
  if (d->dtype == 0) return sums_type<float>(s, d->accumulate, stream);
  if (d->dtype == 1) return sums_type<__nv_bfloat16>(s, d->accumulate, stream);
  if (d->dtype == 2) return sums_type<__half>(s, d->accumulate, stream);
  return "embedding gradient: the type must be fp32, bf16 or fp16";
}

const char* nmtg_embed_rows(const int64_t* tokens, const void* table, void* out, int rows, int vocab, int width, int dtype, float scale,
                            cudaStream_t stream) {
  if (rows <= 0 || width <= 0) return nullptr;
  if (vocab <= 0) return "embedding: the table is empty";
  if (dtype == 0) return gather<float>(tokens, table, out, rows, vocab, width, scale, stream);
  if (dtype == 1) return gather<__nv_bfloat16>(tokens, table, out, rows, vocab, width, scale, stream);
  if (dtype == 2) return gather<__half>(tokens, table, out, rows, vocab, width, scale, stream);
  return "embedding: the type must be fp32, bf16 or fp16";
}

NMTG_BOUNDS_READER(nmtg_bounds_embed_sorted)
