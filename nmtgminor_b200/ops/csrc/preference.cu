// Losses of preference tuning over rows of logits: log-probabilities of target words with their gradient, the clipped policy loss with a
// KL term, and the paired loss over summed log-probabilities (preferred against rejected).  With M = max x, s = sum exp((x - M) / T):
//     lp = (x[y] - M) / T - log s          d lp / d x = (onehot(y) - exp((x - M) / T) / s) / T
// Each loss is a function of the lp of its rows, so a row's gradient is one coefficient times d lp / d x.
//
// One kernel serves all of them (rows_kernel): a block, or a cluster of up to 8 blocks for a long row, takes a whole row, 32 elements of
// 16 bits (16 of 32 bits) a thread, so a row is read from memory once.  Every thread copies the vectors that it will itself use
// (cp.async, two rows ahead of the one in work), which needs no barrier but the one of the row's sum.  Blocks have as few threads as hold a
// row, 1024 threads to an SM in all: 64 KB of rows in work and 128 KB on their way.
//   * the policy loss knows its coefficient once the row is summed: exp((x - max of the thread) / T) stays in registers, and the gradient is
//     one multiplication; each logit is read once, its gradient written once, and one exponential taken (of 16 a cycle and SM, the sum
//     and the gradient together would take three quarters of the time that the row's bytes do).
//   * the paired loss knows it once every row of the pair is summed.  Work is handed out in one order, the sum of row i + lag before the
//     gradient of row i, lag = the longest pair and what is in work elsewhere; the gradient's read then comes from L2 where a
//     pair is small against it.  A gradient waits for its pair only (bounded), and whatever it waits for was handed out before it to a
//     block that runs: no order of blocks can lock.
// A row that no cluster holds is read twice (kLong).
//
// All sums over rows are taken in one order in 64 bits: results do not depend on which block was first.
// This file is compiled without fast math: expf and logf below are the accurate ones, ex2 where it is asked for.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include "b200_ptx.cuh"
#include "tuning_api.h"

namespace b200 {

int num_sms();

namespace {

constexpr int kVecs = 4;              // 16-byte vectors of a row that a thread holds
constexpr int kAhead = 2;             // rows on their way to shared memory
constexpr int kSlots = kAhead + 1;
constexpr int kMaxCluster = 8;
constexpr int kRing = 8;              // numbers of work items known ahead (kAhead + 3 needed)

enum Mode { kScores = 0, kGrad = 1, kPolicy = 2, kPairs = 3 };

struct PairState {          // the head of the workspace
  int ticket, longest, pairs_done, pairs_expected, failed;
};
struct PairWork {
  PairState* state;
  int* cu;                  // [2 pairs + 1] offsets, put in order and into range
  int* seq;                 // [rows] sequence of a row, -1: none
  int* label;               // [rows] label of a row, -1: padding
  int* arrived;             // [pairs] rows summed so far
  int* ready;               // [pairs] 1 once `coef` holds
  float* coef;              // [2 pairs] d loss / d lp of the rows of a sequence
  double* lp;               // [rows]
  double* loss;             // [pairs]
  int* ranked;              // [pairs]
  float2* stat;             // [rows]
};

struct Args {
  const void* x;
  void* g;
  const int64_t* labels;
  long ld, pad;
  int rows, vocab;
  float k, inv_t;           // log2(e) / T, 1 / T
  float* logprobs;
  float2* stat;
  const float* weight;
  const float* scale_at;    // the gradient's factor on the device, or null
  float scale;
  NmtgPolicy policy;
  NmtgPairs pairs;
  PairWork w;
  int slack;                // rows between a pair's end and the gradients taken up, beyond the longest pair
  int* status;
};

template <typename T> struct Num;
template <> struct Num<float> {
  static constexpr int kE = 4;
  static constexpr uint32_t kLow = 0xFF800000u;                   // -inf
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
};
template <> struct Num<__nv_bfloat16> {
  static constexpr int kE = 8;
  static constexpr uint32_t kLow = 0xFF80FF80u;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[2 * j] = __uint_as_float(w[j] << 16); f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u); }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint4 o;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    return o;
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <> struct Num<__half> {
  static constexpr int kE = 8;
  static constexpr uint32_t kLow = 0xFC00FC00u;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j) { const float2 t = __half22float2(h[j]); f[2 * j] = t.x; f[2 * j + 1] = t.y; }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint4 o;
    __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
    return o;
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void copy16(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
template <bool kCluster> __device__ __forceinline__ void meet() {
  if constexpr (kCluster) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
}

// sum of exponentials relative to a reference; a reference of -inf stands for no elements (or only -inf ones) and a sum of 0
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float k) {
  const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
  s = s * ex2((m - base) * k) + s2 * ex2((m2 - base) * k);
  m = top;
}
__device__ __forceinline__ void join_lanes(float& m, float& s, float k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), k);
}

// (x[y] - M) / T - log s in 64 bits; log s as exponent * log 2 + log of a mantissa near 1, whose 32-bit rounding is below 2^-25
__device__ __forceinline__ double log_probability(float xy, float m, float s, float inv_t) {
  const uint32_t bits = __float_as_uint(s);
  if (!(s > 0.f) || bits >= 0x7F800000u || bits < 0x00800000u) return (static_cast<double>(xy) - m) * inv_t - log(static_cast<double>(s));
  int e = static_cast<int>(bits >> 23) - 127;
  float f = __uint_as_float((bits & 0x007FFFFFu) | 0x3F800000u);
  if (f > 1.41421356f) { f *= 0.5f; ++e; }
  return (static_cast<double>(xy) - m) * inv_t - (e * 0.693147180559945309417 + static_cast<double>(logf(f)));
}

// a row as this block's part of it: vectors [v0, v1) after `head` single elements, `tail` single ones at the end
template <typename T> struct Span {
  const T* x;
  T* g;
  int head, tail, nvec, v0, v1;
  __device__ __forceinline__ Span(const Args& a, int row, uint32_t rank, uint32_t parts) {
    x = static_cast<const T*>(a.x) + static_cast<long>(row) * a.ld;
    g = a.g ? static_cast<T*>(a.g) + static_cast<long>(row) * a.ld : nullptr;
    head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)), a.vocab);
    nvec = (a.vocab - head) / Num<T>::kE;
    tail = a.vocab - head - nvec * Num<T>::kE;
    const int each = (nvec + static_cast<int>(parts) - 1) / static_cast<int>(parts);
    v0 = min(nvec, static_cast<int>(rank) * each);
    v1 = min(nvec, v0 + each);
  }
  __device__ __forceinline__ const uint4* xv() const { return reinterpret_cast<const uint4*>(x + head); }
  __device__ __forceinline__ uint4* gv() const { return reinterpret_cast<uint4*>(g + head); }
  // the single element of this thread, -1: none.  Threads 0..7 of the first block have the head, 8..15 of the last the tail.
  __device__ __forceinline__ int single(uint32_t rank, uint32_t parts) const {
    const int t = threadIdx.x;
    if (rank == 0 && t < head) return t;
    if (rank == parts - 1 && t >= 8 && t - 8 < tail) return head + nvec * Num<T>::kE + t - 8;
    return -1;
  }
};

// loss of pair p from the sums of its two sequences: one lane
__device__ __noinline__ void pair_loss(const Args& a, int p, double sw, double sl, int nw, int nl) {
  const NmtgPairs& q = a.pairs;
  q.seq_logprobs[2 * p] = static_cast<float>(sw);
  q.seq_logprobs[2 * p + 1] = static_cast<float>(sl);
  const double cw = q.average && nw > 0 ? 1.0 / nw : 1.0, cl = q.average && nl > 0 ? 1.0 / nl : 1.0;
  const double h = cw * (sw - (q.ref ? q.ref[2 * p] : 0.f)) - cl * (sl - (q.ref ? q.ref[2 * p + 1] : 0.f));
  double loss, slope;                        // slope: d loss / d h
  if (q.kind == 2) {
    const double d = h - 0.5 / q.beta;
    loss = d * d;
    slope = 2.0 * d;
  } else {
    const double z = q.beta * h - q.margin;
    if (q.kind == 1) {
      loss = z < 1.0 ? 1.0 - z : (z >= 1.0 ? 0.0 : z);             // the last: NaN
      slope = z < 1.0 ? -static_cast<double>(q.beta) : 0.0;
    } else {
      const double less = exp(-fabs(z)), soft = log1p(less), eps = q.smoothing;
      const double up = z >= 0.0 ? 1.0 / (1.0 + less) : less / (1.0 + less);      // sigmoid(z)
      loss = (1.0 - eps) * (soft + fmax(-z, 0.0)) + eps * (soft + fmax(z, 0.0));
      if (z != z) loss = z;
      const double down = z >= 0.0 ? less / (1.0 + less) : 1.0 / (1.0 + less);    // sigmoid(-z)
      slope = q.beta * (eps * up - (1.0 - eps) * down);
      if (z != z) slope = z;
    }
  }
  if (q.nll_weight != 0.f) loss -= q.nll_weight * cw * sw;
  a.w.coef[2 * p] = static_cast<float>(cw * (slope - q.nll_weight));
  a.w.coef[2 * p + 1] = static_cast<float>(-cl * slope);
  a.w.loss[p] = loss;
  a.w.ranked[p] = h > 0.0;
}

// all lanes of a warp, after the last pair
__device__ __noinline__ void total_loss(const Args& a) {
  __syncwarp();
  __threadfence();
  double loss = 0.0;
  int ranked = 0;
  for (int p = threadIdx.x & 31; p < a.pairs.pairs; p += 32) { loss += __ldcg(a.w.loss + p); ranked += __ldcg(a.w.ranked + p); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, o);
    ranked += __shfl_xor_sync(0xffffffffu, ranked, o);
  }
  if ((threadIdx.x & 31) == 0) { *a.pairs.loss = static_cast<float>(loss); *a.pairs.ranked = static_cast<float>(ranked); }
}

// all lanes of a warp, after the last row of pair p: sums in one order, coefficients, and at the last pair the loss
__device__ __noinline__ void finish_pair(const Args& a, int p) {
  __syncwarp();
  __threadfence();               // behind lane 0, which has counted the last arrival: the other blocks' rows
  const int lane = threadIdx.x & 31;
  double sum[2];
  int count[2];
  for (int h = 0; h < 2; ++h) {
    double s = 0.0;
    int n = 0;
    for (int r = a.w.cu[2 * p + h] + lane; r < a.w.cu[2 * p + h + 1]; r += 32) {
      s += __ldcg(a.w.lp + r);
      n += a.w.label[r] >= 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); n += __shfl_xor_sync(0xffffffffu, n, o); }
    sum[h] = s;
    count[h] = n;
  }
  int last = 0;
  if (lane == 0) {
    pair_loss(a, p, sum[0], sum[1], count[0], count[1]);
    __threadfence();
    atomicExch(a.w.ready + p, 1);
    last = atomicAdd(&a.w.state->pairs_done, 1) + 1 == a.w.state->pairs_expected;
    __threadfence();
  }
  if (__shfl_sync(0xffffffffu, last, 0)) total_loss(a);
}

// Work item: row and whether it is the gradient's turn; row -1: no more
struct Item { int row; bool grad; };
__device__ __forceinline__ Item pair_item(int t, int rows, int lag, bool grads) {
  if (!grads) return {t < rows ? t : -1, false};
  if (t < lag) return {t, false};
  if (t < 2 * rows - lag) { const int u = t - lag; return (u & 1) ? Item{u >> 1, true} : Item{lag + (u >> 1), false}; }
  return {t < 2 * rows ? t - rows : -1, true};
}

template <typename T, int kThreads, int kMode, bool kCluster, bool kLong>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) rows_kernel(const __grid_constant__ Args a) {
  constexpr int kE = Num<T>::kE, kWarps = kThreads / 32, kParts = kCluster ? kMaxCluster : 1;
  extern __shared__ __align__(16) uint4 slots[];            // [kSlots][kVecs][kThreads]
  __shared__ float2 part[2][kParts * kWarps];
  __shared__ float4 bc[2];                                  // largest logit, factor of the exponentials, coefficient / T
  __shared__ int ring[kRing];
  const uint32_t rank = kCluster ? cluster_rank() : 0, parts = kCluster ? cluster_size() : 1;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int groups = static_cast<int>(gridDim.x / parts), group = static_cast<int>(blockIdx.x / parts);
  const float scale = a.scale_at ? *a.scale_at * a.scale : a.scale;
  const int lag = kMode == kPairs ? min(a.rows, a.w.state->longest + a.slack) : 0;

  const auto item = [&](int i) -> Item {
    if constexpr (kMode == kPairs) {
      return pair_item(ring[i & (kRing - 1)], a.rows, lag, a.g != nullptr);
    } else {
      const long r = group + static_cast<long>(i) * groups;
      return {r < a.rows ? static_cast<int>(r) : -1, kMode == kGrad};
    }
  };
  const auto label_of = [&](int row) -> int {
    if (row < 0) return -1;
    if constexpr (kMode == kPairs) {
      return a.w.label[row];
    } else {
      const int64_t y = a.labels[row];
      return y == a.pad || y < 0 || y >= a.vocab ? -1 : static_cast<int>(y);
    }
  };
  const auto issue = [&](int i, int row, int label) {
    if constexpr (!kLong) {
      if (label >= 0) {
        const Span<T> s(a, row, rank, parts);
        uint4* to = slots + (i % kSlots) * (kVecs * kThreads) + t;
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
          if (s.v0 + t + j * kThreads < s.v1) copy16(to + j * kThreads, s.xv() + s.v0 + t + j * kThreads);
      }
      copies_end();
    }
  };
  const auto single_of = [&](int row) -> float {
    if (row < 0) return -INFINITY;
    const Span<T> s(a, row, rank, parts);
    const int e = s.single(rank, parts);
    return e >= 0 ? Num<T>::get(s.x[e]) : -INFINITY;
  };

  if constexpr (kCluster) meet<true>();     // every block of the cluster runs before the first store to its shared memory
  if constexpr (kMode == kPairs) {
    if (rank == 0 && t == 0) {
      const int first = atomicAdd(&a.w.state->ticket, kAhead + 2);
      for (int i = 0; i < kAhead + 2; ++i) {
        ring[i] = first + i;
        if constexpr (kCluster)
          for (uint32_t c = 1; c < parts; ++c) asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at_rank(ring + i, c)), "r"(first + i) : "memory");
      }
    }
  }
  if constexpr (kMode == kPairs) meet<kCluster>();
#pragma unroll
  for (int i = 0; i < kAhead; ++i) { const int r = item(i).row; issue(i, r, label_of(r)); }
  int label = label_of(item(0).row), label_ahead = label_of(item(kAhead).row);
  float one = single_of(item(0).row);

  for (int i = 0;; ++i) {
    const Item now = item(i);
    if (now.row < 0) break;
    const int row = now.row;
    int ticket = 0;
    if constexpr (kMode == kPairs)
      if (rank == 0 && t == 0) ticket = atomicAdd(&a.w.state->ticket, 1);
    issue(i + kAhead, item(i + kAhead).row, label_ahead);
    label_ahead = label_of(item(i + kAhead + 1).row);
    const int next = item(i + 1).row, next_label = label_of(next);
    const float next_one = single_of(next);

    const Span<T> s(a, row, rank, parts);
    const bool real = label >= 0;
    const bool grads = kMode == kPolicy || now.grad;
    const bool sums = kMode != kGrad && !now.grad;
    const float xy = real ? Num<T>::get(s.x[label]) : 0.f;
    uint4 raw[kLong ? 1 : kVecs];
    float e[kMode == kPolicy && !kLong ? kVecs * kE : 1];
    float m = -INFINITY, sum = 0.f;
    if constexpr (!kLong) {
      copies_wait<kAhead>();
      if (real) {
        const uint4* from = slots + (i % kSlots) * (kVecs * kThreads) + t;
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
          raw[j] = s.v0 + t + j * kThreads < s.v1 ? from[j * kThreads] : make_uint4(Num<T>::kLow, Num<T>::kLow, Num<T>::kLow, Num<T>::kLow);
      }
    }
    if (real && sums) {
      if constexpr (kLong) {
        for (int v = s.v0 + t; v < s.v1; v += kThreads) {
          const uint4 u = s.xv()[v];
          float f[kE], add = 0.f;
          Num<T>::unpack(u, f);
          const float top = fmaxf(m, Num<T>::largest(u)), base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int q = 0; q < kE; ++q) add += ex2((f[q] - base) * a.k);
          sum = sum * ex2((m - base) * a.k) + add;
          m = top;
        }
        join(m, sum, one, one == -INFINITY ? 0.f : ex2((one - one) * a.k), a.k);
      } else {
        m = one;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) m = fmaxf(m, Num<T>::largest(raw[j]));
        const float base = m == -INFINITY ? 0.f : m;
        sum = ex2((one - base) * a.k);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          float f[kE], add = 0.f;
          Num<T>::unpack(raw[j], f);
#pragma unroll
          for (int q = 0; q < kE; ++q) {
            const float v = ex2((f[q] - base) * a.k);
            if constexpr (kMode == kPolicy) e[j * kE + q] = v;
            add += v;
          }
          sum += add;
        }
      }
    }
    const float mine = m;              // reference of this thread's exponentials
    float2* const meeting = part[i & 1];
    if constexpr (kMode != kGrad) {
      if (sums) {
        join_lanes(m, sum, a.k);
        if (lane == 0) {
          const int at = static_cast<int>(rank) * kWarps + warp;
          if constexpr (kCluster) {
            for (uint32_t c = 0; c < parts; ++c)
              asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at_rank(meeting + at, c)), "f"(m), "f"(sum) : "memory");
          } else {
            meeting[at] = make_float2(m, sum);
          }
        }
      }
      if constexpr (kMode == kPairs) {
        if (t == 0 && now.grad && real) {
          const int q = a.w.seq[row], p = q >> 1;
          bool ok = false;
#pragma unroll 1
          for (uint32_t polls = 0; polls < B200_WAIT_POLLS; ++polls) {
            if (ld_acquire_gpu(a.w.ready + p)) { ok = true; break; }
            if ((polls & 63) == 63 && ld_acquire_gpu(&a.w.state->failed)) break;        // one wait in vain is enough
            __nanosleep(polls > 4096 ? 256 : 32);
          }
          if (!ok) { atomicExch(&a.w.state->failed, 1); atomicCAS(a.status, 0, static_cast<int>(kTimeoutPair)); }
          const float2 st = __ldcg(a.w.stat + row);
          const float c = __ldcg(a.w.coef + q) * a.inv_t * scale;
          bc[i & 1] = make_float4(st.x, c / st.y, c, 0.f);
        }
        if (rank == 0 && t == 0) {
          ring[(i + kAhead + 2) & (kRing - 1)] = ticket;
          if constexpr (kCluster)
            for (uint32_t c = 1; c < parts; ++c)
              asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at_rank(ring + ((i + kAhead + 2) & (kRing - 1)), c)), "r"(ticket) : "memory");
        }
      }
      meet<kCluster>();
      if (sums && warp == 0 && (kMode == kPolicy || rank == 0)) {
        m = -INFINITY;
        sum = 0.f;
        for (int j = lane; j < static_cast<int>(parts) * kWarps; j += 32) join(m, sum, meeting[j].x, meeting[j].y, a.k);
        join_lanes(m, sum, a.k);
        const double lp = real ? log_probability(xy, m, sum, a.inv_t) : 0.0;
        if constexpr (kMode == kScores) {
          if (lane == 0) {
            a.logprobs[row] = static_cast<float>(lp);
            if (a.stat) a.stat[row] = real ? make_float2(m, sum) : make_float2(0.f, 1.f);
          }
        } else if constexpr (kMode == kPairs) {
          const int q = a.w.seq[row];
          int last = 0;
          if (lane == 0) {
            a.w.lp[row] = lp;
            a.w.stat[row] = make_float2(m, sum);
            __threadfence();
            if (q >= 0) last = atomicAdd(a.w.arrived + (q >> 1), 1) + 1 == a.w.cu[(q | 1) + 1] - a.w.cu[q & ~1];
            __threadfence();
          }
          if (__shfl_sync(0xffffffffu, last, 0)) finish_pair(a, q >> 1);
        } else if (lane == 0) {
          double loss = 0.0, kl = 0.0, clipped = 0.0;
          float coef = 0.f;
          if (real) {
            const float adv = a.policy.advantages[row];
            const float ratio = expf(static_cast<float>(lp - a.policy.old_logprobs[row]));
            const float held = fminf(fmaxf(ratio, a.policy.clip_low), a.policy.clip_high);
            const bool free = !(ratio * adv > held * adv);         // NaN counts as free, so that it shows
            coef = free ? -ratio * adv : 0.f;
            loss = -static_cast<double>(free ? ratio : held) * adv;
            clipped = free ? 0.0 : 1.0;
            if (a.policy.ref_logprobs) {
              const double d = a.policy.ref_logprobs[row] - lp;
              const float up = expm1f(static_cast<float>(d));
              kl = static_cast<double>(up) - d;
              loss += a.policy.kl_coef * kl;
              coef -= a.policy.kl_coef * up;
            }
          }
          const float c = coef * a.inv_t * scale;
          bc[i & 1] = make_float4(m, c / sum, c, 0.f);
          if (rank == 0) {
            a.logprobs[row] = static_cast<float>(lp);
            a.policy.row_loss[row] = loss;
            a.policy.row_loss[a.rows + static_cast<long>(row)] = kl;
            a.policy.row_loss[2 * static_cast<long>(a.rows) + row] = clipped;
          }
        }
      }
      if constexpr (kMode == kPolicy) __syncthreads();
    }
    if (grads && s.g) {
      float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
      if (real) {
        if constexpr (kMode == kGrad) {
          const float2 st = a.stat[row];
          const float w = a.weight[row] * a.inv_t;
          c = make_float4(st.x, w / st.y, w, 0.f);
        } else {
          c = bc[i & 1];
        }
      }
      uint4* const out = s.gv();
      if (!real) {
        for (int v = s.v0 + t; v < s.v1; v += kThreads) __stcs(out + v, make_uint4(0, 0, 0, 0));
      } else if constexpr (kLong) {
        for (int v = s.v0 + t; v < s.v1; v += kThreads) {
          float f[kE];
          Num<T>::unpack(s.xv()[v], f);
#pragma unroll
          for (int q = 0; q < kE; ++q) f[q] = -c.y * ex2((f[q] - c.x) * a.k);
          __stcs(out + v, Num<T>::pack(f));
        }
      } else {
        const float own = kMode == kPolicy ? -c.y * ex2((mine - c.x) * a.k) : -c.y;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          float f[kE];
          if constexpr (kMode == kPolicy) {
#pragma unroll
            for (int q = 0; q < kE; ++q) f[q] = own * e[j * kE + q];
          } else {
            Num<T>::unpack(raw[j], f);
#pragma unroll
            for (int q = 0; q < kE; ++q) f[q] = own * ex2((f[q] - c.x) * a.k);
          }
          if (s.v0 + t + j * kThreads < s.v1) __stcs(out + s.v0 + t + j * kThreads, Num<T>::pack(f));
        }
      }
      const int e1 = s.single(rank, parts);
      if (e1 >= 0) s.g[e1] = Num<T>::put(real ? (e1 == label ? c.z : 0.f) - c.y * ex2((one - c.x) * a.k) : 0.f);
      if (real) {                       // the label's element again, by the thread that has just written its vector
        const int v = label >= s.head ? (label - s.head) / kE : s.nvec;
        if (v >= s.v0 && v < s.v1 && (v - s.v0) % kThreads == t) s.g[label] = Num<T>::put(c.z - c.y * ex2((xy - c.x) * a.k));
      }
    }
    label = next_label;
    one = next_one;
  }
  if constexpr (!kLong) copies_wait<0>();
  if constexpr (kCluster) meet<true>();     // no block leaves while another may still write to it
}

// Offsets put in order, rows' sequences and labels, the longest pair; pairs without rows get their loss here.  One block: 8 bytes a row
// against the kilobytes that the row has.
__global__ void __launch_bounds__(1024) pairs_setup_kernel(const __grid_constant__ Args a) {
  __shared__ int warp_top[32];
  __shared__ int carry, longest, empty;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = 2 * a.pairs.pairs + 1;
  if (t == 0) { carry = 0; longest = 0; empty = 0; }
  __syncthreads();
  for (int base = 0; base < n; base += 1024) {                 // running maximum of the offsets
    int v = base + t < n ? min(max(a.pairs.cu[base + t], 0), a.rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v = max(v, u); }
    if (lane == 31) warp_top[warp] = v;
    __syncthreads();
    v = max(v, carry);
    for (int w = 0; w < warp; ++w) v = max(v, warp_top[w]);
    if (base + t < n) a.w.cu[base + t] = v;
    __syncthreads();
    if (t == 1023) carry = v;
    __syncthreads();
  }
  const int first = a.w.cu[0], end = a.w.cu[n - 1];
  for (int r = t; r < a.rows; r += 1024)
    if (r < first || r >= end) { a.w.seq[r] = -1; a.w.label[r] = -1; }
  for (int q = warp; q < n - 1; q += 32)
    for (int r = a.w.cu[q] + lane; r < a.w.cu[q + 1]; r += 32) {
      const int64_t y = a.labels[r];
      a.w.seq[r] = q;
      a.w.label[r] = y == a.pad || y < 0 || y >= a.vocab ? -1 : static_cast<int>(y);
    }
  for (int p = t; p < a.pairs.pairs; p += 1024) {
    const int rows = a.w.cu[2 * p + 2] - a.w.cu[2 * p];
    a.w.arrived[p] = 0;
    a.w.ready[p] = 0;
    if (rows == 0) { pair_loss(a, p, 0.0, 0.0, 0, 0); atomicAdd(&empty, 1); }
    atomicMax(&longest, rows);
  }
  __syncthreads();
  if (t == 0) *a.w.state = PairState{0, longest, empty, a.pairs.pairs, 0};
  if (empty == a.pairs.pairs && warp == 0) {
    __threadfence();
    total_loss(a);
  }
}

// a block for each of the sums of v[0 .. 3, 0 .. n), in one order
__global__ void __launch_bounds__(1024) sum_rows_kernel(const double* __restrict__ v, int n, float* out0, float* out1, float* out2) {
  __shared__ double warps[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += v[static_cast<long>(blockIdx.x) * n + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warps[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *(blockIdx.x == 0 ? out0 : blockIdx.x == 1 ? out1 : out2) = static_cast<float>(s);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) scale_rows_kernel(const Args a, const float* __restrict__ factor) {
  constexpr int kE = Num<T>::kE;
  const float f = *factor;
  if (f == 1.f) return;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const Span<T> s(a, r, 0, 1);
    for (int v = threadIdx.x; v < s.nvec; v += 256) {
      float g[kE];
      Num<T>::unpack(s.gv()[v], g);
#pragma unroll
      for (int q = 0; q < kE; ++q) g[q] *= f;
      s.gv()[v] = Num<T>::pack(g);
    }
    const int one = s.single(0, 1);
    if (one >= 0) s.g[one] = Num<T>::put(Num<T>::get(s.g[one]) * f);
  }
}

const char* problem(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

template <typename T, int kThreads, int kMode, bool kCluster, bool kLong>
const char* launch_rows(Args a, int parts, long items, cudaStream_t stream) {
  auto kernel = rows_kernel<T, kThreads, kMode, kCluster, kLong>;
  const size_t smem = kLong ? 0 : static_cast<size_t>(kSlots) * kVecs * kThreads * 16;
  // how many groups of blocks the GPU holds; all GPUs of a machine are alike
  static int groups[kMaxCluster + 1] = {};
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCluster ? 1 : 0;
  // the attribute belongs to a device's context: set at every call, which costs less than keeping account of the devices
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return cudaGetErrorString(e);
  int held = groups[parts];
  if (held == 0) {
    if (kCluster) {
      cfg.gridDim = dim3(parts);
      e = cudaOccupancyMaxActiveClusters(&held, kernel, &cfg);
    } else {
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, kThreads, smem);
      held *= num_sms();
    }
    if (e != cudaSuccess) return cudaGetErrorString(e);
    if (held < 1) return "preference: no block of this shape fits the GPU";
    groups[parts] = held;
  }
  const long g = items < held ? items : held;
  a.slack = 2 * held;
  cfg.gridDim = dim3(static_cast<unsigned>(g * parts));
  e = cudaLaunchKernelEx(&cfg, kernel, a);
  return problem(e);
}

template <typename T, int kMode>
const char* launch_mode(const Args& a, long items, cudaStream_t stream) {
  constexpr int kEach = kVecs * Num<T>::kE;                 // elements of a thread
  if (a.vocab <= 32 * kEach) return launch_rows<T, 32, kMode, false, false>(a, 1, items, stream);
  if (a.vocab <= 128 * kEach) return launch_rows<T, 128, kMode, false, false>(a, 1, items, stream);
  if (a.vocab <= 256 * kEach) return launch_rows<T, 256, kMode, false, false>(a, 1, items, stream);
  if (a.vocab <= 512 * kEach) return launch_rows<T, 512, kMode, false, false>(a, 1, items, stream);
  if (a.vocab <= 1024 * kEach) return launch_rows<T, 1024, kMode, false, false>(a, 1, items, stream);
  for (int parts = 2; parts <= kMaxCluster; parts *= 2)
    if (a.vocab <= parts * 1024 * kEach) return launch_rows<T, 1024, kMode, true, false>(a, parts, items, stream);
  return launch_rows<T, 1024, kMode, true, true>(a, kMaxCluster, items, stream);
}

template <int kMode>
const char* launch_type(const Args& a, int dtype, long items, cudaStream_t stream) {
  if (a.rows <= 0) return nullptr;
  if (dtype == 0) return launch_mode<float, kMode>(a, items, stream);
  if (dtype == 1) return launch_mode<__nv_bfloat16, kMode>(a, items, stream);
  if (dtype == 2) return launch_mode<__half, kMode>(a, items, stream);
  return "preference: logits must be fp32, bf16 or fp16";
}

Args row_args(const NmtgRows* r) {
  Args a = {};
  a.x = r->logits; a.g = r->grad; a.labels = r->labels; a.ld = r->ld; a.pad = r->pad; a.rows = r->rows; a.vocab = r->vocab;
  a.inv_t = r->inv_temperature; a.k = static_cast<float>(1.4426950408889634074 * r->inv_temperature);
  a.scale_at = r->grad_scale_at; a.scale = r->grad_scale;
  a.logprobs = r->logprobs; a.stat = r->stat; a.status = r->status;
  return a;
}

long up16(long n) { return (n + 15) & ~15L; }

}  // namespace
}  // namespace b200

using namespace b200;

const char* nmtg_row_scores(const NmtgRows* r, cudaStream_t stream) {
  return launch_type<kScores>(row_args(r), r->dtype, r->rows, stream);
}

const char* nmtg_row_scores_grad(const NmtgRows* r, const float* weight, cudaStream_t stream) {
  Args a = row_args(r);
  a.weight = weight;
  return launch_type<kGrad>(a, r->dtype, r->rows, stream);
}

const char* nmtg_policy_loss(const NmtgRows* r, const NmtgPolicy* p, cudaStream_t stream) {
  Args a = row_args(r);
  a.policy = *p;
  const char* err = launch_type<kPolicy>(a, r->dtype, r->rows, stream);
  if (err) return err;
  sum_rows_kernel<<<3, 1024, 0, stream>>>(p->row_loss, r->rows, p->loss, p->kl, p->clipped);
  return problem(cudaGetLastError());
}

long nmtg_pairs_workspace(int rows, int pairs) {
  const long r = rows, p = pairs;
  return up16(sizeof(PairState)) + up16(4 * (2 * p + 1)) + 2 * up16(4 * r) + 3 * up16(4 * p) + up16(8 * p) + up16(8 * r) + up16(8 * p) + up16(8 * r);
}

const char* nmtg_preference_loss(const NmtgRows* r, const NmtgPairs* p, cudaStream_t stream) {
  Args a = row_args(r);
  a.pairs = *p;
  char* at = static_cast<char*>(p->workspace);
  const auto take = [&](long bytes) { char* here = at; at += up16(bytes); return static_cast<void*>(here); };
  const long rows = r->rows, pairs = p->pairs;
  a.w.state = static_cast<PairState*>(take(sizeof(PairState)));
  a.w.cu = static_cast<int*>(take(4 * (2 * pairs + 1)));
  a.w.seq = static_cast<int*>(take(4 * rows));
  a.w.label = static_cast<int*>(take(4 * rows));
  a.w.arrived = static_cast<int*>(take(4 * pairs));
  a.w.ready = static_cast<int*>(take(4 * pairs));
  a.w.ranked = static_cast<int*>(take(4 * pairs));
  a.w.coef = static_cast<float*>(take(8 * pairs));
  a.w.lp = static_cast<double*>(take(8 * rows));
  a.w.loss = static_cast<double*>(take(8 * pairs));
  a.w.stat = static_cast<float2*>(take(8 * rows));
  pairs_setup_kernel<<<1, 1024, 0, stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cudaGetErrorString(e);
  return launch_type<kPairs>(a, r->dtype, (r->grad ? 2L : 1L) * rows, stream);
}

const char* nmtg_scale_rows(const NmtgRows* r, const float* factor, cudaStream_t stream) {
  if (r->rows <= 0 || r->vocab <= 0) return nullptr;
  Args a = row_args(r);
  a.x = a.g;
  const int grid = r->rows < 8 * num_sms() ? r->rows : 8 * num_sms();
  if (r->dtype == 0) scale_rows_kernel<float><<<grid, 256, 0, stream>>>(a, factor);
  else if (r->dtype == 1) scale_rows_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a, factor);
  else scale_rows_kernel<__half><<<grid, 256, 0, stream>>>(a, factor);
  return problem(cudaGetLastError());
}
