// Losses of preference tuning over rows of logits: log-probabilities of target words with their gradient, the clipped policy loss with a
// KL term, and the paired loss over summed log-probabilities (preferred against rejected).  With M = max x, s = sum exp((x - M) / T):
//     lp = (x[y] - M) / T - log s          d lp / d x = (onehot(y) - exp((x - M) / T) / s) / T
// Each loss is a function of the lp of its rows, so a row's gradient is one coefficient times d lp / d x.
//
// The policy loss is one pass, a warp, a block or a cluster of blocks to a row, which they hold (rows of up to 896 KB).  Scores of rows in one
// piece are one pass, too.  The paired loss, and the scores and the policy loss of longer rows, are two passes over pieces of rows, sums (sums_kernel, rows_kernel) and
// then gradients (rows_kernel), with a small kernel between that makes rows of the pieces and coefficients of the rows.  (Both at once, the
// gradients some rows behind the sums so that they would find the logits in L2, were built and measured: 353 us against 272 for 8200 rows of 32000 in bf16.
// The coefficient of a pair comes so late that most blocks wait for it.)
// Bound by memory in 32 bits, in every gradient pass and where one pass does all.  The sums of 16-bit logits, two exponentials to a 32-bit word, keep the
// memory at 0.8 of its rate and the exponentials (16 a cycle and SM) at 0.7 of theirs.
// 8200 rows of 32000 in bf16: scores 96 us (floor 81), gradients 165 (163), paired loss 255 (163, of the two passes 244); policy loss of
// 15360 rows 317 (305).  Called without a pause for seconds the policy loss reaches the card's power limit (1014 W, 1620 MHz): 382 us then, the paired loss 260.
//
// All sums over rows are taken in one order in 64 bits: results do not depend on which block was first.
// This file is compiled without fast math: expf and logf below are the accurate ones, ex2 where it is asked for.
// Exponentials, ratios and a row's coefficient are in 32 bits, off by 2^-16 and less: for 16-bit results far below their rounding, for fp32 logits a choice,
// since a row's sum has no more than 2^-19 itself.  Log-probabilities are held in two floats, what is summed of them (scores, losses, KL terms) in 64 bits.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <atomic>
#include <climits>
#include <stdint.h>
#include "b200_ptx.cuh"
#include "launch.cuh"
#include "tuning_api.h"

namespace b200 {


namespace {

constexpr int kVecs = 8;              // 16-byte vectors of an item that a thread holds
constexpr int kSlots = 3;             // items in shared memory or on their way there
constexpr int kRing = 8;              // entries of work known: one behind, kSlots + 3 ahead, and that in hand
constexpr int kFirst = 6;             // items of a block that it need not ask for
constexpr int kBlock = 256, kWide = 512;      // threads of a block for the elements; two or three blocks to an SM, and one
constexpr int kHeldBytes = 112 * 1024;        // of a row that a block holds, two blocks to an SM

// kScores: sums of pieces.  kGrad: gradients from `stat` and a coefficient.  kLocal: the policy loss of rows that a warp holds.
enum Mode { kScores = 0, kGrad = 1, kLocal = 2 };

struct State { int tickets[2], pairs_done; };      // items asked for in the two passes
struct Work {
  State* state;
  int* ticket;              // of this pass, 0 before it; null where every item has its block or warp
  float2* part;             // [rows][pieces] largest logit, sum of exponentials
  float2* stat;             // [rows] the same of a row
  float* coef;              // [2 pairs] or [rows]: d loss / d lp
  int* cu;                  // [2 pairs + 1] offsets, put in order and into range
  int* seq;                 // [rows] sequence of a row, -1: none
  int* label;               // [rows] label of a row, -1: padding
  double* lp;               // [rows]
  double* loss;             // [pairs]
  int* ranked;              // [pairs]
};

struct Args {
  const void* x;
  void* g;
  const int64_t* labels;
  long ld, pad;
  int rows, vocab;
  int pieces, each;         // of a row; vectors of a piece
  int slot;                 // vectors of a slot
  int behind;               // launched while the kernel before it ends
  int stays;                // rows that are to stay in L2 after the sums
  int aligned;              // every row starts on a 16-byte boundary
  float k, inv_t;           // log2(e) / T, 1 / T
  float* logprobs;
  float2* stat;
  const float* weight;      // kGrad: of rows or, where `w.seq` is there, of sequences
  const float* scale_at;    // the gradient's factor on the device, or null
  float scale;
  NmtgPolicy policy;
  NmtgPairs pairs;
  Work w;
};

template <typename T> struct Num;
template <> struct Num<float> {
  static constexpr int kE = 4;
  static constexpr uint32_t kLow = 0xFF800000u;                   // -inf
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
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
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    uint4 o;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[j].x, f[j].y);
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
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __half22float2(h[j]);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    uint4 o;
    __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[j].x, f[j].y);
    return o;
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

// 2^v; below 2^-126 zero: 2^-126 of a sum that is at least 1
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// two 32-bit operations in one instruction
__device__ __forceinline__ uint64_t both(float2 v) { return *reinterpret_cast<const uint64_t*>(&v); }
__device__ __forceinline__ float2 each(uint64_t v) { return *reinterpret_cast<const float2*>(&v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return each(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return each(r);
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void copy16(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
// Rows are gone through from the last to the first where they are read first.  The gradients behind the sums go from the first to the last, and find in L2
// what the sums read last, the first `stays` rows; the others pass through it first out.
// (Paired loss of 8200 rows of 32000 in bf16: 276 us with both in one order, 273 in opposite ones, 261 so; 8200 rows of 8000 in fp32 151, 144, 136.
// 48 to 80 MB alike, 112 of the 126 that L2 has 2 % slower.  From the last row rather than from the first, since what writes logits row by row leaves the last
// rows in L2: behind a copy scores of the 8200 rows 94 us, from the first row 102.  The output layer's product leaves the last columns of all rows
// there, and either order takes 98 behind it, the paired loss 258.)
constexpr long kStaying = 48L << 20;
__device__ __forceinline__ uint64_t policy_of(bool stay) {
  uint64_t first, normal;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
  return stay ? normal : first;
}
__device__ __forceinline__ void copy16(uint4* to, const uint4* from, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "l"(policy) : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy8(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
// sum of exponentials relative to a reference; a reference of -inf stands for no elements (or only -inf ones) and a sum of 0
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float k) {
  const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
  s = s * ex2((m - base) * k) + s2 * ex2((m2 - base) * k);
  m = top;
}
__device__ __forceinline__ void join_lanes(float& m, float& s, float k) {
  const float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  s *= ex2((m - base) * k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = top;
}
// exponentials of a vector relative to a reference: 2^((x - base) k)
template <typename T>
__device__ __forceinline__ void exps(const uint4& u, float minus_base, float k, float2 (&e)[Num<T>::kE / 2]) {
  Num<T>::unpack(u, e);
#pragma unroll
  for (int q = 0; q < Num<T>::kE / 2; ++q) {
    const float2 v = mul2(add2(e[q], make_float2(minus_base, minus_base)), make_float2(k, k));
    e[q] = make_float2(ex2(v.x), ex2(v.y));
  }
}

// A log-probability (x[y] - M) / T - log s as a sum of two floats: log s is an exponent times log 2, whose upper part has 15 bits so that the product is
// exact, and the log of a mantissa near 1, whose rounding is below 2^-26; the rounding of the sum of the large terms is kept.
struct LogProb {
  float hi, lo;
  __device__ __forceinline__ double wide() const { return static_cast<double>(hi) + lo; }
  __device__ __forceinline__ float minus(float v) const { return (hi - v) + lo; }
};
__device__ __forceinline__ LogProb log_probability(float xy, float m, float s, float inv_t) {
  const float t = (xy - m) * inv_t;
  if (!(s > 0.f && s < 3e38f)) return LogProb{t - logf(s), 0.f};           // nothing but -inf, or NaN
  const uint32_t bits = __float_as_uint(s);
  int e = static_cast<int>(bits >> 23) - 127;
  float f = __uint_as_float((bits & 0x007FFFFFu) | 0x3F800000u);
  if (f > 1.41421356f) { f *= 0.5f; ++e; }
  const float n = static_cast<float>(-e), big = n * 0.693145751953125f;     // log 2 = 0.693145751953125 + 1.42860682030941723e-6
  const float hi = t + big, back = hi - t, lost = (t - (hi - back)) + (big - back);
  const float lo = lost + fmaf(n, 1.42860682e-6f, -logf(f)), sum = hi + lo;
  return fabsf(hi) < INFINITY ? LogProb{sum, lo - (sum - hi)} : LogProb{hi, 0.f};
}

// A piece of a row: vectors [v0, v1) behind `head` single elements; `tail` single ones follow the row's last vector.
struct Shape { int head, tail, nvec, v0, v1; };
template <typename T>
__device__ __forceinline__ Shape shape_of(const Args& a, const T* x, int piece) {
  Shape s;
  s.head = a.aligned ? 0 : min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)), a.vocab);
  s.nvec = (a.vocab - s.head) / Num<T>::kE;
  s.tail = a.vocab - s.head - s.nvec * Num<T>::kE;
  s.v0 = min(s.nvec, piece * a.each);
  s.v1 = min(s.nvec, s.v0 + a.each);
  return s;
}
// The single element of this thread, -1: none.  Threads 0..7 have the head with the first piece, 8..15 the tail with the last.
template <typename T>
__device__ __forceinline__ int single_at(const Shape& s, int thread, int piece, int pieces) {
  if (piece == 0 && thread < s.head) return thread;
  if (piece == pieces - 1 && thread >= 8 && thread - 8 < s.tail) return s.head + s.nvec * Num<T>::kE + thread - 8;
  return -1;
}

// a row's sums from those of its pieces
__device__ __forceinline__ void join_pieces(const Args& a, int row, float& m, float& s) {
  const float2* const at = a.w.part + static_cast<long>(row) * a.pieces;
  for (int p = 0; p < a.pieces; p += 8) {
    float2 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p + j < a.pieces ? at[p + j] : make_float2(-INFINITY, 0.f);      // several on their way at a time
#pragma unroll
    for (int j = 0; j < 8; ++j) join(m, s, v[j].x, v[j].y, a.k);
  }
}

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
      slope = z < 1.0 ? -static_cast<double>(q.beta) : (z >= 1.0 ? 0.0 : z);      // so that NaN shows, as under the other kinds
    } else {
      const double less = exp(-fabs(z)), soft = log1p(less), eps = q.smoothing;
      const double up = z >= 0.0 ? 1.0 / (1.0 + less) : less / (1.0 + less);      // sigmoid(z)
      loss = (1.0 - eps) * (soft + fmax(-z, 0.0));
      if (eps != 0.0) loss += eps * (soft + fmax(z, 0.0));                        // without smoothing a pair at z = inf costs 0, not 0 * inf
      if (z != z) loss = z;
      const double down = z >= 0.0 ? less / (1.0 + less) : 1.0 / (1.0 + less);    // sigmoid(-z)
      slope = q.beta * (eps * up - (1.0 - eps) * down);
      if (z != z) slope = z;
    }
  }
  if (q.nll_weight != 0.f) loss -= q.nll_weight * cw * sw;
  a.w.loss[p] = loss;
  a.w.ranked[p] = h > 0.0;
  a.w.coef[2 * p] = static_cast<float>(cw * (slope - q.nll_weight));
  a.w.coef[2 * p + 1] = static_cast<float>(-cl * slope);
}

// An item of work, a piece of a row.  row -1: no more; label -1: padding.
struct __align__(16) Entry { int row, piece, label, unused; };
// What the last warp needs of an entry
struct __align__(16) Mail {
  union { int64_t label; int label32; };
  float2 stat;
  uint32_t word, upper;     // the label's logit, of 16 bits the upper half where `upper`
  int seq;
  float weight;
};

// d loss / d lp of a row under the policy loss
__device__ __forceinline__ float policy_coef(const Args& a, LogProb lp, float old, float adv, float ref) {
  const float ratio = expf(lp.minus(old)), held = fminf(fmaxf(ratio, a.policy.clip_low), a.policy.clip_high);
  const bool free = !(ratio * adv > held * adv);           // NaN counts as free, so that it shows
  const float up = a.policy.ref_logprobs && a.policy.kl_coef != 0.f ? expm1f(-lp.minus(ref)) : 0.f;        // a KL term that is only reported may be infinite
  return (free ? -ratio * adv : 0.f) - a.policy.kl_coef * up;
}

// kCompute threads do the elements' work; one more warp fetches the entries, joins the partial sums and brings the coefficients.  Step i of the
// block: the sums of entry i and the barrier (kScores), or the barrier and the gradient of entry i - 1, its logits in their slot (kGrad).  Between barriers
// i - 1 and i the last warp joins the sums of entry i - 1, or brings its coefficient, and publishes entry i + kLead + 1.
template <typename T, int kCompute, int kMode>
__global__ void __launch_bounds__(kCompute + 32, kCompute == kBlock ? 3 : 1) rows_kernel(const __grid_constant__ Args a) {
  constexpr int kE = Num<T>::kE, kWarps = kCompute / 32;
  constexpr bool kSums = kMode == kScores, kGrads = kMode == kGrad;
  constexpr int kLead = kMode == kScores ? kSlots : kSlots - 1;             // entries whose logits are under way
  extern __shared__ __align__(16) uint4 slots[];            // [kSlots][a.slot]
  if (a.behind) wait_for_previous();
  if (kMode == kScores && a.w.part) let_next_start();
  __shared__ float2 part[2][kWarps];
  __shared__ float4 bc[2];                                  // largest logit, factor of the exponentials, coefficient / T
  __shared__ Entry ring[kRing];
  __shared__ Mail mail[kRing];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* const x0 = static_cast<const T*>(a.x);
  T* const g0 = static_cast<T*>(a.g);

  if (warp == kWarps) {
    // ------------------------------------------------------------------------------------------------ the last warp
    const float scale = a.scale_at ? *a.scale_at * a.scale : a.scale;
    const bool whole = kMode == kScores && !a.w.part;        // an item is a row, and its log-probability wanted
    // What an entry needs comes by asynchronous copies, so that this warp never waits for memory: at step i the label of entry i + kLead + 3, at step
    // i + 2, when its label is there and the entry is published, its logit and the numbers of its row.
    // A block's first kFirst items are its own, the others are handed out one by one, asked for a step ahead: SMs do not get at memory equally fast,
    // and equal shares would wait for the slowest (sums of 8200 rows of 32000: most blocks done after 87 us, the last after 111).
    const auto next_number = [&](int i) -> int {              // of entry i
      if (i < kFirst) return static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
      return a.w.ticket ? kFirst * static_cast<int>(gridDim.x) + atomicAdd(a.w.ticket, 1) : a.rows * a.pieces;
    };
    const auto ask = [&](int i, int number) {                 // lane 0
      const int items = a.rows * a.pieces, n = kMode == kScores ? items - 1 - number : number, q = a.pieces == 1 ? n : n / a.pieces;
      const Entry e = {number < items ? q : -1, n - q * a.pieces, -1, 0};
      Mail& m = mail[i & (kRing - 1)];
      if (e.row < 0) m.label = -1;
      else if (a.w.label) copy4(&m.label32, a.w.label + e.row);
      else copy8(&m.label, a.labels + e.row);
      if (kMode == kGrad && e.row >= 0 && a.w.seq) copy4(&m.seq, a.w.seq + e.row);
      ring[i & (kRing - 1)] = e;
    };
    const auto publish = [&](int i) {                         // lane 0
      Mail& m = mail[i & (kRing - 1)];
      Entry e = ring[i & (kRing - 1)];
      if (e.row >= 0) {
        if (a.w.label) e.label = m.label32;
        else e.label = m.label == a.pad || m.label < 0 || m.label >= a.vocab ? -1 : static_cast<int>(m.label);
      }
      ring[i & (kRing - 1)] = e;
      if (e.label >= 0) {
        if (whole) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(x0 + static_cast<long>(e.row) * a.ld + e.label);
          m.upper = at & 2;
          copy4(&m.word, reinterpret_cast<const void*>(at & ~static_cast<uintptr_t>(3)));
        }
        if constexpr (kMode == kGrad) {
          copy8(&m.stat, a.stat + e.row);
          copy4(&m.weight, a.weight + (a.w.seq ? m.seq : e.row));
        }
      }
    };
    const auto logit_of = [&](const Mail& m) -> float {
      if constexpr (sizeof(T) == 4) return __uint_as_float(m.word);
      else return Num<T>::get(reinterpret_cast<const T*>(&m.word)[m.upper ? 1 : 0]);
    };
    int fresh = 0;                                           // the number of entry i + kLead + 3
    if (lane == 0) {
      int first[kLead + 3];
#pragma unroll
      for (int i = 0; i < kLead + 3; ++i) first[i] = next_number(i);
      fresh = next_number(kLead + 3);
#pragma unroll
      for (int i = 0; i < kLead + 3; ++i) ask(i, first[i]);
      copies_end();
      copies_wait<0>();
      for (int i = 0; i < kLead + 1; ++i) publish(i);
    }
    copies_end();
    __syncthreads();
    Entry before = Entry{-1, 0, -1, 0};                      // entry i - 1
    for (int i = 0;; ++i) {
      const Entry now = ring[i & (kRing - 1)];
      copies_wait<1>();
      if (lane == 0) {
        publish(i + kLead + 1);
        ask(i + kLead + 3, fresh);
        fresh = next_number(i + kLead + 4);
      }
      copies_end();
      if (before.row >= 0) {
        const int row = before.row;
        const bool real = before.label >= 0;
        const Mail& letter = mail[(i - 1) & (kRing - 1)];
        if constexpr (kMode == kGrad) {
          if (lane == 0) {
            const float2 st = letter.stat;
            const float c = real ? letter.weight * a.inv_t * scale : 0.f;
            bc[(i - 1) & 1] = make_float4(st.x, __fdividef(c, st.y), c, 0.f);
          }
        } else {
          float m = -INFINITY, sum = 0.f;
          if (real) {
            if (lane < kWarps) { m = part[(i - 1) & 1][lane].x; sum = part[(i - 1) & 1][lane].y; }
            join_lanes(m, sum, a.k);
          }
          if (lane == 0) {
            if (!whole) {
              a.w.part[static_cast<long>(row) * a.pieces + before.piece] = make_float2(m, sum);
            } else {
              const LogProb lp = real ? log_probability(logit_of(letter), m, sum, a.inv_t) : LogProb{0.f, 0.f};
              a.logprobs[row] = lp.hi;
              if (a.stat) a.stat[row] = real ? make_float2(m, sum) : make_float2(0.f, 1.f);
            }
          }
        }
      }
      __syncthreads();
      if (now.row == -1) break;
      before = now;
    }
    copies_wait<0>();
    return;
  }

  // -------------------------------------------------------------------------------------------------- the elements' warps
  const bool singles = !a.aligned || a.vocab % kE != 0;
  const auto issue = [&](int i) {
    const Entry n = ring[i & (kRing - 1)];
    if (n.label >= 0) {
      const T* x = x0 + static_cast<long>(n.row) * a.ld;
      const Shape s = shape_of(a, x, n.piece);
      const uint4* from = reinterpret_cast<const uint4*>(x + s.head) + s.v0 + t;
      uint4* to = slots + (i % kSlots) * a.slot + t;
      const int left = s.v1 - s.v0 - t;
      if constexpr (kMode == kScores) {
        const uint64_t policy = policy_of(n.row < a.stays);
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
          if (j * kCompute < left) copy16(to + j * kCompute, from + j * kCompute, policy);
      } else {
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
          if (j * kCompute < left) copy16(to + j * kCompute, from + j * kCompute);
      }
    }
    copies_end();
  };
  const auto single_of = [&](int i) -> float {
    if (!singles || warp > 0) return -INFINITY;
    const Entry n = ring[i & (kRing - 1)];
    if (n.label < 0) return -INFINITY;
    const T* x = x0 + static_cast<long>(n.row) * a.ld;
    const int e = single_at<T>(shape_of(a, x, n.piece), t, n.piece, a.pieces);
    return e >= 0 ? Num<T>::get(x[e]) : -INFINITY;
  };
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kLead; ++i) issue(i);
  float one = single_of(0), one_before = -INFINITY;
  Entry before = Entry{-1, 0, -1, 0};
  for (int i = 0;; ++i) {
    const Entry now = ring[i & (kRing - 1)];
    copies_wait<kLead - 1>();
    if (kSums && now.label >= 0) {
      const T* const x = x0 + static_cast<long>(now.row) * a.ld;
      const Shape s = shape_of(a, x, now.piece);
      const int left = s.v1 - s.v0 - t;                          // vectors of this thread: j with j * kCompute < left
      const uint4* const from = slots + (i % kSlots) * a.slot + t;
      uint4 raw[kVecs];
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
        raw[j] = j * kCompute < left ? from[j * kCompute] : make_uint4(Num<T>::kLow, Num<T>::kLow, Num<T>::kLow, Num<T>::kLow);
      float m = one;
#pragma unroll
      for (int j = 0; j < kVecs; ++j) m = fmaxf(m, Num<T>::largest(raw[j]));
      m = warp_max(m);
      const float base = m == -INFINITY ? 0.f : m;
      float2 total[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        if (j > 0 && j * kCompute >= left) break;
        float2 e[kE / 2];
        exps<T>(raw[j], -base, a.k, e);
#pragma unroll
        for (int q = 0; q < kE / 2; ++q) total[q & 1] = add2(total[q & 1], e[q]);
      }
      total[0] = add2(total[0], total[1]);
      float sum = total[0].x + total[0].y;
      if (singles) sum += ex2((one - base) * a.k);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) part[i & 1][warp] = make_float2(m, sum);
    }
    __syncthreads();
    const float next_one = single_of(i + 1);
    if constexpr (kMode == kScores) issue(i + kLead);           // the slot's values are read
    if (kGrads && before.row >= 0 && a.g) {
      T* const g = g0 + static_cast<long>(before.row) * a.ld;
      const T* const x = x0 + static_cast<long>(before.row) * a.ld;
      const Shape s = shape_of(a, x, before.piece);
      const int left = s.v1 - s.v0 - t;
      uint4* const out = reinterpret_cast<uint4*>(g + s.head) + s.v0 + t;
      const int label = before.label;
      const bool real = label >= 0;
      if (!real) {
        for (int v = 0; v < left; v += kCompute) __stcs(out + v, make_uint4(0, 0, 0, 0));
        const int e1 = single_at<T>(s, t, before.piece, a.pieces);
        if (e1 >= 0) g[e1] = Num<T>::put(0.f);
      } else {
        const float4 c = bc[(i - 1) & 1];
        const uint4* const from = slots + ((i - 1) % kSlots) * a.slot + t;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          if (j * kCompute >= left) break;
          float2 e[kE / 2];
          exps<T>(from[j * kCompute], -c.x, a.k, e);
#pragma unroll
          for (int q = 0; q < kE / 2; ++q) e[q] = mul2(e[q], make_float2(-c.y, -c.y));
          __stcs(out + j * kCompute, Num<T>::pack(e));
        }
        if (singles && warp == 0) {
          const int e1 = single_at<T>(s, t, before.piece, a.pieces);
          if (e1 >= 0) g[e1] = Num<T>::put((e1 == label ? c.z : 0.f) - c.y * ex2((one_before - c.x) * a.k));
        }
        const int v = (label - s.head) / kE;                    // the label's element again, by the thread that has just written its vector
        if (label >= s.head && v >= s.v0 && v < s.v1 && (v - s.v0) % kCompute == t) {
          const T* const held = reinterpret_cast<const T*>(slots + ((i - 1) % kSlots) * a.slot + v - s.v0);
          g[label] = Num<T>::put(c.z - c.y * ex2((Num<T>::get(held[(label - s.head) % kE]) - c.x) * a.k));
        }
      }
    }
    if (now.row == -1) break;
    if constexpr (kMode != kScores) issue(i + kLead);           // into the slot of entry i - 1
    before = now;
    one_before = one;
    one = next_one;
  }
  copies_wait<0>();
}

// Sums of pieces of 16-bit rows, a warp to a piece: no barrier, each lane with a running maximum of its own and its own logits on their way by
// asynchronous copies, so that one warp's exponentials run while another's wait.  A block to a piece (above) keeps neither the memory nor the exponentials
// busy all the time: 8200 rows of 32000 in bf16 took 109 us there and take 95 here (floor 81).  32-bit rows have half the exponentials to a byte and
// are at the memory's rate there (159 us; here 165 to 173).
constexpr int kSumWarps = 16, kSumBlocks = 2;               // warps of a block, blocks to an SM
constexpr int kSumVecs = 4, kSumStages = 3, kSumStage = 32 * kSumVecs;      // vectors of a lane in a stage, stages on their way, vectors of a stage
constexpr int kSumRing = 8;                                 // items known: fewer than kSumStages + 3
template <typename T>
__global__ void __launch_bounds__(kSumWarps * 32, kSumBlocks) sums_kernel(const __grid_constant__ Args a) {
  constexpr int kE = Num<T>::kE;
  extern __shared__ __align__(16) uint4 slots[];            // [kSumWarps][kSumStages][kSumStage]
  if (a.behind) wait_for_previous();
  if (a.w.part) let_next_start();
  __shared__ int4 rings[kSumWarps][kSumRing];                      // row, piece, label
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* const x0 = static_cast<const T*>(a.x);
  uint4* const mine = slots + warp * (kSumStages * kSumStage) + lane;
  int4* const ring = rings[warp];
  const int items = a.rows * a.pieces, warps = static_cast<int>(gridDim.x) * kSumWarps;
  const bool singles = !a.aligned || a.vocab % kE != 0;

  // The copying side: lane 0 has the next item's number and label and the number after it, asked for an item ahead.  Rows of padding are passed over.
  int number = static_cast<int>(blockIdx.x) + warp * static_cast<int>(gridDim.x), after = number + warps;
  int label = -1;
  const auto label_of = [&](int of) -> int {
    if (of >= items) return -1;
    const int n = items - 1 - of, row = a.pieces == 1 ? n : n / a.pieces;
    const int64_t y = a.labels[row];
    return y == a.pad || y < 0 || y >= a.vocab ? -1 : static_cast<int>(y);
  };
  if (lane == 0) label = label_of(number);
  int filled = 0, at = 0, end = 0, prow = 0;                // entries of `ring`; the next vectors to copy, -1: none
  const uint4* from = nullptr;
  const auto fetch = [&]() {
    for (;;) {
      const int n = items - 1 - __shfl_sync(0xffffffffu, number, 0), y = __shfl_sync(0xffffffffu, label, 0);
      if (n < 0) { prow = -1; break; }
      if (lane == 0) {
        number = after;
        label = label_of(number);
        after = a.w.ticket ? 2 * warps + atomicAdd(a.w.ticket, 1) : items;
      }
      if (y < 0) {
        if (lane == 0 && !a.w.part) {                       // a row in one piece
          a.logprobs[n] = 0.f;
          if (a.stat) a.stat[n] = make_float2(0.f, 1.f);
        }
        continue;
      }
      prow = a.pieces == 1 ? n : n / a.pieces;
      const int piece = n - prow * a.pieces;
      const T* x = x0 + static_cast<long>(prow) * a.ld;
      const Shape s = shape_of(a, x, piece);
      from = reinterpret_cast<const uint4*>(x + s.head) + lane;
      at = s.v0;
      end = s.v1;
      if (lane == 0) ring[filled & (kSumRing - 1)] = make_int4(prow, piece, y, 0);
      ++filled;
      return;
    }
    if (lane == 0) ring[filled & (kSumRing - 1)] = make_int4(-1, 0, 0, 0);
    ++filled;
  };
  int slot = 0;
  const auto issue = [&](int to) {
    if (prow >= 0) {
      const uint64_t policy = policy_of(prow < a.stays);
#pragma unroll
      for (int j = 0; j < kSumVecs; ++j)
        if (at + lane + j * 32 < end) copy16(mine + to * kSumStage + j * 32, from + at + j * 32, policy);
      at += kSumStage;
      if (at >= end) fetch();
    }
    copies_end();
  };
  fetch();
#pragma unroll
  for (int i = 0; i < kSumStages; ++i) issue(i);
  for (int i = 0;; ++i) {
    __syncwarp();
    const int4 now = ring[i & (kSumRing - 1)];
    if (now.x < 0) break;
    const T* const x = x0 + static_cast<long>(now.x) * a.ld;
    const Shape s = shape_of(a, x, now.y);
    float one = -INFINITY, xy = 0.f;
    if (singles) {
      const int e = single_at<T>(s, lane, now.y, a.pieces);
      if (e >= 0) one = Num<T>::get(x[e]);
    }
    if (!a.w.part) xy = Num<T>::get(x[now.z]);
    float m = -INFINITY, sum = 0.f;
    int v = s.v0;
    do {
      copies_wait<kSumStages - 1>();
      const int left = s.v1 - v - lane;
      uint4 raw[kSumVecs];
#pragma unroll
      for (int j = 0; j < kSumVecs; ++j)
        raw[j] = j * 32 < left ? mine[slot * kSumStage + j * 32] : make_uint4(Num<T>::kLow, Num<T>::kLow, Num<T>::kLow, Num<T>::kLow);
      float top = m;
#pragma unroll
      for (int j = 0; j < kSumVecs; ++j) top = fmaxf(top, Num<T>::largest(raw[j]));
      const float base = top == -INFINITY ? 0.f : top;
      float2 total[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < kSumVecs; ++j) {
        if (j > 0 && v + j * 32 >= s.v1) break;
        float2 e[kE / 2];
        exps<T>(raw[j], -base, a.k, e);
#pragma unroll
        for (int q = 0; q < kE / 2; ++q) total[q & 1] = add2(total[q & 1], e[q]);
      }
      total[0] = add2(total[0], total[1]);
      sum = fmaf(sum, ex2((m - base) * a.k), total[0].x + total[0].y);      // a stage's sum at a time: few roundings in a row
      m = top;
      issue(slot);
      slot = slot + 1 == kSumStages ? 0 : slot + 1;
      v += kSumStage;
    } while (v < s.v1);
    if (singles) join(m, sum, one, one == -INFINITY ? 0.f : 1.f, a.k);
    join_lanes(m, sum, a.k);
    if (lane == 0) {
      if (a.w.part) a.w.part[static_cast<long>(now.x) * a.pieces + now.y] = make_float2(m, sum);
      else {
        a.logprobs[now.x] = log_probability(xy, m, sum, a.inv_t).hi;
        if (a.stat) a.stat[now.x] = make_float2(m, sum);
      }
    }
  }
  copies_wait<0>();
}

// The policy loss of a row that a block's shared memory holds, a block to a row, or a cluster of 2, 4 or 8 to a longer one (kCluster: the blocks read each
// other's sums from shared memory): every thread copies its vectors, adds them up as they arrive in four
// groups, and goes over them again for the gradient.  Nothing is carried from row to row: while a block waits for its row, or for the coefficient, others of the SM
// compute and store, and rows go to SMs as they become free.  (A block that stays and reads the next rows meanwhile, three slots and a warp for the
// coefficients, was built before: 15360 rows of 32000 in bf16 360 us for 317, 3584 of 51865, which it could not hold, 195 for 138.)
constexpr int kHeldGroups = 4, kHeldVecs = 4;             // vectors that a thread has in registers
template <typename T, int kThreads, int kBlocks, bool kCluster>
__global__ void __launch_bounds__(kThreads, kBlocks) held_rows_kernel(const __grid_constant__ Args a) {
  constexpr int kE = Num<T>::kE, kWarps = kThreads / 32;
  extern __shared__ __align__(16) uint4 held[];
  __shared__ float2 part[kWarps], whole;
  __shared__ float4 bc;
  let_next_start();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int pieces = kCluster ? a.pieces : 1, block = static_cast<int>(gridDim.x - 1 - blockIdx.x), row = block / pieces, piece = block - row * pieces;
  const T* const x = static_cast<const T*>(a.x) + static_cast<long>(row) * a.ld;
  T* const g = a.g ? static_cast<T*>(a.g) + static_cast<long>(row) * a.ld : nullptr;
  const Shape s = shape_of(a, x, piece);
  const int nvec = s.v1 - s.v0;                               // of this block
  const uint4* const from = reinterpret_cast<const uint4*>(x + s.head) + s.v0;
  const int64_t y = a.labels[row];
  const int each = (nvec + kHeldGroups * kThreads - 1) / (kHeldGroups * kThreads) * kThreads;      // vectors of a group
#pragma unroll
  for (int q = 0; q < kHeldGroups; ++q) {
    const int end = min(nvec, (q + 1) * each);
#pragma unroll 4
    for (int v = q * each + t; v < end; v += kThreads) copy16(held + v, from + v);
    copies_end();
  }
  const bool real = y != a.pad && y >= 0 && y < a.vocab;
  const int label = real ? static_cast<int>(y) : -1, e1 = single_at<T>(s, t, piece, pieces);
  uint4* const out = reinterpret_cast<uint4*>(g + s.head) + s.v0;
  if (!real) {                                                // for all blocks of the row
    if (t == 0 && piece == 0) { a.logprobs[row] = 0.f; a.w.lp[row] = 0.0; }
    if (g) {
      for (int v = t; v < nvec; v += kThreads) __stcs(out + v, make_uint4(0, 0, 0, 0));
      if (e1 >= 0) g[e1] = Num<T>::put(0.f);
    }
    copies_wait<0>();
    return;
  }
  const float one = e1 >= 0 ? Num<T>::get(x[e1]) : -INFINITY;
  float xy = 0.f, old = 0.f, adv = 0.f, ref = 0.f, scale = 0.f;
  if (warp == 0) {
    xy = Num<T>::get(x[label]);
    old = a.policy.old_logprobs[row];
    adv = a.policy.advantages[row];
    if (a.policy.ref_logprobs) ref = a.policy.ref_logprobs[row];
    scale = a.scale_at ? *a.scale_at * a.scale : a.scale;
  }
  float m = one, sum = one == -INFINITY ? 0.f : 1.f;
#pragma unroll
  for (int q = 0; q < kHeldGroups; ++q) {
    if (q == 0) copies_wait<3>(); else if (q == 1) copies_wait<2>(); else if (q == 2) copies_wait<1>(); else copies_wait<0>();
    const int end = min(nvec, (q + 1) * each);
#pragma unroll 1
    for (int v = q * each + t; v < end; v += kHeldVecs * kThreads) {
      uint4 raw[kHeldVecs];
#pragma unroll
      for (int j = 0; j < kHeldVecs; ++j)
        raw[j] = v + j * kThreads < end ? held[v + j * kThreads] : make_uint4(Num<T>::kLow, Num<T>::kLow, Num<T>::kLow, Num<T>::kLow);
      float top = m;
#pragma unroll
      for (int j = 0; j < kHeldVecs; ++j) top = fmaxf(top, Num<T>::largest(raw[j]));
      const float base = top == -INFINITY ? 0.f : top;
      float2 total[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < kHeldVecs; ++j) {
        if (j > 0 && v + j * kThreads >= end) break;
        float2 e[kE / 2];
        exps<T>(raw[j], -base, a.k, e);
#pragma unroll
        for (int p = 0; p < kE / 2; ++p) total[p & 1] = add2(total[p & 1], e[p]);
      }
      total[0] = add2(total[0], total[1]);
      sum = fmaf(sum, ex2((m - base) * a.k), total[0].x + total[0].y);
      m = top;
    }
  }
  join_lanes(m, sum, a.k);
  if (lane == 0) part[warp] = make_float2(m, sum);
  __syncthreads();
  if (warp == 0) {
    m = lane < kWarps ? part[lane].x : -INFINITY;
    sum = lane < kWarps ? part[lane].y : 0.f;
    join_lanes(m, sum, a.k);
    if (kCluster && lane == 0) whole = make_float2(m, sum);
  }
  if constexpr (kCluster) cooperative_groups::this_cluster().sync();
  if (warp == 0) {
    if constexpr (kCluster) {                                 // every block of the row comes to the same coefficient
      const float2 of = lane < pieces ? *cooperative_groups::this_cluster().map_shared_rank(&whole, lane) : make_float2(-INFINITY, 0.f);
      m = of.x;
      sum = of.y;
      join_lanes(m, sum, a.k);
    }
    const LogProb lp = log_probability(xy, m, sum, a.inv_t);
    const float slope = policy_coef(a, lp, old, adv, ref), c = slope * a.inv_t * scale;
    if (lane == 0) {
      bc = make_float4(m, __fdividef(c, sum), c, 0.f);
      if (piece == 0) {
        a.logprobs[row] = lp.hi;
        a.w.lp[row] = lp.wide();
        if (a.stat) { a.stat[row] = make_float2(m, sum); a.w.coef[row] = slope; }
      }
    }
  }
  if constexpr (kCluster) cooperative_groups::this_cluster().sync();         // `whole` of every block is read
  else __syncthreads();
  if (!g) return;
  const float4 c = bc;
#pragma unroll 4
  for (int v = t; v < nvec; v += kThreads) {
    float2 e[kE / 2];
    exps<T>(held[v], -c.x, a.k, e);
#pragma unroll
    for (int q = 0; q < kE / 2; ++q) e[q] = mul2(e[q], make_float2(-c.y, -c.y));
    __stcs(out + v, Num<T>::pack(e));
  }
  if (e1 >= 0) g[e1] = Num<T>::put((e1 == label ? c.z : 0.f) - c.y * ex2((one - c.x) * a.k));
  const int v = (label - s.head) / kE - s.v0;
  if (label >= s.head && v >= 0 && v < nvec && v % kThreads == t)      // the label's element again, by the thread that has just written its vector
    g[label] = Num<T>::put(c.z - c.y * ex2((Num<T>::get(reinterpret_cast<const T*>(held + v)[(label - s.head) % kE]) - c.x) * a.k));
}

// Rows that a warp holds, kHeld vectors a lane: a warp to a row, everything in registers.  kScores, kGrad, kLocal.  (20000 rows of 2500 in bf16, 16 vectors a lane: scores
// 27 us, gradients 44, paired loss 82; by the kernels for longer rows 74, 64 and 136.  Floors 16 and 31.)
template <typename T, int kMode, int kHeld>
__global__ void __launch_bounds__(256) short_rows_kernel(const __grid_constant__ Args a) {
  constexpr int kE = Num<T>::kE;
  const int lane = threadIdx.x & 31, row = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (a.behind) wait_for_previous();
  if (kMode == kLocal || (kMode == kScores && a.behind)) let_next_start();
  if (row >= a.rows) return;
  const T* const x = static_cast<const T*>(a.x) + static_cast<long>(row) * a.ld;
  T* const g = static_cast<T*>(a.g) + static_cast<long>(row) * a.ld;
  const Shape s = shape_of(a, x, 0);
  const int left = s.nvec - lane, e1 = single_at<T>(s, lane, 0, 1);
  uint4 raw[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    raw[j] = j * 32 < left ? reinterpret_cast<const uint4*>(x + s.head)[lane + j * 32] : make_uint4(Num<T>::kLow, Num<T>::kLow, Num<T>::kLow, Num<T>::kLow);
  const float one = e1 >= 0 ? Num<T>::get(x[e1]) : -INFINITY;
  const int64_t y = a.w.label ? a.w.label[row] : a.labels[row];
  const bool real = y >= 0 && y < a.vocab && (a.w.label || y != a.pad);
  const int label = real ? static_cast<int>(y) : -1;
  const float scale = a.scale_at ? *a.scale_at * a.scale : a.scale;
  float old = 0.f, adv = 0.f, ref = 0.f;
  if (kMode == kLocal && real) {
    old = a.policy.old_logprobs[row];
    adv = a.policy.advantages[row];
    if (a.policy.ref_logprobs) ref = a.policy.ref_logprobs[row];
  }
  const float xy = real ? Num<T>::get(x[label]) : 0.f;
  float m, sum, c = 0.f;
  if constexpr (kMode == kGrad) {
    const float2 st = a.stat[row];
    m = st.x;
    sum = st.y;
    if (real) c = a.weight[a.w.seq ? a.w.seq[row] : row] * scale * a.inv_t;
  } else {
    m = one;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) m = fmaxf(m, Num<T>::largest(raw[j]));
    m = warp_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float2 total = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (j > 0 && j * 32 >= s.nvec) break;
      float2 e[kE / 2];
      exps<T>(raw[j], -base, a.k, e);
#pragma unroll
      for (int q = 0; q < kE / 2; ++q) total = add2(total, e[q]);
    }
    sum = total.x + total.y + ex2((one - base) * a.k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    LogProb lp = {0.f, 0.f};
    if (real) lp = log_probability(xy, m, sum, a.inv_t);
    if constexpr (kMode == kLocal) {
      const float slope = real ? policy_coef(a, lp, old, adv, ref) : 0.f;
      c = slope * a.inv_t * scale;
      if (lane == 0) {
        a.logprobs[row] = lp.hi;
        a.w.lp[row] = lp.wide();
        if (a.stat) { a.stat[row] = make_float2(m, sum); a.w.coef[row] = slope; }
      }
    } else if (lane == 0) {
      if (a.logprobs) a.logprobs[row] = lp.hi;
      if (a.stat) a.stat[row] = real ? make_float2(m, sum) : make_float2(0.f, 1.f);
    }
  }
  if (kMode == kScores || !a.g) return;
  const float f = real ? -c / sum : 0.f;
  uint4* const out = reinterpret_cast<uint4*>(g + s.head) + lane;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    if (j * 32 >= left) break;
    float2 e[kE / 2];
    exps<T>(raw[j], -m, a.k, e);
#pragma unroll
    for (int q = 0; q < kE / 2; ++q) e[q] = real ? mul2(e[q], make_float2(f, f)) : make_float2(0.f, 0.f);
    out[j * 32] = Num<T>::pack(e);
  }
  if (e1 >= 0) g[e1] = Num<T>::put(real ? f * ex2((one - m) * a.k) : 0.f);
  __syncwarp();
  if (lane == 0 && real) g[label] = Num<T>::put(c + f * ex2((xy - m) * a.k));
}

// Offsets put in order (running maximum, within the rows), rows' sequences and labels.  Every block goes through the offsets; its share of the
// sequences it writes.
__global__ void __launch_bounds__(1024) pairs_setup_kernel(const __grid_constant__ Args a) {
  __shared__ int bounds[1025];
  __shared__ int warp_top[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = 2 * a.pairs.pairs + 1;
  let_next_start();
  const auto none = [&](int begin, int end) {                // rows outside every sequence
    for (int r = begin + static_cast<int>(blockIdx.x) * 1024 + t; r < end; r += static_cast<int>(gridDim.x) * 1024) { a.w.seq[r] = -1; a.w.label[r] = -1; }
  };
  if (blockIdx.x == 0 && t == 0) *a.w.state = State{{0, 0}, 0};
  int carry = 0;
  for (int base = 0; base < n; base += 1024) {
    int v = base + t < n ? min(max(a.pairs.cu[base + t], 0), a.rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v = max(v, u); }
    if (lane == 31) warp_top[warp] = v;
    __syncthreads();
    v = max(v, carry);
    for (int w = 0; w < warp; ++w) v = max(v, warp_top[w]);
    bounds[t + 1] = v;
    if (t == 0) bounds[0] = carry;
    if (blockIdx.x == 0 && base + t < n) a.w.cu[base + t] = v;
    __syncthreads();
    if (base == 0) none(0, bounds[1]);
    for (int j = warp + 32 * static_cast<int>(blockIdx.x); j < 1024; j += 32 * static_cast<int>(gridDim.x)) {
      const int q = base + j - 1;                             // between bounds[j] and bounds[j + 1]
      if (q < 0 || q >= n - 1) continue;
      for (int r = bounds[j] + lane; r < bounds[j + 1]; r += 32) {
        const int64_t y = a.labels[r];
        a.w.seq[r] = q;
        a.w.label[r] = y == a.pad || y < 0 || y >= a.vocab ? -1 : static_cast<int>(y);
      }
    }
    carry = bounds[1024];
    __syncthreads();
  }
  none(carry, a.rows);
}

// A block to a pair: its rows' sums from their pieces, their log-probabilities, its loss and coefficients; the last block adds up the losses.
template <typename T>
__global__ void __launch_bounds__(128) pairs_kernel(const __grid_constant__ Args a) {
  __shared__ double sums[2][4];
  __shared__ int counts[2][4];
  __shared__ int last;
  const int p = static_cast<int>(blockIdx.x), t = threadIdx.x, lane = t & 31, warp = t >> 5;
  wait_for_previous();
  let_next_start();
  const int begin = a.w.cu[2 * p], middle = a.w.cu[2 * p + 1], end = a.w.cu[2 * p + 2];
  double sum[2] = {0.0, 0.0};
  int count[2] = {0, 0};
  for (int r = begin + t; r < end; r += 128) {
    const int label = a.w.label[r];
    if (label < 0) continue;
    const float xy = Num<T>::get(static_cast<const T*>(a.x)[static_cast<long>(r) * a.ld + label]);
    float m = -INFINITY, s = 0.f;
    if (a.pieces == 1 && a.stat) {
      m = a.stat[r].x;
      s = a.stat[r].y;
    } else {
      join_pieces(a, r, m, s);
      a.w.stat[r] = make_float2(m, s);
    }
    const double lp = log_probability(xy, m, s, a.inv_t).wide();
    const int which = r >= middle;
    if (which) { sum[1] += lp; ++count[1]; } else { sum[0] += lp; ++count[0]; }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
      count[h] += __shfl_xor_sync(0xffffffffu, count[h], o);
    }
    if (lane == 0) { sums[h][warp] = sum[h]; counts[h][warp] = count[h]; }
  }
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] = sums[h][0] + sums[h][1] + sums[h][2] + sums[h][3];
      count[h] = counts[h][0] + counts[h][1] + counts[h][2] + counts[h][3];
    }
    pair_loss(a, p, sum[0], sum[1], count[0], count[1]);
    __threadfence();
    last = atomicAdd(&a.w.state->pairs_done, 1) + 1 == a.pairs.pairs;
    __threadfence();
  }
  __syncthreads();
  if (!last || warp > 0) return;
  double loss = 0.0;
  int ranked = 0;
  for (int i = lane; i < a.pairs.pairs; i += 32) { loss += __ldcg(a.w.loss + i); ranked += __ldcg(a.w.ranked + i); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, o);
    ranked += __shfl_xor_sync(0xffffffffu, ranked, o);
  }
  if (lane == 0) { *a.pairs.loss = static_cast<float>(loss); *a.pairs.ranked = static_cast<float>(ranked); }
}

// After the sums of rows' pieces: log-probabilities, `stat`, and under the policy loss the coefficient; a thread to a row
template <typename T>
__global__ void __launch_bounds__(128) whole_rows_kernel(const __grid_constant__ Args a) {
  const int row = static_cast<int>(blockIdx.x * 128 + threadIdx.x);
  wait_for_previous();
  if (row >= a.rows) return;
  const int64_t y = a.labels[row];
  const bool real = y != a.pad && y >= 0 && y < a.vocab;
  float m = -INFINITY, s = 0.f;
  LogProb lp = {0.f, 0.f};
  if (real) {
    const float xy = Num<T>::get(static_cast<const T*>(a.x)[static_cast<long>(row) * a.ld + y]);
    join_pieces(a, row, m, s);
    lp = log_probability(xy, m, s, a.inv_t);
  }
  if (a.logprobs) a.logprobs[row] = lp.hi;
  if (a.w.lp) a.w.lp[row] = lp.wide();
  if (a.stat) a.stat[row] = real ? make_float2(m, s) : make_float2(0.f, 1.f);
  if (a.policy.old_logprobs)
    a.w.coef[row] = real ? policy_coef(a, lp, a.policy.old_logprobs[row], a.policy.advantages[row],
                                       a.policy.ref_logprobs ? a.policy.ref_logprobs[row] : 0.f) : 0.f;
}

// The sums of the policy loss from the rows' log-probabilities, in one order: a cluster of 8 blocks, each thread every 8 * kSumThreads-th row, and the
// blocks' sums by the first one, from their shared memory.  (15360 rows: 5.0 us; three blocks, one for each sum over all rows, 16.4.)
constexpr int kSumThreads = 512, kSumEach = 4;
__global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(kSumThreads) policy_sums_kernel(const __grid_constant__ Args a) {
  __shared__ double warps[3][kSumThreads / 32];
  __shared__ double block_sums[3];
  wait_for_previous();
  double sums[3] = {0.0, 0.0, 0.0};                             // the loss, the KL terms, the clipped words
  for (int r0 = blockIdx.x * kSumThreads + threadIdx.x; r0 < a.rows; r0 += kSumEach * 8 * kSumThreads) {
    int64_t y[kSumEach];
    double lp[kSumEach];
    float adv[kSumEach], old[kSumEach], ref[kSumEach];
#pragma unroll
    for (int j = 0; j < kSumEach; ++j) {                        // several rows' numbers are asked for at a time
      const int r = r0 + j * 8 * kSumThreads;
      const bool in = r < a.rows;
      y[j] = in ? a.labels[r] : -1;
      lp[j] = in ? a.w.lp[r] : 0.0;
      adv[j] = in ? a.policy.advantages[r] : 0.f;
      old[j] = in ? a.policy.old_logprobs[r] : 0.f;
      ref[j] = in && a.policy.ref_logprobs ? a.policy.ref_logprobs[r] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kSumEach; ++j) {
      if (y[j] == a.pad || y[j] < 0 || y[j] >= a.vocab) continue;
      const float ratio = expf(static_cast<float>(lp[j] - old[j])), held = fminf(fmaxf(ratio, a.policy.clip_low), a.policy.clip_high);
      const bool free = !(ratio * adv[j] > held * adv[j]);
      double kl = 0.0;
      if (a.policy.ref_logprobs) {
        const double d = ref[j] - lp[j];
        // in 64 bits: it is d^2 / 2 near 0, of which 32 bits leave 2^-23 / d.  inf, not inf - inf, for a word of probability 0
        kl = d < INFINITY ? expm1(d) - d : d;
      }
      sums[0] += (a.policy.kl_coef != 0.f ? a.policy.kl_coef * kl : 0.0) - static_cast<double>(free ? ratio : held) * adv[j];
      sums[1] += kl;
      sums[2] += free ? 0.0 : 1.0;
    }
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sums[q] += __shfl_xor_sync(0xffffffffu, sums[q], o);
    if ((threadIdx.x & 31) == 0) warps[q][threadIdx.x >> 5] = sums[q];
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kSumThreads / 32; ++w) s += warps[threadIdx.x][w];
    block_sums[threadIdx.x] = s;
  }
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x < 3) {
    double s = 0.0;
    for (int b = 0; b < 8; ++b) s += *cluster.map_shared_rank(&block_sums[threadIdx.x], b);
    *(threadIdx.x == 0 ? a.policy.loss : threadIdx.x == 1 ? a.policy.kl : a.policy.clipped) = static_cast<float>(s);
  }
  cluster.sync();                                               // the blocks' shared memory is read
}

template <typename T>
__global__ void __launch_bounds__(256) scale_rows_kernel(const Args a, const float* __restrict__ factor) {
  constexpr int kE = Num<T>::kE;
  const float f = *factor;
  if (f == 1.f) return;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    T* const row = static_cast<T*>(a.g) + static_cast<long>(r) * a.ld;
    const Shape s = shape_of(a, row, 0);
    uint4* const vectors = reinterpret_cast<uint4*>(row + s.head);
    for (int v = threadIdx.x; v < s.nvec; v += 256) {
      float2 g[kE / 2];
      Num<T>::unpack(vectors[v], g);
#pragma unroll
      for (int q = 0; q < kE / 2; ++q) g[q] = mul2(g[q], make_float2(f, f));
      vectors[v] = Num<T>::pack(g);
    }
    const int one = single_at<T>(s, threadIdx.x, 0, 1);
    if (one >= 0) row[one] = Num<T>::put(Num<T>::get(row[one]) * f);
  }
}

const char* problem(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

// The ticket of a pass, unless every block has its items without asking; the paired loss has zeroed it before
const char* set_ticket(Args& a, int pass, bool none, cudaStream_t stream) {
  a.w.ticket = none ? nullptr : a.w.state->tickets + pass;
  return none || a.pairs.pairs > 0 ? nullptr : problem(cudaMemsetAsync(a.w.ticket, 0, sizeof(int), stream));
}

template <typename T, int kCompute, int kMode>
const char* launch_rows(const Args& from, cudaStream_t stream) {
  Args a = from;
  auto kernel = rows_kernel<T, kCompute, kMode>;
  // slots as long as a piece: shorter rows leave room for a third block
  const int across = (a.each < kVecs * kCompute ? (a.each + kCompute - 1) / kCompute * kCompute : kVecs * kCompute);
  const int smem = kSlots * across * 16;
  a.slot = across;
  // the attribute belongs to a device's context: set at every call, which costs less than keeping account of the devices
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlots * kVecs * kCompute * 16);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  static std::atomic<int> blocks[kVecs + 1];      // that an SM holds, 0: not asked for yet; all GPUs of a machine are alike, and all threads find the same
  int held = blocks[across / kCompute].load(std::memory_order_relaxed);
  if (held == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, kCompute + 32, smem);
    if (e != cudaSuccess) return cudaGetErrorString(e);
    if (held < 1) return "preference: no block fits an SM";
    blocks[across / kCompute].store(held, std::memory_order_relaxed);
  }
  const long items = static_cast<long>(a.rows) * a.pieces, most = static_cast<long>(held) * num_sms();
  if (4 * items + (1L << 20) >= 1L << 31) return "preference: too many rows";
  const int grid = static_cast<int>(items < most ? items : most);
  const char* err = set_ticket(a, kMode == kGrad, items <= kFirst * most, stream);
  if (err) return err;
  a.behind = a.pairs.pairs > 0;                             // behind the kernels of the paired loss
  return launch_behind(a.behind, kernel, grid, kCompute + 32, smem, stream, a);
}

template <typename T>
const char* launch_sums(Args a, cudaStream_t stream) {
  const int smem = kSumWarps * kSumStages * kSumStage * 16;
  cudaError_t e = cudaFuncSetAttribute(sums_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  const long items = static_cast<long>(a.rows) * a.pieces, blocks = kSumBlocks * num_sms();
  if (items > INT_MAX / 2) return "preference: too many rows";
  const char* err = set_ticket(a, 0, items <= 2 * blocks * kSumWarps, stream);       // two to a warp without asking
  if (err) return err;
  const int grid = static_cast<int>(items < blocks ? items : blocks);
  a.behind = a.pairs.pairs > 0;
  return launch_behind(a.behind, sums_kernel<T>, grid, kSumWarps * 32, smem, stream, a);
}

template <typename T> constexpr int warp_row() { return 32 * 2 * kVecs * Num<T>::kE; }       // elements that a warp holds

// SMs of the GPU, those in reserve too: how a row is divided decides the bits of a result and the size of the workspace
int all_sms() {
  static const int n = [] {
    int device = 0, sms = 0;
    return cudaGetDevice(&device) == cudaSuccess && cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) == cudaSuccess && sms > 0 ? sms : 148;
  }();
  return n;
}

// Pieces of a row: as many as hold it; for few rows more, of 4 KB at least, until every block that the GPU holds has one.
int pieces_of(int rows, int vocab, int dtype) {
  const int vectors = vocab / (dtype == 0 ? 4 : 8);
  int n = (vectors + kBlock * kVecs - 1) / (kBlock * kVecs);
  if (n < 1) n = 1;
  while (static_cast<long>(n) * rows <= all_sms() && vectors >= 512 * n) n *= 2;
  return n;
}

// Sums by warps: 16-bit logits of 128 MB or more.  With fewer a warp has too little to do before its last piece (4000 rows of 8000 in bf16: 31.7 us by warps,
// 28.0 by blocks; 20000 rows: 64 and 87).
bool by_warps(int rows, int vocab, int dtype) { return dtype != 0 && static_cast<long>(rows) * vocab >= 1L << 26; }
// Pieces of a row for its sums: by warps three to a warp at least, where a row has that many stages, and of no more than 32 stages each: a lane's sum
// is then at most 8 + 32 additions deep, and off by 2^-19 at most
int sums_pieces(int rows, int vocab, int dtype) {
  if (!by_warps(rows, vocab, dtype)) return pieces_of(rows, vocab, dtype);
  const long vectors = vocab / 8, most = vectors / kSumStage > 1 ? vectors / kSumStage : 1, warps = 3L * kSumBlocks * kSumWarps * all_sms();
  const long n = (warps + rows - 1) / rows, least = vectors / (32 * kSumStage) + 1;
  return static_cast<int>(n >= most ? most : n >= least ? n : least);
}
// Scores of no more rows than there are SMs, each no longer than a block holds, are one launch of a block to a row: 37 rows of 32000 in bf16
// take 10.4 us a call, in pieces and a second launch 13.9.
bool few_rows(int rows, int vocab, int dtype) { return rows <= all_sms() && vocab <= kWide * kVecs * (dtype == 0 ? 4 : 8); }

template <typename T, int kMode>
const char* launch_short(Args a, cudaStream_t stream) {
  a.behind = kMode != kLocal && a.pairs.pairs > 0;
  return launch_behind(a.behind, a.vocab <= warp_row<T>() / 2 ? short_rows_kernel<T, kMode, kVecs> : short_rows_kernel<T, kMode, 2 * kVecs>, (a.rows + 7) / 8, 256,
                       0, stream, a);
}

// kMode: kScores or kGrad
template <int kMode>
const char* launch_pass(Args a, int dtype, cudaStream_t stream) {
  if (a.rows <= 0) return nullptr;
  const int size = dtype == 0 ? 4 : 2;
  if (a.vocab <= (dtype == 0 ? warp_row<float>() : warp_row<__half>())) {
    a.pieces = 1;
    a.each = a.vocab / (16 / size);
    return dtype == 0 ? launch_short<float, kMode>(a, stream) : dtype == 1 ? launch_short<__nv_bfloat16, kMode>(a, stream) : launch_short<__half, kMode>(a, stream);
  }
  const bool between = a.pairs.pairs > 0 || a.policy.old_logprobs;         // the paired and the policy loss go on with the sums of the pieces
  if (kMode == kScores && !between && few_rows(a.rows, a.vocab, dtype)) {
    a.pieces = 1;
    a.each = a.vocab / (16 / size);
    a.w.part = nullptr;
    return dtype == 0 ? launch_rows<float, kWide, kScores>(a, stream) : dtype == 1 ? launch_rows<__nv_bfloat16, kWide, kScores>(a, stream)
                                                                                   : launch_rows<__half, kWide, kScores>(a, stream);
  }
  a.pieces = kMode == kScores ? sums_pieces(a.rows, a.vocab, dtype) : pieces_of(a.rows, a.vocab, dtype);
  a.each = (a.vocab / (16 / size) + a.pieces - 1) / a.pieces;
  if (a.pieces == 1 && !between) a.w.part = nullptr;
  const char* err;
  if (kMode == kScores && by_warps(a.rows, a.vocab, dtype))
    err = dtype == 1 ? launch_sums<__nv_bfloat16>(a, stream) : launch_sums<__half>(a, stream);
  else
    err = dtype == 0 ? launch_rows<float, kBlock, kMode>(a, stream) : dtype == 1 ? launch_rows<__nv_bfloat16, kBlock, kMode>(a, stream)
                                                                                 : launch_rows<__half, kBlock, kMode>(a, stream);
  if (kMode != kScores || err || a.pairs.pairs > 0 || !a.w.part) return err;
  const int blocks = (a.rows + 127) / 128;
  return launch_behind(true, dtype == 0 ? whole_rows_kernel<float> : dtype == 1 ? whole_rows_kernel<__nv_bfloat16> : whole_rows_kernel<__half>, blocks, 128, 0,
                       stream, a);
}

template <typename T, int kThreads, int kBlocks, bool kCluster>
const char* launch_held(const Args& a, cudaStream_t stream) {
  if (static_cast<long>(a.rows) * a.pieces > INT_MAX) return "preference: too many rows";
  auto kernel = held_rows_kernel<T, kThreads, kBlocks, kCluster>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldBytes);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows * a.pieces);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = a.each * 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.pieces;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCluster ? 1 : 0;
  return problem(cudaLaunchKernelEx(&cfg, kernel, a));
}

// Threads to a row so that those of an SM, as many rows as its shared memory holds, are 1000 to 1200, what the registers allow.  600 MB of bf16 logits in
// rows of 4000 words (64 threads / 128 / 192 / 384 / 512) 230 / 320 / 390 / 566 / 692 us, 12000 210 / 197 / 223 / 331 / 373, 20000 236 / 210 / 188 / 236 / 296, 32000
// 276 / 228 / 207 / 200 / 242, 56000 338 / 270 / 225 / 213 / 201.  Rows of more
// than 112 KB one to a block, which an SM then holds alone, and to clusters: 64000 words 268 / 230, 128000 292 / 243, 250054 by two passes 300, by a cluster 279.
template <typename T>
const char* launch_local(Args a, cudaStream_t stream) {
  a.pieces = 1;
  a.each = a.vocab / Num<T>::kE;
  if (a.vocab <= warp_row<T>()) return launch_short<T, kLocal>(a, stream);
  const int vectors = a.vocab / Num<T>::kE;
  while (vectors * 16 > kHeldBytes * a.pieces) a.pieces *= 2;          // 2, 4 or 8
  a.each = (vectors + a.pieces - 1) / a.pieces;
  const int kb = a.each / 64;
  if (a.pieces > 1) return kb < 80 ? launch_held<T, 384, 3, true>(a, stream) : launch_held<T, 512, 2, true>(a, stream);
  if (kb < 20) return launch_held<T, 64, 18, false>(a, stream);
  if (kb < 28) return launch_held<T, 128, 9, false>(a, stream);
  if (kb < 52) return launch_held<T, 192, 6, false>(a, stream);
  if (kb < 80) return launch_held<T, 384, 3, false>(a, stream);
  return launch_held<T, 512, 2, false>(a, stream);
}

Args row_args(const NmtgRows* r) {
  Args a = {};
  a.x = r->logits; a.g = r->grad; a.labels = r->labels; a.ld = r->ld; a.pad = r->pad; a.rows = r->rows; a.vocab = r->vocab;
  a.inv_t = r->inv_temperature; a.k = static_cast<float>(1.4426950408889634074 * r->inv_temperature);
  a.scale_at = r->grad_scale_at; a.scale = r->grad_scale;
  const uintptr_t at = reinterpret_cast<uintptr_t>(r->logits ? r->logits : r->grad);
  a.aligned = at % 16 == 0 && (r->rows <= 1 || r->ld * (r->dtype == 0 ? 4 : 2) % 16 == 0);
  a.logprobs = r->logprobs; a.stat = r->stat;
  a.pieces = 1;
  a.each = a.vocab;
  const long staying = kStaying / (r->vocab * (r->dtype == 0 ? 4L : 2L));
  a.stays = r->rows > staying ? static_cast<int>(staying) : r->rows;
  return a;
}

long up16(long n) { return (n + 15) & ~15L; }
const char* bad_type = "preference: logits must be fp32, bf16 or fp16";

// The workspace of a call; null pointers where it is not asked for
Work workspace(char* at, long rows, long pairs, long pieces, long* bytes) {
  char* const begin = at;
  const auto take = [&](long n) { char* here = at; at += up16(n); return static_cast<void*>(here); };
  Work w = {};
  w.state = static_cast<State*>(take(sizeof(State)));
  w.part = static_cast<float2*>(take(8 * rows * pieces));
  w.stat = static_cast<float2*>(take(8 * rows));
  w.coef = static_cast<float*>(take(4 * (2 * pairs > rows ? 2 * pairs : rows)));
  w.cu = static_cast<int*>(take(4 * (2 * pairs + 1)));
  w.seq = static_cast<int*>(take(4 * rows));
  w.label = static_cast<int*>(take(4 * rows));
  w.lp = static_cast<double*>(take(8 * rows));
  w.loss = static_cast<double*>(take(8 * pairs));
  w.ranked = static_cast<int*>(take(4 * pairs));
  *bytes = at - begin;
  return w;
}

}  // namespace
}  // namespace b200

using namespace b200;

long nmtg_rows_workspace(int rows, int vocab, int dtype, int pairs) {
  long bytes = 0;
  workspace(nullptr, rows, pairs, sums_pieces(rows, vocab, dtype), &bytes);
  return bytes;
}

const char* nmtg_row_scores(const NmtgRows* r, cudaStream_t stream) {
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  Args a = row_args(r);
  long bytes;
  const Work w = workspace(static_cast<char*>(r->workspace), r->rows, 0, sums_pieces(r->rows, r->vocab, r->dtype), &bytes);
  a.w.state = w.state;
  a.w.part = w.part;
  return launch_pass<kScores>(a, r->dtype, stream);
}

const char* nmtg_row_scores_grad(const NmtgRows* r, const float* weight, cudaStream_t stream) {
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  Args a = row_args(r);
  a.weight = weight;
  a.scale = 1.f;
  long bytes;
  a.w.state = workspace(static_cast<char*>(r->workspace), r->rows, 0, 1, &bytes).state;
  return launch_pass<kGrad>(a, r->dtype, stream);
}

const char* nmtg_policy_loss(const NmtgRows* r, const NmtgPolicy* p, cudaStream_t stream) {
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  Args a = row_args(r);
  a.policy = *p;
  const int size = r->dtype == 0 ? 4 : 2;
  const char* err = nullptr;
  long bytes;
  const Work w = workspace(static_cast<char*>(r->workspace), r->rows, 0, sums_pieces(r->rows, r->vocab, r->dtype), &bytes);
  a.w.lp = w.lp;
  a.w.state = w.state;
  a.w.coef = p->coef;
  if (r->rows <= 0) {
  } else if (static_cast<long>(r->vocab) * size <= 8L * kHeldBytes) {       // without a gradient, too: the same bits
    err = r->dtype == 0 ? launch_local<float>(a, stream) : r->dtype == 1 ? launch_local<__nv_bfloat16>(a, stream) : launch_local<__half>(a, stream);
  } else {
    a.w.part = w.part;
    if (!a.stat) { a.stat = w.stat; a.w.coef = w.coef; }
    a.weight = a.w.coef;
    err = launch_pass<kScores>(a, r->dtype, stream);
    if (!err && a.g) err = launch_pass<kGrad>(a, r->dtype, stream);
  }
  if (err) return err;
  return launch_behind(r->rows > 0, policy_sums_kernel, 8, kSumThreads, 0, stream, a);
}

const char* nmtg_preference_loss(const NmtgRows* r, const NmtgPairs* p, cudaStream_t stream) {
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  Args a = row_args(r);
  a.pairs = *p;
  long bytes;
  const int pieces = sums_pieces(r->rows, r->vocab, r->dtype);
  const Work w = workspace(static_cast<char*>(r->workspace), r->rows, p->pairs, pieces, &bytes);
  if (p->pairs == 0) {                    // no loss; every row is outside
    cudaError_t e = cudaMemsetAsync(p->loss, 0, sizeof(float), stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(p->ranked, 0, sizeof(float), stream);
    if (e != cudaSuccess) return cudaGetErrorString(e);
  }
  a.w = w;
  const int share = 1 + (p->pairs >= 8) * (p->pairs < 256 ? p->pairs / 8 : 32);
  pairs_setup_kernel<<<share, 1024, 0, stream>>>(a);
  const char* err = problem(cudaGetLastError());
  if (err) return err;
  const bool is_short = r->vocab <= (r->dtype == 0 ? warp_row<float>() : warp_row<__half>());
  if (p->pairs > 0) {
    Args scores = a;
    scores.w.label = scores.w.seq = nullptr;
    scores.stat = is_short ? w.stat : nullptr;
    err = launch_pass<kScores>(scores, r->dtype, stream);
    if (err) return err;
    scores = a;
    scores.pieces = is_short ? 1 : pieces;
    scores.stat = is_short ? w.stat : nullptr;
    err = launch_behind(true, r->dtype == 0 ? pairs_kernel<float> : r->dtype == 1 ? pairs_kernel<__nv_bfloat16> : pairs_kernel<__half>, p->pairs, 128, 0,
                        stream, scores);
    if (err) return err;
  }
  if (!a.g) return nullptr;
  a.weight = w.coef;
  a.stat = w.stat;
  return launch_pass<kGrad>(a, r->dtype, stream);
}

const char* nmtg_preference_grad(const NmtgRows* r, int pairs, cudaStream_t stream) {
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  Args a = row_args(r);
  long bytes;
  a.w = workspace(static_cast<char*>(r->workspace), r->rows, pairs, sums_pieces(r->rows, r->vocab, r->dtype), &bytes);
  a.weight = a.w.coef;
  a.stat = a.w.stat;
  return launch_pass<kGrad>(a, r->dtype, stream);
}

const char* nmtg_scale_rows(const NmtgRows* r, const float* factor, cudaStream_t stream) {
  if (r->rows <= 0 || r->vocab <= 0) return nullptr;
  if (r->dtype < 0 || r->dtype > 2) return bad_type;
  const Args a = row_args(r);
  const int grid = r->rows < 8 * num_sms() ? r->rows : 8 * num_sms();
  if (r->dtype == 0) scale_rows_kernel<float><<<grid, 256, 0, stream>>>(a, factor);
  else if (r->dtype == 1) scale_rows_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a, factor);
  else scale_rows_kernel<__half><<<grid, 256, 0, stream>>>(a, factor);
  return problem(cudaGetLastError());
}
