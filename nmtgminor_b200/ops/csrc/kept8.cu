// Activations that wait for the backward pass in 8 bits.  The 32 elements of a block (along a row; the last block of a row may be shorter)
// share a power of two 2^e, the smallest that brings the largest magnitude to 448 or less; an element is v = x / 2^e as a number of 1 sign,
// 4 exponent and 3 mantissa bits (nearest, ties to even), e a byte of its own (e + 127).  33 bytes for 32 elements instead of 64; a
// restored element is off by at most 2^-4 of itself, or by 2^-10 * 2^e where it is below 2^-6 * 2^e.  Both steps of the arithmetic but the rounding
// are exact, so the codes do not depend on how the work is dealt out.  Infinities and NaN are kept as NaN: a gradient that meets one
// shows it.
//
//   quantise:   x -> codes                         restore:    codes -> x' and, where asked for, dropout(act(x'))
//   forward:    z -> dropout(act(z)), codes        backward:   dy, codes -> dropout-mask(dy) act'(z')
// One pass each, bound by memory.  A thread has one 16-byte vector, 4 (16-bit types) or 8 (fp32) lanes a block, whose largest magnitude
// meets in shuffles.  For 16-bit types GELU takes one exponential and one division for the function and its slope together: with
// t = 1 / (1 + p |z|) the tail Q(|z|) = exp(-z^2 / 2) (c1 t + ... + c7 t^7), fitted over the whole range to 1.1e-6 of itself (the
// form of Hastings' approximation with coefficients of our own), against the 2^-9 and 2^-12 of the rounding that follows; erff and expf
// would take longer than the bytes.  fp32 results use erfcf and expf.  Compiled without fast math: denormals are kept.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <float.h>
#include "b200_ptx.cuh"
#include "tuning_api.h"

namespace b200 {

int num_sms();

namespace {

constexpr int kBlock = 32;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <typename T> __device__ __forceinline__ float most();          // largest finite value
template <> __device__ __forceinline__ float most<float>() { return FLT_MAX; }
template <> __device__ __forceinline__ float most<__nv_bfloat16>() { return 3.38953139e38f; }
template <> __device__ __forceinline__ float most<__half>() { return 65504.f; }

template <typename T, int kN> struct alignas(sizeof(T) * kN) Pack { T v[kN]; };

// exponent of a block's power of two from its largest finite magnitude: 2^e >= largest / 448, at least 2^-127
__device__ __forceinline__ int block_exponent(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  const int e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7);       // 448 = 1.75 * 2^8
  return max(e, -127);
}
__device__ __forceinline__ float power(int e) { return e == -127 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ float inverse_power(int e) { return __uint_as_float(static_cast<uint32_t>(127 - e) << 23); }      // e = -127 .. 120
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// two codes, the first in the low byte
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 decode2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// act: 0 none, 1 ReLU, 2 GELU (erf), 3 SiLU
template <typename T> struct Tail {       // Q(a) and exp(-a^2 / 2), a >= 0
  static __device__ __forceinline__ void get(float a, float& q, float& gauss) {
    const float x = -0.72134752f * a * a;
    asm("ex2.approx.f32 %0, %1;" : "=f"(gauss) : "f"(x));
    float t;
    asm("rcp.approx.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.360624458f, a, 1.f)));
    float h = fmaf(0.0472499409f, t, -0.17956728f);
    h = fmaf(h, t, 0.179222625f);
    h = fmaf(h, t, 0.0275265627f);
    h = fmaf(h, t, 0.139533017f);
    h = fmaf(h, t, 0.142076165f);
    h = fmaf(h, t, 0.143958751f);
    q = h * t * gauss;
  }
};
template <> struct Tail<float> {
  static __device__ __forceinline__ void get(float a, float& q, float& gauss) {
    q = 0.5f * erfcf(a * 0.70710678118654752f);
    gauss = expf(-0.5f * a * a);
  }
};
template <typename T> __device__ __forceinline__ float gate(float z) {        // sigmoid
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(-1.44269504f * z));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}
template <typename T, int kAct> __device__ __forceinline__ float act_of(float z) {
  if constexpr (kAct == 1) return z > 0.f || z != z ? z : 0.f;
  if constexpr (kAct == 2) {
    float q, gauss;
    Tail<T>::get(fabsf(z), q, gauss);
    return z * (z >= 0.f ? 1.f - q : q);
  }
  if constexpr (kAct == 3) return z * gate<T>(z);
  return z;
}
template <typename T, int kAct> __device__ __forceinline__ float slope_of(float z) {
  if constexpr (kAct == 1) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  if constexpr (kAct == 2) {
    float q, gauss;
    Tail<T>::get(fabsf(z), q, gauss);
    return fmaf(z * 0.39894228040143268f, gauss, z >= 0.f ? 1.f - q : q);
  }
  if constexpr (kAct == 3) {
    const float g = gate<T>(z);
    return g * fmaf(z, 1.f - g, 1.f);
  }
  return 1.f;
}

struct Args {
  const void* in;           // x, z or dy
  void* out;                // restored x, activation or gradient
  void* out2;               // restore: dropout(act(x')) or null
  uint8_t* codes;
  uint8_t* scales;
  long rows, width, blocks; // blocks of a row
  long ld_in, ld_codes;
  float p;
  unsigned long long seed, stream_id;
  const unsigned long long* seed_dev;
};

enum Step { kQuantise = 0, kRestore = 1, kForward = 2, kBackward = 3 };

// elements [col, col + kN) of a row; `index` numbers the first for dropout; `lanes` lanes hold a block
template <typename T, int kN, int kStep, int kAct, bool kDrop>
__device__ __forceinline__ void work(const Args& a, const DropRng& rng, long row, long col, bool in_row) {
  constexpr int kLanes = kBlock / kN;
  const long block = col / kBlock, index = row * a.width + col;
  float f[kN];
  uint32_t codes[(kN + 1) / 2];
  float unit = 1.f;
  if constexpr (kStep == kRestore || kStep == kBackward) {
    if (!in_row) return;
    unit = power(static_cast<int>(a.scales[row * a.blocks + block]) - 127);
    const uint8_t* c = a.codes + row * a.ld_codes + col;
    if constexpr (kN == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(c);
      codes[0] = u.x & 0xFFFFu; codes[1] = u.x >> 16; codes[2] = u.y & 0xFFFFu; codes[3] = u.y >> 16;
    } else if constexpr (kN == 4) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(c);
      codes[0] = u & 0xFFFFu; codes[1] = u >> 16;
    } else {
      codes[0] = *c;
    }
  }
  if constexpr (kStep != kRestore) {
    Pack<T, kN> u;
    if (in_row) u = *reinterpret_cast<const Pack<T, kN>*>(static_cast<const T*>(a.in) + row * a.ld_in + col);
#pragma unroll
    for (int j = 0; j < kN; ++j) f[j] = in_row ? to_f<T>(u.v[j]) : 0.f;
  }
  if constexpr (kStep == kQuantise || kStep == kForward) {
    if (a.codes) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < kN; ++j) top = fmaxf(top, finite(f[j]) ? fabsf(f[j]) : 0.f);
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = block_exponent(top);
      const float inv = inverse_power(e);
      if (in_row) {
        float v[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = finite(f[j]) ? f[j] * inv : NAN;
        uint8_t* c = a.codes + row * a.ld_codes + col;
        if constexpr (kN == 8) {
          *reinterpret_cast<uint2*>(c) = make_uint2(encode2(v[0], v[1]) | encode2(v[2], v[3]) << 16, encode2(v[4], v[5]) | encode2(v[6], v[7]) << 16);
        } else if constexpr (kN == 4) {
          *reinterpret_cast<uint32_t*>(c) = encode2(v[0], v[1]) | encode2(v[2], v[3]) << 16;
        } else {
          *c = static_cast<uint8_t>(encode2(v[0], 0.f));
        }
        if (col % kBlock == 0) a.scales[row * a.blocks + block] = static_cast<uint8_t>(e + 127);
      }
    }
  }
  if (!in_row || kStep == kQuantise) return;
  Pack<T, kN> o, o2;
  float z[kN];
  if constexpr (kStep == kRestore || kStep == kBackward) {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      const float2 d = decode2(codes[j / 2]);
      z[j] = fminf(fmaxf(d.x * unit, -most<T>()), most<T>());
      if (d.x != d.x) z[j] = d.x;
      if constexpr (kN > 1) {
        z[j + 1] = fminf(fmaxf(d.y * unit, -most<T>()), most<T>());
        if (d.y != d.y) z[j + 1] = d.y;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    bool keep = true;
    if constexpr (kDrop) {
      const unsigned long long first = static_cast<unsigned long long>(index);      // a multiple of 4 where kN is
      if constexpr (kN % 4 == 0) keep = rng.keep(rng.word((first >> 2) + j / 4), j % 4);
      else keep = rng.keep(rng.word((first + j) >> 2), static_cast<int>((first + j) & 3));
    }
    if constexpr (kStep == kRestore) {
      o.v[j] = from_f<T>(z[j]);
      if (a.out2) {
        const float h = act_of<T, kAct>(to_f<T>(o.v[j]));
        o2.v[j] = from_f<T>(kDrop ? (keep ? h * rng.scale : 0.f) : h);
      }
    } else if constexpr (kStep == kForward) {
      const float h = act_of<T, kAct>(f[j]);
      o.v[j] = from_f<T>(kDrop ? (keep ? h * rng.scale : 0.f) : h);
    } else {
      const float d = kDrop ? (keep ? f[j] * rng.scale : 0.f) : f[j];
      o.v[j] = from_f<T>(d * slope_of<T, kAct>(z[j]));
    }
  }
  if (a.out) *reinterpret_cast<Pack<T, kN>*>(static_cast<T*>(a.out) + index) = o;
  if constexpr (kStep == kRestore)
    if (a.out2) *reinterpret_cast<Pack<T, kN>*>(static_cast<T*>(a.out2) + index) = o2;
}

// kFlat: whole blocks one after another.  Otherwise a warp goes along a row, 8 rows to a block of threads; kN = 1 takes any alignment.
template <typename T, int kN, int kStep, int kAct, bool kDrop, bool kFlat>
__global__ void __launch_bounds__(256) kept_kernel(const __grid_constant__ Args a) {
  const DropRng rng(a.seed + ((kDrop && a.seed_dev) ? *a.seed_dev : 0ull), a.stream_id, a.p);
  if constexpr (kFlat) {
    const long n = a.width / kN, step = static_cast<long>(gridDim.x) * 256;
    const long first = blockIdx.x * 256L + (threadIdx.x & ~31);
    for (long base = first; base < n; base += step) {
      const long v = base + (threadIdx.x & 31);
      work<T, kN, kStep, kAct, kDrop>(a, rng, 0, v * kN, v < n);
    }
  } else {
    const int lane = threadIdx.x & 31;
    const long per = a.blocks * (kBlock / kN);
    for (long row = blockIdx.y * 8L + (threadIdx.x >> 5); row < a.rows; row += gridDim.y * 8L)
      for (long base = blockIdx.x * 32L; base < per; base += gridDim.x * 32L) {
        const long col = (base + lane) * kN;
        work<T, kN, kStep, kAct, kDrop>(a, rng, row, col, col < a.width);
      }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int kStep, int kAct, bool kDrop>
const char* launch(const NmtgKept* k) {
  constexpr int kN = 16 / sizeof(T);
  Args a = {};
  a.in = k->in; a.out = k->out; a.out2 = k->out2; a.codes = k->codes; a.scales = k->scales;
  a.rows = k->rows; a.width = k->width; a.blocks = (k->width + kBlock - 1) / kBlock;
  a.ld_in = k->ld_in; a.ld_codes = a.blocks * kBlock;
  a.p = k->p; a.seed = k->seed; a.stream_id = k->stream_id; a.seed_dev = k->seed_dev;
  if (a.rows <= 0 || a.width <= 0) return nullptr;
  const bool vectors = a.width % kN == 0 && (a.rows == 1 || a.ld_in % kN == 0) && aligned(a.in) && aligned(a.out) && aligned(a.out2);
  if (vectors && a.width % kBlock == 0 && (a.rows == 1 || a.ld_in == a.width)) {
    a.width *= a.rows; a.blocks *= a.rows; a.rows = 1;
    const long blocks = (a.width / kN + 255) / 256, most_blocks = 8L * num_sms();
    kept_kernel<T, kN, kStep, kAct, kDrop, true><<<static_cast<unsigned>(blocks < most_blocks ? blocks : most_blocks), 256, 0, k->stream>>>(a);
  } else {
    const int each = vectors ? kN : 1;
    const long x = (a.blocks * (kBlock / each) + 31) / 32, y = (a.rows + 7) / 8;
    const dim3 grid(static_cast<unsigned>(x < 1024 ? x : 1024), static_cast<unsigned>(y < 65535 ? y : 65535));
    if (vectors) kept_kernel<T, kN, kStep, kAct, kDrop, false><<<grid, 256, 0, k->stream>>>(a);
    else kept_kernel<T, 1, kStep, kAct, kDrop, false><<<grid, 256, 0, k->stream>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

template <int kStep, int kAct>
const char* launch_type(const NmtgKept* k) {
  const bool drop = k->p > 0.f && kStep != kQuantise;
  if (k->dtype == 0) return drop ? launch<float, kStep, kAct, true>(k) : launch<float, kStep, kAct, false>(k);
  if (k->dtype == 1) return drop ? launch<__nv_bfloat16, kStep, kAct, true>(k) : launch<__nv_bfloat16, kStep, kAct, false>(k);
  if (k->dtype == 2) return drop ? launch<__half, kStep, kAct, true>(k) : launch<__half, kStep, kAct, false>(k);
  return "kept: the type must be fp32, bf16 or fp16";
}

template <int kStep>
const char* launch_act(const NmtgKept* k) {
  if (k->act == 0) return launch_type<kStep, 0>(k);
  if (k->act == 1) return launch_type<kStep, 1>(k);
  if (k->act == 2) return launch_type<kStep, 2>(k);
  if (k->act == 3) return launch_type<kStep, 3>(k);
  return "kept: unknown activation";
}

}  // namespace
}  // namespace b200

using namespace b200;

const char* nmtg_kept_quantise(const NmtgKept* k) { return launch_type<kQuantise, 0>(k); }
const char* nmtg_kept_restore(const NmtgKept* k) { return launch_act<kRestore>(k); }
const char* nmtg_kept_forward(const NmtgKept* k) { return launch_act<kForward>(k); }
const char* nmtg_kept_backward(const NmtgKept* k) { return launch_act<kBackward>(k); }
