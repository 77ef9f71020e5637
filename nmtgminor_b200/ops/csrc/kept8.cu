// Activations that wait for the backward pass in 8 bits.  The 32 elements of a block (along a row; the last block of a row may be shorter)
// share a power of two 2^e, the smallest that brings the largest magnitude to 448 or less; an element is v = x / 2^e as a number of 1 sign,
// 4 exponent and 3 mantissa bits (nearest, ties to even), e a byte of its own (e + 127).  33 bytes for 32 elements instead of 64; a
// restored element is off by at most 2^-4 of itself, or by 2^-10 * 2^e where it is below 2^-6 * 2^e.  Both steps of the arithmetic but the rounding
// are exact, so the codes do not depend on how the work is dealt out.  Infinities and NaN are kept as NaN: a gradient that meets one
// shows it.
//
//   quantise:   x -> codes                         restore:    codes -> x' and, where asked for, dropout(act(x'))
//   forward:    z -> dropout(act(z)), codes        backward:   dy, codes -> dropout-mask(dy) act'(z')
// One pass each, bound by memory.  A thread has 32 bytes of a 16-bit type where whole blocks follow one another (2 lanes to a block of 32), otherwise one
// 16-byte vector (4 lanes; of fp32 8) or one element (32); a block's largest magnitude meets in shuffles.  For 16-bit types GELU takes one exponential and one division for the function and its slope together: with
// t = 1 / (1 + p |z|) the tail Q(|z|) = exp(-z^2 / 2) (c1 t + ... + c7 t^7), fitted over the whole range to 1.1e-6 of itself (the
// form of Hastings' approximation with coefficients of our own), against the 2^-9 and 2^-12 of the rounding that follows; erff and expf
// would take longer than the bytes.  fp32 results use erfcf and expf.  Compiled without fast math: codes, restored
// values and fp32 results have their denormals; exponentials of 16-bit results that are below 2^-126 count as 0.
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
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(gauss) : "f"(x));
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.360624458f, a, 1.f)));
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
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.44269504f * z));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
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
__device__ __noinline__ void work(const Args& a, const DropRng& rng, long row, long col, bool in_row) {
  constexpr int kLanes = kBlock / kN;
  const long block = col / kBlock, index = row * a.width + col;
  float f[kN];
  uint32_t codes[(kN + 1) / 2];
  float unit = 1.f;
  if constexpr (kStep == kRestore || kStep == kBackward) {
    if (!in_row) return;
    unit = power(static_cast<int>(a.scales[row * a.blocks + block]) - 127);
    const uint8_t* c = a.codes + row * a.ld_codes + col;
    if constexpr (kN == 16) {
      const uint4 u = *reinterpret_cast<const uint4*>(c);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) codes[j] = (w[j / 2] >> (16 * (j & 1))) & 0xFFFFu;
    } else if constexpr (kN == 8) {
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
        if constexpr (kN == 16) {
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = encode2(v[2 * j], v[2 * j + 1]);
          *reinterpret_cast<uint4*>(c) = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        } else if constexpr (kN == 8) {
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

// ---- 16-bit types, whole vectors: two elements to an instruction wherever there is one for two -----------------------------
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
      "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rcp(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }

__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ uint32_t pack2(float2 v, __nv_bfloat16) { const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack2(float2 v, __half) { const __half2 h = __floats2half2_rn(v.x, v.y); return *reinterpret_cast<const uint32_t*>(&h); }

// Tail::get for two
__device__ __forceinline__ void tails(float2 a, float2& q, float2& gauss) {
  const float2 x = mul2(mul2(a, twice(-0.72134752f)), a);
  gauss = make_float2(ex2(x.x), ex2(x.y));
  const float2 d = fma2(a, twice(0.360624458f), twice(1.f)), t = make_float2(rcp(d.x), rcp(d.y));
  float2 h = fma2(twice(0.0472499409f), t, twice(-0.17956728f));
  h = fma2(h, t, twice(0.179222625f));
  h = fma2(h, t, twice(0.0275265627f));
  h = fma2(h, t, twice(0.139533017f));
  h = fma2(h, t, twice(0.142076165f));
  h = fma2(h, t, twice(0.143958751f));
  q = mul2(mul2(h, t), gauss);
}
template <typename T, int kAct> __device__ __forceinline__ float2 acts_of(float2 z) {
  if constexpr (kAct == 2) {
    const float2 a = make_float2(fabsf(z.x), fabsf(z.y));
    float2 q, gauss;
    tails(a, q, gauss);
    return make_float2(fmaf(-a.x, q.x, fmaxf(z.x, 0.f)), fmaf(-a.y, q.y, fmaxf(z.y, 0.f)));       // z Q(-z) = max(z, 0) - |z| Q(|z|)
  }
  return make_float2(act_of<T, kAct>(z.x), act_of<T, kAct>(z.y));
}
// A restored element has 4 significant bits, so that the slopes of GELU and SiLU have few values: a block makes a table of them, for every exponent,
// 3 bits and sign, and an element costs a look into shared memory.  Between 2^-18 and 2^7 the slopes are computed in full precision; below it is
// 1/2 but for 2^-18, above 0 or 1, and of NaN NaN.  (33.6 M elements with GELU: 46 us with the arithmetic of the forward pass, 38 with a table of that range and
// its ends looked after at every element.)
constexpr int kSlopes = 1 << 12, kSlopeLow = (127 - 18) << 3, kSlopeHigh = (127 + 7) << 3;
template <int kAct> __device__ __forceinline__ void make_slopes(float* table) {
  for (int i = threadIdx.x; i < kSlopes; i += 256) {
    const int at = i & 0x7FF;
    const bool down = i >> 11;
    float v = at < kSlopeLow ? 0.5f : at >= 255 << 3 ? NAN : down ? 0.f : 1.f;
    if (at >= kSlopeLow && at < kSlopeHigh) v = slope_of<float, kAct>(__uint_as_float(static_cast<uint32_t>(i) << 20));
    table[i] = v;
  }
  __syncthreads();
}
template <typename T, int kAct> __device__ __forceinline__ float2 slopes_of(float2 z, const float* table) {
  if constexpr (kAct == 2 || kAct == 3) return make_float2(table[__float_as_uint(z.x) >> 20], table[__float_as_uint(z.y) >> 20]);
  return make_float2(slope_of<T, kAct>(z.x), slope_of<T, kAct>(z.y));
}

// 16 or 32 bytes at a time
template <int kWords> __device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[kWords]) {
  if constexpr (kWords == 8) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
  } else {
    const uint4 u = *static_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
}
template <int kWords> __device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[kWords]) {
  if constexpr (kWords == 8)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7]) : "memory");
  else
    *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// `work` for 8 or 16 elements of 16 bits that are all there and ordinary: no infinity or NaN, nothing that leaves the type when it is restored.  What
// is not ordinary is left to `work`; returns whether it was done.  All lanes of a warp, `in_row` for those with elements.
template <typename T, int kN, int kStep, int kAct, bool kDrop>
__device__ __forceinline__ bool work_pairs(const Args& a, const DropRng& rng, const float* table, long row, long col, bool in_row) {
  constexpr int kWords = kN / 2;
  const long block = col / kBlock, index = row * a.width + col;
  uint32_t w[kWords] = {};
  uint32_t codes[kN / 4] = {};
  int scale = 0;
  bool ordinary = true;
  if constexpr (kStep != kRestore) {
    if (in_row) load_words(static_cast<const T*>(a.in) + row * a.ld_in + col, w);
  }
  if constexpr (kStep == kRestore || kStep == kBackward) {
    if (in_row) {
      const uint8_t* const c = a.codes + row * a.ld_codes + col;
      if constexpr (kN == 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(c);
        codes[0] = u.x; codes[1] = u.y; codes[2] = u.z; codes[3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(c);
        codes[0] = u.x; codes[1] = u.y;
      }
      scale = a.scales[row * a.blocks + block];
      // restored values go to 448 * 2^(scale - 127): below 2^126 in bf16, 57344 in fp16
      ordinary = scale <= (most<T>() > 1e6f ? 244 : 134);
    }
  }
  uint32_t top = 0;
  if constexpr (kStep == kQuantise || kStep == kForward) {
    // magnitudes order as their bits do; infinity and NaN are above every number
#pragma unroll
    for (int j = 0; j < kWords; ++j) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
    top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
    for (int o = 1; o < kBlock / kN; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    ordinary = top < (most<T>() > 1e6f ? 0x7F80u : 0x7C00u);
  }
  if (!__all_sync(0xffffffffu, ordinary)) return false;
  if constexpr (kStep == kQuantise || kStep == kForward) {
    if (a.codes && in_row) {
      const int e = block_exponent(unpack2(top, T()).x);
      const float2 inv = twice(inverse_power(e));
      uint32_t c[kWords];
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const float2 v = mul2(unpack2(w[j], T()), inv);
        c[j] = encode2(v.x, v.y);
      }
      uint8_t* const to = a.codes + row * a.ld_codes + col;
      if constexpr (kN == 16) *reinterpret_cast<uint4*>(to) = make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16);
      else *reinterpret_cast<uint2*>(to) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      if (col % kBlock == 0) a.scales[row * a.blocks + block] = static_cast<uint8_t>(e + 127);
    }
  }
  if (!in_row || kStep == kQuantise) return true;
  const float2 unit = twice(power(scale - 127));
  uint32_t o[kWords], o2[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    float2 keep = twice(1.f);
    if constexpr (kDrop) {
      const uint32_t word = rng.word((static_cast<unsigned long long>(index) >> 2) + j / 2);
      keep = make_float2(rng.keep(word, 2 * (j & 1)) ? rng.scale : 0.f, rng.keep(word, 2 * (j & 1) + 1) ? rng.scale : 0.f);
    }
    float2 z = make_float2(0.f, 0.f);
    if constexpr (kStep == kRestore || kStep == kBackward) z = mul2(decode2(codes[j / 2] >> (16 * (j & 1))), unit);
    float2 v;
    if constexpr (kStep == kRestore) {
      o[j] = pack2(z, T());
      if (a.out2) {
        v = acts_of<T, kAct>(z);
        o2[j] = pack2(kDrop ? mul2(v, keep) : v, T());
      }
    } else if constexpr (kStep == kForward) {
      v = acts_of<T, kAct>(unpack2(w[j], T()));
      o[j] = pack2(kDrop ? mul2(v, keep) : v, T());
    } else {
      v = unpack2(w[j], T());
      if constexpr (kDrop) v = mul2(v, keep);
      o[j] = pack2(mul2(v, slopes_of<T, kAct>(z, table)), T());
    }
  }
  if (a.out) store_words(static_cast<T*>(a.out) + index, o);
  if constexpr (kStep == kRestore)
    if (a.out2) store_words(static_cast<T*>(a.out2) + index, o2);
  return true;
}

template <typename T, int kN, int kStep, int kAct, bool kDrop>
__device__ __forceinline__ void any_work(const Args& a, const DropRng& rng, const float* table, long row, long col, bool in_row) {
  if constexpr (kN >= 8)
    if (work_pairs<T, kN, kStep, kAct, kDrop>(a, rng, table, row, col, in_row)) return;
  work<T, kN, kStep, kAct, kDrop>(a, rng, row, col, in_row);
}

// kFlat: whole blocks one after another.  Otherwise a warp goes along a row, 8 rows to a block of threads; kN = 1 takes any alignment.
template <typename T, int kN, int kStep, int kAct, bool kDrop, bool kFlat>
__global__ void __launch_bounds__(256) kept_kernel(const __grid_constant__ Args a) {
  const DropRng rng(a.seed + ((kDrop && a.seed_dev) ? *a.seed_dev : 0ull), a.stream_id, a.p);
  constexpr bool kTable = kN >= 8 && kStep == kBackward && (kAct == 2 || kAct == 3);
  __shared__ float table[kTable ? kSlopes : 1];
  if constexpr (kTable) make_slopes<kAct>(table);
  if constexpr (kFlat) {
    const long n = a.width / kN, step = static_cast<long>(gridDim.x) * 256;
    const long first = blockIdx.x * 256L + (threadIdx.x & ~31);
    for (long base = first; base < n; base += step) {
      const long v = base + (threadIdx.x & 31);
      any_work<T, kN, kStep, kAct, kDrop>(a, rng, table, 0, v * kN, v < n);
    }
  } else {
    const int lane = threadIdx.x & 31;
    const long per = a.blocks * (kBlock / kN);
    for (long row = blockIdx.y * 8L + (threadIdx.x >> 5); row < a.rows; row += gridDim.y * 8L)
      for (long base = blockIdx.x * 32L; base < per; base += gridDim.x * 32L) {
        const long col = (base + lane) * kN;
        any_work<T, kN, kStep, kAct, kDrop>(a, rng, table, row, col, col < a.width);
      }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool wide_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// as many blocks as the GPU holds: all of them go through the same share
const char* launch_flat(void (*kernel)(const Args), const Args& a, int each, cudaStream_t stream) {
  int held = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, 256, 0);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  const long blocks = (a.width / each + 255) / 256, most = static_cast<long>(held < 1 ? 1 : held) * num_sms();
  kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(a);
  e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

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
    constexpr int kWide = sizeof(T) == 2 ? 16 : kN;              // 32 bytes of a 16-bit type
    const bool wide = kWide > kN && wide_aligned(a.in) && wide_aligned(a.out) && wide_aligned(a.out2) && aligned(a.codes);
    if (wide) return launch_flat(kept_kernel<T, kWide, kStep, kAct, kDrop, true>, a, kWide, k->stream);
    return launch_flat(kept_kernel<T, kN, kStep, kAct, kDrop, true>, a, kN, k->stream);
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
