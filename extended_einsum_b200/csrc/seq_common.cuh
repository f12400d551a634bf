// Shared device helpers of the sequence operators: element types, groups of eight
// consecutive elements, and the exponential family in float32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/xe_b200.h"

namespace xe {
namespace seq {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// Eight consecutive elements as they lie in memory: 16 bytes of a 16-bit type, 32 of float.
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
};

__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// `count` of the eight elements are in bounds (the others read as zero); `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int count, bool vec) {
  Raw8<T> r;
  if (vec && count >= 8) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.q[i] = ldg16(reinterpret_cast<const uint4*>(p) + i);
    return r;
  }
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < count ? reinterpret_cast<const unsigned short*>(p)[2 * i] : 0u;
      const uint32_t hi = 2 * i + 1 < count ? reinterpret_cast<const unsigned short*>(p)[2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = i < count ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.q[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16)) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  } else {
    const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  }
}

template <typename T>
__device__ __forceinline__ void load8f(const T* p, int count, bool vec, float (&v)[8]) {
  unpack8<T>(load8<T>(p, count, vec), v);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int count, bool vec, const float (&v)[8]) {
  if (vec && count >= 8) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) p[i] = from_f32<T>(v[i]);
}

// Copies of 16 bytes into shared memory, awaited by the thread that issued them.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four consecutive elements: 8 bytes of a 16-bit type, 16 of float.  `whole`: one aligned load.
template <typename T>
struct Raw4 {
  uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Raw4<T> load4_if(const T* p, bool in, int count, bool whole) {
  Raw4<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) r.w[i] = 0u;
  if (whole) {
    if (in) {
      if constexpr (sizeof(T) == 2)
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
      else
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p));
    }
  } else if (in) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < count) {
        if constexpr (sizeof(T) == 2)
          r.w[i / 2] |= (uint32_t) reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i % 2));
        else
          r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      }
    }
  }
  return r;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <typename T>
__device__ __forceinline__ float value4(const Raw4<T>& r, int i) {
  if constexpr (__is_same(T, float))
    return __uint_as_float(r.w[i]);
  else if constexpr (__is_same(T, __nv_bfloat16))
    return __uint_as_float(i % 2 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
  else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i / 2]));
    return i % 2 ? f.y : f.x;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int count, bool whole, const float (&v)[4]) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (__is_same(T, __nv_bfloat16)) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) p[i] = from_f32<T>(v[i]);
}

// 2^x and 1/x of the special function unit: relative errors of 2^-22 and 2^-23.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float sigmoid(float v) { return rcp_fast(1.0f + exp2_fast(-kLog2e * v)); }

// Two float32 values in one register pair, for the packed arithmetic instructions.
typedef unsigned long long F2;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return pack2(v, v); }
__device__ __forceinline__ F2 exp2_fast2(F2 v) {
  const float2 f = unpack2(v);
  return pack2(exp2_fast(f.x), exp2_fast(f.y));
}

// 2^(d a), the decay of a recurrence, where errors of one sign add up over as many tokens as the state lasts.  The
// instruction's results lie low: measured on a B200, by 0.6e-8 of themselves on average for exponents above -0.001, by 1.7e-8
// to 2.8e-8 from there to -1 (a result rounded to nearest is off by 1.7e-8, of either sign), so that a state that lasts
// 2048 tokens came out 3.6e-5 too small.  2e-8 more in the exponent are 1.4e-8 more in the result and cost nothing, the
// addition being part of the product's rounding: 0.7e-5, and the error of dA at 2 x 2048 x 2048 x 16 falls from
// 2.1e-6 to 0.9e-6 of its norm.  2^2e-8 itself is one: d = 0 keeps a state as it is.
constexpr float kDecayShift = 2e-8f;
// a in base 2.  It stays finite: a token that does not count has d = 0 and has to leave the state alone, whatever a is.
__device__ __forceinline__ float decay_rate(float a) {
  const float v = a * kLog2e;
  return fabsf(v) > 3.4028235e38f ? copysignf(3.4028235e38f, v) : v;  // a NaN stays
}
__device__ __forceinline__ float decay(float d, float a) { return exp2_fast(fmaf(d, a, kDecayShift)); }
__device__ __forceinline__ F2 decay2(F2 d, F2 a) { return exp2_fast2(fma2(d, a, both(kDecayShift))); }

// softplus(v) = max(v, 0) + log1p(u), u = exp(-|v|) in (0, 1].  log1p(u) / u is a polynomial of degree 8
// (minimax on [0, 1]; with these float32 coefficients within 7.6e-8 of itself): the logarithm instruction would lose
// the small results of negative v, and a reciprocal would cost the special function unit another turn.  The whole is
// within 2^-21 + |v| 2^-23 of itself, the second term from the rounding of v log2(e).
__device__ __forceinline__ F2 softplus2(F2 x) {
  const float2 vw = unpack2(x);
  const float v = vw.x, w = vw.y;
  const F2 u = pack2(exp2_fast(-kLog2e * fabsf(v)), exp2_fast(-kLog2e * fabsf(w)));
  F2 p = fma2(both(5.2326941e-3f), u, both(-2.9505240e-2f));
  p = fma2(p, u, both(7.8225940e-2f));
  p = fma2(p, u, both(-0.13663246f));
  p = fma2(p, u, both(0.19106007f));
  p = fma2(p, u, both(-0.24842982f));
  p = fma2(p, u, both(0.33319098f));
  p = fma2(p, u, both(-0.49999493f));
  p = fma2(p, u, both(0.99999994f));
  return fma2(p, u, pack2(fmaxf(v, 0.0f), fmaxf(w, 0.0f)));  // a NaN stays, in u
}
__device__ __forceinline__ float softplus(float v) { return unpack2(softplus2(both(v))).x; }

// The gate v silu(z) of a pair.
__device__ __forceinline__ F2 gate2(F2 v, F2 z) {
  const float2 d = unpack2(add2(exp2_fast2(mul2(z, both(-kLog2e))), both(1.0f)));
  return mul2(v, mul2(z, pack2(rcp_fast(d.x), rcp_fast(d.y))));
}

// Length of sequence i of a ragged batch, clamped to [0, most]; `lengths` may be null (all whole).
__device__ __forceinline__ int sequence_length(const void* lengths, int is64, int i, int most) {
  if (!lengths) return most;
  const long long n = is64 ? reinterpret_cast<const long long*>(lengths)[i] : reinterpret_cast<const int*>(lengths)[i];
  return (int)(n < 0 ? 0 : (n > most ? most : n));
}

}  // namespace seq
}  // namespace xe
