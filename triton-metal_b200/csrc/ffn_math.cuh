// Element conversions, 16-byte packets, and the activations with their derivatives, in fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ffn_core.h"
#include "sm100_ptx.cuh"

namespace tmc {
namespace ffn {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC consecutive elements as fp32.  VEC > 1 is one 16-byte access (the address must be aligned to
// it); the plain loads go through the read-only path with no cache hint.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(*p);
  } else {
    static_assert(VEC * sizeof(T) == 16, "one packet");
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(e[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(v[0]);
  } else {
    static_assert(VEC * sizeof(T) == 16, "one packet");
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
}

// 1 / (1 + exp(-z)): exp overflows to infinity for z < -88 and the quotient is then 0, its limit.
// __expf and __fdividef err by a few units in the last place of fp32, far below a 16-bit rounding;
// fp32 operands (PRECISE) take expf and the exact quotient.
template <bool PRECISE>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (PRECISE) return 1.f / (1.f + expf(-z));
  return __fdividef(1.f, 1.f + __expf(-z));
}
// z kept inside the range where the derivatives still change (a comparison lets a NaN through):
// beyond it exp(-z^2/2) and s(1-s) are 0 in fp32 and would meet an overflowed factor.
__device__ __forceinline__ float bounded(float z) { return z > 100.f ? 100.f : (z < -100.f ? -100.f : z); }

constexpr float kSqrtHalf = 0.70710678118654752440f;
constexpr float kInvSqrt2Pi = 0.39894228040143267794f;
constexpr float kTanhA = 0.79788456080286535588f;   // sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The normal distribution's upper tail at |z|, 1 - Phi(|z|), for 16-bit results, without a branch where erff and
// erfcf have several: exp(-z^2 / 2) t (c0 + c1 t + ... + c5 t^5) with t = 1 / (1 + kTailT |z|).  The coefficients
// are this file's own: a least-squares fit, reweighted towards the least largest error, of the tail over its
// exponential on |z| <= 13.6, where the tail leaves fp32's range.  In fp32 it is off by at most 3e-7, and by
// 2.2e-5 of itself wherever that is less - a twentieth of f16's half step far out, where a bound of the first
// kind alone leaves gelu(-5) a step or more off.  `density` is exp(-z^2 / 2), which the derivative needs too.
constexpr float kTailT = 0.297f;
constexpr float kTail0 = 0.11908809f, kTail1 = 0.10998656f, kTail2 = 0.15484719f, kTail3 = -0.041209962f,
                kTail4 = 0.23927316f, kTail5 = -0.08198507f;
__device__ __forceinline__ float normal_tail(float z, float& density) {
  const float a = fabsf(z);
  density = __expf(-0.5f * a * a);
  const float t = __fdividef(1.f, fmaf(kTailT, a, 1.f));
  float poly = fmaf(kTail5, t, kTail4);
  poly = fmaf(poly, t, kTail3);
  poly = fmaf(poly, t, kTail2);
  poly = fmaf(poly, t, kTail1);
  poly = fmaf(poly, t, kTail0);
  return poly * t * density;
}

// gelu_tanh(z) = z/2 (1 + tanh(a(z + b z^3))) = z sigmoid(2a(z + b z^3)): no cancellation for z < 0.
template <bool PRECISE>
__device__ __forceinline__ float act_forward(Act act, float z) {
  switch (act) {
    case Act::Relu: return z != z ? z : fmaxf(z, 0.f);          // fmaxf alone would drop a NaN
    case Act::Gelu: {
      // erfc keeps the tail's relative accuracy where 1 + erf cancels (z = -5: four per cent off, z < -5.6: 0);
      // z is bounded below where erfc is 0, so that minus infinity gives 0, the limit
      if constexpr (PRECISE) return 0.5f * (z < -100.f ? -100.f : z) * erfcf(-z * kSqrtHalf);
      // z Phi(z) = max(z, 0) - |z| tail(|z|); |z| bounded where the tail is 0, so that infinities give the limits
      float density;
      const float a = min_nan(fabsf(z), 100.f);
      return max_nan(z, 0.f) - a * normal_tail(a, density);
    }
    case Act::GeluTanh: return z * sigmoid<PRECISE>(2.f * kTanhA * (z + kTanhB * z * z * z));
    case Act::Silu: return z * sigmoid<PRECISE>(z);
    case Act::Sigmoid: return sigmoid<PRECISE>(z);
    default: return z;
  }
}
template <bool PRECISE>
__device__ __forceinline__ float act_derivative(Act act, float z) {
  z = bounded(z);
  switch (act) {
    case Act::Relu: return z != z ? z : (z > 0.f ? 1.f : 0.f);
    case Act::Gelu: {
      if constexpr (PRECISE) return 0.5f * erfcf(-z * kSqrtHalf) + z * kInvSqrt2Pi * expf(-0.5f * z * z);
      float density;
      const float tail = normal_tail(z, density);
      return fmaf(z * kInvSqrt2Pi, density, z < 0.f ? tail : 1.f - tail);
    }
    case Act::GeluTanh: {
      const float s = sigmoid<PRECISE>(2.f * kTanhA * (z + kTanhB * z * z * z));
      return s + z * s * (1.f - s) * 2.f * kTanhA * (1.f + 3.f * kTanhB * z * z);
    }
    case Act::Silu: {
      const float s = sigmoid<PRECISE>(z);
      return s * (1.f + z * (1.f - s));
    }
    case Act::Sigmoid: {
      const float s = sigmoid<PRECISE>(z);
      return s * (1.f - s);
    }
    default: return 1.f;
  }
}

// Value and derivative together: what both need - the sigmoid, the tail - is computed once.
template <bool PRECISE>
__device__ __forceinline__ void act_both(Act act, float z, float& value, float& slope) {
  const float zb = bounded(z);
  switch (act) {
    case Act::Gelu: {
      if constexpr (PRECISE) break;
      float density;
      const float tail = normal_tail(zb, density);
      value = max_nan(z, 0.f) - fabsf(zb) * tail;
      slope = fmaf(zb * kInvSqrt2Pi, density, zb < 0.f ? tail : 1.f - tail);
      return;
    }
    case Act::GeluTanh: {
      const float s = sigmoid<PRECISE>(2.f * kTanhA * (zb + kTanhB * zb * zb * zb));
      value = z * s;
      slope = s + zb * s * (1.f - s) * 2.f * kTanhA * (1.f + 3.f * kTanhB * zb * zb);
      return;
    }
    case Act::Silu: {
      const float s = sigmoid<PRECISE>(zb);
      value = z * s;
      slope = s * (1.f + zb * (1.f - s));
      return;
    }
    case Act::Sigmoid: {
      value = sigmoid<PRECISE>(zb);
      slope = value * (1.f - value);
      return;
    }
    default: break;
  }
  value = act_forward<PRECISE>(act, z);
  slope = act_derivative<PRECISE>(act, z);
}

// The activation of a row's registers: gelu of 16-bit results two-wide (it is the dearest: with scalar
// arithmetic 16384 x 1024 x 4096 ran at 1069 TFLOP/s, this way at 1169), the others element by element.
template <Act ACT, int N>
__device__ __forceinline__ void act_row(float (&v)[N]) {
  if constexpr (ACT == Act::Gelu) {
    auto both = [](float c) { return ptx::pack_f32x2(c, c); };
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float a0 = min_nan(fabsf(v[i]), 100.f), a1 = min_nan(fabsf(v[i + 1]), 100.f);
      const uint64_t a = ptx::pack_f32x2(a0, a1);
      // exp(-z^2 / 2) as a power of two
      const uint64_t power = ptx::mul_f32x2(ptx::mul_f32x2(a, a), both(-0.5f * 1.44269504088896341f));
      const uint64_t below = ptx::fma_f32x2(a, both(kTailT), both(1.f));
      float p0, p1, b0, b1;
      ptx::unpack_f32x2(power, p0, p1);
      ptx::unpack_f32x2(below, b0, b1);
      const uint64_t density = ptx::pack_f32x2(ptx::fast_exp2(p0), ptx::fast_exp2(p1));
      const uint64_t t = ptx::pack_f32x2(fast_rcp(b0), fast_rcp(b1));
      uint64_t poly = ptx::fma_f32x2(both(kTail5), t, both(kTail4));
      poly = ptx::fma_f32x2(poly, t, both(kTail3));
      poly = ptx::fma_f32x2(poly, t, both(kTail2));
      poly = ptx::fma_f32x2(poly, t, both(kTail1));
      poly = ptx::fma_f32x2(poly, t, both(kTail0));
      const uint64_t tail = ptx::mul_f32x2(ptx::mul_f32x2(poly, t), density);
      const uint64_t out = ptx::fma_f32x2(ptx::pack_f32x2(-a0, -a1), tail, ptx::pack_f32x2(max_nan(v[i], 0.f), max_nan(v[i + 1], 0.f)));
      ptx::unpack_f32x2(out, v[i], v[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_forward<false>(ACT, v[i]);
  }
}

// Calls f with the activation as a compile-time constant.
template <typename F>
__device__ __forceinline__ void with_act(Act act, F&& f) {
  switch (act) {
    case Act::Relu: f(std::integral_constant<Act, Act::Relu>{}); break;
    case Act::Gelu: f(std::integral_constant<Act, Act::Gelu>{}); break;
    case Act::GeluTanh: f(std::integral_constant<Act, Act::GeluTanh>{}); break;
    case Act::Silu: f(std::integral_constant<Act, Act::Silu>{}); break;
    case Act::Sigmoid: f(std::integral_constant<Act, Act::Sigmoid>{}); break;
    default: f(std::integral_constant<Act, Act::None>{}); break;
  }
}

}  // namespace ffn
}  // namespace tmc
