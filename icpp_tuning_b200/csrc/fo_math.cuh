// fo_math.cuh -- paired fp32 arithmetic, and the gated activations built on it.
#pragma once
#include "fo_kernel.cuh"

namespace fo {

enum : int { ACT_SILU = 4 };  // beside ACT_RELU, ACT_GELU_TANH, ACT_GELU_ERF

// Two fp32 values in one 64-bit register: sm_100 adds and multiplies both in one
// instruction.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ float2 both(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ float sum(Two a) {
  const float2 f = both(a);
  return f.x + f.y;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(Two a) {
  const float2 f = both(a);
  return pack2<DT>(f.x, f.y);
}

// What 16 bits leave of v, high being its first part: nothing where that is not finite, so that
// the parts of an infinity add up to it.
__device__ __forceinline__ float low_part(float v, float high) {
  const float rest = v - high;
  return fabsf(rest) < __builtin_huge_valf() ? rest : 0.f;
}

// The gated activations and their derivatives, in forms whose error stays at fp32's: the
// sigmoid ones take one exponential and one reciprocal a value (gelu_tanh(g) = g sigmoid(2 w),
// w = sqrt(2 / pi) (g + 0.044715 g^3)), the erf one a reciprocal (erf by Abramowitz & Stegun
// 7.1.28, |error| <= 3e-7) and, for the derivative, an exponential.
__device__ __forceinline__ Two exp_of(Two x) {
  const float2 f = both(mul2(x, two(1.4426950408889634f)));
  float a, b;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(f.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(f.y));
  return two(a, b);
}
__device__ __forceinline__ Two rcp_of(Two x) {
  const float2 f = both(x);
  float a, b;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(f.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(f.y));
  return two(a, b);
}
__device__ __forceinline__ Two sigmoid(Two x) { return rcp_of(add2(two(1.0f), exp_of(mul2(x, two(-1.0f))))); }

__device__ __forceinline__ Two normal_cdf(Two g) {  // (1 + erf(g / sqrt 2)) / 2
  const Two z = mul2(g, two(0.7071067811865476f));
  const float2 f = both(z);
  const Two az = two(fabsf(f.x), fabsf(f.y));
  Two p = fma2(two(4.30638e-5f), az, two(2.765672e-4f));
  p = fma2(p, az, two(1.520143e-4f));
  p = fma2(p, az, two(9.2705272e-3f));
  p = fma2(p, az, two(4.22820123e-2f));
  p = fma2(p, az, two(7.05230784e-2f));
  p = fma2(p, az, two(1.0f));
  Two r = rcp_of(p);
  r = mul2(r, r);
  r = mul2(r, r);
  r = mul2(r, r);
  r = mul2(r, r);
  const float2 e = both(fma2(r, two(-1.0f), two(1.0f)));
  return fma2(two(0.5f), two(copysignf(e.x, f.x), copysignf(e.y, f.y)), two(0.5f));
}

template <int ACT>
__device__ __forceinline__ Two gate_act(Two g) {
  if constexpr (ACT == ACT_SILU) return mul2(g, sigmoid(g));
  if constexpr (ACT == ACT_GELU_TANH)
    return mul2(g, sigmoid(mul2(mul2(two(1.5957691216057308f), g), fma2(two(0.044715f), mul2(g, g), two(1.0f)))));
  if constexpr (ACT == ACT_GELU_ERF) return mul2(g, normal_cdf(g));
  const float2 f = both(g);
  return two(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);
}

__device__ __forceinline__ Two gate_act(int act, Two g) {
  if (act == ACT_SILU) return gate_act<ACT_SILU>(g);
  if (act == ACT_GELU_TANH) return gate_act<ACT_GELU_TANH>(g);
  if (act == ACT_GELU_ERF) return gate_act<ACT_GELU_ERF>(g);
  return gate_act<ACT_RELU>(g);
}

// From dh: dg = dh u act'(g), du = dh act(g), and h = act(g) u.
template <int ACT>
__device__ __forceinline__ void gate_grad(Two dh, Two g, Two u, Two& dg, Two& du, Two& h) {
  Two s, ds;
  if constexpr (ACT == ACT_SILU) {
    const Two p = sigmoid(g);
    s = mul2(g, p);
    ds = fma2(s, fma2(p, two(-1.0f), two(1.0f)), p);
  } else if constexpr (ACT == ACT_GELU_TANH) {
    // s = g p, p = sigmoid(2 w): s' = p + s (1 - p) 2 w'
    const Two g2 = mul2(g, g);
    const Two p = sigmoid(mul2(mul2(two(1.5957691216057308f), g), fma2(two(0.044715f), g2, two(1.0f))));
    s = mul2(g, p);
    const Two w = mul2(two(1.5957691216057308f), fma2(two(0.134145f), g2, two(1.0f)));
    ds = fma2(mul2(s, fma2(p, two(-1.0f), two(1.0f))), w, p);
  } else if constexpr (ACT == ACT_GELU_ERF) {
    const Two c = normal_cdf(g);
    s = mul2(g, c);
    ds = fma2(mul2(g, two(0.3989422804014327f)), exp_of(mul2(mul2(g, two(-0.5f)), g)), c);
  } else {
    const float2 f = both(g);
    s = two(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);
    ds = two(f.x > 0.f ? 1.f : 0.f, f.y > 0.f ? 1.f : 0.f);
  }
  dg = mul2(mul2(dh, u), ds);
  du = mul2(dh, s);
  h = mul2(s, u);
}

}  // namespace fo
