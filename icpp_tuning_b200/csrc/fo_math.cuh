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

// The gated activations and their derivatives.  The sigmoid ones take one exponential and one
// reciprocal a value (gelu_tanh(g) = g sigmoid(2 w), w = sqrt(2 / pi) (g + 0.044715 g^3)); the
// erf one takes the same two.  Errors are a few units of fp32, relative to the value, the
// exponential's argument x adding |x| 2^-24: tests/test_gate_math_gpu.py holds the bounds.
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

// (1 + erf(g / sqrt 2)) / 2 and bell = e^(-g^2 / 2): the tail below -|g| is bell times a
// polynomial in t = 1 / (1 + 0.3 |g|), the minimax fit of degree 8 to the tail / bell over |g| <=
// 14 (relative error 6e-8; a Remez iteration on 0.5 erfcx(|g| / sqrt 2)).  So the tail keeps its
// relative accuracy where 1 + erf cancels.
__device__ __forceinline__ Two normal_cdf(Two g, Two& bell) {
  const float2 f = both(g);
  const Two t = rcp_of(fma2(two(0.3f), two(fabsf(f.x), fabsf(f.y)), two(1.0f)));
  Two p = fma2(two(3.837832828e-2f), t, two(-1.691660597e-1f));
  p = fma2(p, t, two(2.286599804e-1f));
  p = fma2(p, t, two(-7.650637060e-2f));
  p = fma2(p, t, two(1.425354567e-1f));
  p = fma2(p, t, two(9.468354909e-2f));
  p = fma2(p, t, two(1.219203362e-1f));
  p = fma2(p, t, two(1.194876897e-1f));
  p = fma2(p, t, two(7.168838789e-6f));
  bell = exp_of(mul2(mul2(g, two(-0.5f)), g));
  const Two tail = mul2(p, bell);
  const float2 lo = both(tail), hi = both(fma2(tail, two(-1.0f), two(1.0f)));
  return two(f.x < 0.f ? lo.x : hi.x, f.y < 0.f ? lo.y : hi.y);
}

template <int ACT>
__device__ __forceinline__ Two gate_act(Two g) {
  if constexpr (ACT == ACT_SILU) return mul2(g, sigmoid(g));
  if constexpr (ACT == ACT_GELU_TANH)
    return mul2(g, sigmoid(mul2(mul2(two(1.5957691216057308f), g), fma2(two(0.044715f), mul2(g, g), two(1.0f)))));
  if constexpr (ACT == ACT_GELU_ERF) {
    Two bell;
    return mul2(g, normal_cdf(g, bell));
  }
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
    // (past +-64, where p is 1 or 0 and s' with it, g^3 and w' stay those of 64: an infinity would
    // meet 1 - p = 0)
    const float2 f = both(g);
    const Two near = two(fminf(fmaxf(f.x, -64.f), 64.f), fminf(fmaxf(f.y, -64.f), 64.f)), g2 = mul2(near, near);
    const Two p = sigmoid(mul2(mul2(two(1.5957691216057308f), near), fma2(two(0.044715f), g2, two(1.0f))));
    s = mul2(g, p);
    const Two w = mul2(two(1.5957691216057308f), fma2(two(0.134145f), g2, two(1.0f)));
    ds = fma2(mul2(s, fma2(p, two(-1.0f), two(1.0f))), w, p);
  } else if constexpr (ACT == ACT_GELU_ERF) {
    Two bell;
    const Two c = normal_cdf(g, bell);
    s = mul2(g, c);
    ds = fma2(mul2(g, two(0.3989422804014327f)), bell, c);
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
