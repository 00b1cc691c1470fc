// What a product's epilogue can do to a float32 element before its one rounding: bias, activation,
// residual, or the slope of an activation (the gradient passing through it).  Shared by the
// tensor-core kernel, the CUDA-core kernel, the kernels that sum the parts of a cut contraction
// and the elementwise activation gradient, so that every path computes the same function.
//
//   z    = product + bias                 value  = act(z) + residual          (pre, if kept, = z)
//   gradient form:                        value  = product * act'(grad_pre)
//
// All of it happens in float32 on the unrounded product; each stored tensor is rounded once.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace hc {

// Every activation but ReLU is z * S(z) with S rising from 0 to 1:
//   SILU       S = sigma(z), sigma(t) = 1 / (1 + e^-t)
//   GELU_TANH  S = sigma(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which is (1 + tanh u) / 2 without its
//              cancellation in the lower tail, where float16 still has 11 bits to fill
//   GELU       S = Phi, the normal distribution function
// and the slope is S + z S'.
//
// Phi(-y) = e^(-y^2/2) Q(y) for y >= 0 and Phi(y) = 1 - Phi(-y), where Q falls slowly from 1/2 and is fitted
// by t R(t), t = 1/(1 + 0.3 y), R a polynomial of degree 7, with least largest relative error over y <= 14 (Phi(-14) is 8e-45,
// below float32's normals): 1.7e-7.  The exponent's rounding dominates: 6e-7 of Phi at z = -3, 1.3e-6 at -6.
// kFast, for float16 results, takes the hardware's exponential and reciprocal (a few 2^-23).
__device__ __forceinline__ float exp2_approx(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// e^(c t), t's factor c folded into the base change where the exponential is the hardware's.
template <bool kFast>
__device__ __forceinline__ float exp_f(float c, float t) { return kFast ? exp2_approx(c * 1.4426950408889634f * t) : expf(c * t); }
template <bool kFast>
__device__ __forceinline__ float recip_f(float d) {
  if (!kFast) return 1.0f / d;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// Two float32 operations in one instruction; each lane rounds as its scalar form does.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*(unsigned long long*)&r)
      : "l"(*(const unsigned long long*)&a), "l"(*(const unsigned long long*)&b), "l"(*(const unsigned long long*)&c));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(unsigned long long*)&r) : "l"(*(const unsigned long long*)&a), "l"(*(const unsigned long long*)&b));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*(unsigned long long*)&r) : "l"(*(const unsigned long long*)&a), "l"(*(const unsigned long long*)&b));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

constexpr float kTanh1 = 1.5957691216057308f, kTanh3 = kTanh1 * 0.044715f;   // 2 sqrt(2/pi), and times 0.044715

// Phi(z), and e^(-z^2/2) for the slope.
template <bool kFast>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float y = fabsf(z);
  const float t = recip_f<kFast>(fmaf(0.3f, y, 1.0f));
  float r = 0.035674773156642914f;
  r = fmaf(r, t, -0.1572030782699585f);
  r = fmaf(r, t, 0.20635350048542023f);
  r = fmaf(r, t, -0.05368364229798317f);
  r = fmaf(r, t, 0.12856163084506989f);
  r = fmaf(r, t, 0.09991349279880524f);
  r = fmaf(r, t, 0.12075395882129669f);
  r = fmaf(r, t, 0.11962930113077164f);
  e = kFast ? exp2_approx(-0.72134752044448170f * y * y) : expf(-0.5f * y * y);
  const float tail = t * r * e;
  return z < 0.0f ? tail : 1.0f - tail;   // NaN: 1 - NaN
}

// The same for two values, as float16 results take it: 15 instructions a value instead of 26.
__device__ __forceinline__ float2 normal_cdf_pair(float2 z, float2& e) {
  const float2 y = make_float2(fabsf(z.x), fabsf(z.y));
  const float2 d = fma2(both(0.3f), y, both(1.0f));
  const float2 t = make_float2(recip_f<true>(d.x), recip_f<true>(d.y));
  float2 r = fma2(both(0.035674773156642914f), t, both(-0.1572030782699585f));
  r = fma2(r, t, both(0.20635350048542023f));
  r = fma2(r, t, both(-0.05368364229798317f));
  r = fma2(r, t, both(0.12856163084506989f));
  r = fma2(r, t, both(0.09991349279880524f));
  r = fma2(r, t, both(0.12075395882129669f));
  r = fma2(r, t, both(0.11962930113077164f));
  const float2 q = mul2(mul2(y, both(-0.72134752044448170f)), y);
  e = make_float2(exp2_approx(q.x), exp2_approx(q.y));
  const float2 tail = mul2(mul2(t, r), e), rest = fma2(both(-1.0f), tail, both(1.0f));
  return make_float2(z.x < 0.0f ? tail.x : rest.x, z.y < 0.0f ? tail.y : rest.y);
}

template <int kAct, bool kFast, int W>
__device__ __forceinline__ void act_apply_t(float (&x)[W]) {
  if constexpr (kAct == HC_ACT_GELU && kFast && W % 2 == 0) {
#pragma unroll
    for (int e = 0; e < W; e += 2) {
      const float2 z = make_float2(x[e], x[e + 1]);
      float2 g;
      const float2 v = mul2(z, normal_cdf_pair(z, g));
      x[e] = v.x;
      x[e + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; e++) {
      const float z = x[e];
      if (kAct == HC_ACT_RELU) x[e] = z < 0.0f ? 0.0f : z;   // keeps NaN
      if (kAct == HC_ACT_SILU) x[e] = z * recip_f<kFast>(1.0f + exp_f<kFast>(-1.0f, z));
      if (kAct == HC_ACT_GELU_TANH) {
        const float q = kFast ? exp2_approx(z * fmaf(-1.4426950408889634f * kTanh3 * z, z, -1.4426950408889634f * kTanh1))
                              : expf(-z * fmaf(kTanh3 * z, z, kTanh1));
        x[e] = z * recip_f<kFast>(1.0f + q);
      }
      if (kAct == HC_ACT_GELU) {
        float g;
        x[e] = z * normal_cdf<kFast>(z, g);
      }
    }
  }
}

// x *= act'(pre).  sigma and 1 - sigma underflow together with the exponential's overflow, and inf * 0 must
// not arise: beyond |z| = 16 (SILU 80) the slope is 0 or 1 to float32, so z is bounded there first.
template <int kAct, bool kFast, int W>
__device__ __forceinline__ void act_scale_t(float (&x)[W], const float (&pre)[W]) {
  if constexpr (kAct == HC_ACT_GELU && kFast && W % 2 == 0) {
#pragma unroll
    for (int e = 0; e < W; e += 2) {
      // bounded as below; min and max drop a NaN, which is put back at the end
      const float2 z = make_float2(fminf(fmaxf(pre[e], -16.0f), 16.0f), fminf(fmaxf(pre[e + 1], -16.0f), 16.0f));
      float2 g;
      const float2 s = normal_cdf_pair(z, g);
      const float2 v = fma2(mul2(z, both(0.39894228040143268f)), g, s);
      x[e] = pre[e] != pre[e] ? pre[e] : x[e] * v.x;
      x[e + 1] = pre[e + 1] != pre[e + 1] ? pre[e + 1] : x[e + 1] * v.y;
    }
  } else {
    constexpr float kBound = kAct == HC_ACT_SILU ? 80.0f : 16.0f;
    constexpr float k1 = kAct == HC_ACT_SILU ? 1.0f : kTanh1, k3 = kAct == HC_ACT_SILU ? 0.0f : kTanh3;
#pragma unroll
    for (int e = 0; e < W; e++) {
      if (kAct == HC_ACT_RELU) x[e] = pre[e] <= 0.0f ? 0.0f : x[e];
      const float z = pre[e] != pre[e] ? pre[e] : fminf(fmaxf(pre[e], -kBound), kBound);
      if (kAct == HC_ACT_SILU || kAct == HC_ACT_GELU_TANH) {
        const float q = exp_f<kFast>(-1.0f, fabsf(z) * fmaf(k3 * z, z, k1));   // in (0, 1]: both sigmas from it
        const float d = recip_f<kFast>(1.0f + q);
        const float s = z < 0.0f ? q * d : d;
        x[e] *= fmaf(z * fmaf(3.0f * k3 * z, z, k1), q * d * d, s);
      }
      if (kAct == HC_ACT_GELU) {
        float g;
        const float s = normal_cdf<kFast>(z, g);
        x[e] *= fmaf(z * 0.39894228040143268f, g, s);
      }
    }
  }
}

// A launch's epilogue as one number, so that a loop over a tile can be chosen once: the activation, plus
// kGradCode in the gradient form.
constexpr int kGradCode = 8;
template <typename F>
__device__ __forceinline__ void with_code(int act, int grad, F&& f) {
  switch (act + (grad ? kGradCode : 0)) {
    case HC_ACT_RELU: f(std::integral_constant<int, HC_ACT_RELU>()); break;
    case HC_ACT_GELU: f(std::integral_constant<int, HC_ACT_GELU>()); break;
    case HC_ACT_GELU_TANH: f(std::integral_constant<int, HC_ACT_GELU_TANH>()); break;
    case HC_ACT_SILU: f(std::integral_constant<int, HC_ACT_SILU>()); break;
    case kGradCode + HC_ACT_NONE: f(std::integral_constant<int, kGradCode + HC_ACT_NONE>()); break;
    case kGradCode + HC_ACT_RELU: f(std::integral_constant<int, kGradCode + HC_ACT_RELU>()); break;
    case kGradCode + HC_ACT_GELU: f(std::integral_constant<int, kGradCode + HC_ACT_GELU>()); break;
    case kGradCode + HC_ACT_GELU_TANH: f(std::integral_constant<int, kGradCode + HC_ACT_GELU_TANH>()); break;
    case kGradCode + HC_ACT_SILU: f(std::integral_constant<int, kGradCode + HC_ACT_SILU>()); break;
    default: f(std::integral_constant<int, HC_ACT_NONE>()); break;
  }
}

template <typename T> __device__ __forceinline__ float widen_f(T v);
template <> __device__ __forceinline__ float widen_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow_f(float v);
template <> __device__ __forceinline__ float narrow_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow_f<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of T, widened and narrowed.
template <typename T> struct Pack16;
template <> struct Pack16<float> {
  static constexpr int W = 4;
  __device__ static void widen(const uint4& u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 narrow(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <> struct Pack16<__half> {
  static constexpr int W = 8;
  __device__ static void widen(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  __device__ static uint4 narrow(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *(const uint32_t*)&h;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The epilogue over W consecutive elements of a row, x the float32 product; `bias` and `aux` the W elements of those
// tensors, widened (zero where a tensor is absent or the element lies outside).  z is what `pre` keeps.
template <int kCode, bool kFast, int W>
__device__ __forceinline__ void fused_values(float (&x)[W], const float (&bias)[W], const float (&aux)[W], float (&z)[W]) {
  if constexpr (kCode >= kGradCode) {
    act_scale_t<kCode - kGradCode, kFast, W>(x, aux);
  } else {
#pragma unroll
    for (int e = 0; e < W; e++) z[e] = x[e] = x[e] + bias[e];
    act_apply_t<kCode, kFast, W>(x);
#pragma unroll
    for (int e = 0; e < W; e++) x[e] += aux[e];
  }
}

// The same over four consecutive columns in memory, element by element: for the CUDA-core kernel and for the kernel that sums
// the parts of a cut contraction, whose time goes elsewhere.  `off` is the element offset in every [M, N] tensor.
template <typename T, int W>
__device__ __forceinline__ void fused_direct(const FusedEpilogue& f, int64_t off, int64_t col, int n, float (&x)[W]) {
  constexpr bool kFast = sizeof(T) == 2;
  float a[W], b[W], z[W];
#pragma unroll
  for (int e = 0; e < W; e++) {
    a[e] = (f.aux && e < n) ? widen_f<T>(((const T*)f.aux)[off + e]) : 0.0f;
    b[e] = (f.bias && e < n) ? widen_f<T>(((const T*)f.bias)[col + e]) : 0.0f;
    z[e] = 0.0f;
  }
  with_code(f.act, f.grad, [&](auto code) { fused_values<decltype(code)::value, kFast, W>(x, b, a, z); });
  if (f.pre)
#pragma unroll
    for (int e = 0; e < W; e++)
      if (e < n) ((T*)f.pre)[off + e] = narrow_f<T>(z[e]);
}

}  // namespace hc
