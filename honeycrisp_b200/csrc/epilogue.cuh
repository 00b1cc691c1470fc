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
#include "common.cuh"

namespace hc {

// Every activation but ReLU is z * S(z) with S rising from 0 to 1:
//   SILU       S = sigma(z), sigma(t) = 1 / (1 + e^-t)
//   GELU_TANH  S = sigma(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which is (1 + tanh u) / 2 without its
//              cancellation in the lower tail, where float16 still has 11 bits to fill
//   GELU       S = Phi, the normal distribution function
// so SILU and GELU_TANH share their code, sigma(k1 z + k3 z^3), and the slope is S + z S'.
//
// Phi(-y) = e^(-y^2/2) Q(y) for y >= 0 and Phi(y) = 1 - Phi(-y), where Q falls slowly from 1/2 and is fitted
// by t R(t), t = 1/(1 + p y), R a polynomial, with least largest relative error over y <= 14 (Phi(-14) is
// 8e-45, below float32's normals): degree 7, p = 0.3, 1.5e-7, for float32 results; degree 5, p = 0.31, 4.7e-6, for float16
// ones, whose rounding is 4.9e-4.  In float32 the exponent's rounding dominates: 6e-7 of Phi at z = -3,
// 1.3e-6 at -6.  kFast also takes the hardware's exponential and reciprocal (a few 2^-23).
template <bool kFast>
__device__ __forceinline__ float exp_f(float t) { return kFast ? __expf(t) : expf(t); }
template <bool kFast>
__device__ __forceinline__ float recip_f(float d) { return kFast ? __fdividef(1.0f, d) : 1.0f / d; }

// Phi(z), and e^(-z^2/2) for the slope.
template <bool kFast>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float y = fabsf(z);
  const float t = recip_f<kFast>(fmaf(kFast ? 0.31f : 0.3f, y, 1.0f));
  float r;
  if (kFast) {
    r = -0.07392915338277817f;
    r = fmaf(r, t, 0.18045039474964142f);
    r = fmaf(r, t, 0.015744661912322044f);
    r = fmaf(r, t, 0.13342981040477753f);
    r = fmaf(r, t, 0.12044127285480499f);
    r = fmaf(r, t, 0.12386070191860199f);
  } else {
    r = 0.035674773156642914f;
    r = fmaf(r, t, -0.1572030782699585f);
    r = fmaf(r, t, 0.20635350048542023f);
    r = fmaf(r, t, -0.05368364229798317f);
    r = fmaf(r, t, 0.12856163084506989f);
    r = fmaf(r, t, 0.09991349279880524f);
    r = fmaf(r, t, 0.12075395882129669f);
    r = fmaf(r, t, 0.11962930113077164f);
  }
  e = exp_f<kFast>(-0.5f * y * y);
  const float tail = t * r * e;
  return z < 0.0f ? tail : 1.0f - tail;   // NaN: 1 - NaN
}

// The activation as the constants its code takes, so that one launch's choice costs a uniform branch:
// kind 0 none, 1 ReLU, 2 sigma(k1 z + k3 z^3), 3 Phi.
struct ActCode { int kind; float k1, k3; };
__device__ __forceinline__ ActCode act_code(int act) {
  ActCode c = {0, 1.0f, 0.0f};
  if (act == HC_ACT_RELU) c.kind = 1;
  if (act == HC_ACT_SILU) c.kind = 2;
  if (act == HC_ACT_GELU_TANH) { c.kind = 2; c.k1 = 1.5957691216057308f; c.k3 = 1.5957691216057308f * 0.044715f; }
  if (act == HC_ACT_GELU) c.kind = 3;
  return c;
}

template <bool kFast, int W>
__device__ __forceinline__ void act_apply(int act, float (&x)[W]) {
  const ActCode c = act_code(act);
  if (c.kind == 2) {
#pragma unroll
    for (int e = 0; e < W; e++) {
      const float z = x[e];
      const float t = c.k3 != 0.0f ? z * fmaf(c.k3 * z, z, c.k1) : z;   // (0 z^3 is NaN at infinity)
      x[e] = z * recip_f<kFast>(1.0f + exp_f<kFast>(-t));
    }
  } else if (c.kind == 3) {
#pragma unroll
    for (int e = 0; e < W; e++) {
      float g;
      const float s = normal_cdf<kFast>(x[e], g);
      x[e] *= s;
    }
  } else if (c.kind == 1) {
#pragma unroll
    for (int e = 0; e < W; e++) x[e] = x[e] < 0.0f ? 0.0f : x[e];   // keeps NaN
  }
}

// x *= act'(pre).  sigma and 1 - sigma underflow together with the exponential's overflow, and inf * 0 must
// not arise: beyond |z| = 16 (SILU 80) the slope is 0 or 1 to float32, so z is bounded there first.
template <bool kFast, int W>
__device__ __forceinline__ void act_scale(int act, float (&x)[W], const float (&pre)[W]) {
  const ActCode c = act_code(act);
  if (c.kind == 2) {
    const float bound = c.k3 != 0.0f ? 16.0f : 80.0f;
#pragma unroll
    for (int e = 0; e < W; e++) {
      const float z = pre[e] != pre[e] ? pre[e] : fminf(fmaxf(pre[e], -bound), bound);
      const float q = exp_f<kFast>(-fabsf(z) * fmaf(c.k3 * z, z, c.k1));   // in (0, 1]: both sigmas from it
      const float d = recip_f<kFast>(1.0f + q);
      const float s = z < 0.0f ? q * d : d;
      x[e] *= fmaf(z * fmaf(3.0f * c.k3 * z, z, c.k1), q * d * d, s);
    }
  } else if (c.kind == 3) {
#pragma unroll
    for (int e = 0; e < W; e++) {
      const float z = pre[e] != pre[e] ? pre[e] : fminf(fmaxf(pre[e], -16.0f), 16.0f);
      float g;
      const float s = normal_cdf<kFast>(z, g);
      x[e] *= fmaf(z * 0.39894228040143268f, g, s);
    }
  } else if (c.kind == 1) {
#pragma unroll
    for (int e = 0; e < W; e++) x[e] = pre[e] <= 0.0f ? 0.0f : x[e];
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

// The 16 bytes of elements [0, n) at p, the rest zero.
template <typename T>
__device__ __forceinline__ uint4 load16_partial(const T* p, int n) {
  float x[Pack16<T>::W];
#pragma unroll
  for (int e = 0; e < Pack16<T>::W; e++) x[e] = e < n ? widen_f<T>(p[e]) : 0.0f;
  return Pack16<T>::narrow(x);   // exact: the values came from T (a NaN's payload may change)
}

// One 16-byte chunk of a result row: x holds the float32 product of W columns, of which `n` exist
// (n <= 0: none; nothing is read or written).  `off` is the chunk's element offset in every [M, N]
// tensor, `col` its first column; `aux` its 16 bytes of the auxiliary tensor.
template <typename T, int W>
__device__ __forceinline__ void fused_chunk(const FusedEpilogue& f, int64_t off, int64_t col, int n, const uint4& aux,
                                            float (&x)[W]) {
  static_assert(W == Pack16<T>::W, "one 16-byte chunk");
  constexpr bool kFast = sizeof(T) == 2;
  if (f.grad) {
    float pre[W];
    Pack16<T>::widen(aux, pre);
    act_scale<kFast, W>(f.act, x, pre);
    return;
  }
  if (f.bias) {
    const T* b = (const T*)f.bias + col;
    float bv[W];
    if (n >= W && ((uintptr_t)b & 15) == 0) {
      Pack16<T>::widen(__ldg((const uint4*)b), bv);
    } else {
#pragma unroll
      for (int e = 0; e < W; e++) bv[e] = e < n ? widen_f<T>(b[e]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < W; e++) x[e] += bv[e];
  }
  if (f.pre) {
    T* dst = (T*)f.pre + off;
    if (n >= W && f.vec) {
      *(uint4*)dst = Pack16<T>::narrow(x);
    } else {
#pragma unroll
      for (int e = 0; e < W; e++)
        if (e < n) dst[e] = narrow_f<T>(x[e]);
    }
  }
  act_apply<kFast, W>(f.act, x);
  if (f.aux) {
    float r[W];
    Pack16<T>::widen(aux, r);
#pragma unroll
    for (int e = 0; e < W; e++) x[e] += r[e];
  }
}

// kChunks consecutive 16-byte chunks of one row of the auxiliary tensor, of which `n` elements exist.
template <typename T, int kChunks>
__device__ __forceinline__ void load_aux(const FusedEpilogue& f, int64_t off, int64_t n, uint4 (&u)[kChunks]) {
  constexpr int W = Pack16<T>::W;
  if (f.aux && n > 0) {
    const T* src = (const T*)f.aux + off;
    if (f.vec && n >= kChunks * W) {
#pragma unroll
      for (int q = 0; q < kChunks; q++) u[q] = *(const uint4*)(src + q * W);   // not __ldg: it may be the result's own buffer
    } else {
#pragma unroll
      for (int q = 0; q < kChunks; q++) {
        const int64_t left = n - q * W;
        u[q] = load16_partial<T>(src + q * W, left > W ? W : left < 0 ? 0 : (int)left);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < kChunks; q++) u[q] = make_uint4(0, 0, 0, 0);
  }
}

// The same over 32 consecutive columns of a row, for the paths that store from registers.
template <typename T>
__device__ __forceinline__ void fused_row32(const FusedEpilogue& f, int64_t off, int64_t col, int64_t n, float (&v)[32]) {
  constexpr int W = Pack16<T>::W;
  uint4 aux[32 / W];
  load_aux<T, 32 / W>(f, off, n, aux);
#pragma unroll
  for (int q = 0; q < 32 / W; q++) {
    float x[W];
#pragma unroll
    for (int e = 0; e < W; e++) x[e] = v[q * W + e];
    const int64_t left = n - q * W;
    fused_chunk<T, W>(f, off + q * W, col + q * W, left > W ? W : left < 0 ? 0 : (int)left, aux[q], x);
#pragma unroll
    for (int e = 0; e < W; e++) v[q * W + e] = x[e];
  }
}

// The same over four consecutive columns, element by element: for the kernel that sums the parts of a
// cut contraction, whose time goes into reading the parts.
template <typename T>
__device__ __forceinline__ void fused_four(const FusedEpilogue& f, int64_t off, int64_t col, int n, float (&x)[4]) {
  constexpr bool kFast = sizeof(T) == 2;
  float a[4];
#pragma unroll
  for (int e = 0; e < 4; e++) a[e] = (f.aux && e < n) ? widen_f<T>(((const T*)f.aux)[off + e]) : 0.0f;
  if (f.grad) {
    act_scale<kFast, 4>(f.act, x, a);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (f.bias && e < n) x[e] += widen_f<T>(((const T*)f.bias)[col + e]);
    if (f.pre && e < n) ((T*)f.pre)[off + e] = narrow_f<T>(x[e]);
  }
  act_apply<kFast, 4>(f.act, x);
  if (f.aux)
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += a[e];
}

}  // namespace hc
