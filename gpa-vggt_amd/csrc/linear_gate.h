// y = residual + gate act(x w^T + bias): what its kernels share.
#pragma once

#include <algorithm>
#include <math.h>

#include "gpa_common.h"

namespace gpa {

enum Act { kActNone = 0, kActGelu = 1, kActGeluTanh = 2, kActSilu = 3, kActRelu = 4 };

// How a product of I x J over K is cut: tiles (0: 256 x 256, 1: 128 x 256, 2: 128 x 128, 3: 64 x 64
// of i and j), parts along k, and the fp32 partials' bytes.
struct GemmPlan { int tile; int64_t ti, tj, splits; size_t bytes; };
GemmPlan gemm_plan(int64_t I, int64_t J, int64_t K, bool turned);

// x and w as the products take them: K a multiple of 8 and rows that are 16-byte aligned, so or as
// padded copies in the workspace (`bytes` of it, x's first).  `turned`: as the gradients' products take them.
struct Laid {
  int64_t K;
  bool copy_x, copy_w;
  size_t w_at, bytes;
};
Laid linear_laid(const gpa_linear_gate_args* a, bool x, bool w, bool turned);
struct Matrix { const uint16_t* p; int64_t stride; };
hipError_t linear_lay(const gpa_linear_gate_args* a, const Laid& l, void* ws, Matrix& x, Matrix& w, hipStream_t s);
int linear_check(const char* fn, int dtype, int pdtype, const gpa_linear_gate_args* a);
bool linear_launchable(const GemmPlan& x, int64_t I, int64_t J);

// What becomes of a sum.
struct Finish {
  void* out;              // 16-bit, rows out_s apart
  const void *bias, *gate;
  const void* residual;
  float* z;               // the sums before the activation, rows of J (nullable)
  const float* unscale;   // a factor for each row (nullable)
  float* part;            // parts along k: [part][I][J rounded up to 8]
  int64_t out_s, res_s, I, J;
  int32_t act, pf32;      // pf32: bias and gate are fp32
  int32_t wide;           // whole 16-byte groups of 8 can be loaded and stored
};

namespace {

// Cumulative normal distribution, off by 8e-8 absolutely: Abramowitz and Stegun 7.1.26 for
// erfc(|z| / sqrt 2) / 2.  A third of the instructions of the library's erf, which a
// product of 10,992 x 4,096 x 1,024 spent as long in as in its matrix instructions.
__device__ __forceinline__ float normal_cdf(float z, float& density) {
  const float a = fabsf(z);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.3275911f * 0.70710678f, 1.0f));
  density = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504f));   // e^(-z^2 / 2)
  float p = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  p = __builtin_fmaf(t, p, 0.5f * 1.421413741f);
  p = __builtin_fmaf(t, p, 0.5f * -0.284496736f);
  p = __builtin_fmaf(t, p, 0.5f * 0.254829592f);
  const float q = p * t * density;
  return z > 0.f ? 1.0f - q : q;
}
__device__ __forceinline__ float logistic(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
constexpr float kTanhC = 0.7978845608f, kTanhD = 0.044715f;   // gelu's tanh form: z logistic(2 c (z + d z^3))

// act(z).  (z is kept finite from below for the product: -inf times the 0 of its distribution
// is 0, as the limit is.  A NaN comes out by the other factor.)
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kActNone) return z;
  if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;     // NaN stays
  float s, d;
  if constexpr (ACT == kActGelu) {
    s = normal_cdf(z, d);
  } else {
    constexpr float l2e = 1.44269504f;
    float t = -l2e * z;
    if constexpr (ACT == kActGeluTanh) t = z * __builtin_fmaf(z * z, -2.0f * l2e * kTanhC * kTanhD, -2.0f * l2e * kTanhC);
    s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
  }
  return fmaxf(z, -3.0e38f) * s;
}
// act(z) and its derivative.
template <int ACT>
__device__ __forceinline__ float act_both(float z, float& slope) {
  if constexpr (ACT == kActNone) {
    slope = 1.f;
    return z;
  }
  if constexpr (ACT == kActRelu) {
    slope = z > 0.f ? 1.f : 0.f;
    return z < 0.f ? 0.f : z;
  }
  if constexpr (ACT == kActGelu) {
    float d;
    const float s = normal_cdf(z, d);
    slope = d == 0.f ? s : __builtin_fmaf(0.3989422804f * z, d, s);
    return s == 0.f ? 0.f : z * s;
  }
  float s, dt;
  if constexpr (ACT == kActSilu) {
    s = logistic(z);
    dt = z;
  } else {
    s = logistic(2.0f * kTanhC * z * __builtin_fmaf(kTanhD * z, z, 1.0f));
    dt = 2.0f * kTanhC * z * __builtin_fmaf(3.0f * kTanhD * z, z, 1.0f);
  }
  const float both = s * (1.0f - s);
  slope = both == 0.f ? s : __builtin_fmaf(dt, both, s);
  return s == 0.f ? 0.f : z * s;
}

// Eight values at `at` of a parameter (fp32 or of the operands' format), n of them there.
template <bool F16>
__device__ __forceinline__ void param8(const void* p, int pf32, int wide, int64_t at, int n, float (&x)[8]) {
  if (wide && pf32) {
    const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 lo = q[0], hi = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = lo[e];
      x[4 + e] = hi[e];
    }
  } else if (wide) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = half_to_f32<F16>(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = e >= n ? 0.f : pf32 ? static_cast<const float*>(p)[at + e]
                                 : half_to_f32<F16>(static_cast<const __bf16*>(p)[at + e]);
  }
}

// n sums (8: whole groups) kept at `at` of z for the backward, in fp32: a slope takes the relative error of
// z times z act'' / act', which is 5 and more where an activation runs out (as fp16, half the bytes, sums of -10
// cost a SiLU's gradients up to 0.4 %, as much as rounding dz to bf16, and alike in all rows of a column).
__device__ __forceinline__ void keep8(const Finish& f, int64_t at, int n, const float (&v)[8]) {
  float* z = f.z + at;
  if (n == 8 && f.wide) {
    reinterpret_cast<f32x4*>(z)[0] = f32x4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4*>(z)[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) z[e] = v[e];
  }
}

template <int ACT>
__device__ __forceinline__ void act8(float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = act_of<ACT>(v[e]);
}

// act's eight values, chosen at run time.
__device__ __forceinline__ void act8_of(int act, float (&v)[8]) {
  switch (act) {
    case kActGelu: act8<kActGelu>(v); break;
    case kActGeluTanh: act8<kActGeluTanh>(v); break;
    case kActSilu: act8<kActSilu>(v); break;
    case kActRelu: act8<kActRelu>(v); break;
    default: break;
  }
}

// The sums v of row i, columns j .. j + 7 of a part.
__device__ __forceinline__ void part8(const Finish& f, int64_t i, int64_t j, int split, const float (&v)[8]) {
  if (i >= f.I || j >= f.J) return;
  f32x4* to = reinterpret_cast<f32x4*>(f.part + ((int64_t)split * f.I + i) * ((f.J + 7) / 8 * 8) + j);
  to[0] = f32x4{v[0], v[1], v[2], v[3]};
  to[1] = f32x4{v[4], v[5], v[6], v[7]};
}

// The sums v of column j, rows i, i + STEP, ...
template <bool F16, int STEP>
__device__ __forceinline__ void finish_down(const Finish& f, int64_t i, int64_t j, float (&v)[8]) {
  if (j >= f.J) return;
  auto param = [&](const void* p) {
    return f.pf32 ? static_cast<const float*>(p)[j] : half_to_f32<F16>(static_cast<const __bf16*>(p)[j]);
  };
  const float bias = f.bias ? param(f.bias) : 0.f, gate = f.gate ? param(f.gate) : 1.f;
  const int n = f.I <= i ? 0 : (f.I - i + STEP - 1) / STEP < 8 ? (int)((f.I - i + STEP - 1) / STEP) : 8;
  __bf16 res[8];
  if (f.residual)
#pragma unroll
    for (int e = 0; e < 8; ++e) res[e] = e < n ? static_cast<const __bf16*>(f.residual)[(i + e * STEP) * f.res_s + j] : (__bf16)0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (f.unscale && e < n) v[e] *= f.unscale[i + e * STEP];
    if (f.bias) v[e] += bias;
  }
  if (f.z)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) f.z[(i + e * STEP) * f.J + j] = v[e];
  act8_of(f.act, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (f.gate) v[e] *= gate;
    if (f.residual) v[e] += half_to_f32<F16>(res[e]);
    if (e < n) static_cast<__bf16*>(f.out)[(i + e * STEP) * f.out_s + j] = f32_to_half<F16>(v[e]);
  }
}

// The sums v of row i, columns j .. j + 7.
template <bool F16>
__device__ __forceinline__ void finish8(const Finish& f, int64_t i, int64_t j, float (&v)[8]) {
  if (i >= f.I || j >= f.J) return;
  const int n = f.J - j < 8 ? (int)(f.J - j) : 8;
  float x[8];
  if (f.unscale) {
    const float s = f.unscale[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
  }
  if (f.bias) {
    param8<F16>(f.bias, f.pf32, f.wide, j, n, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
  }
  if (f.z) keep8(f, i * f.J + j, n, v);
  act8_of(f.act, v);
  if (f.gate) {
    param8<F16>(f.gate, f.pf32, f.wide, j, n, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= x[e];
  }
  if (f.residual) {
    param8<F16>(static_cast<const uint16_t*>(f.residual) + i * f.res_s, 0, f.wide, j, n, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
  }
  uint16_t* out = static_cast<uint16_t*>(f.out) + i * f.out_s + j;
  bf16x8 y;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const bf16x2 w = pack2<F16>(v[e], v[e + 1]);
    y[e] = w[0];
    y[e + 1] = w[1];
  }
  if (f.wide) {
    *reinterpret_cast<bf16x8*>(out) = y;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) reinterpret_cast<__bf16*>(out)[e] = y[e];
  }
}

}  // namespace
}  // namespace gpa
