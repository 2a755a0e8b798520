// The norms around a transformer block fused with its gate and residual:
//
//   u   = N(y) * w1 + b1            (the norm after the block; w1 absent: u = y)
//   h   = x + scale * gate * u      (gate absent: 1; one row of C for each group of rows)
//   out = N(h) * w2 + b2            (the norm before the next block)
//
// N(t) = (t - mean) * rsqrt(var + eps) (LayerNorm) or t * rsqrt(mean t^2 + eps)
// (RMS), and their gradients.  Everything between a load and a store is fp32;
// h and out are each rounded once, out from the unrounded h.
//
// Both kernels are bound by HBM: the forward reads x and y and writes h and
// out; the backward reads x, y, dh and dout, forms u and h again (the row is
// in registers; only the four row statistics come from the forward) and
// writes dx and dy.  A row belongs to one wave (up to 1,024 features, or 2,048
// in the forward) or to four, 8 features a lane and step.  The column sums of
// the parameters' gradients stay in the registers of a workgroup over all its
// rows, then are added over its waves in LDS and over workgroups by a second
// kernel, in a fixed order: two calls give the same bits.
//
// Measured at 16,384 x 4,096 bf16: forward 95 us (5.6 TB/s), backward 173 (4.7 TB/s)
// and 11 for the column sums; at 8 rows of 2,048 the forward takes 4.2, a launch.
#include "gpa_common.h"

#include <math.h>

#include <algorithm>

namespace gpa {
namespace {

struct NormArgs {
  const void *x, *y, *gate, *w1, *b1, *w2, *b2;
  void *h, *out;
  float* stats;                 // [rows][4]: mean and rstd of y, of h
  const void *dh, *dout;
  void *dx, *dy;
  float* part;                  // [workgroups][sums][C]
  int64_t rows, per;            // rows; rows of a gate's group
  int64_t x_sn, y_sn, h_sn, out_sn, dh_sn, dout_sn, dx_sn, dy_sn;
  int64_t chunk, cpg;           // rows of a workgroup; workgroups of a group (0: several groups each)
  void* dgate;                  // written by the workgroups where cpg is 0
  int32_t C, layer, pf32;       // pf32: parameters are fp32, not of the rows' type
  float scale, eps;
};

// Column sums of the backward, in the order of a workgroup's partials.
enum { kDGate = 0, kDW1 = 1, kDW2 = 2, kDB1 = 3, kDB2 = 4 };

// A descriptor over one row of n features (n = 0, or no tensor: empty).  Loads
// past it give zeros and stores past it are dropped, so neither the end of a row
// nor a row past the last one needs a branch.  The row is the same for a wave.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* base, int64_t at, int n) {
  return make_rsrc(static_cast<const T*>(base) + at, base ? (uint32_t)n * sizeof(T) : 0u);
}

// Features i .. i + 7 of a row as fp32; those past its end are zeros.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t r, int i, float (&f)[8]) {
  constexpr int E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E)));
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < 8 / E; ++k) {
      const vec v = __builtin_bit_cast(vec, buf_load16(r, (uint32_t)(i + k * E) * sizeof(T)));
#pragma unroll
      for (int e = 0; e < E; ++e) f[k * E + e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t at = (uint32_t)(i + e) * sizeof(T);
      if constexpr (sizeof(T) == 4)
        f[e] = __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
      else
        f[e] = (float)__builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(__amdgpu_buffer_rsrc_t r, int i, const float (&f)[8]) {
  constexpr int E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E)));
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < 8 / E; ++k) {
      vec v;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = (T)f[k * E + e];
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r,
                                             (uint32_t)(i + k * E) * sizeof(T), 0, 0);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t at = (uint32_t)(i + e) * sizeof(T);
      const T v = (T)f[e];
      if constexpr (sizeof(T) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, at, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), r, at, 0, 0);
    }
  }
}

// Eight values of a parameter's row at `at`; without the parameter, `none`.
template <typename T, bool VEC>
__device__ __forceinline__ void param8(const NormArgs& a, const void* p, int64_t at, int i, float none,
                                       float (&f)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = none;
  } else if (sizeof(T) == 4 || a.pf32) {
    load8<float, VEC>(row_rsrc<float>(p, at, a.C), i, f);
  } else {
    load8<T, VEC>(row_rsrc<T>(p, at, a.C), i, f);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// Sums over the lanes of a row: a wave, or several through LDS.  Two
// buffers in turn make one barrier enough: whoever writes a buffer again has
// passed the barrier of the other one, after everybody's reads of this.
template <int LANES, int ROWS>
struct RowSum {
  static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
  float (*buf)[ROWS][WAVES][2];  // [2] of them
  int turn = 0;
  __device__ __forceinline__ void sum2(float& a, float& b, int slot, int wave) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (LANES > 64) {
      if ((threadIdx.x & 63) == 0) {
        buf[turn][slot][wave][0] = a;
        buf[turn][slot][wave][1] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        a += buf[turn][slot][i][0];
        b += buf[turn][slot][i][1];
      }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ float sum(float a, int slot, int wave) {
    float none = 0.f;
    sum2(a, none, slot, wave);
    return a;
  }
};

template <typename T, int LANES, int NV, bool VEC>
__global__ __launch_bounds__(256) void norm_gate_kernel(NormArgs a) {
  constexpr int ROWS = 256 / LANES;
  using Sum = RowSum<LANES, ROWS>;
  __shared__ float buf[2][ROWS][Sum::WAVES][2];
  Sum red{buf};
  const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  const int lane = threadIdx.x % LANES, wave = lane / 64;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + slot;
  const bool live = row < a.rows;
  const int n = live ? a.C : 0;
  const float inv_c = 1.0f / a.C;

  float u[NV][8], h[NV][8];
  const __amdgpu_buffer_rsrc_t xr = row_rsrc<T>(a.x, row * a.x_sn, n), yr = row_rsrc<T>(a.y, row * a.y_sn, n);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load8<T, VEC>(yr, (v * LANES + lane) * 8, u[v]);
    load8<T, VEC>(xr, (v * LANES + lane) * 8, h[v]);
  }
  // Mean and reciprocal deviation of a row held in t.
  auto moments = [&](const float (&t)[NV][8], float& mean, float& rstd) {
    mean = 0.f;
    if (a.layer) {
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += t[v][e];
      mean = red.sum(s, slot, wave) * inv_c;
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = (v * LANES + lane) * 8 + e < a.C ? t[v][e] - mean : 0.f;
        ss = __builtin_fmaf(d, d, ss);
      }
    rstd = 1.0f / sqrtf(red.sum(ss, slot, wave) * inv_c + a.eps);
  };
  float my = 0.f, ry = 1.f, mh, rh;
  if (a.w1) {
    moments(u, my, ry);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float w[8], b[8];
      param8<T, VEC>(a, a.w1, 0, (v * LANES + lane) * 8, 1.f, w);
      param8<T, VEC>(a, a.b1, 0, (v * LANES + lane) * 8, 0.f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[v][e] = __builtin_fmaf((u[v][e] - my) * ry, w[e], b[e]);
    }
  }
  const int64_t gate_at = a.gate && live ? row / a.per * a.C : 0;
  const __amdgpu_buffer_rsrc_t hr = row_rsrc<T>(a.h, row * a.h_sn, n), or_ = row_rsrc<T>(a.out, row * a.out_sn, n);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float g[8];
    param8<T, VEC>(a, a.gate, gate_at, (v * LANES + lane) * 8, 1.f, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[v][e] = __builtin_fmaf(a.scale * g[e], u[v][e], h[v][e]);
    store8<T, VEC>(hr, (v * LANES + lane) * 8, h[v]);
  }
  moments(h, mh, rh);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float w[8], b[8];
    param8<T, VEC>(a, a.w2, 0, (v * LANES + lane) * 8, 1.f, w);
    param8<T, VEC>(a, a.b2, 0, (v * LANES + lane) * 8, 0.f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[v][e] = __builtin_fmaf((h[v][e] - mh) * rh, w[e], b[e]);
    store8<T, VEC>(or_, (v * LANES + lane) * 8, h[v]);
  }
  if (a.stats && live && lane == 0)
    *reinterpret_cast<f32x4*>(a.stats + 4 * row) = f32x4{my, ry, mh, rh};
}

// Threads of a backward workgroup: rows in hand share its partial sums.
template <int LANES> constexpr int kBwdThreads = LANES > 512 ? LANES : 512;

// Inside a group of rows the gate is constant, so the group's sums of dh * N(y) and
// of dh (dh: the whole gradient of h) give three of the five column sums:
//   dgate = scale (w1 A + b1 D),  dw1 = scale gate A,  db1 = scale gate D.
// WHOLE: a workgroup has whole groups, whose gate's gradient it finishes (few rows
// a group); else a part of one.
template <typename T, int LANES, bool VEC, bool WHOLE>
__global__ __launch_bounds__(kBwdThreads<LANES>, WHOLE ? 2 : 4) void norm_gate_bwd_kernel(NormArgs a) {
  constexpr int ROWS = kBwdThreads<LANES> / LANES;
  using Sum = RowSum<LANES, ROWS>;
  __shared__ float buf[2][ROWS][Sum::WAVES][2];
  __shared__ __attribute__((aligned(16))) float tot[ROWS > 1 ? ROWS - 1 : 1][LANES * 8];
  Sum red{buf};
  const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  const int lane = threadIdx.x % LANES, wave = lane / 64;
  const int i = lane * 8;                      // this lane's features
  const float inv_c = 1.0f / a.C;

  // A sum over the workgroup's rows in hand, in slot 0's registers.
  auto join = [&](float (&v)[8]) {
    if constexpr (ROWS > 1) {
      __syncthreads();
      if (slot > 0) {
        *reinterpret_cast<f32x4*>(&tot[slot - 1][i]) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(&tot[slot - 1][i + 4]) = f32x4{v[4], v[5], v[6], v[7]};
      }
      __syncthreads();
      if (slot == 0) {
#pragma unroll
        for (int s = 0; s < ROWS - 1; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += tot[s][i + e];
      }
    }
  };

  float A[8] = {}, D[8] = {}, dw2[8] = {}, db2[8] = {}, dw1[8] = {}, db1[8] = {}, w2[8];
  param8<T, VEC>(a, a.w2, 0, i, 1.f, w2);
  auto partial = [&](int k, float (&v)[8], bool used) {
    if (!used) return;
    join(v);
    if (slot == 0) store8<float, false>(row_rsrc<float>(a.part, ((int64_t)blockIdx.x * 5 + k) * a.C, a.C), i, v);
  };

  const int64_t g0 = WHOLE ? (int64_t)blockIdx.x * a.chunk / a.per : blockIdx.x / a.cpg;
  const int64_t g1 = WHOLE ? std::min(g0 + a.chunk / a.per, a.rows / a.per) : g0 + 1;
  const int64_t skip = WHOLE ? 0 : blockIdx.x % a.cpg * a.chunk;
  for (int64_t g = g0; g < g1; ++g) {
    float gw[8], gb[8];                        // scale * gate * w1, scale * gate * b1
    {
      float w1[8], b1[8], gt[8];
      param8<T, VEC>(a, a.w1, 0, i, 1.f, w1);
      param8<T, VEC>(a, a.b1, 0, i, 0.f, b1);
      param8<T, VEC>(a, a.gate, g * a.C, i, 1.f, gt);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        gw[e] = a.scale * gt[e] * w1[e];
        gb[e] = a.b1 ? a.scale * gt[e] * b1[e] : 0.f;
      }
    }
    const int64_t end = (g + 1) * a.per, first = g * a.per + skip;
    const int64_t last = WHOLE ? end : std::min(first + a.chunk, end);
    for (int64_t r0 = first; r0 < last; r0 += ROWS) {
      const int64_t row = r0 + slot;
      const int n = row < last ? a.C : 0;
      float u[8], h[8], d[8], o[8];            // normed y, normed h, dh, dout
      const f32x4 st = __builtin_bit_cast(
          f32x4, buf_load16(make_rsrc(a.stats + 4 * row, row < last ? 16u : 0u), 0));
      load8<T, VEC>(row_rsrc<T>(a.y, row * a.y_sn, n), i, u);
      load8<T, VEC>(row_rsrc<T>(a.x, row * a.x_sn, n), i, h);
      load8<T, VEC>(row_rsrc<T>(a.dout, row * a.dout_sn, n), i, o);
      load8<T, VEC>(row_rsrc<T>(a.dh, row * a.dh_sn, n), i, d);
      // A norm that is absent, or whose output has no gradient, is left out, and a mean that
      // RMS does not take is not multiplied by 0: where a value or a sum is not finite, 0
      // times it is NaN for the whole row.  Features past C: o, gate and weights are zeros
      // there (a weight or gate that is absent is 1), so no sum of the row has them.
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = (u[e] - st[0]) * st[1];
      if (a.dout) {
        float s1 = 0.f, s0 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[e] = (h[e] + __builtin_fmaf(gw[e], u[e], gb[e]) - st[2]) * st[3];
          dw2[e] = __builtin_fmaf(o[e], h[e], dw2[e]);
          db2[e] += o[e];
          o[e] *= w2[e];
          s1 = __builtin_fmaf(o[e], h[e], s1);
          s0 += o[e];
        }
        red.sum2(s1, s0, slot, wave);
        s1 *= inv_c;
        s0 = a.layer ? s0 * inv_c : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] += st[3] * (o[e] - s0 - h[e] * s1);
      }
      float t1 = 0.f, t0 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        A[e] = __builtin_fmaf(d[e], u[e], A[e]);
        D[e] += d[e];
        o[e] = gw[e] * d[e];
        t1 = __builtin_fmaf(o[e], u[e], t1);
        t0 += o[e];
      }
      store8<T, VEC>(row_rsrc<T>(a.dx, row * a.dx_sn, n), i, d);
      if (a.w1) {
        red.sum2(t1, t0, slot, wave);
        t1 *= inv_c;
        t0 = a.layer ? t0 * inv_c : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = st[1] * (o[e] - t0 - u[e] * t1);
      }
      store8<T, VEC>(row_rsrc<T>(a.dy, row * a.dy_sn, n), i, o);
    }
    float w1[8], b1[8], gt[8];
    param8<T, VEC>(a, a.w1, 0, i, 1.f, w1);
    param8<T, VEC>(a, a.b1, 0, i, 0.f, b1);
    param8<T, VEC>(a, a.gate, g * a.C, i, 1.f, gt);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dw1[e] = __builtin_fmaf(a.scale * gt[e], A[e], dw1[e]);
      db1[e] = __builtin_fmaf(a.scale * gt[e], D[e], db1[e]);
      A[e] = a.scale * (a.b1 ? __builtin_fmaf(w1[e], A[e], b1[e] * D[e]) : w1[e] * A[e]);   // dgate
      D[e] = 0.f;
    }
    if constexpr (WHOLE) {
      join(A);
      if (slot == 0 && a.dgate) {
        if (sizeof(T) == 4 || a.pf32) store8<float, VEC>(row_rsrc<float>(a.dgate, g * a.C, a.C), i, A);
        else store8<T, VEC>(row_rsrc<T>(a.dgate, g * a.C, a.C), i, A);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) A[e] = 0.f;
    }
  }
  partial(kDGate, A, !WHOLE && a.gate);
  partial(kDW1, dw1, a.w1);
  partial(kDB1, db1, a.b1);
  partial(kDW2, dw2, true);
  partial(kDB2, db2, a.b2);
}

// The partials of a column sum added up: 64 columns a workgroup, 16 waves over
// the workgroups' rows.  Group g's gate has the partials [g cpg, (g + 1) cpg).
struct ColArgs {
  const float* part;
  void* out[5];                 // null: not wanted
  int64_t wgs, cpg, groups;
  int32_t C;
};

template <typename P>
__global__ __launch_bounds__(1024) void norm_gate_cols_kernel(ColArgs a) {
  __shared__ float tot[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, k = blockIdx.y == 0 ? (int)blockIdx.z : 0;
  const int64_t g = blockIdx.y == 0 ? 0 : blockIdx.y - 1;
  // blockIdx.y 0: the five sums over all rows (the gate's only where it has one
  // row); y > 0: the gate of group y - 1.
  int64_t lo = 0, hi = a.wgs;
  if (blockIdx.y > 0) {
    if (blockIdx.z > 0) return;
    lo = g * a.cpg;
    hi = lo + a.cpg;
  } else if (k == kDGate) {
    return;
  }
  P* out = static_cast<P*>(a.out[k]);
  if (!out) return;
  float s = 0.f;
  if (c < a.C)
    for (int64_t i = lo + wave; i < hi; i += 16) s += a.part[(i * 5 + k) * a.C + c];
  tot[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < a.C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += tot[i][lane];
    out[g * a.C + c] = (P)s;
  }
}

// Rows of a backward workgroup, as ColArgs and NormArgs have them.  Two workgroups
// of 512 threads a CU hold its registers; more would only write more partials.
constexpr int64_t kBwdWgs = 512;
struct Split { int64_t chunk, cpg, wgs; };
Split split_rows(int64_t rows, int64_t per) {
  Split s;
  s.chunk = std::max<int64_t>((rows + kBwdWgs - 1) / kBwdWgs, 8);
  if (per >= s.chunk) {
    s.cpg = (per + s.chunk - 1) / s.chunk;
    s.wgs = rows / per * s.cpg;
  } else {
    s.chunk = s.chunk / per * per;
    s.cpg = 0;
    s.wgs = (rows + s.chunk - 1) / s.chunk;
  }
  return s;
}

template <typename T, int LANES, int NV, bool VEC>
void forward(const NormArgs& a, hipStream_t s) {
  // A dimension of a grid has less than 2^32 threads; workgroups past the rows do nothing.
  const int64_t wgs = (a.rows * LANES + 255) / 256, most = (int64_t)1 << 23;
  hipLaunchKernelGGL((norm_gate_kernel<T, LANES, NV, VEC>),
                     dim3((unsigned)std::min(wgs, most), (unsigned)((wgs + most - 1) / most)), dim3(256), 0, s, a);
}
template <typename T>
void launch_forward(const NormArgs& a, bool vec, hipStream_t s) {
  if (!vec) return forward<T, 256, 4, false>(a, s);
  // A wave a row up to 2,048 features (32 a lane), unless there are few rows:
  // those are spread over four waves each.
  if (a.rows >= 1024) {
    if (a.C <= 512) return forward<T, 64, 1, true>(a, s);
    if (a.C <= 1024) return forward<T, 64, 2, true>(a, s);
    if (a.C <= 2048) return forward<T, 64, 4, true>(a, s);
  }
  if (a.C <= 2048) return forward<T, 256, 1, true>(a, s);
  if (a.C <= 4096) return forward<T, 256, 2, true>(a, s);
  forward<T, 256, 4, true>(a, s);
}

template <typename T, int LANES, bool VEC>
void backward(const NormArgs& a, int64_t wgs, hipStream_t s) {
  const dim3 grid((unsigned)wgs), block(kBwdThreads<LANES>);
  if (a.cpg > 0) hipLaunchKernelGGL((norm_gate_bwd_kernel<T, LANES, VEC, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((norm_gate_bwd_kernel<T, LANES, VEC, true>), grid, block, 0, s, a);
}
template <typename T>
void launch_backward(const NormArgs& a, int64_t wgs, bool vec, hipStream_t s) {
  if (!vec) {
    if (a.C <= 512) return backward<T, 64, false>(a, wgs, s);
    return backward<T, 1024, false>(a, wgs, s);
  }
  if (a.C <= 512) return backward<T, 64, true>(a, wgs, s);
  if (a.C <= 1024) return backward<T, 128, true>(a, wgs, s);
  if (a.C <= 2048) return backward<T, 256, true>(a, wgs, s);
  if (a.C <= 4096) return backward<T, 512, true>(a, wgs, s);
  backward<T, 1024, true>(a, wgs, s);
}

constexpr int64_t kMaxC = 8192;

int check(const char* fn, int dtype, int pdtype, const gpa_norm_gate_args* a) {
  if (!a) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (dtype < GPA_DTYPE_F32 || dtype > GPA_DTYPE_F16 || (pdtype != dtype && pdtype != GPA_DTYPE_F32)) {
    gpa_set_error("%s: dtypes %d and %d (parameters have the rows' type or fp32)", fn, dtype, pdtype);
    return GPA_E_INVALID;
  }
  if (a->rows < 0 || a->C < 0 || a->groups < 1 || a->rows % a->groups != 0) {
    gpa_set_error("%s: negative size, or rows that do not divide into the gate's groups", fn);
    return GPA_E_INVALID;
  }
  if (a->C < 1 || a->C > kMaxC) {
    gpa_set_error("%s: C=%lld unsupported (1 to %lld)", fn, (long long)a->C, (long long)kMaxC);
    return GPA_E_UNSUPPORTED;
  }
  if (a->rows >= (int64_t)1 << 31) {
    gpa_set_error("%s: too many rows", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (!(a->eps >= 0.f) || !isfinite(a->eps) || !isfinite(a->scale)) {
    gpa_set_error("%s: eps must be finite and >= 0, scale finite", fn);
    return GPA_E_INVALID;
  }
  if (a->rows > 0 && (!a->x || !a->y || !a->w2 || (a->b1 && !a->w1))) {
    gpa_set_error("%s: null pointer (x, y, w2; w1 with b1)", fn);
    return GPA_E_INVALID;
  }
  return GPA_OK;
}

struct RowPtr { const void* p; int64_t sn; };

// Whether whole 16-byte groups of 8 features can be loaded and stored.
bool vectors(const gpa_norm_gate_args* a, int dtype, std::initializer_list<RowPtr> rows,
             std::initializer_list<const void*> params) {
  const int64_t per16 = dtype == GPA_DTYPE_F32 ? 4 : 8;
  bool ok = a->C % 8 == 0;
  for (const RowPtr& r : rows)
    ok = ok && (!r.p || ((uintptr_t)r.p % 16 == 0 && (a->rows <= 1 || r.sn % per16 == 0)));
  for (const void* p : params) ok = ok && (uintptr_t)p % 16 == 0;
  return ok;
}

NormArgs fill(const gpa_norm_gate_args* a, int pdtype) {
  NormArgs f{};
  f.x = a->x; f.y = a->y; f.gate = a->gate;
  f.w1 = a->w1; f.b1 = a->b1; f.w2 = a->w2; f.b2 = a->b2;
  f.rows = a->rows;
  f.per = a->rows / a->groups;
  f.x_sn = a->x_sn; f.y_sn = a->y_sn;
  f.stats = a->stats;
  f.C = (int32_t)a->C;
  f.layer = a->layer != 0;
  f.pf32 = pdtype == GPA_DTYPE_F32;
  f.scale = a->scale;
  f.eps = a->eps;
  return f;
}

}  // namespace
}  // namespace gpa

using namespace gpa;

extern "C" int gpa_norm_gate(int dtype, int param_dtype, const gpa_norm_gate_args* a, void* h,
                             int64_t h_sn, void* out, int64_t out_sn, void* stream) {
  const char* fn = "gpa_norm_gate";
  gpa_clear_error();
  const int rc = check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK || a->rows == 0) return rc;
  if (!h || !out || (a->stats && (uintptr_t)a->stats % 16)) {
    gpa_set_error("%s: null output, or stats that are not 16-byte aligned", fn);
    return GPA_E_INVALID;
  }
  NormArgs f = fill(a, param_dtype);
  f.h = h; f.h_sn = h_sn;
  f.out = out; f.out_sn = out_sn;
  const bool vec = vectors(a, dtype,
                           {{a->x, a->x_sn}, {a->y, a->y_sn}, {h, h_sn}, {out, out_sn}},
                           {a->gate, a->w1, a->b1, a->w2, a->b2});
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == GPA_DTYPE_F32) launch_forward<float>(f, vec, s);
  else if (dtype == GPA_DTYPE_BF16) launch_forward<__bf16>(f, vec, s);
  else launch_forward<_Float16>(f, vec, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}

extern "C" size_t gpa_norm_gate_bwd_workspace_bytes(int64_t rows, int64_t C, int64_t groups) {
  if (rows <= 0 || C <= 0 || groups <= 0 || rows % groups) return 0;
  return (size_t)split_rows(rows, rows / groups).wgs * 5 * C * sizeof(float);
}

extern "C" int gpa_norm_gate_bwd(int dtype, int param_dtype, const gpa_norm_gate_args* a,
                                 const gpa_norm_gate_grads* g, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_norm_gate_bwd";
  gpa_clear_error();
  const int rc = check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK) return rc;
  if (!g) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (a->rows == 0) {
    if (g->dgate || g->dw1 || g->db1 || g->dw2 || g->db2) {
      gpa_set_error("%s: no row, so the parameters' gradients are zeros that the caller writes", fn);
      return GPA_E_INVALID;
    }
    return GPA_OK;
  }
  if (!g->dx || !g->dy || !a->stats || (uintptr_t)a->stats % 16 || (g->dgate && !a->gate) ||
      (g->dw1 && !a->w1) || (g->db1 && !a->b1) || (g->db2 && !a->b2)) {
    gpa_set_error("%s: dx, dy and 16-byte aligned stats are needed, and no gradient of an absent "
                  "parameter", fn);
    return GPA_E_INVALID;
  }
  const Split sp = split_rows(a->rows, a->rows / a->groups);
  const size_t need = gpa_norm_gate_bwd_workspace_bytes(a->rows, a->C, a->groups);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, need);
    return GPA_E_WORKSPACE;
  }
  if (sp.wgs > 0x7fffffff || (sp.cpg > 0 && a->groups >= 65535)) {
    gpa_set_error("%s: too many groups", fn);
    return GPA_E_UNSUPPORTED;
  }
  NormArgs f = fill(a, param_dtype);
  f.dh = g->dh; f.dh_sn = g->dh_sn;
  f.dout = g->dout; f.dout_sn = g->dout_sn;
  f.dx = g->dx; f.dx_sn = g->dx_sn;
  f.dy = g->dy; f.dy_sn = g->dy_sn;
  f.part = (float*)workspace;
  f.chunk = sp.chunk; f.cpg = sp.cpg;
  f.dgate = sp.cpg == 0 ? g->dgate : nullptr;
  const bool vec = vectors(a, dtype,
                           {{a->x, a->x_sn}, {a->y, a->y_sn}, {g->dh, g->dh_sn}, {g->dout, g->dout_sn},
                            {g->dx, g->dx_sn}, {g->dy, g->dy_sn}},
                           {a->gate, a->w1, a->b1, a->w2, a->b2, g->dgate});
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == GPA_DTYPE_F32) launch_backward<float>(f, sp.wgs, vec, s);
  else if (dtype == GPA_DTYPE_BF16) launch_backward<__bf16>(f, sp.wgs, vec, s);
  else launch_backward<_Float16>(f, sp.wgs, vec, s);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    ColArgs c{};
    c.part = f.part;
    c.out[kDGate] = sp.cpg > 0 ? g->dgate : nullptr;
    c.out[kDW1] = g->dw1; c.out[kDW2] = g->dw2; c.out[kDB1] = g->db1; c.out[kDB2] = g->db2;
    c.wgs = sp.wgs; c.cpg = sp.cpg; c.groups = a->groups;
    c.C = (int32_t)a->C;
    const dim3 grid((unsigned)((a->C + 63) / 64), c.out[kDGate] ? (unsigned)(a->groups + 1) : 1u, 5), block(1024);
    if (param_dtype == GPA_DTYPE_F32) hipLaunchKernelGGL((norm_gate_cols_kernel<float>), grid, block, 0, s, c);
    else if (param_dtype == GPA_DTYPE_BF16) hipLaunchKernelGGL((norm_gate_cols_kernel<__bf16>), grid, block, 0, s, c);
    else hipLaunchKernelGGL((norm_gate_cols_kernel<_Float16>), grid, block, 0, s, c);
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
