// A projection with what follows it: y = residual + gate act(x w^T + bias), 16-bit
// operands, fp32 from the products to the one rounding of y.  act: none, GELU (erf and
// tanh forms), SiLU, ReLU.  For gradients the sum before the activation is kept (z), in fp32 or,
// where the gradients are coarser anyway, in fp16 (linear_gate.h, keep8).
//
// Many rows: linear_gemm.h.  Up to 64 rows (a decode step) the weight's bytes bound it,
// and linear_rows_kernel streams them: 16 of its rows a workgroup, straight into the
// matrix instructions' registers, the eight waves taking every eighth 32 features, so that
// they read 512 bytes of a row together; the waves' sums meet in LDS.  x comes out of the L2.
#include "linear_gemm.h"

namespace gpa {

// A product's time, roughly, in microseconds.  A CU has `held` workgroups at once; a stage of 32 k takes
// one of them `alone`, and all together not less than `each` for every one; `ends` is what comes
// before and after the stages.  As measured (8,192 x 4,096 x 4,096, us: 210, 252, 300, 500 by
// tile; 2,048 x 2,048 x 1,024: 45, 22, 15, 19).  Parts along k pay where few tiles have long sums;
// they cost a launch and their fp32 sums' bytes.
GemmPlan gemm_plan(int64_t I, int64_t J, int64_t K, bool turned) {
  struct Shape { int64_t i, j; int held; double alone, each, ends; };
  static const Shape shapes[4] = {{256, 256, 1, 0.86, 0.86, 15}, {128, 256, 2, 0.62, 0.49, 7}, {128, 128, 3, 0.38, 0.27, 6},
                                  {64, 64, 5, 0.2, 0.13, 2}};
  const int64_t nk = std::max<int64_t>((K + 31) / 32, 1);
  GemmPlan best{};
  double least = 0;
  for (int t = 0; t < 4; ++t) {
    // Two turned operands' addresses do not fit beside 4 x 8 blocks: 440 to 710 us for 205.
    if (t == 1 && turned) continue;
    const Shape& s = shapes[t];
    const int64_t ti = (I + s.i - 1) / s.i, tj = (J + s.j - 1) / s.j;
    for (int64_t z = 1; z <= 128 && (z == 1 || nk / z >= 8); z *= 2) {
      const double n = std::ceil((double)ti * tj * z / 256), rounds = std::floor(n / s.held), rest = n - rounds * s.held;
      const double stages = std::ceil((double)nk / z);
      double time = rounds * (stages * std::max(s.alone, s.held * s.each) + s.ends);
      if (rest > 0) time += stages * std::max(s.alone, rest * s.each) + s.ends;
      if (z > 1) time += 5 + (double)I * J * 4 * (2 * z + 1) / 4e6;
      if (best.ti == 0 || time < least) {
        least = time;
        best = GemmPlan{t, ti, tj, z, z > 1 ? (size_t)z * I * ((J + 7) / 8 * 8) * sizeof(float) : 0};
      }
    }
  }
  return best;
}

namespace {

constexpr int kRowsMost = 64;
constexpr int kRowWaves = 8;

template <int MB, bool F16>
__global__ __launch_bounds__(kRowWaves * 64) void linear_rows_kernel(const uint16_t* x, int64_t x_s, const uint16_t* w, int64_t w_s,
                                                                     int K, Finish f) {
  constexpr int U = MB == 1 ? 8 : 4;           // steps whose loads are in flight together
  __shared__ f32x4 sum[kRowWaves][MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4, l16 = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16, n = n0 + l16;
  const uint16_t* W = w + n * w_s + 8 * quad;
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = f32x4{};
  const int steps = (K + 31) / 32;
  for (int s0 = wave; s0 < steps; s0 += U * kRowWaves) {
    bf16x8 p[U], q[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s0 + u * kRowWaves) * 32;
      const bool in = k + 8 * quad < K;
      p[u] = in && n < f.J ? *reinterpret_cast<const bf16x8*>(W + k) : bf16x8{};
#pragma unroll
      for (int b = 0; b < MB; ++b)
        q[u][b] = in && 16 * b + l16 < f.I ? *reinterpret_cast<const bf16x8*>(x + (16 * b + l16) * x_s + k + 8 * quad) : bf16x8{};
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[b] = mfma16x16x32_t<F16>(p[u], q[u][b], acc[b]);
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) sum[wave][b][lane] = acc[b];
  __syncthreads();
  // Lane (quad, l16) of block b has row 16 b + l16, columns 4 quad .. +3: eight of a row to a thread.
  const int t = threadIdx.x;
  if (t >= MB * 32) return;
  const int b = t >> 5, half = t >> 4 & 1, at = half * 32 + (t & 15);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) {
    const f32x4 lo = sum[i][b][at], hi = sum[i][b][at + 16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += lo[e];
      v[4 + e] += hi[e];
    }
  }
  finish8<F16>(f, 16 * b + (t & 15), n0 + 8 * half, 0, 1, v);
}

template <bool F16>
hipError_t rows_launch(const gpa_linear_gate_args* a, const Finish& f, hipStream_t s) {
  const dim3 grid((unsigned)((a->N + 15) / 16)), block(kRowWaves * 64);
  const auto *x = (const uint16_t*)a->x, *w = (const uint16_t*)a->w;
  if (a->M <= 16) hipLaunchKernelGGL((linear_rows_kernel<1, F16>), grid, block, 0, s, x, a->x_s, w, a->w_s, (int)a->K, f);
  else if (a->M <= 32) hipLaunchKernelGGL((linear_rows_kernel<2, F16>), grid, block, 0, s, x, a->x_s, w, a->w_s, (int)a->K, f);
  else hipLaunchKernelGGL((linear_rows_kernel<4, F16>), grid, block, 0, s, x, a->x_s, w, a->w_s, (int)a->K, f);
  return hipGetLastError();
}

}  // namespace

int linear_check(const char* fn, int dtype, int pdtype, const gpa_linear_gate_args* a) {
  if (!a) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if ((dtype != GPA_DTYPE_BF16 && dtype != GPA_DTYPE_F16) || (pdtype != dtype && pdtype != GPA_DTYPE_F32)) {
    gpa_set_error("%s: dtypes %d and %d (bf16 or fp16; bias and gate of that or fp32)", fn, dtype, pdtype);
    return GPA_E_INVALID;
  }
  if (a->M < 0 || a->N < 0 || a->K < 0) {
    gpa_set_error("%s: negative size", fn);
    return GPA_E_INVALID;
  }
  if (a->act < kActNone || a->act > kActRelu) {
    gpa_set_error("%s: unknown activation %d", fn, a->act);
    return GPA_E_INVALID;
  }
  const int64_t lim = (int64_t)1 << 21, most = (int64_t)1 << 30;
  if (a->M >= most || a->N >= most || a->K >= lim) {
    gpa_set_error("%s: %lld x %lld x %lld is too large (2^30 rows, 2^21 features)", fn, (long long)a->M, (long long)a->N, (long long)a->K);
    return GPA_E_UNSUPPORTED;
  }
  if (a->M == 0 || a->N == 0) return GPA_OK;
  if (!a->x || !a->w) {
    gpa_set_error("%s: null pointer", fn);
    return GPA_E_INVALID;
  }
  auto fine = [&](const void* p, int64_t n, int64_t s) { return (uintptr_t)p % 16 == 0 && (n < 2 || s % 8 == 0); };
  if (a->K < 8 || a->K % 8 || !fine(a->x, a->M, a->x_s) || !fine(a->w, a->N, a->w_s)) {
    gpa_set_error("%s: K must be a positive multiple of 8, rows of x and w 16-byte aligned", fn);
    return GPA_E_INVALID;
  }
  // Rows of a tile are addressed by 32-bit offsets from its first one.
  if ((a->M > 1 && (a->x_s < 0 || a->x_s >= lim)) || (a->N > 1 && (a->w_s < 0 || a->w_s >= lim))) {
    gpa_set_error("%s: row strides from 0 to 2^21 are supported", fn);
    return GPA_E_UNSUPPORTED;
  }
  return GPA_OK;
}

bool linear_launchable(const GemmPlan& x, int64_t I, int64_t J) {
  const int64_t most = ((int64_t)1 << 32) / 256 - 8;   // a launch has less than 2^32 threads
  return x.ti <= most / x.tj / x.splits && (x.splits == 1 || (J + 7) / 8 <= most * 255 / I);
}

}  // namespace gpa

using namespace gpa;

extern "C" size_t gpa_linear_gate_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= kRowsMost || N <= 0 || K <= 0) return 0;
  return gemm_plan(M, N, K, false).bytes;
}

extern "C" int gpa_linear_gate(int dtype, int param_dtype, const gpa_linear_gate_args* a, void* y, int64_t y_s, void* z,
                               int z_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_linear_gate";
  gpa_clear_error();
  const int rc = linear_check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK || a->M == 0 || a->N == 0) return rc;
  if (!y || (z && ((uintptr_t)z % 16 || (z_dtype != GPA_DTYPE_F32 && z_dtype != GPA_DTYPE_F16)))) {
    gpa_set_error("%s: null output, or z that is not 16-byte aligned fp32 or fp16", fn);
    return GPA_E_INVALID;
  }
  const int64_t psize = param_dtype == GPA_DTYPE_F32 ? 4 : 2;
  Finish f{};
  f.out = y; f.out_s = y_s;
  f.bias = a->bias; f.gate = a->gate; f.residual = a->residual; f.res_s = a->residual_s;
  f.z = z; f.z16 = z_dtype == GPA_DTYPE_F16;
  f.I = a->M; f.J = a->N;
  f.act = a->act; f.pf32 = psize == 4;
  auto fine = [&](const void* p, int64_t s) { return !p || ((uintptr_t)p % 16 == 0 && (a->M < 2 || s % 8 == 0)); };
  f.wide = a->N % 8 == 0 && fine(y, y_s) && fine(a->residual, a->residual_s) && fine(a->bias, 0) && fine(a->gate, 0);
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype == GPA_DTYPE_F16;
  hipError_t e;
  if (a->M <= kRowsMost) {
    e = f16 ? rows_launch<true>(a, f, s) : rows_launch<false>(a, f, s);
  } else {
    const GemmPlan x = gemm_plan(a->M, a->N, a->K, false);
    if (!linear_launchable(x, a->M, a->N)) {
      gpa_set_error("%s: problem exceeds the grid limit", fn);
      return GPA_E_UNSUPPORTED;
    }
    if (x.bytes > 0 && (!workspace || workspace_bytes < x.bytes || (uintptr_t)workspace % 16)) {
      gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, x.bytes);
      return GPA_E_WORKSPACE;
    }
    GemmArgs g{};
    g.P = Operand{(const uint16_t*)a->w, a->N > 1 ? a->w_s : a->K, a->N, a->K};
    g.Q = Operand{(const uint16_t*)a->x, a->M > 1 ? a->x_s : a->K, a->M, a->K};
    g.nk = (int32_t)((a->K + 31) / 32);
    f.part = (float*)workspace;
    g.out = f;
    e = f16 ? gemm<false, false, true>(g, x, s) : gemm<false, false, false>(g, x, s);
  }
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
