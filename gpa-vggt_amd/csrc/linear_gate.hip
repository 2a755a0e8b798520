// A projection with what follows it: y = residual + gate act(x w^T + bias), 16-bit
// operands, fp32 from the products to the one rounding of y.  act: none, GELU (erf and
// tanh forms), SiLU, ReLU.  For gradients the sum before the activation is kept (z, fp32).
//
// Many rows: linear_gemm.h.  Up to 16 rows (a decode step) the weight's bytes bound it,
// and linear_rows_kernel streams them: 16 of its rows a workgroup, straight into the
// matrix instructions' registers, eight waves taking every eighth 32 features, so that
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

constexpr int kRowsMost = 16;

// Up to 16 rows.  WAVES waves take the steps of 32 k in turn.  Measured, us: 8 rows of 4,096 x 4,096
// 10.5 (3.2 TB/s, launch and all; 256 workgroups, one a CU), 16,384 x 4,096 33 (4.1 TB/s), and of
// 4,096 outputs over 16,384 features 43 with eight waves, 36 with sixteen.  More rows would
// read x once for each 16 outputs: 32 and 64 rows took 16 and 23 us here, 64 x 64 tiles take 12 to 15.
template <int WAVES, bool F16>
__global__ __launch_bounds__(WAVES * 64) void linear_rows_kernel(Matrix x, Matrix w, int K, Finish f) {
  constexpr int U = 4;                         // steps whose loads are in flight together
  __shared__ f32x4 sum[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4, l16 = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const bool mine = n0 + l16 < f.J, row = l16 < f.I;
  const uint16_t* W = w.p + (mine ? n0 + l16 : 0) * w.stride + 8 * quad;
  const uint16_t* X = x.p + (row ? l16 : 0) * x.stride + 8 * quad;
  f32x4 acc{};
  for (int k0 = wave * 32; k0 < K; k0 += U * WAVES * 32) {
    bf16x8 p[U], q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * WAVES * 32;
      const bool in = k + 8 * quad < K;
      p[u] = in && mine ? *reinterpret_cast<const bf16x8*>(W + k) : bf16x8{};
      q[u] = in && row ? *reinterpret_cast<const bf16x8*>(X + k) : bf16x8{};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc = mfma16x16x32_t<F16>(p[u], q[u], acc);
  }
  sum[wave][lane] = acc;
  __syncthreads();
  // Lane (quad, l16) has row l16, columns 4 quad .. +3: eight of a row to a thread.
  const int t = threadIdx.x;
  if (t >= 32) return;
  const int half = t >> 4, at = half * 32 + (t & 15);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const f32x4 lo = sum[i][at], hi = sum[i][at + 16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += lo[e];
      v[4 + e] += hi[e];
    }
  }
  finish8<F16>(f, t & 15, n0 + 8 * half, v);
}

template <bool F16>
hipError_t rows_launch(const Matrix& x, const Matrix& w, int64_t K, const Finish& f, hipStream_t s) {
  const dim3 grid((unsigned)((f.J + 15) / 16));
  if (K > 4096) hipLaunchKernelGGL((linear_rows_kernel<16, F16>), grid, dim3(1024), 0, s, x, w, (int)K, f);
  else hipLaunchKernelGGL((linear_rows_kernel<8, F16>), grid, dim3(512), 0, s, x, w, (int)K, f);
  return hipGetLastError();
}

// Rows of C values to rows of C8, the columns past C zeros: x's, then w's.
struct LayArgs { const uint16_t *x, *w; uint16_t *to_x, *to_w; int64_t x_rows, w_rows, x_s, w_s; int32_t C, C8; };
__global__ __launch_bounds__(256) void linear_lay_kernel(LayArgs a) {
  const int64_t wave = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (wave >= a.x_rows + a.w_rows) return;
  const bool x = wave < a.x_rows;
  const int64_t row = x ? wave : wave - a.x_rows;
  const uint16_t* from = x ? a.x + row * a.x_s : a.w + row * a.w_s;
  uint16_t* to = (x ? a.to_x : a.to_w) + row * a.C8;
#pragma unroll 8
  for (int c = threadIdx.x & 63; c < a.C8; c += 64) to[c] = c < a.C ? from[c] : (uint16_t)0;
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
  if (a->M >= most || a->N >= most || a->K >= lim - 8) {
    gpa_set_error("%s: %lld x %lld x %lld is too large (2^30 rows, 2^21 features)", fn, (long long)a->M, (long long)a->N, (long long)a->K);
    return GPA_E_UNSUPPORTED;
  }
  if (a->M == 0 || a->N == 0) return GPA_OK;
  if (a->K > 0 && (!a->x || !a->w)) {
    gpa_set_error("%s: null pointer", fn);
    return GPA_E_INVALID;
  }
  return GPA_OK;
}

Laid linear_laid(const gpa_linear_gate_args* a, bool x, bool w, bool turned) {
  Laid l{};
  l.K = std::max<int64_t>((a->K + 7) / 8 * 8, 8);
  // Rows of a tile are addressed by 32-bit offsets from its first one: strides below 2^21.  Turned
  // operands' rows lie apart (linear_gemm.h, Feed).
  const int64_t least = turned ? l.K : 0;
  auto copied = [&](const void* p, int64_t n, int64_t st) {
    return a->K != l.K || (uintptr_t)p % 16 || (n > 1 && (st % 8 || st < least || st >= (int64_t)1 << 21));
  };
  l.copy_x = x && copied(a->x, a->M, a->x_s);
  l.copy_w = w && copied(a->w, a->N, a->w_s);
  l.w_at = l.copy_x ? (size_t)a->M * l.K * 2 : 0;
  l.bytes = l.w_at + (l.copy_w ? (size_t)a->N * l.K * 2 : 0);
  return l;
}

hipError_t linear_lay(const gpa_linear_gate_args* a, const Laid& l, void* ws, Matrix& x, Matrix& w, hipStream_t s) {
  char* const at = (char*)ws;
  x = Matrix{(const uint16_t*)(l.copy_x ? at : a->x), l.copy_x || a->M < 2 ? l.K : a->x_s};
  w = Matrix{(const uint16_t*)(l.copy_w ? at + l.w_at : a->w), l.copy_w || a->N < 2 ? l.K : a->w_s};
  if (!l.copy_x && !l.copy_w) return hipSuccess;
  const LayArgs p{(const uint16_t*)a->x, (const uint16_t*)a->w, (uint16_t*)x.p, (uint16_t*)w.p, l.copy_x ? a->M : 0, l.copy_w ? a->N : 0,
                  a->M > 1 ? a->x_s : 0, a->N > 1 ? a->w_s : 0, (int32_t)a->K, (int32_t)l.K};
  const int64_t wgs = (p.x_rows + p.w_rows + 3) / 4, most = (int64_t)1 << 22;
  hipLaunchKernelGGL(linear_lay_kernel, dim3((unsigned)std::min(wgs, most), (unsigned)((wgs + most - 1) / most)), dim3(256), 0, s, p);
  return hipGetLastError();
}

bool linear_launchable(const GemmPlan& x, int64_t I, int64_t J) {
  const int64_t most = ((int64_t)1 << 32) / 256 - 8;   // a launch has less than 2^32 threads
  return x.ti <= most / x.tj / x.splits && (x.splits == 1 || (J + 7) / 8 <= most * 255 / I);
}

}  // namespace gpa

using namespace gpa;

extern "C" size_t gpa_linear_gate_workspace_bytes(const gpa_linear_gate_args* a) {
  if (!a || a->M <= 0 || a->N <= 0 || a->K < 0) return 0;
  const Laid l = linear_laid(a, true, true, false);
  return l.bytes + (a->M <= kRowsMost ? 0 : gemm_plan(a->M, a->N, l.K, false).bytes);
}

extern "C" int gpa_linear_gate(int dtype, int param_dtype, const gpa_linear_gate_args* a, void* y, int64_t y_s, void* z,
                               int z_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_linear_gate";
  gpa_clear_error();
  const int rc = linear_check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK || a->M == 0 || a->N == 0) return rc;
  if (!y || (z && ((uintptr_t)z % 16 || z_dtype != GPA_DTYPE_F32))) {
    gpa_set_error("%s: null output, or z that is not 16-byte aligned fp32", fn);
    return GPA_E_INVALID;
  }
  const int64_t psize = param_dtype == GPA_DTYPE_F32 ? 4 : 2;
  Finish f{};
  f.out = y; f.out_s = y_s;
  f.bias = a->bias; f.gate = a->gate; f.residual = a->residual; f.res_s = a->residual_s;
  f.z = (float*)z;
  f.I = a->M; f.J = a->N;
  f.act = a->act; f.pf32 = psize == 4;
  auto fine = [&](const void* p, int64_t s) { return !p || ((uintptr_t)p % 16 == 0 && (a->M < 2 || s % 8 == 0)); };
  f.wide = a->N % 8 == 0 && fine(y, y_s) && fine(a->residual, a->residual_s) && fine(a->bias, 0) && fine(a->gate, 0);
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype == GPA_DTYPE_F16;
  const bool few = a->M <= kRowsMost;
  const Laid l = linear_laid(a, true, true, false);
  const GemmPlan x = few ? GemmPlan{} : gemm_plan(a->M, a->N, l.K, false);
  // (A launch has less than 2^32 threads: of a few rows up to 1,024 for 16 columns.)
  if (few ? a->N > (int64_t)1 << 25 : !linear_launchable(x, a->M, a->N)) {
    gpa_set_error("%s: problem exceeds the grid limit", fn);
    return GPA_E_UNSUPPORTED;
  }
  const size_t need = l.bytes + x.bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, need);
    return GPA_E_WORKSPACE;
  }
  Matrix mx, mw;
  hipError_t e = linear_lay(a, l, workspace, mx, mw, s);
  if (e == hipSuccess && few) {
    e = f16 ? rows_launch<true>(mx, mw, l.K, f, s) : rows_launch<false>(mx, mw, l.K, f, s);
  } else if (e == hipSuccess) {
    GemmArgs g{};
    g.P = Operand{mw.p, mw.stride, a->N, l.K};
    g.Q = Operand{mx.p, mx.stride, a->M, l.K};
    g.nk = (int32_t)((l.K + 31) / 32);
    f.part = (float*)((char*)workspace + l.bytes);
    g.out = f;
    e = f16 ? gemm<false, false, true>(g, x, s) : gemm<false, false, false>(g, x, s);
  }
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
