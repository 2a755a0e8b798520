// The gradients of y = residual + gate act(z), z = x w^T + bias:
//
//   dz = dy gate act'(z)     dx = dz w     dw = dz^T x     dbias = sum dz     dgate = sum dy act(z)
//
// (the residual's is dy itself).  One pass over dy and z makes dz, rounded once to the
// operands' format for the two products, and the column sums from the unrounded values, in fixed
// parts.  Without activation and gate dz is dy as it lies.  Both products take w and x as they
// lie in memory, turned on their way out of LDS (linear_gemm.h): no transposed copy.
//
// fp16: a gate may be as small as it likes (1e-5 is usual where it begins), and dz would
// leave the format's range with it; the gate goes into dz times a power of two that makes its
// largest value one to two, and the products are multiplied by its inverse.
#include "linear_gemm.h"

namespace gpa {
namespace {

struct DzArgs {
  const void* dy;
  const void* z;
  const void* gate;
  const float* scale;     // fp16 with a gate: (scale, 1 / scale)
  void* dz;               // rows of J8, the columns past J zeros; null: sums alone
  float* part;            // [chunk][2][J]; null: no sums
  int64_t dy_s, I, J, J8, chunk;
  int32_t pf32, wide, z16;
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) v = fmaxf(v, __shfl_xor(v, i));
  return v;
}

__global__ __launch_bounds__(1024) void linear_scale_kernel(const void* gate, int pf32, int64_t J, float* scale) {
  __shared__ float top[16];
  float m = 0.f;
  for (int64_t j = threadIdx.x; j < J; j += 1024) {
    const float x = fabsf(pf32 ? static_cast<const float*>(gate)[j] : (float)static_cast<const _Float16*>(gate)[j]);
    m = x < INFINITY ? fmaxf(m, x) : m;
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x > 0) return;
  for (int i = 1; i < 16; ++i) m = fmaxf(m, top[i]);
  int e = 0;
  if (m > 0.f) frexpf(m, &e);                  // m = [0.5, 1) 2^e
  e = min(max(e - 1, -100), 100);
  scale[0] = ldexpf(1.0f, -e);
  scale[1] = ldexpf(1.0f, e);
}

// 512 columns (eight a lane) of `chunk` rows a workgroup, a wave every fourth row.
template <int ACT, bool F16>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs a) {
  __shared__ __attribute__((aligned(16))) float red[4][2][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 512 + lane * 8, i0 = blockIdx.y * a.chunk;
  const int64_t i1 = i0 + a.chunk < a.I ? i0 + a.chunk : a.I;
  const int n = a.J - j >= 8 ? 8 : a.J > j ? (int)(a.J - j) : 0;
  float g[8], db[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    g[e] = 1.f;
    db[e] = dg[e] = 0.f;
  }
  const bool wide = a.wide && n == 8;
  if (a.gate) param8<F16>(a.gate, a.pf32, wide, j, n, g);
  const float scale = a.scale ? *a.scale : 1.f;
  if (n > 0)
    for (int64_t i = i0 + wave; i < i1; i += 4) {
      float dy[8], z[8], out[8];
      param8<F16>(static_cast<const uint16_t*>(a.dy) + i * a.dy_s, 0, wide, j, n, dy);
      if (a.z) {
        if (a.z16) param8<true>(static_cast<const uint16_t*>(a.z) + i * a.J, 0, wide, j, n, z);
        else param8<true>(static_cast<const float*>(a.z) + i * a.J, 1, wide, j, n, z);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float slope = 1.f;
        if (ACT != kActNone || a.z) {
          const float v = act_both<ACT>(z[e], slope);
          dg[e] = __builtin_fmaf(dy[e], v, dg[e]);
        }
        const float d = ACT != kActNone ? dy[e] * slope : dy[e];
        db[e] = a.gate ? __builtin_fmaf(d, g[e], db[e]) : db[e] + d;
        out[e] = a.gate ? d * (g[e] * scale) : d;
      }
      if (!a.dz) continue;
      bf16x8 y;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const bf16x2 w = pack2<F16>(out[e], out[e + 1]);
        y[e] = e < n ? w[0] : (__bf16)0.f;
        y[e + 1] = e + 1 < n ? w[1] : (__bf16)0.f;
      }
      *reinterpret_cast<bf16x8*>(static_cast<uint16_t*>(a.dz) + i * a.J8 + j) = y;
    }
  if (!a.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    red[wave][0][lane * 8 + e] = db[e];
    red[wave][1][lane * 8 + e] = dg[e];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 1024; c += 256) {
    const int k = c >> 9, at = c & 511;
    const int64_t col = (int64_t)blockIdx.x * 512 + at;
    if (col < a.J) a.part[((int64_t)blockIdx.y * 2 + k) * a.J + col] = red[0][k][at] + red[1][k][at] + red[2][k][at] + red[3][k][at];
  }
}

// The chunks' sums added up: 64 columns a workgroup, 16 waves over the chunks.
template <typename P>
__global__ __launch_bounds__(1024) void linear_cols_kernel(const float* part, int64_t J, int chunks, P* db, P* dg) {
  __shared__ float tot[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  P* out = blockIdx.y ? dg : db;
  if (!out) return;
  float s = 0.f;
  if (c < J)
#pragma unroll 4
    for (int i = wave; i < chunks; i += 16) s += part[((int64_t)i * 2 + blockIdx.y) * J + c];
  tot[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < J) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += tot[i][lane];
    out[c] = (P)s;
  }
}

// Rows of a workgroup of the pass over dy: 1,024 workgroups in all, 16 rows at least.
int64_t dz_chunk(int64_t I, int64_t J) {
  const int64_t cols = (J + 511) / 512, rows = std::max<int64_t>(1, 1024 / cols);
  return std::max<int64_t>(16, (I + rows - 1) / rows);
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct BwdPlan {
  GemmPlan x, w;
  int64_t chunk, chunks, J8;
  size_t dz, part, scale, split, bytes;        // where each begins
};
BwdPlan bwd_plan(int64_t M, int64_t N, int64_t K, bool dz, bool sums, bool dx, bool dw) {
  BwdPlan p{};
  p.J8 = (N + 7) / 8 * 8;
  p.chunk = dz_chunk(M, N);
  p.chunks = (M + p.chunk - 1) / p.chunk;
  if (dx) p.x = gemm_plan(M, K, N, true);
  if (dw) p.w = gemm_plan(N, K, M, true);
  p.scale = dz ? (size_t)round16(M * p.J8 * 2) : 0;
  p.part = p.scale + 16;
  p.split = p.part + (sums ? (size_t)round16(p.chunks * 2 * N * 4) : 0);
  p.bytes = p.split + std::max(p.x.bytes, p.w.bytes);
  return p;
}

}  // namespace

int linear_check(const char* fn, int dtype, int pdtype, const gpa_linear_gate_args* a);
bool linear_launchable(const GemmPlan& x, int64_t I, int64_t J);

namespace {

template <bool F16>
hipError_t dz_launch(const DzArgs& d, int act, dim3 grid, hipStream_t s) {
  const dim3 block(256);
  switch (act) {
    case kActGelu: hipLaunchKernelGGL((linear_dz_kernel<kActGelu, F16>), grid, block, 0, s, d); break;
    case kActGeluTanh: hipLaunchKernelGGL((linear_dz_kernel<kActGeluTanh, F16>), grid, block, 0, s, d); break;
    case kActSilu: hipLaunchKernelGGL((linear_dz_kernel<kActSilu, F16>), grid, block, 0, s, d); break;
    case kActRelu: hipLaunchKernelGGL((linear_dz_kernel<kActRelu, F16>), grid, block, 0, s, d); break;
    default: hipLaunchKernelGGL((linear_dz_kernel<kActNone, F16>), grid, block, 0, s, d); break;
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace gpa

using namespace gpa;

// Whether dy itself is not dz as the products take it.
static bool needs_dz(const gpa_linear_gate_args* a, const gpa_linear_gate_grads* g) {
  const bool aligned = a->N % 8 == 0 && (uintptr_t)g->dy % 16 == 0 && (a->M < 2 || (g->dy_s % 8 == 0 && g->dy_s >= 0 && g->dy_s < 1 << 21));
  return (g->dx || g->dw) && (a->act != kActNone || a->gate || !aligned);
}

extern "C" size_t gpa_linear_gate_bwd_workspace_bytes(const gpa_linear_gate_args* a, const gpa_linear_gate_grads* g) {
  if (!a || !g || a->M <= 0 || a->N <= 0 || a->K <= 0) return 0;
  return bwd_plan(a->M, a->N, g->K_out, needs_dz(a, g), g->dbias || g->dgate, g->dx, g->dw).bytes;
}

extern "C" int gpa_linear_gate_bwd(int dtype, int param_dtype, const gpa_linear_gate_args* a, const gpa_linear_gate_grads* g,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_linear_gate_bwd";
  gpa_clear_error();
  const int rc = linear_check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK) return rc;
  if (!g) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (!g->dx && !g->dw && !g->dbias && !g->dgate) return GPA_OK;
  if (a->M == 0 || a->N == 0) {
    gpa_set_error("%s: nothing to sum, so the gradients are zeros that the caller writes", fn);
    return GPA_E_INVALID;
  }
  if (!g->dy || (g->dgate && !a->gate) || (g->z && ((uintptr_t)g->z % 16 || (g->z_dtype != GPA_DTYPE_F32 && g->z_dtype != GPA_DTYPE_F16))) ||
      (!g->z && (a->act != kActNone || g->dgate))) {
    gpa_set_error("%s: dy is needed, z with an activation or the gate's gradient, and there is none of an absent gate", fn);
    return GPA_E_INVALID;
  }
  if (g->K_out < 1 || g->K_out > a->K || a->K - g->K_out >= 8) {
    gpa_set_error("%s: %lld columns of gradients for K = %lld", fn, (long long)g->K_out, (long long)a->K);
    return GPA_E_INVALID;
  }
  if (a->N >= (int64_t)1 << 21) {
    gpa_set_error("%s: %lld output features (below 2^21)", fn, (long long)a->N);
    return GPA_E_UNSUPPORTED;
  }
  const bool f16 = dtype == GPA_DTYPE_F16, need_dz = needs_dz(a, g), sums = g->dbias || g->dgate;
  const BwdPlan p = bwd_plan(a->M, a->N, g->K_out, need_dz, sums, g->dx, g->dw);
  if ((g->dx && !linear_launchable(p.x, a->M, g->K_out)) || (g->dw && !linear_launchable(p.w, a->N, g->K_out))) {
    gpa_set_error("%s: problem exceeds the grid limit", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, p.bytes);
    return GPA_E_WORKSPACE;
  }
  char* ws = (char*)workspace;
  const hipStream_t s = (hipStream_t)stream;
  float* const scale = need_dz && f16 && a->gate ? (float*)(ws + p.scale) : nullptr;
  hipError_t e = hipSuccess;
  if (scale) {
    hipLaunchKernelGGL(linear_scale_kernel, dim3(1), dim3(1024), 0, s, a->gate, (int)(param_dtype == GPA_DTYPE_F32), a->N, scale);
    e = hipGetLastError();
  }
  if (e == hipSuccess && (need_dz || sums)) {
    DzArgs d{};
    d.dy = g->dy; d.dy_s = a->M > 1 ? g->dy_s : 0;
    d.z = g->z; d.z16 = g->z_dtype == GPA_DTYPE_F16; d.gate = a->gate; d.scale = scale;
    d.dz = need_dz ? ws : nullptr;
    d.part = sums ? (float*)(ws + p.part) : nullptr;
    d.I = a->M; d.J = a->N; d.J8 = p.J8; d.chunk = p.chunk;
    d.pf32 = param_dtype == GPA_DTYPE_F32;
    d.wide = a->N % 8 == 0 && (uintptr_t)g->dy % 16 == 0 && d.dy_s % 8 == 0 && (uintptr_t)a->gate % 16 == 0;
    const dim3 grid((unsigned)((a->N + 511) / 512), (unsigned)p.chunks);
    e = f16 ? dz_launch<true>(d, a->act, grid, s) : dz_launch<false>(d, a->act, grid, s);
    if (e == hipSuccess && sums) {
      const dim3 cols((unsigned)((a->N + 63) / 64), 2);
      auto go = [&](auto type) {
        typedef decltype(type) P;
        hipLaunchKernelGGL((linear_cols_kernel<P>), cols, dim3(1024), 0, s, d.part, a->N, (int)p.chunks, (P*)g->dbias, (P*)g->dgate);
      };
      if (param_dtype == GPA_DTYPE_F32) go(0.f);
      else if (f16) go((_Float16)0.f);
      else go((__bf16)0.f);
      e = hipGetLastError();
    }
  }
  const Operand dz_rows{need_dz ? (const uint16_t*)ws : (const uint16_t*)g->dy, need_dz ? p.J8 : a->M > 1 ? g->dy_s : p.J8, a->M, p.J8};
  auto fine = [](const void* q, int64_t n, int64_t st) { return (uintptr_t)q % 16 == 0 && (n < 2 || st % 8 == 0); };
  GemmArgs m{};
  m.out.unscale = scale ? scale + 1 : nullptr;
  m.out.part = (float*)(ws + p.split);
  m.out.J = g->K_out;
  if (e == hipSuccess && g->dx) {              // over the output features: w turned
    m.P = Operand{(const uint16_t*)a->w, a->N > 1 ? a->w_s : a->K, a->N, a->K};
    m.Q = dz_rows;
    m.nk = (int32_t)((p.J8 + 31) / 32);
    m.out.out = g->dx; m.out.out_s = g->dx_s; m.out.I = a->M;
    m.out.wide = g->K_out % 8 == 0 && fine(g->dx, a->M, g->dx_s);
    e = f16 ? gemm<true, false, true>(m, p.x, s) : gemm<true, false, false>(m, p.x, s);
  }
  if (e == hipSuccess && g->dw) {              // over the rows: both turned
    m.P = Operand{(const uint16_t*)a->x, a->M > 1 ? a->x_s : a->K, a->M, a->K};
    m.Q = dz_rows;
    m.nk = (int32_t)((a->M + 31) / 32);
    m.out.out = g->dw; m.out.out_s = g->dw_s; m.out.I = a->N;
    m.out.wide = g->K_out % 8 == 0 && fine(g->dw, a->N, g->dw_s);
    e = f16 ? gemm<true, true, true>(m, p.w, s) : gemm<true, true, false>(m, p.w, s);
  }
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
