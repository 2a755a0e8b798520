// The gradients of y = residual + gate act(z), z = x w^T + bias:
//
//   dz = dy gate act'(z)     dx = dz w     dw = dz^T x     dbias = sum dz     dgate = sum dy act(z)
//
// (the residual's is dy itself).  One pass over dy and z makes dz, rounded once to the
// operands' format for the two products, and the column sums from the unrounded values, in fixed
// parts.  Without activation and gate dz is dy as it lies.  Both products take w and x as they
// lie in memory, turned on their way out of LDS (linear_gemm.h): no transposed copy.
//
// fp16: a gate may be as small as it likes (1e-5 is usual where it begins), or of any size in
// one column and another, and dz would leave the format's range with it.  A row of dw has one gate: its
// product takes dy act'(z), and the gate multiplies the sums.  A row of dx has them all: its dz are
// scaled by a power of two that brings the row's largest dy gate (dz is no larger than 1.13 of it,
// whatever the activation) to 2^13 .. 2^14, and the sums by its inverse; what lies 2^27 below
// the largest keeps every bit.  (One scale for both products, by the largest gate: under gates of 300 and 0.3
// and a dy of 1e-3 the small one's row of dw was off by 3 % of its norm.)
#include "linear_gemm.h"

namespace gpa {
namespace {

struct DzArgs {
  const void* dy;
  const float* z;
  const void* gate;
  void* dz;               // rows of J8, the columns past J zeros; null: not wanted
  void* bare;             // fp16 with a gate: dw's, without it; null: not wanted
  float* unscale;         // fp16 with a gate: the inverse of each row's scale in dz
  float* gate32;          // where the gate goes, the scales of dw's rows; null: not wanted
  float* part;            // [chunk][2][J]; null: no sums
  int64_t dy_s, I, J, J8, chunk;
  int32_t pf32, gate_wide;
};

// The scale of each row of dz in fp16, by its largest finite dy gate: a workgroup a row (a wave a
// row: 8.4 us for 4.3 at 1,374 rows of 1,001).
template <bool WIDE>
__global__ __launch_bounds__(256) void linear_scale_kernel(DzArgs a) {
  __shared__ float top[4];
  const int64_t i = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (i >= a.I) return;
  const __bf16* DY = static_cast<const __bf16*>(a.dy) + i * a.dy_s;
  float m = 0.f;
  constexpr int AT = WIDE ? 8 : 1;
  for (int64_t j = threadIdx.x * AT; j < a.J; j += 256 * AT) {
    float dy[8], g[8];
    if constexpr (WIDE) {
      param8<true>(DY + j, 0, 1, 0, 8, dy);
      param8<true>(a.gate, a.pf32, a.gate_wide, j, 8, g);
    } else {
      dy[0] = half_to_f32<true>(DY[j]);
      g[0] = a.pf32 ? static_cast<const float*>(a.gate)[j] : half_to_f32<true>(static_cast<const __bf16*>(a.gate)[j]);
    }
#pragma unroll
    for (int e = 0; e < AT; ++e) {
      const float x = fabsf(dy[e] * g[e]);
      m = x < INFINITY ? fmaxf(m, x) : m;
    }
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  int e = 14;
  if (m > 0.f) frexpf(m, &e);                  // m = [0.5, 1) 2^e
  if (threadIdx.x == 0) a.unscale[i] = ldexpf(1.0f, max(e - 14, -126));
}

// 512 columns (eight a lane: side by side where they come in aligned groups (WIDE), else each 64
// from the next, so that a wave's loads lie together) of `chunk` rows a workgroup, a wave every
// fourth row.
template <int ACT, bool F16, bool WIDE, bool GATE>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs a) {
  __shared__ __attribute__((aligned(16))) float red[4][2][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int STEP = WIDE ? 1 : 64;
  const int64_t j = (int64_t)blockIdx.x * 512 + (WIDE ? lane * 8 : lane), i0 = blockIdx.y * a.chunk;
  const int64_t i1 = i0 + a.chunk < a.I ? i0 + a.chunk : a.I;
  float g[8], db[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    g[e] = 1.f;
    if (GATE && j + e * STEP < a.J)
      g[e] = a.pf32 ? static_cast<const float*>(a.gate)[j + e * STEP] : half_to_f32<F16>(static_cast<const __bf16*>(a.gate)[j + e * STEP]);
    db[e] = dg[e] = 0.f;
    if (GATE && F16 && a.gate32 && blockIdx.y == 0 && wave == 0 && j + e * STEP < a.J) a.gate32[j + e * STEP] = g[e];
  }
  auto put = [&](void* rows, int64_t i, const float (&v)[8]) __attribute__((always_inline)) {
    __bf16* to = static_cast<__bf16*>(rows) + i * a.J8 + j;
    if constexpr (WIDE) {
      bf16x8 y;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const bf16x2 w = pack2<F16>(v[e], v[e + 1]);
        y[e] = w[0];
        y[e + 1] = w[1];
      }
      *reinterpret_cast<bf16x8*>(to) = y;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e * 64 < a.J8) to[e * 64] = j + e * 64 < a.J ? f32_to_half<F16>(v[e]) : (__bf16)0.f;
    }
  };
  if (j < a.J8)
    for (int64_t i = i0 + wave; i < i1; i += 4) {
      float dy[8], z[8], d[8];
      const __bf16* DY = static_cast<const __bf16*>(a.dy) + i * a.dy_s + j;
      if constexpr (WIDE) {
        param8<F16>(DY, 0, 1, 0, 8, dy);
        if (a.z) param8<F16>(a.z + i * a.J + j, 1, 1, 0, 8, z);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = j + e * 64 < a.J;
          dy[e] = in ? half_to_f32<F16>(DY[e * 64]) : 0.f;
          z[e] = a.z && in ? a.z[i * a.J + j + e * 64] : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float slope = 1.f;
        if (ACT != kActNone || (GATE && a.z)) {
          const float v = act_both<ACT>(z[e], slope);
          if (GATE) dg[e] = __builtin_fmaf(dy[e], v, dg[e]);
        }
        d[e] = ACT != kActNone ? dy[e] * slope : dy[e];
      }
      if (GATE && F16 && a.bare) put(a.bare, i, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        db[e] = GATE ? __builtin_fmaf(d[e], g[e], db[e]) : db[e] + d[e];
        if (GATE) d[e] *= g[e];
      }
      if (!a.dz) continue;
      if (GATE && F16) {
        const float scale = 1.0f / a.unscale[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= scale;
      }
      put(a.dz, i, d);
    }
  if (!a.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = WIDE ? lane * 8 + e : lane + e * 64;
    red[wave][0][at] = db[e];
    red[wave][1][at] = dg[e];
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

// Rows of a workgroup of the pass over dy: 1,024 workgroups in all, 8 rows at least.
int64_t dz_chunk(int64_t I, int64_t J) {
  const int64_t cols = (J + 511) / 512, rows = std::max<int64_t>(1, 1024 / cols);
  return std::max<int64_t>(8, (I + rows - 1) / rows);
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct BwdPlan {
  GemmPlan x, w;
  Laid laid;
  int64_t chunk, chunks, J8;
  size_t bare, rows, gate, part, split, lay, bytes;   // where each begins, dz at 0
};
BwdPlan bwd_plan(const gpa_linear_gate_args* a, bool dz, bool sums, bool dx, bool dw) {
  BwdPlan p{};
  const int64_t M = a->M, N = a->N, K = std::max<int64_t>(a->K, 1);
  p.J8 = (N + 7) / 8 * 8;
  p.chunk = dz_chunk(M, N);
  p.chunks = (M + p.chunk - 1) / p.chunk;
  if (dx) p.x = gemm_plan(M, K, N, true);
  if (dw) p.w = gemm_plan(N, K, M, true);
  // (With a gate as fp16 needs it: the formats are not known here.)
  const size_t one = dz ? (size_t)round16(M * p.J8 * 2) : 0;
  const bool gate = dz && a->gate;
  p.bare = gate && dx ? one : 0;
  p.rows = gate && dx && dw ? 2 * one : one;
  p.gate = p.rows + (gate ? round16(M * 4) : 0);
  p.part = p.gate + (gate ? round16(N * 4) : 0);
  p.split = p.part + (sums ? (size_t)round16(p.chunks * 2 * N * 4) : 0);
  p.laid = linear_laid(a, dw, dx, true);
  p.lay = p.split + round16(std::max(p.x.bytes, p.w.bytes));
  p.bytes = p.lay + p.laid.bytes;
  return p;
}

}  // namespace

namespace {

template <bool F16, bool WIDE, bool GATE>
void dz_go(const DzArgs& d, int act, dim3 grid, hipStream_t s) {
  const dim3 block(256);
  switch (act) {
    case kActGelu: hipLaunchKernelGGL((linear_dz_kernel<kActGelu, F16, WIDE, GATE>), grid, block, 0, s, d); break;
    case kActGeluTanh: hipLaunchKernelGGL((linear_dz_kernel<kActGeluTanh, F16, WIDE, GATE>), grid, block, 0, s, d); break;
    case kActSilu: hipLaunchKernelGGL((linear_dz_kernel<kActSilu, F16, WIDE, GATE>), grid, block, 0, s, d); break;
    case kActRelu: hipLaunchKernelGGL((linear_dz_kernel<kActRelu, F16, WIDE, GATE>), grid, block, 0, s, d); break;
    default: hipLaunchKernelGGL((linear_dz_kernel<kActNone, F16, WIDE, GATE>), grid, block, 0, s, d); break;
  }
}
template <bool F16, bool WIDE>
void dz_gate(const DzArgs& d, int act, dim3 grid, hipStream_t s) {
  d.gate ? dz_go<F16, WIDE, true>(d, act, grid, s) : dz_go<F16, WIDE, false>(d, act, grid, s);
}
hipError_t dz_launch(const DzArgs& d, int act, bool f16, bool wide, dim3 grid, hipStream_t s) {
  if (d.dz && d.unscale) {
    const int64_t wgs = d.I, most = (int64_t)1 << 22;   // (a dimension has less than 2^32 threads)
    const dim3 rows((unsigned)std::min(wgs, most), (unsigned)((wgs + most - 1) / most));
    if (wide) hipLaunchKernelGGL((linear_scale_kernel<true>), rows, dim3(256), 0, s, d);
    else hipLaunchKernelGGL((linear_scale_kernel<false>), rows, dim3(256), 0, s, d);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (f16) wide ? dz_gate<true, true>(d, act, grid, s) : dz_gate<true, false>(d, act, grid, s);
  else wide ? dz_gate<false, true>(d, act, grid, s) : dz_gate<false, false>(d, act, grid, s);
  return hipGetLastError();
}

}  // namespace
}  // namespace gpa

using namespace gpa;

// Whether dy itself is not dz as the products take it (turned, for dw: linear_gemm.h, Feed).
static bool needs_dz(const gpa_linear_gate_args* a, const gpa_linear_gate_grads* g) {
  const int64_t least = g->dw ? a->N : 0;
  const bool aligned = a->N % 8 == 0 && (uintptr_t)g->dy % 16 == 0 && (a->M < 2 || (g->dy_s % 8 == 0 && g->dy_s >= least && g->dy_s < 1 << 21));
  return (g->dx || g->dw) && (a->act != kActNone || a->gate || !aligned);
}

extern "C" size_t gpa_linear_gate_bwd_workspace_bytes(const gpa_linear_gate_args* a, const gpa_linear_gate_grads* g) {
  if (!a || !g || a->M <= 0 || a->N <= 0 || a->K < 0) return 0;
  return bwd_plan(a, needs_dz(a, g), g->dbias || g->dgate, g->dx, g->dw).bytes;
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
  if (!g->dy || (g->dgate && !a->gate) || (g->z && ((uintptr_t)g->z % 16 || g->z_dtype != GPA_DTYPE_F32)) ||
      (!g->z && (a->act != kActNone || g->dgate))) {
    gpa_set_error("%s: dy is needed, z with an activation or the gate's gradient, and there is none of an absent gate", fn);
    return GPA_E_INVALID;
  }
  if ((g->dx || g->dw) && a->K == 0) {
    gpa_set_error("%s: no feature, so there are no gradients of x and w", fn);
    return GPA_E_INVALID;
  }
  if (a->N >= (int64_t)1 << 21) {
    gpa_set_error("%s: %lld output features (below 2^21)", fn, (long long)a->N);
    return GPA_E_UNSUPPORTED;
  }
  const bool f16 = dtype == GPA_DTYPE_F16, need_dz = needs_dz(a, g), sums = g->dbias || g->dgate;
  const BwdPlan p = bwd_plan(a, need_dz, sums, g->dx, g->dw);
  if ((g->dx && !linear_launchable(p.x, a->M, a->K)) || (g->dw && !linear_launchable(p.w, a->N, a->K))) {
    gpa_set_error("%s: problem exceeds the grid limit", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16)) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, p.bytes);
    return GPA_E_WORKSPACE;
  }
  char* ws = (char*)workspace;
  const hipStream_t s = (hipStream_t)stream;
  const bool apart = need_dz && f16 && a->gate;          // dw's dz without the gate, dx's with its rows' scales
  float* const rows = apart && g->dx ? (float*)(ws + p.rows) : nullptr;
  float* const gates = apart && g->dw ? (float*)(ws + p.gate) : nullptr;
  Matrix x, w;
  hipError_t e = linear_lay(a, p.laid, ws + p.lay, x, w, s);
  if (e == hipSuccess && (need_dz || sums)) {
    DzArgs d{};
    d.dy = g->dy; d.dy_s = a->M > 1 ? g->dy_s : 0;
    d.z = (const float*)g->z; d.gate = a->gate;
    d.gate_wide = (uintptr_t)a->gate % 16 == 0;
    d.dz = need_dz && (!apart || g->dx) ? ws : nullptr;
    d.bare = gates ? ws + p.bare : nullptr;
    d.unscale = rows; d.gate32 = gates;
    d.part = sums ? (float*)(ws + p.part) : nullptr;
    d.I = a->M; d.J = a->N; d.J8 = p.J8; d.chunk = p.chunk;
    d.pf32 = param_dtype == GPA_DTYPE_F32;
    const bool wide = a->N % 8 == 0 && (uintptr_t)g->dy % 16 == 0 && d.dy_s % 8 == 0;
    const dim3 grid((unsigned)((a->N + 511) / 512), (unsigned)p.chunks);
    e = dz_launch(d, a->act, f16, wide, grid, s);
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
  Operand dz_rows{need_dz ? (const uint16_t*)ws : (const uint16_t*)g->dy, need_dz ? p.J8 : a->M > 1 ? g->dy_s : p.J8, a->M, p.J8};
  auto fine = [](const void* q, int64_t n, int64_t st) { return (uintptr_t)q % 16 == 0 && (n < 2 || st % 8 == 0); };
  GemmArgs m{};
  m.out.unscale = rows;
  m.out.part = (float*)(ws + p.split);
  m.out.J = a->K;
  if (e == hipSuccess && g->dx) {              // over the output features: w turned
    m.P = Operand{w.p, w.stride, a->N, p.laid.K};
    m.Q = dz_rows;
    m.nk = (int32_t)((p.J8 + 31) / 32);
    m.out.out = g->dx; m.out.out_s = g->dx_s; m.out.I = a->M;
    m.out.wide = a->K % 8 == 0 && fine(g->dx, a->M, g->dx_s);
    e = f16 ? gemm<true, false, true>(m, p.x, s) : gemm<true, false, false>(m, p.x, s);
  }
  if (e == hipSuccess && g->dw) {              // over the rows: both turned
    m.P = Operand{x.p, x.stride, a->M, p.laid.K};
    if (apart) dz_rows.p = (const uint16_t*)(ws + p.bare);
    m.Q = dz_rows;
    m.out.unscale = gates;
    m.nk = (int32_t)((a->M + 31) / 32);
    m.out.out = g->dw; m.out.out_s = g->dw_s; m.out.I = a->N;
    m.out.wide = a->K % 8 == 0 && fine(g->dw, a->N, g->dw_s);
    e = f16 ? gemm<true, true, true>(m, p.w, s) : gemm<true, true, false>(m, p.w, s);
  }
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
