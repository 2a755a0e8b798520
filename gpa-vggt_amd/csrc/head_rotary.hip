// The norm of every head and its rotation by positions of one or more axes, and
// their gradients: what a block's queries and keys go through between the
// projection and the attention, of any head dim, over one or two tensors.
//
//   n = N(x) w + b                          N: none, RMS or LayerNorm over the head
//   angle_j = p[axis_j] freq_j              of pair j of features (a_j, b_j)
//   y_a = n_a cos - n_b sin                 y_b = n_b cos + n_a sin
//
// and with g = dn w, dn being dy turned by the negative angles:
//   dx = (g - hat mean(g hat) [- mean(g)]) / sigma      dw = sum dn hat      db = sum dn
//
// Features that belong to no pair are not turned (and not multiplied by one and
// zero: an infinity there stays with itself).
//
// Angles.  Positions reach millions, where an angle in fp32 is off by tenths: the
// product is formed in 64 bits, in turns, and what is left of it after whole turns
// is taken to fp32 (off by 2^-25 of a turn at most), whose sine and cosine are
// good to an ulp or two.  One sine and cosine costs what half a head's row does, so
// a workgroup forms them once a token, in LDS, for all of its heads.
//
// Lanes.  A head is cut into chunks of eight pairs: a lane has both features of
// each, so the rotation needs no exchange; the moments go over the chunks' lanes
// by DPP.  A chunk is 32 bytes in two 16-byte pieces (fp32: four) where its
// features lie so, whole and aligned (VEC); otherwise single elements.
//
// Bound by HBM: the forward reads and writes each value once, the backward
// reads x and dy and writes dx (the moments are formed again, which costs less than
// keeping them).  Parameters' gradients go through one fp32 partial a workgroup,
// in a fixed order.
#include <algorithm>
#include <math.h>

#include "gpa_common.h"

namespace gpa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxD = 256;
constexpr int kMaxChunks = 32;
constexpr int kMaxTokens = 16;            // of a workgroup's tile
constexpr int kCsFloats = 4096;           // cosines and sines of a tile
constexpr int64_t kBwdWgs = 1024;

// Eight pairs of a head: their features begin at o0 and o1 (neighbours: all at
// o0), the first pair's number (-1: they are not turned), how many there are.
struct Chunk { int16_t o0, o1, p0, n; };

struct Side {
  const void* x;          // [B, heads, N, D]
  const void* dy;         // backward
  void* out;              // y, or dx
  int64_t x_sb, x_sh, x_sn, y_sb, y_sh, y_sn, o_sb, o_sh, o_sn;
  const void *w, *b;
  float* part;            // backward: [workgroup][2][D]
  int32_t heads, wgs;     // wgs: the backward's workgroups of this side
};

struct RotArgs {
  Side side[2];
  const void* pos;
  int64_t pos_sb, pos_sn;
  const double* freqs;
  const int32_t* axes;
  int64_t N, tokens, tiles;
  uint32_t rows_magic;    // 2^32 / heads of both, rounded up (one head: not used)
  int32_t D, pairs, count, pos_kind, chunks, lanes, per_tile, norm, pf32;
  float eps, inv_d;
  Chunk chunk[kMaxChunks];
};

enum { kNone = 0, kRms = 1, kLayer = 2 };

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// Sum over the `lanes` (a power of two up to 32) of a row.
__device__ __forceinline__ float row_sum(float v, int lanes) {
  if (lanes > 1) v = dpp_add<0xB1>(v);         // lane ^ 1
  if (lanes > 2) v = dpp_add<0x4E>(v);         // lane ^ 2
  if (lanes > 4) v = dpp_add<0x141>(v);        // the mirror of eight: the other four's sum
  if (lanes > 8) v = dpp_add<0x140>(v);        // the mirror of sixteen
  if (lanes > 16) v += __shfl_xor(v, 16);
  return v;
}

template <typename T> struct Piece;            // 16 bytes
template <> struct Piece<float> { typedef f32x4 type; };
template <> struct Piece<__bf16> { typedef bf16x8 type; };
template <> struct Piece<_Float16> { typedef f16x8 type; };

// A chunk's sixteen values as they lie in memory.
template <typename T, bool VEC, bool INTER>
struct Raw {
  typedef typename Piece<T>::type V;
  static constexpr int PER = 16 / sizeof(T), HALF = 8 / PER;   // values of a piece; pieces of eight values
  V v[2 * HALF];
  __device__ __forceinline__ void load(const T* row, const Chunk& c) {
    if constexpr (VEC) {
      const V* a = reinterpret_cast<const V*>(row + c.o0);
      const V* b = INTER ? a + HALF : reinterpret_cast<const V*>(row + c.o1);
#pragma unroll
      for (int i = 0; i < HALF; ++i) v[i] = c.n ? a[i] : V{};
#pragma unroll
      for (int i = 0; i < HALF; ++i) v[HALF + i] = c.n ? b[i] : V{};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = i < c.n;
        put(INTER ? 2 * i : i, in ? row[c.o0 + (INTER ? 2 * i : i)] : (T)0.f);
        put(INTER ? 2 * i + 1 : 8 + i, in ? row[INTER ? c.o0 + 2 * i + 1 : c.o1 + i] : (T)0.f);
      }
    }
  }
  __device__ __forceinline__ void put(int i, T x) { v[i / PER][i % PER] = x; }
  __device__ __forceinline__ void get(float (&a)[8], float (&b)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = INTER ? 2 * i : i, q = INTER ? 2 * i + 1 : 8 + i;
      a[i] = (float)v[p / PER][p % PER];
      b[i] = (float)v[q / PER][q % PER];
    }
  }
  __device__ __forceinline__ void set(const float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      put(INTER ? 2 * i : i, (T)a[i]);
      put(INTER ? 2 * i + 1 : 8 + i, (T)b[i]);
    }
  }
  __device__ __forceinline__ void store(T* row, const Chunk& c) const {
    if constexpr (VEC) {
      if (c.n == 0) return;
      V* a = reinterpret_cast<V*>(row + c.o0);
      V* b = INTER ? a + HALF : reinterpret_cast<V*>(row + c.o1);
#pragma unroll
      for (int i = 0; i < HALF; ++i) a[i] = v[i];
#pragma unroll
      for (int i = 0; i < HALF; ++i) b[i] = v[HALF + i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= c.n) continue;
        const int p = INTER ? 2 * i : i, q = INTER ? 2 * i + 1 : 8 + i;
        row[c.o0 + p] = v[p / PER][p % PER];
        row[INTER ? c.o0 + q : c.o1 + i] = v[q / PER][q % PER];
      }
    }
  }
};

// Eight values of LDS.
__device__ __forceinline__ void take8(const float* p, float (&x)[8]) {
  const f32x4 lo = reinterpret_cast<const f32x4*>(p)[0], hi = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = lo[i];
    x[4 + i] = hi[i];
  }
}

struct Tile {
  float cs[kCsFloats];    // [token][chunk][cos 8, sin 8]
  int64_t at[kMaxTokens][2];   // a token's batch element and number
};

// The tokens of a tile, and the cosines and sines of their chunks.
template <bool INTER>
__device__ __forceinline__ void place_tile(const RotArgs& a, Tile& t, int64_t first, int live) {
  for (int i = threadIdx.x; i < live; i += kThreads) {
    const uint32_t tok = (uint32_t)(first + i), b = tok / (uint32_t)a.N;
    t.at[i][0] = b;
    t.at[i][1] = tok - b * (uint32_t)a.N;
  }
  const int width = a.chunks * 8;
  for (int i = threadIdx.x; i < live * width; i += kThreads) {
    const int k = i / width, c = i % width;
    const Chunk ch = a.chunk[c >> 3];
    if (ch.p0 < 0 || (c & 7) >= ch.n) continue;
    const int j = ch.p0 + (c & 7);
    const uint32_t tok = (uint32_t)(first + k), b = tok / (uint32_t)a.N, n = tok - b * (uint32_t)a.N;
    int ax = a.axes[j];
    ax = ax < 0 ? 0 : ax >= a.count ? a.count - 1 : ax;
    const int64_t at = b * a.pos_sb + n * a.pos_sn + ax;
    const double p = a.pos_kind == 0 ? (double)static_cast<const int32_t*>(a.pos)[at]
                     : a.pos_kind == 1 ? (double)static_cast<const int64_t*>(a.pos)[at]
                                       : (double)static_cast<const float*>(a.pos)[at];
    const double turns = p * a.freqs[j] * 0.15915494309189533577;
    const float rest = (float)(turns - __builtin_rint(turns));
    float s, co;
    sincospif(2.0f * rest, &s, &co);
    t.cs[(k * a.chunks + (c >> 3)) * 16 + (c & 7)] = co;
    t.cs[(k * a.chunks + (c >> 3)) * 16 + 8 + (c & 7)] = s;
  }
}

// A parameter in a lane's order: its sixteen values, `none` where there are none.
template <typename T, bool INTER>
__device__ __forceinline__ void take_param(const RotArgs& a, const void* p, const Chunk& c, float none, float (&x)[8], float (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = y[i] = none;
    if (!p || i >= c.n) continue;
    const int u = INTER ? c.o0 + 2 * i : c.o0 + i, v = INTER ? c.o0 + 2 * i + 1 : c.o1 + i;
    const bool wide = sizeof(T) == 4 || a.pf32;
    x[i] = wide ? static_cast<const float*>(p)[u] : (float)static_cast<const T*>(p)[u];
    y[i] = wide ? static_cast<const float*>(p)[v] : (float)static_cast<const T*>(p)[v];
  }
}

// Both moments of a row; x, y centred under LayerNorm.  Returns 1 / sigma.
__device__ __forceinline__ float moments(const RotArgs& a, const Chunk& c, bool vec, float (&x)[8], float (&y)[8]) {
  if (a.norm == kLayer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] + y[i];
    const float mean = row_sum(s, a.lanes) * a.inv_d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {              // values that are not there stay 0
      const bool in = vec ? c.n != 0 : i < c.n;
      x[i] = in ? x[i] - mean : 0.f;
      y[i] = in ? y[i] - mean : 0.f;
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], __builtin_fmaf(y[i], y[i], ss));
  return rsqrtf(__builtin_fmaf(row_sum(ss, a.lanes), a.inv_d, a.eps));
}

// A lane's chunk (none past the last), and its row of the workgroup's.
struct Lane { Chunk c; int row, rows; };
__device__ __forceinline__ Lane lane_of(const RotArgs& a) {
  Lane l;
  const int at = threadIdx.x % a.lanes;
  l.c = a.chunk[at < a.chunks ? at : 0];
  if (at >= a.chunks) l.c.n = 0;
  l.row = threadIdx.x / a.lanes;
  l.rows = kThreads / a.lanes;
  return l;
}

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void head_rotary_kernel(RotArgs a) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;    // rows a lane has in flight
  __shared__ __attribute__((aligned(16))) Tile t;
  __shared__ __attribute__((aligned(16))) float par[2][2][kMaxChunks * 16];
  const Lane l = lane_of(a);
  const int at = threadIdx.x % a.lanes, both = a.side[0].heads + a.side[1].heads;
  if (a.norm && l.row < 2) {                   // a row of lanes for each side (a wave has two at least)
    const Side& s = a.side[l.row];
    float x[8], y[8];
    for (int k = 0; k < 2; ++k) {
      take_param<T, INTER>(a, k ? s.b : s.w, l.c, k ? 0.f : 1.f, x, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        par[l.row][k][at * 16 + i] = x[i];
        par[l.row][k][at * 16 + 8 + i] = y[i];
      }
    }
  }
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t first = tile * a.per_tile;
    const int live = (int)(a.tokens - first < a.per_tile ? a.tokens - first : a.per_tile);
    const int rows = live * both;
    __syncthreads();
    place_tile<INTER>(a, t, first, live);
    __syncthreads();
    for (int r0 = l.row; r0 < rows + l.row; r0 += U * l.rows) {
      Raw<T, VEC, INTER> raw[U];
      T* out[U];
      const float *cs[U], *w[U];
      bool biased[U], fine[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * l.rows;
        fine[u] = r < rows;
        const int rc = fine[u] ? r : rows - 1;
        const int k = both == 1 ? rc : (int)__umulhi((uint32_t)rc, a.rows_magic), hh = rc - k * both;
        const bool which = hh >= a.side[0].heads;
        const int h = which ? hh - a.side[0].heads : hh;
        // Selected, not indexed: a lane's own index would be a load from the arguments.
        const Side &s0 = a.side[0], &s1 = a.side[1];
        const int64_t b = t.at[k][0], n = t.at[k][1];
        raw[u].load(static_cast<const T*>(which ? s1.x : s0.x) + b * (which ? s1.x_sb : s0.x_sb) +
                        h * (which ? s1.x_sh : s0.x_sh) + n * (which ? s1.x_sn : s0.x_sn), l.c);
        out[u] = static_cast<T*>(which ? s1.out : s0.out) + b * (which ? s1.o_sb : s0.o_sb) +
                 h * (which ? s1.o_sh : s0.o_sh) + n * (which ? s1.o_sn : s0.o_sn);
        cs[u] = t.cs + (k * a.chunks + (at < a.chunks ? at : 0)) * 16;
        w[u] = par[which][0] + at * 16;
        biased[u] = which ? s1.b != nullptr : s0.b != nullptr;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8], y[8];
        raw[u].get(x, y);
        if (a.norm) {
          const float inv = moments(a, l.c, VEC, x, y);
          float p[8], q[8];
          take8(w[u], p);
          take8(w[u] + 8, q);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * inv * p[i];
            y[i] = y[i] * inv * q[i];
          }
          if (biased[u]) {
            take8(w[u] + kMaxChunks * 16, p);
            take8(w[u] + kMaxChunks * 16 + 8, q);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              x[i] += p[i];
              y[i] += q[i];
            }
          }
        }
        if (l.c.p0 >= 0) {
          float c[8], s[8];
          take8(cs[u], c);
          take8(cs[u] + 8, s);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = x[i];
            x[i] = __builtin_fmaf(v, c[i], -(y[i] * s[i]));
            y[i] = __builtin_fmaf(y[i], c[i], v * s[i]);
          }
        }
        if (!fine[u]) continue;
        raw[u].set(x, y);
        raw[u].store(out[u], l.c);
      }
    }
  }
}

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void head_rotary_bwd_kernel(RotArgs a) {
  constexpr int U = sizeof(T) == 4 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) Tile t;
  const Lane l = lane_of(a);
  const int at = threadIdx.x % a.lanes;
  const int which = (int)blockIdx.x >= a.side[0].wgs;
  const Side& s = a.side[which];
  const int wg = which ? (int)blockIdx.x - a.side[0].wgs : (int)blockIdx.x;
  float wa[8], wb[8], dwa[8], dwb[8], dba[8], dbb[8];
  take_param<T, INTER>(a, s.w, l.c, 1.f, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) dwa[i] = dwb[i] = dba[i] = dbb[i] = 0.f;

  for (int64_t tile = wg; tile < a.tiles; tile += s.wgs) {
    const int64_t first = tile * a.per_tile;
    const int live = (int)(a.tokens - first < a.per_tile ? a.tokens - first : a.per_tile);
    const int rows = live * s.heads;
    __syncthreads();
    place_tile<INTER>(a, t, first, live);
    __syncthreads();
    for (int r0 = l.row; r0 < rows + l.row; r0 += U * l.rows) {
      Raw<T, VEC, INTER> rx[U], ry[U];
      T* out[U];
      const float* cs[U];
      bool fine[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * l.rows;
        fine[u] = r < rows;
        const int rc = fine[u] ? r : rows - 1, k = rc / s.heads, h = rc - k * s.heads;
        ry[u].load(static_cast<const T*>(s.dy) + t.at[k][0] * s.y_sb + h * s.y_sh + t.at[k][1] * s.y_sn, l.c);
        if (a.norm) rx[u].load(static_cast<const T*>(s.x) + t.at[k][0] * s.x_sb + h * s.x_sh + t.at[k][1] * s.x_sn, l.c);
        out[u] = static_cast<T*>(s.out) + t.at[k][0] * s.o_sb + h * s.o_sh + t.at[k][1] * s.o_sn;
        cs[u] = t.cs + (k * a.chunks + (at < a.chunks ? at : 0)) * 16;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float ga[8], gb[8];
        ry[u].get(ga, gb);
        if (l.c.p0 >= 0) {                     // turned back
          float c[8], sn[8];
          take8(cs[u], c);
          take8(cs[u] + 8, sn);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = ga[i];
            ga[i] = __builtin_fmaf(v, c[i], gb[i] * sn[i]);
            gb[i] = __builtin_fmaf(gb[i], c[i], -(v * sn[i]));
          }
        }
        if (a.norm) {
          float x[8], y[8];
          rx[u].get(x, y);
          const float inv = moments(a, l.c, VEC, x, y);
          float s1 = 0.f, s0 = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= inv;
            y[i] *= inv;
            if (fine[u]) {
              dwa[i] = __builtin_fmaf(ga[i], x[i], dwa[i]);
              dwb[i] = __builtin_fmaf(gb[i], y[i], dwb[i]);
              dba[i] += ga[i];
              dbb[i] += gb[i];
            }
            ga[i] *= wa[i];
            gb[i] *= wb[i];
            s1 = __builtin_fmaf(ga[i], x[i], __builtin_fmaf(gb[i], y[i], s1));
            s0 += ga[i] + gb[i];
          }
          s1 = row_sum(s1, a.lanes) * a.inv_d;
          s0 = a.norm == kLayer ? row_sum(s0, a.lanes) * a.inv_d : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ga[i] = inv * (ga[i] - s0 - x[i] * s1);
            gb[i] = inv * (gb[i] - s0 - y[i] * s1);
          }
        }
        if (!fine[u]) continue;
        ry[u].set(ga, gb);
        ry[u].store(out[u], l.c);
      }
    }
  }
  if (!s.part) return;

  // The rows' sums: over a wave's rows, then over the four waves in LDS.
  float* red = t.cs;                           // [wave][lane of a row][4][8], at most 4 * 32 * 32 floats
  float* sums[4] = {dwa, dwb, dba, dbb};
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      for (int m = a.lanes; m < 64; m <<= 1) sums[k][i] += __shfl_xor(sums[k][i], m);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane < a.lanes)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) red[((wave * a.lanes + lane) * 4 + k) * 8 + i] = sums[k][i];
  __syncthreads();
  float* part = s.part + (int64_t)wg * 2 * a.D;
  for (int i = threadIdx.x; i < a.chunks * 32; i += kThreads) {
    const Chunk c = a.chunk[i >> 5];
    const int e = i & 7, side = i >> 3 & 1, bias = i >> 4 & 1;
    if (e >= c.n) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v += red[(w * a.lanes + (i >> 5)) * 32 + (i & 31)];
    const int f = INTER ? c.o0 + 2 * e + side : side ? c.o1 + e : c.o0 + e;
    part[bias * a.D + f] = v;
  }
}

// A side's partials added up: 64 columns a workgroup, 16 waves over the partials.
struct SumArgs {
  const float* part[2];
  void* out[2][2];        // [side][w, b]; null: not wanted
  int32_t wgs[2], D;
};
template <typename P>
__global__ __launch_bounds__(1024) void head_rotary_sum_kernel(SumArgs a) {
  __shared__ float tot[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, side = blockIdx.y, k = blockIdx.z;
  P* out = static_cast<P*>(a.out[side][k]);
  if (!out) return;
  float s = 0.f;
  if (c < a.D)
#pragma unroll 4
    for (int i = wave; i < a.wgs[side]; i += 16) s += a.part[side][((int64_t)i * 2 + k) * a.D + c];
  tot[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < a.D) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += tot[i][lane];
    out[c] = (P)s;
  }
}

// Chunks of eight pairs; false: more than kMaxChunks.
bool cut(const gpa_head_rotary_args* a, RotArgs& r) {
  int n = 0;
  auto add = [&](int first, int second, int pairs, int p0, bool neighbours) {
    for (int i = 0; i < pairs; i += 8) {
      if (n == kMaxChunks) return false;
      r.chunk[n++] = Chunk{(int16_t)(first + (neighbours ? 2 * i : i)), (int16_t)(second + i),
                           (int16_t)(p0 < 0 ? -1 : p0 + i), (int16_t)std::min(8, pairs - i)};
    }
    return true;
  };
  const int P = (int)a->pairs, rest = (int)a->D - 2 * P;
  const bool next = a->pairing == GPA_PAIRS_NEIGHBOURS;
  bool ok = true;
  if (a->pairing == GPA_PAIRS_BLOCKS) {
    for (int i = 0, p = 0; i < a->sections_count; p += a->sections[i++])
      ok = ok && add(2 * p, 2 * p + a->sections[i], a->sections[i], p, false);
  } else {
    ok = add(0, P, P, 0, next);
  }
  ok = ok && add(2 * P, 2 * P + rest / 2, rest / 2, -1, next);
  r.chunks = n;
  r.lanes = 1;
  while (r.lanes < n) r.lanes *= 2;
  return ok;
}

int check(const char* fn, int dtype, int pdtype, const gpa_head_rotary_args* a) {
  if (!a) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (dtype < GPA_DTYPE_F32 || dtype > GPA_DTYPE_F16 || (pdtype != dtype && pdtype != GPA_DTYPE_F32)) {
    gpa_set_error("%s: dtypes %d and %d (parameters have the heads' type or fp32)", fn, dtype, pdtype);
    return GPA_E_INVALID;
  }
  if (a->B < 0 || a->N < 0 || a->H < 0 || a->Hk < 0 || a->D < 0 || a->pairs < 0) {
    gpa_set_error("%s: negative size", fn);
    return GPA_E_INVALID;
  }
  if (a->D < 2 || a->D > kMaxD || a->D % 2) {
    gpa_set_error("%s: head dim %lld unsupported (even, 2 to %d)", fn, (long long)a->D, kMaxD);
    return GPA_E_UNSUPPORTED;
  }
  if (2 * a->pairs > a->D || a->pairing < GPA_PAIRS_HALVES || a->pairing > GPA_PAIRS_BLOCKS) {
    gpa_set_error("%s: %lld pairs of %lld features, pairing %d", fn, (long long)a->pairs,
                  (long long)a->D, a->pairing);
    return GPA_E_INVALID;
  }
  if (a->pairs > 0) {
    if (a->sections_count < 1 || a->sections_count > GPA_MAX_AXES) {
      gpa_set_error("%s: %d axes (1 to %d)", fn, a->sections_count, GPA_MAX_AXES);
      return GPA_E_INVALID;
    }
    int64_t sum = 0;
    for (int i = 0; i < a->sections_count; ++i) {
      sum += a->sections[i];
      if (a->sections[i] < 0 || sum > a->pairs) break;
    }
    for (int i = 0; i < a->sections_count; ++i)
      if (a->sections[i] < 0) sum = -1;
    if (sum != a->pairs) {
      gpa_set_error("%s: the axes' sections do not add to %lld pairs", fn, (long long)a->pairs);
      return GPA_E_INVALID;
    }
  }
  if (a->norm < kNone || a->norm > kLayer || !(a->eps >= 0.f) || !isfinite(a->eps)) {
    gpa_set_error("%s: norm %d (0 to 2), or eps that is not finite and >= 0", fn, a->norm);
    return GPA_E_INVALID;
  }
  // Token numbers are 32-bit; heads of a tile's tokens below 2^16.
  if (a->N >= (int64_t)1 << 31 || a->B >= (int64_t)1 << 31 || a->B * a->N >= (int64_t)1 << 31 ||
      a->H >= 2048 || a->Hk >= 2048) {
    gpa_set_error("%s: too many tokens or heads", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (a->B == 0 || a->N == 0) return GPA_OK;
  if ((a->H > 0 && !a->q) || (a->Hk > 0 && !a->k) ||
      (a->pairs > 0 && (!a->positions || !a->freqs || !a->axes))) {
    gpa_set_error("%s: null pointer", fn);
    return GPA_E_INVALID;
  }
  if (a->positions_kind < 0 || a->positions_kind > 2) {
    gpa_set_error("%s: positions of kind %d (0 int32, 1 int64, 2 fp32)", fn, a->positions_kind);
    return GPA_E_INVALID;
  }
  if (!a->norm && (a->q_w || a->k_w || a->q_b || a->k_b)) {
    gpa_set_error("%s: parameters without a norm", fn);
    return GPA_E_INVALID;
  }
  return GPA_OK;
}

struct Rows { const void* p; int64_t heads, sb, sh, sn; };

// Fills everything but the outputs; returns whether chunks are whole 16-byte pieces.
bool fill(const gpa_head_rotary_args* a, int dtype, int pdtype, std::initializer_list<Rows> all, RotArgs& r) {
  const int64_t esize = dtype == GPA_DTYPE_F32 ? 4 : 2, per16 = 16 / esize;
  auto st = [](int64_t n, int64_t s) { return n > 1 ? s : 0; };
  Side &q = r.side[0], &k = r.side[1];
  q.x = a->q; k.x = a->k;
  q.x_sb = st(a->B, a->q_sb); q.x_sh = st(a->H, a->q_sh); q.x_sn = st(a->N, a->q_sn);
  k.x_sb = st(a->B, a->k_sb); k.x_sh = st(a->Hk, a->k_sh); k.x_sn = st(a->N, a->k_sn);
  q.w = a->q_w; q.b = a->q_b; k.w = a->k_w; k.b = a->k_b;
  q.heads = (int32_t)a->H; k.heads = (int32_t)a->Hk;
  r.pos = a->positions; r.pos_sb = st(a->B, a->pos_sb); r.pos_sn = st(a->N, a->pos_sn);
  r.pos_kind = a->positions_kind;
  r.freqs = a->freqs; r.axes = a->axes;
  r.N = a->N; r.tokens = a->B * a->N;
  r.D = (int32_t)a->D; r.pairs = (int32_t)a->pairs; r.count = a->sections_count;
  r.norm = a->norm; r.pf32 = pdtype == GPA_DTYPE_F32;
  r.eps = a->eps; r.inv_d = 1.0f / (float)a->D;
  bool vec = true;
  for (int i = 0; i < r.chunks; ++i) {
    const Chunk& c = r.chunk[i];
    vec = vec && c.n == 8 && c.o0 % 8 == 0 && (a->pairing == GPA_PAIRS_NEIGHBOURS || c.o1 % 8 == 0);
  }
  for (const Rows& x : all)
    if (x.p && x.heads > 0)
      vec = vec && (uintptr_t)x.p % 16 == 0 && st(a->B, x.sb) % per16 == 0 &&
            st(x.heads, x.sh) % per16 == 0 && st(a->N, x.sn) % per16 == 0;
  return vec;
}

// Tokens of a workgroup's tile: four rounds of its rows, unless that leaves CUs
// without a workgroup.  (Cosines and sines are formed for a whole tile at once.)
int tile_tokens(const RotArgs& r, int64_t heads, int64_t rounds) {
  const int64_t rows = kThreads / r.lanes;
  int64_t n = std::min<int64_t>({rounds * rows / std::max<int64_t>(heads, 1), r.tokens / 1024, kMaxTokens,
                                 kCsFloats / (16 * std::max(r.chunks, 1))});
  return (int)std::max<int64_t>(n, 1);
}

template <typename T, bool VEC>
hipError_t forward(const RotArgs& r, bool inter, hipStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>(r.tiles, 1 << 22)), block(kThreads);
  if (inter) hipLaunchKernelGGL((head_rotary_kernel<T, VEC, true>), grid, block, 0, s, r);
  else hipLaunchKernelGGL((head_rotary_kernel<T, VEC, false>), grid, block, 0, s, r);
  return hipGetLastError();
}
template <typename T, bool VEC>
hipError_t backward(const RotArgs& r, bool inter, hipStream_t s) {
  const dim3 grid((unsigned)(r.side[0].wgs + r.side[1].wgs)), block(kThreads);
  if (inter) hipLaunchKernelGGL((head_rotary_bwd_kernel<T, VEC, true>), grid, block, 0, s, r);
  else hipLaunchKernelGGL((head_rotary_bwd_kernel<T, VEC, false>), grid, block, 0, s, r);
  return hipGetLastError();
}
template <bool BWD>
hipError_t launch(const RotArgs& r, int dtype, bool vec, bool inter, hipStream_t s) {
  auto go = [&](auto type) {
    typedef decltype(type) T;
    if constexpr (BWD) return vec ? backward<T, true>(r, inter, s) : backward<T, false>(r, inter, s);
    else return vec ? forward<T, true>(r, inter, s) : forward<T, false>(r, inter, s);
  };
  return dtype == GPA_DTYPE_F32 ? go(0.f) : dtype == GPA_DTYPE_BF16 ? go((__bf16)0.f) : go((_Float16)0.f);
}

int refuse_launch(const char* fn, hipError_t e) {
  if (e == hipSuccess) return GPA_OK;
  gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
  return GPA_E_LAUNCH;
}

// Workgroups of the backward's two sides, by their share of the heads; none has more than tiles.
struct Wgs { int64_t q, k; };
Wgs bwd_wgs(int64_t tokens, int64_t H, int64_t Hk, bool q, bool k) {
  if (tokens <= 0) return {0, 0};
  const int64_t h = q ? H : 0, hk = k ? Hk : 0, all = std::max<int64_t>(h + hk, 1);
  auto share = [&](int64_t n) {
    return n == 0 ? 0 : std::max<int64_t>(1, std::min(tokens, (kBwdWgs * n + all - 1) / all));
  };
  return {share(h), share(hk)};
}

}  // namespace
}  // namespace gpa

using namespace gpa;

extern "C" int gpa_head_rotary(int dtype, int param_dtype, const gpa_head_rotary_args* a, void* q_out,
                               int64_t qo_sb, int64_t qo_sh, int64_t qo_sn, void* k_out, int64_t ko_sb,
                               int64_t ko_sh, int64_t ko_sn, void* stream) {
  const char* fn = "gpa_head_rotary";
  gpa_clear_error();
  const int rc = check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK || a->B == 0 || a->N == 0 || a->H + a->Hk == 0) return rc;
  if ((a->H > 0 && !q_out) || (a->Hk > 0 && !k_out)) {
    gpa_set_error("%s: null output", fn);
    return GPA_E_INVALID;
  }
  RotArgs r{};
  if (!cut(a, r)) {
    gpa_set_error("%s: too many sections for this head dim", fn);
    return GPA_E_UNSUPPORTED;
  }
  const bool vec = fill(a, dtype, param_dtype,
                        {{a->q, a->H, a->q_sb, a->q_sh, a->q_sn}, {a->k, a->Hk, a->k_sb, a->k_sh, a->k_sn},
                         {q_out, a->H, qo_sb, qo_sh, qo_sn}, {k_out, a->Hk, ko_sb, ko_sh, ko_sn}}, r);
  r.side[0].out = q_out; r.side[0].o_sb = qo_sb; r.side[0].o_sh = qo_sh; r.side[0].o_sn = qo_sn;
  r.side[1].out = k_out; r.side[1].o_sb = ko_sb; r.side[1].o_sh = ko_sh; r.side[1].o_sn = ko_sn;
  const int64_t both = a->H + a->Hk;
  r.per_tile = tile_tokens(r, both, dtype == GPA_DTYPE_F32 ? 2 : 4);
  r.tiles = (r.tokens + r.per_tile - 1) / r.per_tile;
  r.rows_magic = both == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + both - 1) / both);
  return refuse_launch(fn, launch<false>(r, dtype, vec, a->pairing == GPA_PAIRS_NEIGHBOURS, (hipStream_t)stream));
}

extern "C" size_t gpa_head_rotary_bwd_workspace_bytes(int64_t B, int64_t N, int64_t H, int64_t Hk,
                                                      int64_t D, int norm) {
  if (B <= 0 || N <= 0 || H < 0 || Hk < 0 || D <= 0 || !norm) return 0;
  const Wgs w = bwd_wgs(B * N, H, Hk, true, true), q = bwd_wgs(B * N, H, Hk, true, false),
            k = bwd_wgs(B * N, H, Hk, false, true);
  return (size_t)std::max({w.q + w.k, q.q, k.k}) * 2 * D * sizeof(float);
}

extern "C" int gpa_head_rotary_bwd(int dtype, int param_dtype, const gpa_head_rotary_args* a,
                                   const gpa_head_rotary_grads* g, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_head_rotary_bwd";
  gpa_clear_error();
  const int rc = check(fn, dtype, param_dtype, a);
  if (rc != GPA_OK) return rc;
  if (!g) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  const bool hq = g->d_q_out && a->H > 0, hk = g->d_k_out && a->Hk > 0;
  if ((g->dq_w && (!a->q_w || !hq)) || (g->dk_w && (!a->k_w || !hk)) || (g->dq_b && (!a->q_b || !hq)) ||
      (g->dk_b && (!a->k_b || !hk)) || (hq && !g->dq) || (hk && !g->dk)) {
    gpa_set_error("%s: a gradient of an output needs that of its input, and there is none of an "
                  "absent parameter", fn);
    return GPA_E_INVALID;
  }
  const bool sums = g->dq_w || g->dk_w || g->dq_b || g->dk_b;
  if (a->B == 0 || a->N == 0 || (!hq && !hk)) {
    if (!sums) return GPA_OK;
    gpa_set_error("%s: no row, so the parameters' gradients are zeros that the caller writes", fn);
    return GPA_E_INVALID;
  }
  const size_t need = sums ? gpa_head_rotary_bwd_workspace_bytes(a->B, a->N, a->H, a->Hk, a->D, a->norm) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, need);
    return GPA_E_WORKSPACE;
  }
  RotArgs r{};
  if (!cut(a, r)) {
    gpa_set_error("%s: too many sections for this head dim", fn);
    return GPA_E_UNSUPPORTED;
  }
  const int64_t H = hq ? a->H : 0, Hk = hk ? a->Hk : 0;
  const bool vec = fill(a, dtype, param_dtype,
                        {{a->norm ? a->q : nullptr, H, a->q_sb, a->q_sh, a->q_sn},
                         {a->norm ? a->k : nullptr, Hk, a->k_sb, a->k_sh, a->k_sn},
                         {g->d_q_out, H, g->dqo_sb, g->dqo_sh, g->dqo_sn}, {g->d_k_out, Hk, g->dko_sb, g->dko_sh, g->dko_sn},
                         {g->dq, H, g->dq_sb, g->dq_sh, g->dq_sn}, {g->dk, Hk, g->dk_sb, g->dk_sh, g->dk_sn}}, r);
  Side &q = r.side[0], &k = r.side[1];
  q.heads = (int32_t)H; k.heads = (int32_t)Hk;
  q.dy = g->d_q_out; q.y_sb = g->dqo_sb; q.y_sh = g->dqo_sh; q.y_sn = g->dqo_sn;
  k.dy = g->d_k_out; k.y_sb = g->dko_sb; k.y_sh = g->dko_sh; k.y_sn = g->dko_sn;
  q.out = g->dq; q.o_sb = g->dq_sb; q.o_sh = g->dq_sh; q.o_sn = g->dq_sn;
  k.out = g->dk; k.o_sb = g->dk_sb; k.o_sh = g->dk_sh; k.o_sn = g->dk_sn;
  const Wgs w = bwd_wgs(r.tokens, a->H, a->Hk, hq, hk);
  q.wgs = (int32_t)w.q; k.wgs = (int32_t)w.k;
  if (sums) {
    q.part = g->dq_w || g->dq_b ? (float*)workspace : nullptr;
    k.part = g->dk_w || g->dk_b ? (float*)workspace + w.q * 2 * a->D : nullptr;
  }
  r.per_tile = tile_tokens(r, std::max(H, Hk), 2);
  r.tiles = (r.tokens + r.per_tile - 1) / r.per_tile;
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e = launch<true>(r, dtype, vec, a->pairing == GPA_PAIRS_NEIGHBOURS, s);
  if (e == hipSuccess && sums) {
    SumArgs c{};
    c.part[0] = q.part; c.part[1] = k.part;
    c.out[0][0] = g->dq_w; c.out[0][1] = g->dq_b; c.out[1][0] = g->dk_w; c.out[1][1] = g->dk_b;
    c.wgs[0] = q.wgs; c.wgs[1] = k.wgs;
    c.D = (int32_t)a->D;
    const dim3 grid((unsigned)((a->D + 63) / 64), 2, 2), block(1024);
    if (param_dtype == GPA_DTYPE_F32) hipLaunchKernelGGL((head_rotary_sum_kernel<float>), grid, block, 0, s, c);
    else if (param_dtype == GPA_DTYPE_BF16) hipLaunchKernelGGL((head_rotary_sum_kernel<__bf16>), grid, block, 0, s, c);
    else hipLaunchKernelGGL((head_rotary_sum_kernel<_Float16>), grid, block, 0, s, c);
    e = hipGetLastError();
  }
  return refuse_launch(fn, e);
}
