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
// in a fixed order.  16,384 tokens of 32 + 8 heads of 128 in bf16: forward 74 us
// (4.5 TB/s), backward 117 (4.3) and 6 for the sums; a copy runs at 4.9.
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
// Workgroups: what 256 CUs hold at once, each walking its tiles with the next rows' loads in flight
// (four to a CU forward; as many as tiles took 77 us for 71 at 16,384 tokens of 32 + 8 heads of
// 128, and 38 for 28 at 10,992 of 16 + 16 of 64).
constexpr int64_t kFwdWgs = 1024;
constexpr int64_t kBwdWgs = 1024;        // three to a CU, 768, with a bias's sums or in fp32 (10,992 tokens of 16 + 16 heads of 64:
                                         // 36.4 us on 1,024, 34.6; 20,000: 56, 51; fp32 12.6, 11.2)

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
  int32_t heads, wgs, per_tile;   // wgs: the backward's workgroups of this side; per_tile: a tile's tokens
  int64_t tiles;
  uint32_t magic;         // 2^32 / heads, rounded up
};

struct RotArgs {
  Side side[2];
  const void* pos;
  int64_t pos_sb, pos_sn;
  const double* freqs;
  const int32_t* axes;
  int64_t N, tokens;
  uint32_t rows_magic;    // 2^32 / heads of a row's tensors, rounded up (one head: not used)
  uint32_t n_magic;       // 2^32 / N, rounded up (N == 1: not used)
  int32_t D, pairs, count, pos_kind, chunks, lanes, norm, pf32, bias, par16;   // par16: parameters are 16-byte aligned
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

// A chunk's sixteen values as they lie in memory, V of them at a time: 8 whole 16-byte
// pieces, 2 a pair of values, 1 each by itself.
template <typename T, int V, bool INTER>
struct Raw {
  typedef typename Piece<T>::type P16;
  static constexpr int PER = 16 / sizeof(T), HALF = 8 / PER;   // values of a piece; pieces of eight values
  P16 v[2 * HALF];
  __device__ __forceinline__ void put(int i, T x) { v[i / PER][i % PER] = x; }
  __device__ __forceinline__ T at(int i) const { return v[i / PER][i % PER]; }
  __device__ __forceinline__ void load(const T* row, const Chunk& c) {
    if constexpr (V == 8) {
      const P16* a = reinterpret_cast<const P16*>(row + c.o0);
      const P16* b = INTER ? a + HALF : reinterpret_cast<const P16*>(row + c.o1);
#pragma unroll
      for (int i = 0; i < HALF; ++i) v[i] = c.n ? a[i] : P16{};
#pragma unroll
      for (int i = 0; i < HALF; ++i) v[HALF + i] = c.n ? b[i] : P16{};
    } else {
      typedef T Some __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 16; i += V) {        // value i of the chunk, in its order in registers
        const bool in = (INTER ? i / 2 : i & 7) < c.n;
        const T* from = row + (INTER || i < 8 ? c.o0 + i : c.o1 + i - 8);
        if constexpr (V == 2) {
          const Some x = in ? *reinterpret_cast<const Some*>(from) : Some{};
          put(i, x[0]);
          put(i + 1, x[1]);
        } else {
          put(i, in ? *from : (T)0.f);
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&a)[8], float (&b)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = (float)at(INTER ? 2 * i : i);
      b[i] = (float)at(INTER ? 2 * i + 1 : 8 + i);
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
    if constexpr (V == 8) {
      if (c.n == 0) return;
      P16* a = reinterpret_cast<P16*>(row + c.o0);
      P16* b = INTER ? a + HALF : reinterpret_cast<P16*>(row + c.o1);
#pragma unroll
      for (int i = 0; i < HALF; ++i) a[i] = v[i];
#pragma unroll
      for (int i = 0; i < HALF; ++i) b[i] = v[HALF + i];
    } else {
      typedef T Some __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 16; i += V) {
        if ((INTER ? i / 2 : i & 7) >= c.n) continue;
        T* to = row + (INTER || i < 8 ? c.o0 + i : c.o1 + i - 8);
        if constexpr (V == 2) *reinterpret_cast<Some*>(to) = Some{at(i), at(i + 1)};
        else *to = at(i);
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

// Where a tile's tokens lie: its first one's batch element and number.
struct Place { uint32_t b, n; };
__device__ __forceinline__ Place place_of(const RotArgs& a, uint32_t first) {
  const uint32_t b = first / (uint32_t)a.N;
  return {b, first - b * (uint32_t)a.N};
}
// Token k (below kMaxTokens) of the tile.  (Sequences of kMaxTokens or more: it
// lies in the first one's or the next.)
__device__ __forceinline__ Place token_at(const RotArgs& a, Place p, uint32_t k) {
  const uint32_t n = p.n + k, N = (uint32_t)a.N;
  const uint32_t d = N >= kMaxTokens ? (n >= N ? 1 : 0) : N == 1 ? n : __umulhi(n, a.n_magic);
  return {p.b + d, n - d * N};
}

// A thread's pair of features, whose angles it forms for every tile.
struct Turner {
  int pair, slot, slots, to;   // pair: -1 none; the tokens slot, slot + slots, ...
  double speed;                // turns a unit of position
  int64_t axis;
  __device__ __forceinline__ explicit Turner(const RotArgs& a) {
    const int width = a.lanes * 8, c = threadIdx.x % width;
    slot = threadIdx.x / width;
    slots = kThreads / width;
    pair = -1;
    to = 0;
    speed = 0.0;
    axis = 0;
    if (c >= a.chunks * 8) return;
    const Chunk ch = a.chunk[c >> 3];
    if (ch.p0 < 0 || (c & 7) >= ch.n) return;
    pair = ch.p0 + (c & 7);
    to = (c >> 3) * 16 + (c & 7);
    speed = a.freqs[pair] * 0.15915494309189533577;
    const int ax = a.axes[pair];
    axis = ax < 0 ? 0 : ax >= a.count ? a.count - 1 : ax;
  }
  __device__ __forceinline__ void turn(const RotArgs& a, Place first, int live, float* cs) const {
    if (pair < 0) return;
    for (int k = slot; k < live; k += slots) {
      const Place t = token_at(a, first, k);
      const int64_t at = t.b * a.pos_sb + t.n * a.pos_sn + axis;
      const double p = a.pos_kind == 0 ? (double)static_cast<const int32_t*>(a.pos)[at]
                       : a.pos_kind == 1 ? (double)static_cast<const int64_t*>(a.pos)[at]
                                         : (double)static_cast<const float*>(a.pos)[at];
      const double turns = p * speed;
      float s, c;
      sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &c);
      cs[k * a.chunks * 16 + to] = c;
      cs[k * a.chunks * 16 + to + 8] = s;
    }
  }
};

// A parameter in a lane's order: its sixteen values, `none` where there are none.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void take_param(const RotArgs& a, const void* p, const Chunk& c, float none, float (&x)[8], float (&y)[8]) {
  const bool wide = sizeof(T) == 4 || a.pf32;
  if (V == 8 && a.par16 && p) {
    if (wide) {
      Raw<float, 8, INTER> r;
      r.load(static_cast<const float*>(p), c);
      r.get(x, y);
    } else {
      Raw<T, 8, INTER> r;
      r.load(static_cast<const T*>(p), c);
      r.get(x, y);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = y[i] = none;
    if (!p || i >= c.n) continue;
    const int u = INTER ? c.o0 + 2 * i : c.o0 + i, v = INTER ? c.o0 + 2 * i + 1 : c.o1 + i;
    x[i] = wide ? static_cast<const float*>(p)[u] : (float)static_cast<const T*>(p)[u];
    y[i] = wide ? static_cast<const float*>(p)[v] : (float)static_cast<const T*>(p)[v];
  }
}

// Both moments of a row; x, y centred under LayerNorm.  Returns 1 / sigma.
template <bool WHOLE>
__device__ __forceinline__ float moments(const RotArgs& a, const Chunk& c, float (&x)[8], float (&y)[8]) {
  if (a.norm == kLayer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] + y[i];
    const float mean = row_sum(s, a.lanes) * a.inv_d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {              // values that are not there stay 0
      const bool in = WHOLE ? c.n != 0 : i < c.n;
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

// Rows of a workgroup: those of its tiles, `all` heads of each token, U * l.rows at a time; the next
// ones' loads are issued before this one's arithmetic, a tile's first before its angles.
struct Walk {
  int64_t tile;
  int r0, rows;           // the next rows' first, of `rows` of the tile
  uint32_t first;         // the tile's first token
  int live;
  __device__ __forceinline__ void open(const RotArgs& a, const Side& s, int64_t at, int all) {
    tile = at;
    r0 = 0;
    first = (uint32_t)(at * s.per_tile);
    live = at < s.tiles ? (int)(a.tokens - first < s.per_tile ? a.tokens - first : s.per_tile) : 0;
    rows = live * all;
  }
  // Whether the next rows are another tile's.
  __device__ __forceinline__ bool on(const RotArgs& a, const Side& s, int step, int64_t stride, int all) {
    r0 += step;
    if (r0 < rows) return false;
    open(a, s, tile + stride, all);
    return true;
  }
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(kThreads, 4) void head_rotary_kernel(RotArgs a) {
  constexpr int U = sizeof(T) == 4 ? 1 : 2;    // rows a lane has in flight, twice
  __shared__ __attribute__((aligned(16))) float cs[kCsFloats];    // [token][chunk][cos 8, sin 8]
  __shared__ __attribute__((aligned(16))) float par[2][2][kMaxChunks * 16];
  const Lane l = lane_of(a);
  const int at = threadIdx.x % a.lanes, both = a.side[0].heads + a.side[1].heads, cat = at < a.chunks ? at : 0;
  struct Some {
    Raw<T, V, INTER> raw[U];
    T* out[U];
    int k[U];
    bool which[U], fine[U];
  };
  // (Selected, not indexed: a lane's own index would be a load from the arguments.)
  auto fetch = [&](const Walk& w, Some& m) __attribute__((always_inline)) {
    const Place first = place_of(a, w.first);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = w.r0 + l.row + u * l.rows;
      m.fine[u] = r < w.rows;
      const int rc = m.fine[u] ? r : 0;
      const int k = both == 1 ? rc : (int)__umulhi((uint32_t)rc, a.rows_magic), hh = rc - k * both;
      const bool which = hh >= a.side[0].heads;
      const int h = which ? hh - a.side[0].heads : hh;
      const Side &s0 = a.side[0], &s1 = a.side[1];
      const Place t = token_at(a, first, k);
      m.k[u] = k;
      m.which[u] = which;
      m.out[u] = static_cast<T*>(which ? s1.out : s0.out) + t.b * (which ? s1.o_sb : s0.o_sb) +
                 h * (which ? s1.o_sh : s0.o_sh) + t.n * (which ? s1.o_sn : s0.o_sn);
      Chunk c = l.c;
      if (!m.fine[u]) c.n = 0;
      m.raw[u].load(static_cast<const T*>(which ? s1.x : s0.x) + t.b * (which ? s1.x_sb : s0.x_sb) +
                        h * (which ? s1.x_sh : s0.x_sh) + t.n * (which ? s1.x_sn : s0.x_sn), c);
    }
  };
  Walk w;
  w.open(a, a.side[0], blockIdx.x, both);     // (both sides together, in the first one's tiles)
  Some now;
  fetch(w, now);
  if (a.norm && l.row < 2) {                   // a row of lanes for each side (a wave has two at least)
    const Side& s = a.side[l.row];
    float x[8], y[8];
    for (int k = 0; k < 2; ++k) {
      take_param<T, V, INTER>(a, k ? s.b : s.w, l.c, k ? 0.f : 1.f, x, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        par[l.row][k][at * 16 + i] = x[i];
        par[l.row][k][at * 16 + 8 + i] = y[i];
      }
    }
  }
  const Turner turner(a);
  bool fresh = true;
  while (w.live > 0) {
    if (fresh) {
      __syncthreads();                         // the tile before is done with its angles
      turner.turn(a, place_of(a, w.first), w.live, cs);
      __syncthreads();
    }
    Some cur = now;
    fresh = w.on(a, a.side[0], U * l.rows, gridDim.x, both);
    if (w.live > 0) fetch(w, now);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8], y[8];
      cur.raw[u].get(x, y);
      if (a.norm) {
        const float inv = moments<V == 8>(a, l.c, x, y);
        const float* pw = par[cur.which[u]][0] + at * 16;
        float p[8], q[8];
        take8(pw, p);
        take8(pw + 8, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * inv * p[i];
          y[i] = y[i] * inv * q[i];
        }
        if (a.side[0].b || a.side[1].b) {      // (of one alone: the other adds zeros)
          take8(pw + kMaxChunks * 16, p);
          take8(pw + kMaxChunks * 16 + 8, q);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] += p[i];
            y[i] += q[i];
          }
        }
      }
      if (l.c.p0 >= 0) {
        float c[8], s[8];
        take8(cs + (cur.k[u] * a.chunks + cat) * 16, c);
        take8(cs + (cur.k[u] * a.chunks + cat) * 16 + 8, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = x[i];
          x[i] = __builtin_fmaf(v, c[i], -(y[i] * s[i]));
          y[i] = __builtin_fmaf(y[i], c[i], v * s[i]);
        }
      }
      if (!cur.fine[u]) continue;
      cur.raw[u].set(x, y);
      cur.raw[u].store(cur.out[u], l.c);
    }
  }
}

// BIAS: a bias's gradient is wanted (its sums take 16 registers, with which a CU holds three
// workgroups instead of four).
template <typename T, int V, bool INTER, bool BIAS>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && V == 8 && !BIAS ? 4 : 3) void head_rotary_bwd_kernel(RotArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[kCsFloats];
  const Lane l = lane_of(a);
  const int at = threadIdx.x % a.lanes, cat = at < a.chunks ? at : 0;
  const int which = (int)blockIdx.x >= a.side[0].wgs;
  const Side& s = a.side[which];
  const int wg = which ? (int)blockIdx.x - a.side[0].wgs : (int)blockIdx.x;
  struct Some {
    Raw<T, V, INTER> x, dy;
    T* out;
    int k;
    bool fine;
  };
  auto fetch = [&](const Walk& w, Some& m) __attribute__((always_inline)) {
    const Place first = place_of(a, w.first);
    const int r = w.r0 + l.row;
    m.fine = r < w.rows;
    const int rc = m.fine ? r : 0;
    m.k = s.heads == 1 ? rc : (int)__umulhi((uint32_t)rc, s.magic);
    const int h = rc - m.k * s.heads;
    const Place t = token_at(a, first, m.k);
    Chunk c = l.c;
    if (!m.fine) c.n = 0;
    m.dy.load(static_cast<const T*>(s.dy) + t.b * s.y_sb + h * s.y_sh + t.n * s.y_sn, c);
    if (a.norm) m.x.load(static_cast<const T*>(s.x) + t.b * s.x_sb + h * s.x_sh + t.n * s.x_sn, c);
    m.out = static_cast<T*>(s.out) + t.b * s.o_sb + h * s.o_sh + t.n * s.o_sn;
  };
  Walk w;
  w.open(a, s, wg, s.heads);
  Some now;
  fetch(w, now);
  const Turner turner(a);
  float wa[8], wb[8], dwa[8], dwb[8], dba[8], dbb[8];
  take_param<T, V, INTER>(a, s.w, l.c, 1.f, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) dwa[i] = dwb[i] = dba[i] = dbb[i] = 0.f;
  bool fresh = true;
  while (w.live > 0) {
    if (fresh) {
      __syncthreads();
      turner.turn(a, place_of(a, w.first), w.live, cs);
      __syncthreads();
    }
    Some cur = now;
    fresh = w.on(a, s, l.rows, s.wgs, s.heads);
    if (w.live > 0) fetch(w, now);
    float ga[8], gb[8];
    cur.dy.get(ga, gb);
    if (l.c.p0 >= 0) {                         // turned back
      float c[8], sn[8];
      take8(cs + (cur.k * a.chunks + cat) * 16, c);
      take8(cs + (cur.k * a.chunks + cat) * 16 + 8, sn);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = ga[i];
        ga[i] = __builtin_fmaf(v, c[i], gb[i] * sn[i]);
        gb[i] = __builtin_fmaf(gb[i], c[i], -(v * sn[i]));
      }
    }
    if (a.norm) {
      float x[8], y[8];
      cur.x.get(x, y);
      const float inv = moments<V == 8>(a, l.c, x, y);
      float s1 = 0.f, s0 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= inv;
        y[i] *= inv;
        if (cur.fine) {
          dwa[i] = __builtin_fmaf(ga[i], x[i], dwa[i]);
          dwb[i] = __builtin_fmaf(gb[i], y[i], dwb[i]);
          if (BIAS) {
            dba[i] += ga[i];
            dbb[i] += gb[i];
          }
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
    if (!cur.fine) continue;
    cur.dy.set(ga, gb);
    cur.dy.store(cur.out, l.c);
  }
  if (!s.part) return;

  // The rows' sums: over a wave's rows, then over the four waves in LDS.
  float* red = cs;                             // [wave][lane of a row][4][8], at most 4 * 32 * 32 floats
  float* sums[4] = {dwa, dwb, dba, dbb};
  auto each = [&](auto op) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < (BIAS ? 4 : 2); ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[k][i] = op(sums[k][i]);
  };
  // (By DPP and swaps: as shuffles through LDS these sums cost a pass 7 to 10 us.)
  if (a.lanes <= 8) each([](float v) { return dpp_add<0x128>(v); });     // the lane eight on in a row of sixteen
  if (a.lanes <= 4) each([](float v) { return dpp_add<0x124>(v); });
  if (a.lanes <= 2) each([](float v) { return dpp_add<0x122>(v); });
  if (a.lanes <= 1) each([](float v) { return dpp_add<0x121>(v); });
  if (a.lanes <= 16)
    each([](float v) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    });
  each([](float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  });
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
#pragma unroll 16
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

uint32_t magic_of(int64_t n) { return n < 2 ? 0 : (uint32_t)((((uint64_t)1 << 32) + n - 1) / n); }

// Fills everything but the outputs; returns how many values can be loaded and stored together (8, 2, 1).
int fill(const gpa_head_rotary_args* a, int dtype, int pdtype, std::initializer_list<Rows> all, RotArgs& r) {
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
  r.par16 = ((uintptr_t)a->q_w | (uintptr_t)a->k_w | (uintptr_t)a->q_b | (uintptr_t)a->k_b) % 16 == 0;
  r.eps = a->eps; r.inv_d = 1.0f / (float)a->D;
  r.n_magic = magic_of(a->N);
  q.magic = magic_of(a->H); k.magic = magic_of(a->Hk);
  bool vec = true, two = true;
  const bool next = a->pairing == GPA_PAIRS_NEIGHBOURS;
  for (int i = 0; i < r.chunks; ++i) {
    const Chunk& c = r.chunk[i];
    vec = vec && c.n == 8 && c.o0 % 8 == 0 && (next || c.o1 % 8 == 0);
    two = two && (next || (c.n % 2 == 0 && c.o0 % 2 == 0 && c.o1 % 2 == 0));
  }
  for (const Rows& x : all) {
    if (!x.p || x.heads == 0) continue;
    const int64_t some = st(a->B, x.sb) | st(x.heads, x.sh) | st(a->N, x.sn);   // divisible by a power of two where all are
    vec = vec && (uintptr_t)x.p % 16 == 0 && some % per16 == 0;
    two = two && (uintptr_t)x.p % (2 * esize) == 0 && some % 2 == 0;
  }
  return vec ? 8 : two ? 2 : 1;
}

// Tokens of a workgroup's tile.  Each has `heads` rows, `step` of them go at a time: of what the
// angles' LDS holds and `wgs` workgroups leave to each, the number that leaves the fewest lanes idle
// (5,476 tokens of 16 heads of 64 on 2,048 workgroups, 32 rows each where 128 go at a time: 15 us;
// on 685, 128 each: 9.5).  Few tokens are spread over the chip.
void tile(const RotArgs& r, Side& s, int64_t heads, int64_t step, int64_t wgs) {
  wgs = std::max<int64_t>(wgs, 1);
  const int64_t most = std::min<int64_t>(kMaxTokens, kCsFloats / (16 * std::max(r.chunks, 1)));
  const int64_t fill = std::min<int64_t>((step + heads - 1) / std::max<int64_t>(heads, 1), std::max<int64_t>(r.tokens / 256, 1));
  const int64_t top = std::min(most, std::max((r.tokens + wgs - 1) / wgs, fill));
  int64_t best = 1;
  double least = 1e30;
  for (int64_t n = 1; n <= top; ++n) {         // rounds a token; more tokens share a tile's ends
    const double cost = (double)((n * heads + step - 1) / step) / n * (1.0 + 0.5 / n);
    if (cost <= least) {
      least = cost;
      best = n;
    }
  }
  s.per_tile = (int32_t)best;
  s.tiles = (r.tokens + best - 1) / best;
}

template <typename T, int V, bool BWD>
hipError_t go(const RotArgs& r, bool inter, hipStream_t s) {
  const dim3 grid((unsigned)(BWD ? r.side[0].wgs + r.side[1].wgs : std::min(r.side[0].tiles, kFwdWgs))), block(kThreads);
  if constexpr (BWD) {
    if (inter && r.bias) hipLaunchKernelGGL((head_rotary_bwd_kernel<T, V, true, true>), grid, block, 0, s, r);
    else if (inter) hipLaunchKernelGGL((head_rotary_bwd_kernel<T, V, true, false>), grid, block, 0, s, r);
    else if (r.bias) hipLaunchKernelGGL((head_rotary_bwd_kernel<T, V, false, true>), grid, block, 0, s, r);
    else hipLaunchKernelGGL((head_rotary_bwd_kernel<T, V, false, false>), grid, block, 0, s, r);
  } else {
    if (inter) hipLaunchKernelGGL((head_rotary_kernel<T, V, true>), grid, block, 0, s, r);
    else hipLaunchKernelGGL((head_rotary_kernel<T, V, false>), grid, block, 0, s, r);
  }
  return hipGetLastError();
}
template <bool BWD>
hipError_t launch(const RotArgs& r, int dtype, int some, bool inter, hipStream_t s) {
  auto of = [&](auto type) {
    typedef decltype(type) T;
    return some == 8 ? go<T, 8, BWD>(r, inter, s) : some == 2 ? go<T, 2, BWD>(r, inter, s) : go<T, 1, BWD>(r, inter, s);
  };
  return dtype == GPA_DTYPE_F32 ? of(0.f) : dtype == GPA_DTYPE_BF16 ? of((__bf16)0.f) : of((_Float16)0.f);
}

int refuse_launch(const char* fn, hipError_t e) {
  if (e == hipSuccess) return GPA_OK;
  gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
  return GPA_E_LAUNCH;
}

// Workgroups of the backward's two sides, by their share of the heads; none has more than tiles.
struct Wgs { int64_t q, k; };
Wgs bwd_wgs(int64_t tokens, int64_t H, int64_t Hk, bool q, bool k, int64_t total = kBwdWgs) {
  if (tokens <= 0) return {0, 0};
  const int64_t h = q ? H : 0, hk = k ? Hk : 0, all = std::max<int64_t>(h + hk, 1);
  auto share = [&](int64_t n) {
    return n == 0 ? 0 : std::max<int64_t>(1, std::min(tokens, (total * n + all - 1) / all));
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
  const int some = fill(a, dtype, param_dtype,
                        {{a->q, a->H, a->q_sb, a->q_sh, a->q_sn}, {a->k, a->Hk, a->k_sb, a->k_sh, a->k_sn},
                         {q_out, a->H, qo_sb, qo_sh, qo_sn}, {k_out, a->Hk, ko_sb, ko_sh, ko_sn}}, r);
  r.side[0].out = q_out; r.side[0].o_sb = qo_sb; r.side[0].o_sh = qo_sh; r.side[0].o_sn = qo_sn;
  r.side[1].out = k_out; r.side[1].o_sb = ko_sb; r.side[1].o_sh = ko_sh; r.side[1].o_sn = ko_sn;
  const int64_t both = a->H + a->Hk;
  tile(r, r.side[0], both, (dtype == GPA_DTYPE_F32 ? 1 : 2) * (kThreads / r.lanes), kFwdWgs);
  r.rows_magic = magic_of(both);
  return refuse_launch(fn, launch<false>(r, dtype, some, a->pairing == GPA_PAIRS_NEIGHBOURS, (hipStream_t)stream));
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
  const int some = fill(a, dtype, param_dtype,
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
  r.bias = g->dq_b || g->dk_b;
  const Wgs w = bwd_wgs(r.tokens, a->H, a->Hk, hq, hk, r.bias || dtype == GPA_DTYPE_F32 ? kBwdWgs * 3 / 4 : kBwdWgs);
  q.wgs = (int32_t)w.q; k.wgs = (int32_t)w.k;
  if (sums) {
    q.part = g->dq_w || g->dq_b ? (float*)workspace : nullptr;
    k.part = g->dk_w || g->dk_b ? (float*)workspace + w.q * 2 * a->D : nullptr;
  }
  tile(r, q, H, kThreads / r.lanes, w.q);
  tile(r, k, Hk, kThreads / r.lanes, w.k);
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e = launch<true>(r, dtype, some, a->pairing == GPA_PAIRS_NEIGHBOURS, s);
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
