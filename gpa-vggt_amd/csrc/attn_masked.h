// Shared by the masked attention's forward (attn_masked.hip) and backward
// (attn_masked_bwd.hip) kernels: rows and their key ranges, the score
// function, the tiles in LDS.
//
//   x_ij = sm_scale q_i.k_j
//   s_ij = cap tanh(x_ij / cap) - slope_h |p_i - p_j|      (both optional)
//   o_i  = sum_j softmax_j(s_ij) v_j over the keys that query i sees
//
// Rows.  The G = H / Hk query heads of a key head are rows of one problem:
// row r of problem (b, key head) is token r / G, head r % G of the group, so
// K and V are read once for the group and a block of rows spans few tokens.
//
// Masks are ranges.  A document is a run of queries [q0, q1) and one of keys
// [k0, k1); query m stands at key coordinate at = m + k1 - q1 (the last query
// at the last key).  It sees the keys [k0, hi), hi = k1, or under a causal
// mask min(k1, max(k0 + prefix, at + 1)): ONE range, and the queries that see
// a key are one range too.  So a tile is outside, inside or on the edge of a
// block's ranges, and only edge tiles compare indices.
#pragma once

#include <math.h>

#include "gpa_common.h"

namespace gpa {

constexpr int kMTile = 32;          // keys (forward, dq) or rows (dk, dv) of a tile
constexpr int kMWaves = 4;
constexpr int kMThreads = kMWaves * 64;
constexpr int kMRows = kMWaves * 32;
constexpr int64_t kMostWgs = 0xffffffff / kMThreads;
constexpr float kMLog2e = 1.4426950408889634f;
constexpr uint32_t kNoRow = 0x40000000u;   // a DMA offset outside every descriptor: zeros

// Where documents lie, and what limits a query's keys.
struct MaskArgs {
  const int32_t* q_off;   // nullable: one document, all queries
  const int32_t* k_off;   // nullable: one document, all keys
  const int32_t* lens;    // nullable: key counts of a batch (one document)
  const int32_t* prefix;  // nullable: prefix_len for every document
  int64_t qo_sb, ko_sb, prefix_sb;
  int32_t docs, prefix_len, causal;
  int32_t M, N;
};

struct DocSpan { int q0, q1, k0, k1, pre; };

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// The last of `docs` runs that begins at or before `at` (-1: none), of the
// run borders off[0 .. docs]; docs where off[docs] lies at or before it.
__device__ __forceinline__ int find_run(const int32_t* off, int docs, int at) {
  int lo = 0, hi = docs + 1;        // off[i] <= at holds for i < lo, not for i >= hi
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= at) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

// The document of batch element b's run d, or an empty one.  Whatever the
// offsets hold, the ranges stay inside the queries and the keys.
__device__ __forceinline__ DocSpan doc_span(const MaskArgs& a, int64_t b, int d) {
  DocSpan s{0, 0, 0, 0, 0};
  if (d < 0 || d >= a.docs) return s;
  s.q1 = a.M;
  s.k1 = a.N;
  if (a.q_off) {
    const int32_t* q = a.q_off + b * a.qo_sb + d;
    s.q0 = clampi(q[0], 0, a.M);
    s.q1 = clampi(q[1], s.q0, a.M);
  }
  if (a.k_off) {
    const int32_t* k = a.k_off + b * a.ko_sb + d;
    s.k0 = clampi(k[0], 0, a.N);
    s.k1 = clampi(k[1], s.k0, a.N);
  }
  if (a.lens) s.k1 = clampi(a.lens[b], 0, a.N);
  if (a.causal) s.pre = a.prefix ? clampi(a.prefix[b * a.prefix_sb + d], 0, a.N) : a.prefix_len;
  return s;
}

// Keys [lo, hi) that query m of batch element b sees, and its key coordinate.
struct RowSpan { int lo, hi, at; };
__device__ __forceinline__ RowSpan row_span(const MaskArgs& a, int64_t b, int m) {
  const int d = a.q_off ? find_run(a.q_off + b * a.qo_sb, a.docs, m) : 0;
  const DocSpan s = doc_span(a, b, d);
  RowSpan r{s.k0, s.k1, m + s.k1 - s.q1};
  if (a.causal) r.hi = clampi(s.k0 + s.pre > r.at + 1 ? s.k0 + s.pre : r.at + 1, s.k0, s.k1);
  if (m < s.q0 || m >= s.q1) r.hi = r.lo;
  return r;
}

// Queries [lo, hi) that see key j, and what m is added to for its coordinate.
struct KeySpan { int lo, hi, shift; };
__device__ __forceinline__ KeySpan key_span(const MaskArgs& a, int64_t b, int j) {
  const int d = a.k_off ? find_run(a.k_off + b * a.ko_sb, a.docs, j) : 0;
  const DocSpan s = doc_span(a, b, d);
  KeySpan k{s.q0, s.q1, s.k1 - s.q1};
  if (a.causal && j - s.k0 >= s.pre) k.lo = clampi(j - k.shift, s.q0, s.q1);
  if (j < s.k0 || j >= s.k1) k.hi = k.lo;
  return k;
}

// Scores, in log2 units.  c1 = sm_scale log2(e).  With a cap: ce = 2 log2(e)
// sm_scale / cap (the exponent of e^(2u), u = x / cap), capl = cap log2(e), and for
// |u| <= kPolyMax, a product |q.k| <= lim, the coefficients of an odd polynomial;
// half = 1 / (2 capl).
struct ScoreArgs { float c1, ce, capl, lim, half, poly[4]; };

// tanh(u) = 1 - 2 / (1 + e^(2u)): right at both ends (e^(2u) = 0 or inf), and
// off by about 2^-23 absolutely, 1e-5 of a score at a cap of 50.
__device__ __forceinline__ float cap_tanh(float s, float ce) {
  const float e = __builtin_amdgcn_exp2f(s * ce);
  return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
}

// tanh(u) / u as a polynomial in u^2, for |u| <= 0.5 off by less than 1.3e-7 of
// tanh (weighted least squares towards the smallest largest error).  Four FMA-rate
// instructions and the one that subtracts the offset, where the exponential and
// the reciprocal above (half rate each) take the time of eight: scores seldom
// come nearer to their cap, and a tile in which one does takes the other form.
constexpr float kPolyMax = 0.5f;
constexpr double kPoly[4] = {0.999997676, -0.333206552, 0.131451453, -0.043372476};
// The score of a product s over s, in log2 units, by the polynomial.
__device__ __forceinline__ float cap_poly(float s, const ScoreArgs& a) {
  const float z = s * s;
  return __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(a.poly[3], z, a.poly[2]), z, a.poly[1]), z, a.poly[0]);
}

// One tile of a tensor in LDS: 32 rows of HD 16-bit values, row-major, their
// 16-byte chunks XOR-swizzled by row so that both kinds of read are free of
// bank conflicts: fragments of one chunk of 16 consecutive rows (all 16 slots
// of 256 bytes are hit once) and ds_read_b64_tr_b16 of 4 chunks of 4 rows.
template <int HD>
__device__ __forceinline__ constexpr int tile_swz(int row) {
  if constexpr (HD == 64) return ((row >> 1 & 1) << 2) | (row >> 2 & 3);   // two rows per 256 bytes
  else return ((row & 3) << 2) | (row >> 2 & 3);
}
// Element offset of a row's 16-byte chunk.
template <int HD>
__device__ __forceinline__ constexpr int tile_at(int row, int chunk) {
  return row * HD + ((chunk ^ tile_swz<HD>(row)) << 3);
}

// Where part k of n equal parts of `tiles` begins: the same for all lanes, which the
// compiler does not see through a division.
__device__ __forceinline__ int share_of(int tiles, int k, int n) {
  return __builtin_amdgcn_readfirstlane((int)((int64_t)tiles * k / n));
}

// Item L of blocks x problems: heavy blocks first (the last rows of a causal
// document see the most keys, so a launch's tail is short), and the blocks of one
// problem on one XCD (workgroups go round the eight of them), whose L2 then holds
// the problem's tiles.
__device__ __forceinline__ void item_of(int L, int blocks, int problems, int& block, int& prob) {
  const int per = problems / 8;
  if (problems % 8 == 0) {
    prob = L % 8 + 8 * (L / 8 % per);
    block = L / 8 / per;
  } else {
    prob = L % problems;
    block = L / problems;
  }
}

// DMA of 4 / 16 bytes per lane into LDS at lds + 4 * lane / lds + 16 * lane.
__device__ __forceinline__ void m_dma4(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void*)lds, 4, voff, 0, 0, 0);
}
__device__ __forceinline__ void m_dma16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}
// Wait until at most N vector-memory instructions of this wave are in flight.
template <int N>
__device__ __forceinline__ void m_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// The same, then the workgroup's barrier.  (__syncthreads is a fence as well: the
// compiler waits for every DMA in flight before it, and the ring hides nothing.)
template <int N>
__device__ __forceinline__ void m_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A descriptor over the rows [row, row + 32) of a tensor that ends at `end`
// (rows; none: nothing is read).  Its base moves in 64 bits, so a tensor may
// be longer than a 32-bit offset reaches.
template <int HD>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint16_t* base, int64_t stride,
                                                            int row, int end) {
  int n = end - row;
  n = n > kMTile ? kMTile : n;
  const uint32_t bytes = n > 0 ? (uint32_t)(n - 1) * (uint32_t)(stride * 2) + HD * 2 : 0u;
  return make_rsrc(base + (int64_t)row * stride, bytes);
}

// Reads of a tile's operands.  A lane's offsets inside a tile are kept, and the
// tile's own place goes into the instructions' offset fields: `fresh`, once a
// tile, keeps the compiler from holding the sums of both in registers (a set of
// them for each of the ring's slots).
template <int HD>
struct TileReader {
  uint32_t row[HD / 16], tr[HD / 32][2];       // bytes
  __device__ __forceinline__ explicit TileReader(int lane) {
    const int hi = lane >> 5, l32 = lane & 31, v4 = (lane & 15) >> 2, a = lane & 3, bit4 = (lane >> 4) & 1;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) row[ks] = 2 * tile_at<HD>(l32, 2 * ks + hi);
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        tr[db][e] = 2 * (tile_at<HD>(8 * e + 4 * hi + v4, 4 * db + 2 * bit4 + (a >> 1)) + (a & 1) * 4);
  }
  __device__ __forceinline__ void fresh() {
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) asm volatile("" : "+v"(row[ks]));
#pragma unroll
    for (int db = 0; db < HD / 32; ++db) asm volatile("" : "+v"(tr[db][0]), "+v"(tr[db][1]));
  }
  typedef __attribute__((address_space(3))) const char* lds_ptr;
  static __device__ __forceinline__ lds_ptr lds(const uint16_t* t) { return (lds_ptr)t; }
  // The A operand of a product over the tile's features: lane (hi, l32) has row
  // l32, features 16 ks + 8 hi .. +7.
  __device__ __forceinline__ bf16x8 rows(const uint16_t* t, int ks) const {
    return *reinterpret_cast<__attribute__((address_space(3))) const bf16x8*>(lds(t) + row[ks]);
  }
  // The A operand of a product over the tile's rows, transposed: lane (hi, l32)
  // has feature 32 db + l32 of the rows 16 s + 8 e + 4 hi + 0 .. 3 (e = 0, 1), the
  // order in which the score MFMA's result registers hold them, so that its
  // results are the B operand as they stand.
  __device__ __forceinline__ bf16x8 turned(const uint16_t* t, int db, int s) const {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4* tr_ptr;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(lds(t) + tr[db][0] + 32 * s * HD));
    const i16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(lds(t) + tr[db][1] + 32 * s * HD));
    const bf16x4 l4 = __builtin_bit_cast(bf16x4, lo), u4 = __builtin_bit_cast(bf16x4, up);
    return bf16x8{l4[0], l4[1], l4[2], l4[3], u4[0], u4[1], u4[2], u4[3]};
  }
};

// Sixteen fp32 values of a lane as the B operand's two fragments.
template <bool F16>
__device__ __forceinline__ void pack_frags(const float (&p)[16], bf16x8 (&out)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const bf16x2 v = pack2<F16>(p[8 * s + e], p[8 * s + e + 1]);
      out[s][e] = v[0];
      out[s][e + 1] = v[1];
    }
}

// What rounding took from the first fragment's values, as one more.
template <bool F16>
__device__ __forceinline__ bf16x8 rest_frag(const float (&p)[16], const bf16x8& x) {
  bf16x8 out;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const bf16x2 v = pack2<F16>(p[e] - half_to_f32<F16>(x[e]), p[e + 1] - half_to_f32<F16>(x[e + 1]));
    out[e] = v[0];
    out[e + 1] = v[1];
  }
  return out;
}

// sum + the sum of a fragment's values, as the matrix instructions take them.
template <bool F16>
__device__ __forceinline__ float sum_frag(const bf16x8& x, float sum) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  const u32x4 y = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = y[i];                   // a bit_cast of the element itself reads another one
    if constexpr (F16)
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{1, 1}, sum, false);
    else
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b16x2, w), b16x2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
  }
  return sum;
}

// acc += A^T . P over a tile's rows where a row that a lane does not see may
// hold infinities or NaN: 0 times them is NaN, so such values are taken out of
// the product and the rows that do see them get them back by their sign: an
// indicator product over the seen rows tells which (both signs: NaN).
template <int HD, bool F16>
__device__ __forceinline__ f32x16 careful_mfma(const TileReader<HD>& rd, const uint16_t* t, int db,
                                               const bf16x8 (&p)[2], const bf16x8 (&seen)[2],
                                               f32x16 acc) {
  const uint16_t expo = F16 ? 0x7c00 : 0x7f80, one = F16 ? 0x3c00 : 0x3f80;
  f32x16 up{}, down{};
  __builtin_amdgcn_sched_barrier(0);           // one feature block at a time: registers, not speed
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 x = __builtin_bit_cast(u16x8, rd.turned(t, db, s)), xp, xn;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t w = x[e];
      const bool odd = (w & expo) == expo, nan = odd && (w & (0x7fff ^ expo)) != 0;
      xp[e] = odd && (nan || !(w & 0x8000)) ? one : 0;
      xn[e] = odd && (nan || (w & 0x8000)) ? one : 0;
      x[e] = odd ? 0 : w;
    }
    acc = mfma32x32x16_t<F16>(__builtin_bit_cast(bf16x8, x), p[s], acc);
    up = mfma32x32x16_t<F16>(__builtin_bit_cast(bf16x8, xp), seen[s], up);
    down = mfma32x32x16_t<F16>(__builtin_bit_cast(bf16x8, xn), seen[s], down);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    if (up[r] > 0.f) acc[r] += INFINITY;
    if (down[r] > 0.f) acc[r] -= INFINITY;
  }
  return acc;
}

// Whether the rows of a [n0, n1, n2, D] tensor of 16-bit values are 16-byte aligned;
// a dimension of one has any stride.
inline bool rows_aligned(const void* p, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2,
                         int64_t s2) {
  return (uintptr_t)p % 16 == 0 && (n0 < 2 || s0 % 8 == 0) && (n1 < 2 || s1 % 8 == 0) &&
         (n2 < 2 || s2 % 8 == 0);
}

// Shared by the entry points: the checks of their arguments (has_o: an output
// is written to a->o), and the kernels' form of them.
int masked_check(const char* fn, int dtype, const gpa_attn_masked_args* a, bool has_o);
// The arguments with a plain stride for every dimension of one.
gpa_attn_masked_args masked_plain(const gpa_attn_masked_args* a);
void masked_fill(const gpa_attn_masked_args* a, MaskArgs* m, ScoreArgs* s);

}  // namespace gpa
