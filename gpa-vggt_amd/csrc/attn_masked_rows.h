// The rows of a wave in the attention's forward kernels: their queries, softmax state
// and outputs (attn_masked.hip has the method and what it measured).
#pragma once
#include "attn_masked.h"

namespace gpa {

struct Deal;

namespace {

template <bool F16> constexpr float kUp = F16 ? 15.0f : 64.0f;
// Outputs up to here, in 2^9 parts at once, add up to a finite sum.  Weights of 2^-30
// keep those of 2^30 keys finite whatever the values are.
constexpr float kBig = 0x1p100f, kDown = -30.0f;

// One set of rows over one set of keys.
struct FwdSet {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  int32_t N;              // keys
  int32_t R;              // rows of a problem
  int32_t blocks, problems, splits, z0;   // row blocks, problems, splits and the first split's number
  int32_t folded;         // the rows of all sequences over one sequence of keys, all seen
};

template <int HD> constexpr int kPerCu = HD == 64 ? 3 : 2;   // workgroups to a CU

struct FwdArgs {
  const uint16_t* q;
  uint16_t* o;
  uint16_t* rest;         // what rounding took from o (nullable), laid out as it
  float* lse;             // nullable
  int64_t q_sb, q_sh, q_sm, o_sb, o_sh, o_sm, lse_sb, lse_sh;
  const float* slopes;
  int64_t slopes_sb;
  float* part;            // partial outputs [splits][rows][HD]; null: none
  float* stat;            // their (offset, sum) [splits][rows][2]
  Deal* deal;             // null: splits.  Otherwise parts are [part][key head][128 rows]
  int64_t rows;           // B * Hk * M * G
  int32_t B, Hk, G, splits;
  MaskArgs mask;
  ScoreArgs score;
  FwdSet set[2];          // the own keys; the shared prefix (no blocks: none)
};

// A lane's row of a set's problem, and the ranges of a wave's 32 rows.
struct Row {
  bool live;
  int b, h, kvh, tok;
  int lo, hi, at;         // keys [lo, hi) are seen; the row's key coordinate
  int w_lo, w_hi;         // keys that some row of the wave sees
  int a_lo, a_hi;         // keys that every row sees
};

__device__ __forceinline__ Row locate(const FwdArgs& p, const FwdSet& S, int prob, int r) {
  Row x;
  x.live = r < S.R;
  const int rc = x.live ? r : S.R - 1;
  const int per = p.mask.M * p.G;
  x.kvh = S.folded ? prob : prob % p.Hk;
  x.b = S.folded ? rc / per : prob / p.Hk;
  const int rr = S.folded ? rc % per : rc;
  x.tok = rr / p.G;
  x.h = x.kvh * p.G + rr % p.G;
  const RowSpan s = row_span(p.mask, x.b, x.tok);
  x.lo = S.folded ? 0 : s.lo;
  x.hi = S.folded ? S.N : s.hi;
  x.at = S.folded ? s.at + S.N : s.at;
  const bool any = x.live && x.hi > x.lo;
  x.w_lo = any ? x.lo : 0x7fffffff;
  x.w_hi = any ? x.hi : 0;
  x.a_lo = x.live ? x.lo : 0;
  x.a_hi = !x.live ? 0x7fffffff : any ? x.hi : 0;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    x.w_lo = min(x.w_lo, __shfl_xor(x.w_lo, i));
    x.w_hi = max(x.w_hi, __shfl_xor(x.w_hi, i));
    x.a_lo = max(x.a_lo, __shfl_xor(x.a_lo, i));
    x.a_hi = min(x.a_hi, __shfl_xor(x.a_hi, i));
  }
  x.w_lo = __builtin_amdgcn_readfirstlane(x.w_lo);
  x.w_hi = __builtin_amdgcn_readfirstlane(x.w_hi);
  x.a_lo = __builtin_amdgcn_readfirstlane(x.a_lo);
  x.a_hi = __builtin_amdgcn_readfirstlane(x.a_hi);
  return x;
}

// What rounding took from four values, rounded itself; none of a value that is not finite.
template <bool F16>
__device__ __forceinline__ u32x2 rest_of(f32x4 x, bf16x2 lo, bf16x2 hi) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] -= half_to_f32<F16>(e < 2 ? lo[e] : hi[e - 2]);
    x[e] = fabsf(x[e]) < INFINITY ? x[e] : 0.f;
  }
  const bf16x2 a = pack2<F16>(x[0], x[1]), b = pack2<F16>(x[2], x[3]);
  return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// Where a row's unnormalised outputs, offset and sum go (null: to no partial).
struct Part {
  float* o;
  float2* stat;
};
template <int HD>
__device__ __forceinline__ Part part_at(const FwdArgs& p, int64_t i) {
  return {p.part + i * HD, reinterpret_cast<float2*>(p.stat) + i};
}
// Split z of a set, in which a row's number is that of (sequence, key head, token, head).
template <int HD>
__device__ __forceinline__ Part split_part(const FwdArgs& p, const FwdSet& S, const Row& x, int z) {
  if (!p.part) return {};
  const int64_t row = (((int64_t)x.b * p.Hk + x.kvh) * p.mask.M + x.tok) * p.G + (x.h - x.kvh * p.G);
  return part_at<HD>(p, (int64_t)(S.z0 + z) * p.rows + row);
}

// A wave's 32 rows: their queries, softmax state and outputs.
template <int HD, bool F16, bool CAP, bool SLOPE>
struct Rows {
  static constexpr int KS = HD / 16, DB = HD / 32;
  const ScoreArgs& sc;
  TileReader<HD> rd;
  const int hi;
  int lo, end, at;
  float slope, lift;       // lift: what a key of distance 1 gains, 0 but for slopes below zero
  bf16x8 qf[KS];
  f32x16 o[DB];
  float m, l, n;           // offset; sums of the weights, and of the rounded ones

  __device__ __forceinline__ Rows(const FwdArgs& p, const Row& x, int lane)
      : sc(p.score), rd(lane), hi(lane >> 5), lo(x.lo), end(x.hi), at(x.at), slope(0.f), lift(0.f) {
    if constexpr (SLOPE) {
      slope = p.slopes[x.b * p.slopes_sb + x.h] * kMLog2e;
      lift = fmaxf(-slope, 0.f);
    }
    const uint16_t* Q = p.q + x.b * p.q_sb + x.h * p.q_sh + x.tok * p.q_sm;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(Q + 16 * ks + 8 * hi);
  }
  __device__ __forceinline__ void restart() {
    m = -1.0e30f;                              // finite: -inf - m is -inf
    l = n = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  }
  // The products of a tile's 32 keys (registers) and this lane's query.
  __device__ __forceinline__ f32x16 products(const uint16_t* k) const {
    f32x16 s{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma32x32x16_t<F16>(rd.rows(k, ks), qf[ks], s);
    return s;
  }
  // Scores in log2 units, less `off`.  (AHEAD: the distances are formed anew, so that
  // the two uses in a tile share no values, which would live across a branch.)
  template <bool AHEAD, bool DIST = SLOPE>
  __device__ __forceinline__ void scores(const f32x16& s, int n0, bool poly, float off, float (&x)[16]) const {
    if (!CAP) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(s[i], sc.c1, -off);
    } else if (poly) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(s[i], cap_poly(s[i], sc), -off);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(cap_tanh(s[i], sc.ce), sc.capl, -off);
    }
    if constexpr (DIST) {
      int own = at;
      if constexpr (AHEAD) asm volatile("" : "+v"(own));
      const float dist = (float)(own - n0 - 4 * hi);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(-slope, fabsf(dist - (float)mfma_row(i, 0)), x[i]);
    }
  }
  // `none` where the row does not see the key.
  __device__ __forceinline__ void masked(float (&x)[16], int n0, float none) const {
    const int from = lo - n0 - 4 * hi, to = end - n0 - 4 * hi;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (mfma_row(i, 0) < from || mfma_row(i, 0) >= to) x[i] = none;
  }
  // Before a tile's weights: where its largest |product| (and distance) does not tell that
  // all scores lie below the offset's reach, the offset follows the row's maximum, and
  // the sum and the output with it (two branches, the second with nothing but the
  // scaling: as one, the outputs had other registers after it, and every tile that
  // took the other way copied them, 32 moves).  Whether the polynomial serves all
  // products.
  // `up`: how far scores may lie above the offset (below zero: have to lie below it).
  __device__ __forceinline__ bool settle(const f32x16& s, int n0, bool edge, float up = kUp<F16>) {
    float a = fmaxf(fabsf(s[0]), fabsf(s[1]));
#pragma unroll
    for (int i = 2; i < 16; i += 2) a = fmaxf(fmaxf(a, fabsf(s[i])), fabsf(s[i + 1]));
    const bool poly = CAP && __builtin_amdgcn_ballot_w64(!(a <= sc.lim)) == 0;
    float m_new = m, bound = a * sc.c1;
    if constexpr (SLOPE) {
      const float dist = (float)(at - n0);     // of the tile's first key; its last: 31 less
      bound = __builtin_fmaf(lift, fmaxf(fabsf(dist), fabsf(dist - (kMTile - 1))), bound);
    }
    if (__builtin_amdgcn_ballot_w64(!(bound <= m + up))) {
      float x[16];
      scores<true>(s, n0, poly, 0.f, x);
      if (edge) masked(x, n0, -INFINITY);
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      mx = max_halves(mx);
      if (mx > m + up) m_new = mx - fminf(up, 0.f);
    }
    if (__builtin_amdgcn_ballot_w64(m_new != m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
      n *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    return poly;
  }
  __device__ __forceinline__ void weigh(int n0, bool edge, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(x[i]);
    if (edge) masked(x, n0, 0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) l += x[i];
  }
  __device__ __forceinline__ void add(const uint16_t* v, const float (&x)[16]) {
    bf16x8 pb[2];
    pack_frags<F16>(x, pb);
#pragma unroll
    for (int s = 0; s < 2; ++s) n = sum_frag<F16>(pb[s], n);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int s = 0; s < 2; ++s) o[db] = mfma32x32x16_t<F16>(rd.turned(v, db, s), pb[s], o[db]);
  }
  // A tile whose values may hold infinities or NaN that a row does not see.
  __device__ __forceinline__ void careful(const uint16_t* k, const uint16_t* v, int n0, float up) {
    float x[16], seen[16];
    const f32x16 s = products(k);
    const bool poly = settle(s, n0, true, up);
    scores<false>(s, n0, poly, m, x);
    weigh(n0, true, x);
    const int from = lo - n0 - 4 * hi, to = end - n0 - 4 * hi;
#pragma unroll
    for (int i = 0; i < 16; ++i) seen[i] = mfma_row(i, 0) < from || mfma_row(i, 0) >= to ? 0.f : 1.f;
    bf16x8 pb[2], sb[2];
    pack_frags<F16>(x, pb);
    pack_frags<F16>(seen, sb);
#pragma unroll
    for (int s = 0; s < 2; ++s) n = sum_frag<F16>(pb[s], n);
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = careful_mfma<HD, F16>(rd, v, db, pb, sb, o[db]);
  }
  __device__ __forceinline__ bool odd() const {
    bool x = false;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) x |= !(fabsf(o[db][i]) < kBig);
    return x;
  }
  // The rows' outputs, or with `to` this lane's part of them; `total` and `norm` are l
  // and n over both halves.  Outputs are divided by the sum of the weights as they
  // were rounded, so a weight that stands alone loses nothing: 0.6 to 1.0 instead of
  // 1.7 thousandths of the output's norm in bf16.  The LSE has the exact weights;
  // parts are scaled to go with their sum.
  __device__ __forceinline__ void finish(const FwdArgs& p, const Row& x, Part to, float total, float norm) {
    if (!x.live) return;
    if (to.o) {
      const float a = norm == 0.f ? 0.f : total / norm;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= a;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(to.o + db * 32 + 8 * g + 4 * hi) =
              f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
      if (hi == 0) *to.stat = float2{m, total};
      return;
    }
    const float inv = norm == 0.f ? 0.f : 1.0f / norm;   // no key seen: zeros
    uint16_t* O = p.o + x.b * p.o_sb + x.h * p.o_sh + x.tok * p.o_sm;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const bf16x2 a = pack2<F16>(o[db][4 * g + 0] * inv, o[db][4 * g + 1] * inv);
        const bf16x2 b = pack2<F16>(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
        *reinterpret_cast<u32x2*>(O + db * 32 + 8 * g + 4 * hi) =
            u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
        if (p.rest)
          *reinterpret_cast<u32x2*>(p.rest + (O - p.o) + db * 32 + 8 * g + 4 * hi) =
              rest_of<F16>(f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]} * inv, a, b);
      }
    if (p.lse && hi == 0)
      p.lse[x.b * p.lse_sb + x.h * p.lse_sh + x.tok] = total == 0.f ? -INFINITY : m + __log2f(total);
  }
};

template <int HD>
struct Slot {
  uint16_t k[kMTile * HD];
  uint16_t v[kMTile * HD];
};

// Four values of a row's outputs.
template <bool F16>
__device__ __forceinline__ void emit(const FwdArgs& p, int64_t b, int64_t h, int64_t tok, int at, f32x4 o, float total) {
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  const bf16x2 lo = pack2<F16>(o[0] * inv, o[1] * inv), hi = pack2<F16>(o[2] * inv, o[3] * inv);
  const int64_t to = b * p.o_sb + h * p.o_sh + tok * p.o_sm + 4 * at;
  *reinterpret_cast<u32x2*>(p.o + to) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  if (p.rest) *reinterpret_cast<u32x2*>(p.rest + to) = rest_of<F16>(o * inv, lo, hi);
}

}  // namespace
}  // namespace gpa
