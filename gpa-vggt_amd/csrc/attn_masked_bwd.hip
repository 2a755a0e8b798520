// Masked attention, backward (attn_masked.h has the formulas and the masks).
//
//   P_ij  = 2^(s_ij log2(e) - lse_i)             (recomputed from q, k and the LSE)
//   dP_ij = dO_i . V_j,   delta_i = dO_i . O_i - log2(e) dlse_i
//   dS_ij = P_ij (dP_ij - delta_i) (1 - tanh^2(x_ij / cap))
//   dV_j  = sum_i P_ij dO_i,   dK_j = sm_scale sum_i dS_ij Q_i,
//   dQ_i  = sm_scale sum_j dS_ij K_j
//
// attn_masked_delta_kernel writes a record of every 64 rows: their LSE, -delta,
// token (counted from the first row's, so that it is exact in fp32) and slope.  delta comes from O and what rounding took from it: where a
// row's weights are sharp, dP - delta is small beside both, and delta from the
// rounded O alone put dq and dk 1.9 to 2.5 roundings off (1.55 with the rest).
//
// attn_masked_dkdv_kernel: a workgroup has 64 keys and walks the rows that see
// them, all query heads of the key head, so a shared head's gradient is one sum
// in one order.  A wave owns 32 of the keys (K, V, dK and dV in registers) and
// one half of each 64-row tile; the two halves are added at the end.  (With 128
// keys to a workgroup, one row tile for all four waves, a launch of 4,096 keys
// and 8 heads had 256 workgroups of very different lengths.)  S = Q . K^T puts a
// key in each lane, and P and dS are used in place as the B operands of dV^T +=
// dO^T . P and dK^T += Q^T . dS.
//
// attn_masked_dq_kernel mirrors it: a wave owns 32 rows and walks the keys, dQ^T +=
// K^T . dS^T.  In both the next tile's S and dP are computed beside this one's
// weights.  No atomics: two kernels compute S and dP twice (7 products instead of
// 5), and in return the results repeat bit by bit and no fp32 copy of dQ goes
// through memory.
//
// Where few key blocks decide how long a launch lasts, blocks are cut and taken by
// length as in the forward pass; attn_masked_grad_join_kernel adds up the parts.
//
// With a cap, r = 1 / (1 + e^(2u)) gives both: tanh = 1 - 2r, 1 - tanh^2 = 4 (r - r^2).
// Scores that are small beside the cap lose what r rounds away, so with caps above kNarrow
// they come from the forward's polynomial.
//
// P and dS are rounded to the operand format for the products (the same
// relative error as the gradients' own rounding); sums are fp32.  Of the two
// fragments that dS of a tile makes, one goes into a second product with what
// rounding took from it.  dq and dk are then off by 1.4 times what their own
// rounding does, against 1.55 without and 1.15 with both fragments; the two passes
// take 505 us against 487 and 532 (2 x 16 heads of 128 on 2 x 4, 4,096 tokens), and
// 545 against 500 and 582 (8 heads of 64, 8,191 tokens).  In fp16 small weights
// would lose bits below 2^-14, so P is scaled by 2^14 and dS by a power of two that
// follows its largest finite value; the sums are scaled back.
//
// Measured (us a kernel after 200 passes; the first ten of a process take a seventh
// longer): dk, dv 235 and dq 114 at 2 x 16 heads of 128 on 2 x 4, four causal documents of
// 4,096 tokens in all, capped (420 and 650 TFLOP/s, four and three products); 197 and 178
// at 8 of 64, 8,191 tokens, causal with a prefix and slopes (720 and 590).  At head
// dim 128 dk and dv are bound by latency: the ring's 135 KB leave one workgroup a CU, so
// one wave a SIMD (416 registers, of which dK, dV, K and V are 192); it waits 43 % of its
// time, vector issue takes 29 % of a SIMD's, matrix instructions run 23 %, and LDS is
// busy 13 % of a CU's.  With two waves a SIMD, at 64, these are 35, 48, 37 and 34 %; dq
// at 128 36, 47, 38 and 17 %.  delta reads 100 MB in 17.6.
#include "attn_masked_deal.h"

#include <algorithm>

namespace gpa {
namespace {

constexpr int kRowTile = 64;                   // rows of a record, and of a dk, dv tile
constexpr int kRec = 4 * kRowTile;             // lse (kNarrowCap: less cap log2(e)), -delta, token, slope
constexpr int kKeys = 64;                      // keys of a dk, dv workgroup
static_assert(kRowTile == 64 && kKeys == 64, "attn_masked_count_kernel counts these");

struct BwdArgs {
  const uint16_t *q, *k, *v, *o, *rest, *d_o;
  const float *lse, *d_lse;
  uint16_t *dq, *dk, *dv;
  int64_t q_sb, q_sh, q_sm, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, o_sb, o_sh, o_sm;
  int64_t do_sb, do_sh, do_sm, dq_sb, dq_sh, dq_sm, dk_sb, dk_sh, dk_sn, dv_sb, dv_sh, dv_sn;
  int64_t lse_sb, lse_sh;
  const float* slopes;
  int64_t slopes_sb;
  float* rec;                                  // [B * Hk][tiles][kRec]
  int32_t Hk, G, R, tiles;                     // R = M * G rows of a problem
  float sm_scale, lse_off;
  const Deal *keys, *rows;                     // null: every block whole, heavy ones first
  float *kpart, *qpart;                        // [part][key head][dk, dv of 64 keys; dq of 128 rows][HD]
  MaskArgs mask;
  ScoreArgs score;
};

// Workgroup L's piece of a block (k of n), and where its part goes (-1: it is whole).
struct Piece { int block, prob, k, n, part; };
__device__ __forceinline__ Piece piece_of(const Deal* d, int L, int blocks, int problems, int Hk) {
  Piece x{0, 0, 0, 1, -1};
  if (!d) {
    item_of(L, blocks, problems, x.block, x.prob);
    return x;
  }
  x.n = 0;
  if (L / Hk >= d->pieces) return x;
  const int4 y = same(d->piece[L / Hk]);
  const int b = y.x / blocks, kvh = L % Hk;
  return {y.x - b * blocks, b * Hk + kvh, y.y, y.z, y.w < 0 ? -1 : y.w * Hk + kvh};
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void attn_masked_delta_kernel(BwdArgs p) {
  constexpr int CH = HD / 8;                   // lanes of a row
  const int tile = blockIdx.x % p.tiles, prob = blockIdx.x / p.tiles;
  const int b = prob / p.Hk, kvh = prob % p.Hk;
  float* rec = p.rec + ((int64_t)prob * p.tiles + tile) * kRec;
  const int ch = threadIdx.x % CH;
  for (int i = threadIdx.x / CH; i < kRowTile; i += 256 / CH) {
    const int r = tile * kRowTile + i;
    float lse = INFINITY, delta = 0.f, slope = 0.f;   // past the rows: weights of zero
    float tok = 0.f;
    if (r < p.R) {
      const int m = r / p.G;
      tok = (float)(m - tile * kRowTile / p.G);
      const int h = kvh * p.G + r % p.G;
      const int64_t at = b * p.o_sb + h * p.o_sh + m * p.o_sm + 8 * ch;
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(p.o + at);
      const bf16x8 y = *reinterpret_cast<const bf16x8*>(p.d_o + b * p.do_sb + h * p.do_sh + m * p.do_sm + 8 * ch);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta = __builtin_fmaf(half_to_f32<F16>(x[e]), half_to_f32<F16>(y[e]), delta);
      if (p.rest) {
        const bf16x8 z = *reinterpret_cast<const bf16x8*>(p.rest + at);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          delta = __builtin_fmaf(half_to_f32<F16>(z[e]), half_to_f32<F16>(y[e]), delta);
      }
      lse = p.lse[b * p.lse_sb + h * p.lse_sh + m];
      if (lse == -INFINITY) lse = INFINITY;    // a row that sees nothing
      if (p.slopes) slope = p.slopes[b * p.slopes_sb + h] * kMLog2e;
      if (p.d_lse && ch == 0)
        delta -= kMLog2e * p.d_lse[((int64_t)b * p.Hk * p.G + h) * p.mask.M + m];
    }
#pragma unroll
    for (int s = 1; s < CH; s <<= 1) delta += __shfl_xor(delta, s);
    if (ch == 0) {
      rec[i] = lse - p.lse_off;
      rec[kRowTile + i] = -delta;
      rec[2 * kRowTile + i] = tok;
      rec[3 * kRowTile + i] = slope;
    }
  }
}

constexpr float kPScale = 16384.0f;            // of P in fp16

// The power of two by which a wave's dS are scaled in fp16: the largest one, lowered
// where values would pass the format's range.
struct DsScale {
  float s = 0x1p100f;
  // Whether it has to move for these values; `ratio` rescales the sums.
  __device__ __forceinline__ bool follow(const float (&ds)[16], float& ratio) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(ds[i]));
    if (!__builtin_amdgcn_ballot_w64(mx * s > 32768.0f)) return false;
    // Infinities, of rows and keys that are lost, leave the scale to the others.
    mx = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fabsf(ds[i]) < INFINITY ? fmaxf(mx, fabsf(ds[i])) : mx;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
    if (!(mx * s > 32768.0f)) return false;
    const float to = __builtin_amdgcn_ldexpf(1.0f, 13 - __builtin_amdgcn_frexp_expf(mx));   // 2^13 at most
    ratio = to / s;
    s = to;
    return true;
  }
};

// How scores are capped.  From r alone they are off by about 5 2^-24 cap (log2 units): for
// caps up to kNarrow P by less than a seventeenth of what rounding takes from it.  Above,
// products within `lim` go through the polynomial, selected one by one.  Measured (us,
// forward and backward, cap 100 and 200 with kNarrow between): 1,005 and 1,122 at
// 2 x 16 heads of 128 on 2 x 4, 4,096 tokens, causal; 592 and 762 at 8 of 64, 8,191 tokens.
template <bool F16> constexpr float kNarrow = F16 ? 128.0f : 1024.0f;
enum Cap { kNoCap, kNarrowCap, kWideCap };

// log2 of P, and 1 - tanh^2 (of which a quarter with a cap), of one product s; `lse` is a record's.
struct Pair { float x, der; };
template <Cap CAP>
__device__ __forceinline__ Pair log_weight(float s, float lse, const ScoreArgs& a) {
  if constexpr (CAP == kNoCap) return {__builtin_fmaf(s, a.c1, -lse), 1.0f};
  const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * a.ce));
  if constexpr (CAP == kNarrowCap) return {__builtin_fmaf(r, -2.0f * a.capl, -lse), __builtin_fmaf(-r, r, r)};
  const float near = s * cap_poly(s, a), t = near * a.half;
  const bool in = fabsf(s) <= a.lim;
  return {(in ? near : __builtin_fmaf(r, -2.0f * a.capl, a.capl)) - lse,
          in ? __builtin_fmaf(-t, t, 0.25f) : __builtin_fmaf(-r, r, r)};
}

template <int HD>
struct RowSlot {
  uint16_t q[kRowTile * HD];
  uint16_t d[kRowTile * HD];
  float st[kRec];
};

template <int HD, bool F16, Cap CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, HD == 64 ? 2 : 1) void attn_masked_dkdv_kernel(BwdArgs p) {
  constexpr int KS = HD / 16, DB = HD / 32, CH = HD / 8;
  constexpr int DJ = kRowTile * CH / kMThreads;
  __shared__ __attribute__((aligned(16))) RowSlot<HD> r0, r1, r2, r3;
  __shared__ int range[2][kMWaves];

  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave >> 1;                  // of a row tile
  const int blocks = (p.mask.N + kKeys - 1) / kKeys;
  const Piece piece = piece_of(p.keys, blockIdx.x, blocks, gridDim.x / blocks, p.Hk);
  if (piece.n == 0) return;
  const int kb = piece.block, prob = __builtin_amdgcn_readfirstlane(piece.prob);
  const int b = __builtin_amdgcn_readfirstlane(prob / p.Hk), kvh = __builtin_amdgcn_readfirstlane(prob % p.Hk);
  const int j = kb * kKeys + (wave & 1) * 32 + l32;
  const bool live = j < p.mask.N;
  const int jc = live ? j : p.mask.N - 1;
  const KeySpan ks_ = key_span(p.mask, b, jc);
  const int lo = ks_.lo * p.G, hi_r = ks_.hi * p.G;   // rows that see this lane's key
  // A tile's first token, as a distance from this lane's key.
  auto place_of = [&](int t) { return t * kRowTile / p.G + ks_.shift - jc; };

  bf16x8 kf[KS], vf[KS];
  {
    const uint16_t* K = p.k + b * p.k_sb + kvh * p.k_sh + jc * p.k_sn;
    const uint16_t* V = p.v + b * p.v_sb + kvh * p.v_sh + jc * p.v_sn;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = *reinterpret_cast<const bf16x8*>(K + 16 * ks + 8 * hi);
      vf[ks] = *reinterpret_cast<const bf16x8*>(V + 16 * ks + 8 * hi);
    }
  }

  const bool any = live && hi_r > lo;
  int w_lo = any ? lo : 0x7fffffff, w_hi = any ? hi_r : 0;
  int a_lo = live ? lo : 0, a_hi = live ? (any ? hi_r : 0) : 0x7fffffff;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    w_lo = min(w_lo, __shfl_xor(w_lo, i));
    w_hi = max(w_hi, __shfl_xor(w_hi, i));
    a_lo = max(a_lo, __shfl_xor(a_lo, i));
    a_hi = min(a_hi, __shfl_xor(a_hi, i));
  }
  w_lo = __builtin_amdgcn_readfirstlane(w_lo);
  w_hi = __builtin_amdgcn_readfirstlane(w_hi);
  a_lo = __builtin_amdgcn_readfirstlane(a_lo);
  a_hi = __builtin_amdgcn_readfirstlane(a_hi);
  if (lane == 0) {
    range[0][wave] = w_lo;
    range[1][wave] = w_hi;
  }
  __syncthreads();
  int n_lo = range[0][0], n_hi = range[1][0];
#pragma unroll
  for (int i = 1; i < kMWaves; ++i) {
    n_lo = min(n_lo, range[0][i]);
    n_hi = max(n_hi, range[1][i]);
  }
  n_lo = __builtin_amdgcn_readfirstlane(n_lo);
  n_hi = __builtin_amdgcn_readfirstlane(n_hi);
  const int t_lo = n_hi > n_lo ? n_lo / kRowTile : 0;
  const int all_tiles = n_hi > n_lo ? (n_hi + kRowTile - 1) / kRowTile - t_lo : 0;
  const int t_begin = t_lo + share_of(all_tiles, piece.k, piece.n);
  const int t_end = t_lo + share_of(all_tiles, piece.k + 1, piece.n);

  // Rows of a tile: token and head of row 64 t + i follow from (64 t) / G; where
  // G divides 64 the offsets inside a tile are the same for all tiles.
  const uint16_t* Q = p.q + b * p.q_sb + (int64_t)kvh * p.G * p.q_sh;
  const uint16_t* D = p.d_o + b * p.do_sb + (int64_t)kvh * p.G * p.do_sh;
  const bool even = kRowTile % p.G == 0;
  uint32_t q_voff[DJ], d_voff[DJ];
  auto offsets = [&](int first) {              // first: (64 t) % G
#pragma unroll
    for (int i = 0; i < DJ; ++i) {
      const int pos = (wave * DJ + i) * 64 + lane, row = pos / CH;
      const uint32_t ch = (uint32_t)((pos % CH) ^ tile_swz<HD>(row)) * 16u;
      const uint32_t tok = (uint32_t)(first + row) / (uint32_t)p.G, g = (uint32_t)(first + row) % (uint32_t)p.G;
      q_voff[i] = tok * (uint32_t)(p.q_sm * 2) + g * (uint32_t)(p.q_sh * 2) + ch;
      d_voff[i] = tok * (uint32_t)(p.do_sm * 2) + g * (uint32_t)(p.do_sh * 2) + ch;
    }
  };
  offsets(0);
  const float* rec = p.rec + (int64_t)prob * p.tiles * kRec;
  auto issue = [&](int t, RowSlot<HD>& T) {
    const int base = min(t, p.tiles) * kRowTile;   // tiles past the rows: all lanes idle
    if (!even) offsets(base % p.G);
    const int64_t tok = base / p.G;
    const __amdgpu_buffer_rsrc_t qr = make_rsrc(Q + tok * p.q_sm, kNoRow);
    const __amdgpu_buffer_rsrc_t dr = make_rsrc(D + tok * p.do_sm, kNoRow);
    const int left = p.R - base;
    const __amdgpu_buffer_rsrc_t rr = make_rsrc(rec + (int64_t)base / kRowTile * kRec, left > 0 ? kRec * 4 : 0);
#pragma unroll
    for (int i = 0; i < DJ; ++i) {
      const bool in = ((wave * DJ + i) * 64 + lane) / CH < left;
      m_dma16(qr, &T.q[(wave * DJ + i) * 512], in ? q_voff[i] : kNoRow);
    }
#pragma unroll
    for (int i = 0; i < DJ; ++i) {
      const bool in = ((wave * DJ + i) * 64 + lane) / CH < left;
      m_dma16(dr, &T.d[(wave * DJ + i) * 512], in ? d_voff[i] : kNoRow);
    }
    m_dma4(rr, &T.st[wave * 64], (uint32_t)(wave * 64 + lane) * 4u);
  };

  TileReader<HD> rd(lane);
  f32x16 dk[DB], dv[DB];
  DsScale sc;
  auto restart = [&]() {
    sc = DsScale{};
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = f32x16{};
  };
  // S and dP - delta of the rows of this wave's half (registers) and this lane's key.
  auto products = [&](const RowSlot<HD>& T, f32x16& s, f32x16& dp) {
    s = f32x16{};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 nd = *reinterpret_cast<const f32x4*>(&T.st[kRowTile + half * 32 + 8 * g + 4 * hi]);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * g + e] = nd[e];
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mfma32x32x16_t<F16>(rd.rows(T.q + half * 32 * HD, ks), kf[ks], s);
      dp = mfma32x32x16_t<F16>(rd.rows(T.d + half * 32 * HD, ks), vf[ks], dp);
    }
  };
  // P and dS.
  auto weights = [&](const RowSlot<HD>& T, const f32x16& s, const f32x16& dp, int row0, bool edge,
                     float first_at, float (&w)[16], float (&ds)[16]) {
    const float* st = &T.st[half * 32 + 4 * hi];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(&st[8 * g]);
      f32x4 tok, sl;
      if constexpr (SLOPE) {
        tok = *reinterpret_cast<const f32x4*>(&st[2 * kRowTile + 8 * g]);
        sl = *reinterpret_cast<const f32x4*>(&st[3 * kRowTile + 8 * g]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e;
        const Pair y = log_weight<CAP>(s[i], ls[e], p.score);
        float x = y.x;
        if constexpr (SLOPE) x = __builtin_fmaf(-sl[e], fabsf(tok[e] + first_at), x);
        w[i] = __builtin_amdgcn_exp2f(x);
        ds[i] = w[i] * dp[i];
        if constexpr (CAP != kNoCap) ds[i] *= y.der;
      }
    }
    if (edge) {
      const int from = lo - row0 - 4 * hi, to = hi_r - row0 - 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (mfma_row(i, 0) < from || mfma_row(i, 0) >= to) w[i] = ds[i] = 0.f;
    }
    if constexpr (F16) {
      float ratio;
      if (sc.follow(ds, ratio)) {
#pragma unroll
        for (int db = 0; db < DB; ++db) dk[db] *= ratio;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w[i] *= kPScale;
        ds[i] *= sc.s;
      }
    }
  };

  f32x16 s, dp;
  int place = SLOPE ? place_of(t_begin) : 0;
  const int step = kRowTile / p.G;             // from tile to tile, where G divides one
  auto iter = [&](int t, const RowSlot<HD>& cur, const RowSlot<HD>& nxt, RowSlot<HD>& dst) {
    m_wait_barrier<2 * DJ + 1>();              // tile t + 1 landed (t + 2 in flight) for every wave
    issue(t + 3, dst);
    rd.fresh();
    const float first_at = (float)place;
    if constexpr (SLOPE) place = even ? place + step : place_of(t + 1);
    const int row0 = t * kRowTile + half * 32;
    if (row0 < w_hi && row0 + 32 > w_lo) {
      f32x16 s_next, dp_next;
      products(nxt, s_next, dp_next);
      float w[16], ds[16];
      weights(cur, s, dp, row0, row0 < a_lo || row0 + 32 > a_hi, first_at, w, ds);
      bf16x8 wb[2], db_[2];
      pack_frags<F16>(w, wb);
      pack_frags<F16>(ds, db_);
      const bf16x8 dr = rest_frag<F16>(ds, db_[0]);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8 qt = rd.turned(cur.q + half * 32 * HD, db, i);
          if (i == 0) dk[db] = mfma32x32x16_t<F16>(qt, dr, dk[db]);
          dv[db] = mfma32x32x16_t<F16>(rd.turned(cur.d + half * 32 * HD, db, i), wb[i], dv[db]);
          dk[db] = mfma32x32x16_t<F16>(qt, db_[i], dk[db]);
        }
      s = s_next;
      dp = dp_next;
    } else {
      products(nxt, s, dp);
    }
  };
  restart();
  issue(t_begin, r0);
  issue(t_begin + 1, r1);
  issue(t_begin + 2, r2);
  m_wait_barrier<2 * (2 * DJ + 1)>();
  products(r0, s, dp);
  for (int t = t_begin; t < t_end; t += 4) {
    iter(t, r0, r1, r3);
    if (t + 1 >= t_end) break;
    iter(t + 1, r1, r2, r0);
    if (t + 2 >= t_end) break;
    iter(t + 2, r2, r3, r1);
    if (t + 3 >= t_end) break;
    iter(t + 3, r3, r0, r2);
  }
  m_wait<0>();

  bool odd = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      odd |= !(fabsf(dk[db][i]) < INFINITY) || !(fabsf(dv[db][i]) < INFINITY);
  if (__syncthreads_or(odd && live)) {
    restart();
    for (int t = t_begin; t < t_end; ++t) {
      __syncthreads();
      issue(t, r0);
      m_wait<0>();
      __syncthreads();
      const int row0 = t * kRowTile + half * 32, from = lo - row0 - 4 * hi, to = hi_r - row0 - 4 * hi;
      float w[16], ds[16], sx[16];
      products(r0, s, dp);
      weights(r0, s, dp, row0, true, SLOPE ? (float)place_of(t) : 0.f, w, ds);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sx[i] = mfma_row(i, 0) < from || mfma_row(i, 0) >= to ? 0.f : 1.f;
      bf16x8 wb[2], db_[2], sb[2];
      pack_frags<F16>(w, wb);
      pack_frags<F16>(ds, db_);
      pack_frags<F16>(sx, sb);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dv[db] = careful_mfma<HD, F16>(rd, r0.d + half * 32 * HD, db, wb, sb, dv[db]);
        dk[db] = careful_mfma<HD, F16>(rd, r0.q + half * 32 * HD, db, db_, sb, dk[db]);
      }
    }
    __syncthreads();
  }

  // The second half's sums by way of the ring, slots of 16 bytes a lane.
  const float kx = (CAP != kNoCap ? 4.0f : 1.0f) * p.sm_scale * (F16 ? 1.0f / sc.s : 1.0f);
  const float vx = F16 ? 1.0f / kPScale : 1.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    dk[db] *= kx;
    dv[db] *= vx;
  }
  static_assert(sizeof(RowSlot<HD>) >= 2 * DB * 4 * 64 * 16, "two waves' sums of one tensor in a slot");
  auto give = [&](uint16_t* to, const f32x16 (&v)[DB]) {
    f32x4* at = reinterpret_cast<f32x4*>(to) + (wave & 1) * DB * 4 * 64 + lane;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at[(db * 4 + g) * 64] = f32x4{v[db][4 * g], v[db][4 * g + 1], v[db][4 * g + 2], v[db][4 * g + 3]};
  };
  auto take = [&](const uint16_t* from, f32x16 (&v)[DB]) {
    const f32x4* at = reinterpret_cast<const f32x4*>(from) + (wave & 1) * DB * 4 * 64 + lane;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = at[(db * 4 + g) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[db][4 * g + e] += x[e];
      }
  };
  if (half == 1) {
    give(r0.q, dk);
    give(r1.q, dv);
  }
  __syncthreads();
  if (half == 1 || !live) return;
  take(r0.q, dk);
  take(r1.q, dv);
  if (piece.part >= 0) {
    float* P = p.kpart + ((int64_t)piece.part * 2 * kKeys + (wave & 1) * 32 + l32) * HD;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = db * 32 + 8 * g + 4 * hi;
        *reinterpret_cast<f32x4*>(P + at) = f32x4{dk[db][4 * g], dk[db][4 * g + 1], dk[db][4 * g + 2], dk[db][4 * g + 3]};
        *reinterpret_cast<f32x4*>(P + kKeys * HD + at) =
            f32x4{dv[db][4 * g], dv[db][4 * g + 1], dv[db][4 * g + 2], dv[db][4 * g + 3]};
      }
    return;
  }
  uint16_t* DK = p.dk + b * p.dk_sb + kvh * p.dk_sh + j * p.dk_sn;
  uint16_t* DV = p.dv + b * p.dv_sb + kvh * p.dv_sh + j * p.dv_sn;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = db * 32 + 8 * g + 4 * hi;
      const bf16x2 k0 = pack2<F16>(dk[db][4 * g], dk[db][4 * g + 1]);
      const bf16x2 k1 = pack2<F16>(dk[db][4 * g + 2], dk[db][4 * g + 3]);
      const bf16x2 v0 = pack2<F16>(dv[db][4 * g], dv[db][4 * g + 1]);
      const bf16x2 v1 = pack2<F16>(dv[db][4 * g + 2], dv[db][4 * g + 3]);
      *reinterpret_cast<u32x2*>(DK + at) =
          u32x2{__builtin_bit_cast(uint32_t, k0), __builtin_bit_cast(uint32_t, k1)};
      *reinterpret_cast<u32x2*>(DV + at) =
          u32x2{__builtin_bit_cast(uint32_t, v0), __builtin_bit_cast(uint32_t, v1)};
    }
}

template <int HD>
struct KeySlot {
  uint16_t k[kMTile * HD];
  uint16_t v[kMTile * HD];
};

template <int HD, bool F16, Cap CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, 2) void attn_masked_dq_kernel(BwdArgs p) {
  constexpr int KS = HD / 16, DB = HD / 32, CH = HD / 8;
  constexpr int DJ = kMTile * CH / kMThreads;
  __shared__ __attribute__((aligned(16))) KeySlot<HD> r0, r1, r2, r3;
  __shared__ int range[2][kMWaves];

  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (p.R + kMRows - 1) / kMRows;
  const Piece piece = piece_of(p.rows, blockIdx.x, blocks, gridDim.x / blocks, p.Hk);
  if (piece.n == 0) return;
  const int qb = p.rows ? piece.block : blocks - 1 - piece.block;
  const int prob = __builtin_amdgcn_readfirstlane(piece.prob);
  const int b = __builtin_amdgcn_readfirstlane(prob / p.Hk), kvh = __builtin_amdgcn_readfirstlane(prob % p.Hk);
  const int r = qb * kMRows + wave * 32 + l32;
  const bool live = r < p.R;
  const int rc = live ? r : p.R - 1;
  const int m_tok = rc / p.G, h = kvh * p.G + rc % p.G;
  const RowSpan span = row_span(p.mask, b, m_tok);
  const float* rec = p.rec + ((int64_t)prob * p.tiles + rc / kRowTile) * kRec + rc % kRowTile;
  const float lse = rec[0], ndelta = rec[kRowTile], slope = SLOPE ? rec[3 * kRowTile] : 0.f;

  bf16x8 qf[KS], df[KS];
  {
    const uint16_t* Q = p.q + b * p.q_sb + h * p.q_sh + m_tok * p.q_sm;
    const uint16_t* D = p.d_o + b * p.do_sb + h * p.do_sh + m_tok * p.do_sm;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = *reinterpret_cast<const bf16x8*>(Q + 16 * ks + 8 * hi);
      df[ks] = *reinterpret_cast<const bf16x8*>(D + 16 * ks + 8 * hi);
    }
  }

  const bool any = live && span.hi > span.lo;
  int w_lo = any ? span.lo : 0x7fffffff, w_hi = any ? span.hi : 0;
  int a_lo = live ? span.lo : 0, a_hi = live ? (any ? span.hi : 0) : 0x7fffffff;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    w_lo = min(w_lo, __shfl_xor(w_lo, i));
    w_hi = max(w_hi, __shfl_xor(w_hi, i));
    a_lo = max(a_lo, __shfl_xor(a_lo, i));
    a_hi = min(a_hi, __shfl_xor(a_hi, i));
  }
  w_lo = __builtin_amdgcn_readfirstlane(w_lo);
  w_hi = __builtin_amdgcn_readfirstlane(w_hi);
  a_lo = __builtin_amdgcn_readfirstlane(a_lo);
  a_hi = __builtin_amdgcn_readfirstlane(a_hi);
  if (lane == 0) {
    range[0][wave] = w_lo;
    range[1][wave] = w_hi;
  }
  __syncthreads();
  int n_lo = range[0][0], n_hi = range[1][0];
#pragma unroll
  for (int i = 1; i < kMWaves; ++i) {
    n_lo = min(n_lo, range[0][i]);
    n_hi = max(n_hi, range[1][i]);
  }
  n_lo = __builtin_amdgcn_readfirstlane(n_lo);
  n_hi = __builtin_amdgcn_readfirstlane(n_hi);
  if (n_hi <= n_lo) n_lo = n_hi = 0;
  const int all_tiles = (n_hi - n_lo + kMTile - 1) / kMTile;
  const int t_begin = share_of(all_tiles, piece.k, piece.n), t_end = share_of(all_tiles, piece.k + 1, piece.n);

  const uint16_t* K = p.k + b * p.k_sb + kvh * p.k_sh;
  const uint16_t* V = p.v + b * p.v_sb + kvh * p.v_sh;
  uint32_t k_voff[DJ], v_voff[DJ];
#pragma unroll
  for (int i = 0; i < DJ; ++i) {
    const int pos = (wave * DJ + i) * 64 + lane, key = pos / CH;
    const uint32_t ch = (uint32_t)((pos % CH) ^ tile_swz<HD>(key)) * 16u;
    k_voff[i] = key * (uint32_t)(p.k_sn * 2) + ch;
    v_voff[i] = key * (uint32_t)(p.v_sn * 2) + ch;
  }
  auto issue = [&](int t, KeySlot<HD>& T) {
    const int n0 = n_lo + t * kMTile;
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc<HD>(K, p.k_sn, n0, n_hi);
    const __amdgpu_buffer_rsrc_t vr = tile_rsrc<HD>(V, p.v_sn, n0, n_hi);
#pragma unroll
    for (int i = 0; i < DJ; ++i) m_dma16(kr, &T.k[(wave * DJ + i) * 512], k_voff[i]);
#pragma unroll
    for (int i = 0; i < DJ; ++i) m_dma16(vr, &T.v[(wave * DJ + i) * 512], v_voff[i]);
  };

  TileReader<HD> rd(lane);
  f32x16 dq[DB];
  DsScale sc;
  auto restart = [&]() {
    sc = DsScale{};
#pragma unroll
    for (int db = 0; db < DB; ++db) dq[db] = f32x16{};
  };
  auto products = [&](const KeySlot<HD>& T, f32x16& s, f32x16& dp) {
    s = f32x16{};
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = ndelta;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mfma32x32x16_t<F16>(rd.rows(T.k, ks), qf[ks], s);
      dp = mfma32x32x16_t<F16>(rd.rows(T.v, ks), df[ks], dp);
    }
  };
  auto weights = [&](const f32x16& s, const f32x16& dp, int n0, bool edge, float (&ds)[16]) {
    const float dist = (float)(span.at - n0 - 4 * hi);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const Pair y = log_weight<CAP>(s[i], lse, p.score);
      float x = y.x;
      if constexpr (SLOPE) x = __builtin_fmaf(-slope, fabsf(dist - (float)mfma_row(i, 0)), x);
      ds[i] = __builtin_amdgcn_exp2f(x) * dp[i];
      if constexpr (CAP != kNoCap) ds[i] *= y.der;
    }
    if (edge) {
      const int from = span.lo - n0 - 4 * hi, to = span.hi - n0 - 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (mfma_row(i, 0) < from || mfma_row(i, 0) >= to) ds[i] = 0.f;
    }
    if constexpr (F16) {
      float ratio;
      if (sc.follow(ds, ratio)) {
#pragma unroll
        for (int db = 0; db < DB; ++db) dq[db] *= ratio;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] *= sc.s;
    }
  };
  f32x16 s, dp;
  auto iter = [&](int t, const KeySlot<HD>& cur, const KeySlot<HD>& nxt, KeySlot<HD>& dst) {
    m_wait_barrier<2 * DJ>();                  // tile t + 1 landed (t + 2 in flight) for every wave
    issue(t + 3, dst);
    rd.fresh();
    const int n0 = n_lo + t * kMTile;
    if (n0 < w_hi && n0 + kMTile > w_lo) {
      f32x16 s_next, dp_next;
      products(nxt, s_next, dp_next);
      float ds[16];
      weights(s, dp, n0, n0 < a_lo || n0 + kMTile > a_hi, ds);
      bf16x8 db_[2];
      pack_frags<F16>(ds, db_);
      const bf16x8 dr = rest_frag<F16>(ds, db_[0]);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8 kt = rd.turned(cur.k, db, i);
          if (i == 0) dq[db] = mfma32x32x16_t<F16>(kt, dr, dq[db]);
          dq[db] = mfma32x32x16_t<F16>(kt, db_[i], dq[db]);
        }
      s = s_next;
      dp = dp_next;
    } else {
      products(nxt, s, dp);
    }
  };
  restart();
  issue(t_begin, r0);
  issue(t_begin + 1, r1);
  issue(t_begin + 2, r2);
  m_wait_barrier<4 * DJ>();
  products(r0, s, dp);
  for (int t = t_begin; t < t_end; t += 4) {
    iter(t, r0, r1, r3);
    if (t + 1 >= t_end) break;
    iter(t + 1, r1, r2, r0);
    if (t + 2 >= t_end) break;
    iter(t + 2, r2, r3, r1);
    if (t + 3 >= t_end) break;
    iter(t + 3, r3, r0, r2);
  }
  m_wait<0>();

  bool odd = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd |= !(fabsf(dq[db][i]) < INFINITY);
  if (__syncthreads_or(odd && live)) {
    restart();
    for (int t = t_begin; t < t_end; ++t) {
      __syncthreads();
      issue(t, r0);
      m_wait<0>();
      __syncthreads();
      const int n0 = n_lo + t * kMTile, from = span.lo - n0 - 4 * hi, to = span.hi - n0 - 4 * hi;
      float ds[16], sx[16];
      products(r0, s, dp);
      weights(s, dp, n0, true, ds);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sx[i] = mfma_row(i, 0) < from || mfma_row(i, 0) >= to ? 0.f : 1.f;
      bf16x8 db_[2], sb[2];
      pack_frags<F16>(ds, db_);
      pack_frags<F16>(sx, sb);
#pragma unroll
      for (int db = 0; db < DB; ++db) dq[db] = careful_mfma<HD, F16>(rd, r0.k, db, db_, sb, dq[db]);
    }
  }
  if (!live) return;
  const float x = (CAP != kNoCap ? 4.0f : 1.0f) * p.sm_scale * (F16 ? 1.0f / sc.s : 1.0f);
  if (piece.part >= 0) {
    float* P = p.qpart + ((int64_t)piece.part * kMRows + wave * 32 + l32) * HD;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(P + db * 32 + 8 * g + 4 * hi) =
            f32x4{dq[db][4 * g] * x, dq[db][4 * g + 1] * x, dq[db][4 * g + 2] * x, dq[db][4 * g + 3] * x};
    return;
  }
  uint16_t* DQ = p.dq + b * p.dq_sb + h * p.dq_sh + m_tok * p.dq_sm;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const bf16x2 a = pack2<F16>(dq[db][4 * g] * x, dq[db][4 * g + 1] * x);
      const bf16x2 c = pack2<F16>(dq[db][4 * g + 2] * x, dq[db][4 * g + 3] * x);
      *reinterpret_cast<u32x2*>(DQ + db * 32 + 8 * g + 4 * hi) =
          u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, c)};
    }
}

// The parts of blocks that were cut, added up: of dk and dv in the first `key_cuts`
// workgroups, then of dq; HD / 4 lanes a row.
template <int HD, bool F16>
__global__ __launch_bounds__(256) void attn_masked_grad_join_kernel(BwdArgs p, int key_cuts) {
  constexpr int L = HD / 4;
  const bool of_keys = (int)blockIdx.x < key_cuts;
  const int i = blockIdx.x - (of_keys ? 0 : key_cuts), kvh = i % p.Hk;
  const Deal* d = of_keys ? p.keys : p.rows;
  if (i / p.Hk >= d->cuts) return;
  const int4 c = d->cut[i / p.Hk];
  const int row = blockIdx.y * (256 / L) + threadIdx.x / L, at = threadIdx.x % L;
  const f32x4* P = reinterpret_cast<const f32x4*>(of_keys ? p.kpart : p.qpart) +
                   (((int64_t)c.z * p.Hk + kvh) * kMRows + row) * L + at;
  f32x4 x = P[0];
#pragma unroll 4
  for (int k = 1; k < c.y; ++k) x += P[(int64_t)k * p.Hk * kMRows * L];
  uint16_t* to;
  if (of_keys) {
    const int blocks = (p.mask.N + kKeys - 1) / kKeys, b = c.x / blocks;
    const int64_t j = c.x % blocks * kKeys + row % kKeys;
    if (j >= p.mask.N) return;
    to = row < kKeys ? p.dk + b * p.dk_sb + kvh * p.dk_sh + j * p.dk_sn
                     : p.dv + b * p.dv_sb + kvh * p.dv_sh + j * p.dv_sn;
  } else {
    const int blocks = (p.R + kMRows - 1) / kMRows, b = c.x / blocks, r = c.x % blocks * kMRows + row;
    if (r >= p.R) return;
    to = p.dq + b * p.dq_sb + ((int64_t)kvh * p.G + r % p.G) * p.dq_sh + (int64_t)(r / p.G) * p.dq_sm;
  }
  const bf16x2 lo = pack2<F16>(x[0], x[1]), hi = pack2<F16>(x[2], x[3]);
  *reinterpret_cast<u32x2*>(to + 4 * at) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// Workgroups that are resident at once.
template <int HD> constexpr int kKeySpans = kCus * (HD == 64 ? 2 : 1);
constexpr int kRowSpans = kCus * 2;

template <int HD, bool F16, Cap CAP, bool SLOPE>
hipError_t launch_one(const BwdArgs& a, int64_t problems, hipStream_t s) {
  const int64_t kb = (a.mask.N + kKeys - 1) / kKeys, qb = (a.R + kMRows - 1) / kMRows, B = problems / a.Hk;
  // As in the forward: a head's pieces are fewer than its blocks and spans / Hk.
  const int64_t k_cuts = kKeySpans<HD> / a.Hk * a.Hk, q_cuts = kRowSpans / a.Hk * a.Hk;
  hipError_t e;
  if (a.rows) {
    e = deal_out(a.mask, (int)B, a.Hk, a.G, {const_cast<Deal*>(a.rows), (int)qb, kRowSpans},
                 {const_cast<Deal*>(a.keys), (int)kb, kKeySpans<HD>}, s);
    if (e != hipSuccess) return e;
  }
  if (kb > 0)
    hipLaunchKernelGGL((attn_masked_dkdv_kernel<HD, F16, CAP, SLOPE>),
                       dim3((unsigned)(kb * problems + (a.keys ? k_cuts : 0))), dim3(kMThreads), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_masked_dq_kernel<HD, F16, CAP, SLOPE>),
                     dim3((unsigned)(qb * problems + (a.rows ? q_cuts : 0))), dim3(kMThreads), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || !a.rows || k_cuts + q_cuts == 0) return e;
  hipLaunchKernelGGL((attn_masked_grad_join_kernel<HD, F16>), dim3((unsigned)(k_cuts + q_cuts), kMRows * HD / 4 / 256),
                     dim3(256), 0, s, a, (int)k_cuts);
  return hipGetLastError();
}

template <int HD, bool F16>
hipError_t launch(const BwdArgs& a, int64_t problems, Cap cap, hipStream_t s) {
  hipLaunchKernelGGL((attn_masked_delta_kernel<HD, F16>), dim3((unsigned)(problems * a.tiles)),
                     dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (cap == kWideCap) return a.slopes ? launch_one<HD, F16, kWideCap, true>(a, problems, s)
                                       : launch_one<HD, F16, kWideCap, false>(a, problems, s);
  if (cap == kNarrowCap) return a.slopes ? launch_one<HD, F16, kNarrowCap, true>(a, problems, s)
                                         : launch_one<HD, F16, kNarrowCap, false>(a, problems, s);
  return a.slopes ? launch_one<HD, F16, kNoCap, true>(a, problems, s)
                  : launch_one<HD, F16, kNoCap, false>(a, problems, s);
}

// Whether the blocks are counted, cut and sorted first, as far as the rows decide it,
// and then.  It costs 17 us in all, and pays where the key blocks are few enough for
// the longest to decide (shared key heads above all).  Measured (us of all kernels,
// without and with; bf16, causal):
//   2 x 16 heads of 64 on 2 x 4, 2,048 tokens (256 key blocks)       157   115
//   8 of 64, 4,096 tokens (512)                                      143   122
//   16 of 64, 4,096 tokens (1,024)                                   177   184
//   8 of 64, 8,192 tokens (1,024)                                    315   305
//   4 x 16 of 64, 2,048 tokens, four documents (2,048)               131   152
//   8 of 128, 4,096 tokens (512)                                     247   214
//   2 x 16 of 128 on 2 x 4, 2,048 tokens, four documents (256)       229   185
bool may_deal(int64_t problems, int64_t B, int64_t R) {
  const int64_t qb = (R + kMRows - 1) / kMRows;
  return qb * problems >= 128 && R >= 2048 && R < (int64_t)1 << 24 && qb * B <= kDealItems;
}
bool deals(Unequal u, int64_t problems, int64_t B, int64_t R, int64_t N) {
  const int64_t kb = (N + kKeys - 1) / kKeys;
  return u != Unequal::no && may_deal(problems, B, R) && N >= 2048 && kb * problems < 4 * kCus && kb * B <= kDealItems;
}
size_t record_floats(int64_t problems, int64_t R) { return (size_t)problems * ((R + kRowTile - 1) / kRowTile) * kRec; }
// Parts of the lists at most: two for each resident workgroup.
template <int HD> constexpr size_t kKeyPart = (size_t)2 * kKeySpans<HD> * 2 * kKeys * HD;
template <int HD> constexpr size_t kRowPart = (size_t)2 * kRowSpans * kMRows * HD;

}  // namespace
}  // namespace gpa

using namespace gpa;

extern "C" size_t gpa_attn_masked_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t M) {
  if (B <= 0 || H <= 0 || Hk <= 0 || M <= 0 || H % Hk) return 0;
  const int64_t R = H / Hk * M;
  const size_t rec = record_floats(B * Hk, R) * sizeof(float);
  return may_deal(B * Hk, B, R) ? rec + 2 * sizeof(Deal) + (kKeyPart<128> + kRowPart<128>) * sizeof(float) : rec;
}

extern "C" int gpa_attn_masked_bwd(int dtype, const gpa_attn_masked_args* args,
                                   const gpa_attn_masked_grads* g, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_attn_masked_bwd";
  gpa_clear_error();
  const int rc = masked_check(fn, dtype, args, true);
  if (rc != GPA_OK) return rc;
  const gpa_attn_masked_args plain_args = masked_plain(args), *a = &plain_args;
  if (!g) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (a->P > 0 || a->lens) {
    gpa_set_error("%s: no gradients of a shared prefix or of padded batches by lens", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (a->B == 0 || a->H == 0 || a->M == 0) {
    if (a->B > 0 && a->Hk > 0 && a->N > 0 && a->H > 0 && (g->dk || g->dv)) {
      gpa_set_error("%s: no query, so dk and dv are zeros that the caller writes", fn);
      return GPA_E_INVALID;
    }
    return GPA_OK;
  }
  const bool keys = a->N > 0;
  if (!a->lse || !g->d_o || !g->dq || (keys && (!g->dk || !g->dv))) {
    gpa_set_error("%s: null pointer (lse, d_o, dq, dk, dv)", fn);
    return GPA_E_INVALID;
  }
  if (!rows_aligned(g->d_o, a->B, g->do_sb, a->H, g->do_sh, a->M, g->do_sm) ||
      !rows_aligned(g->dq, a->B, g->dq_sb, a->H, g->dq_sh, a->M, g->dq_sm) ||
      (keys && (!rows_aligned(g->dk, a->B, g->dk_sb, a->Hk, g->dk_sh, a->N, g->dk_sn) ||
                !rows_aligned(g->dv, a->B, g->dv_sb, a->Hk, g->dv_sh, a->N, g->dv_sn)))) {
    gpa_set_error("%s: rows must be 16-byte aligned", fn);
    return GPA_E_INVALID;
  }
  const int64_t G = a->H / a->Hk, problems = a->B * a->Hk;
  // A tile's 64 rows (at most 65 tokens, G heads) by 32-bit offsets below kNoRow.
  for (int i = 0; i < 2; ++i) {
    const int64_t sm = a->M < 2 ? a->D : i ? g->do_sm : a->q_sm, sh = G < 2 ? 0 : i ? g->do_sh : a->q_sh;
    if (sm < 0 || sh < 0 || (G - 1) * sh + (kRowTile + 1) * sm + a->D >= (int64_t)1 << 29) {
      gpa_set_error("%s: the query heads of a key head span 2^29 elements or more", fn);
      return GPA_E_UNSUPPORTED;
    }
  }
  const int64_t tiles = (a->M * G + kRowTile - 1) / kRowTile, kb = (a->N + kKeys - 1) / kKeys;
  if (problems * std::max({tiles, kb, (a->M * G + kMRows - 1) / kMRows}) > kMostWgs) {
    gpa_set_error("%s: too many rows", fn);
    return GPA_E_UNSUPPORTED;
  }
  const size_t need = gpa_attn_masked_bwd_workspace_bytes(a->B, a->H, a->Hk, a->M);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, need);
    return GPA_E_WORKSPACE;
  }
  BwdArgs f{};
  f.q = (const uint16_t*)a->q; f.k = (const uint16_t*)a->k; f.v = (const uint16_t*)a->v;
  f.o = (const uint16_t*)a->o; f.rest = (const uint16_t*)a->o_rest; f.d_o = (const uint16_t*)g->d_o;
  f.lse = a->lse; f.d_lse = g->d_lse;
  f.dq = (uint16_t*)g->dq; f.dk = (uint16_t*)g->dk; f.dv = (uint16_t*)g->dv;
  f.q_sb = a->q_sb; f.q_sh = a->q_sh; f.q_sm = a->q_sm;
  f.k_sb = a->k_sb; f.k_sh = a->k_sh; f.k_sn = a->k_sn;
  f.v_sb = a->v_sb; f.v_sh = a->v_sh; f.v_sn = a->v_sn;
  f.o_sb = a->o_sb; f.o_sh = a->o_sh; f.o_sm = a->o_sm;
  f.do_sb = a->B < 2 ? 0 : g->do_sb; f.do_sh = a->H < 2 ? 0 : g->do_sh; f.do_sm = a->M < 2 ? a->D : g->do_sm;
  f.dq_sb = g->dq_sb; f.dq_sh = g->dq_sh; f.dq_sm = g->dq_sm;
  f.dk_sb = g->dk_sb; f.dk_sh = g->dk_sh; f.dk_sn = g->dk_sn;
  f.dv_sb = g->dv_sb; f.dv_sh = g->dv_sh; f.dv_sn = g->dv_sn;
  f.lse_sb = a->lse_sb; f.lse_sh = a->lse_sh;
  f.slopes = a->slopes; f.slopes_sb = a->slopes_sb;
  f.rec = (float*)workspace;
  if (deals(unequal_of(*a), problems, a->B, a->M * G, a->N)) {
    Deal* d = (Deal*)(f.rec + record_floats(problems, a->M * G));
    f.rows = d;
    f.keys = d + 1;
    f.kpart = (float*)(d + 2);
    f.qpart = f.kpart + (a->D == 64 ? kKeyPart<64> : kKeyPart<128>);
  }
  f.Hk = (int32_t)a->Hk; f.G = (int32_t)G; f.R = (int32_t)(a->M * G); f.tiles = (int32_t)tiles;
  f.sm_scale = a->sm_scale;
  masked_fill(a, &f.mask, &f.score);
  const bool f16 = dtype == GPA_DTYPE_F16;
  const Cap cap = a->cap > (f16 ? kNarrow<true> : kNarrow<false>) ? kWideCap : a->cap > 0.f ? kNarrowCap : kNoCap;
  if (cap == kNarrowCap) f.lse_off = f.score.capl;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t e =
      a->D == 64 ? (f16 ? launch<64, true>(f, problems, cap, s) : launch<64, false>(f, problems, cap, s))
                 : (f16 ? launch<128, true>(f, problems, cap, s) : launch<128, false>(f, problems, cap, s));
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
