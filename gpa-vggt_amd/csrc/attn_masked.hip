// Masked attention, forward: packed documents, causal and prefix masks,
// tanh-capped scores, a bias by distance, shared key heads, and a prefix of
// keys that a whole batch shares (attn_masked.h has the formulas and the
// ranges that the masks are).
//
// attn_masked_kernel.  A workgroup has 128 rows (32 a wave) of one problem
// and walks the keys that any of them sees, 32 a tile, through a four-slot
// LDS ring filled by DMA three tiles ahead.  Scores are computed transposed,
// S^T = K . Q^T on v_mfma_f32_32x32x16, so that a lane owns one row and the
// softmax needs no exchange but one between lane halves; P^T is used in place
// as the B operand of O^T += V^T . P^T.  The softmax offset starts at the first
// tile's row max and moves only where a later one exceeds it by more than
// the format of P allows (64 for bf16, 15 for fp16, in log2 units).  Sums are
// fp32; P is rounded to the operand format for the product with V, as the
// framework's other attention does (its relative error, 2^-9 or 2^-12, is
// that of the output's own rounding).
//
// Few rows and many keys leave most of the chip without work: the key range
// of a block is then split over workgroups, whose unnormalised outputs, offsets
// and sums (fp32) attn_masked_join_kernel puts together.  A shared prefix
// is one more set of rows, those of all sequences, over its own keys, joined
// the same way.
//
// A masked key's value does not reach a row: its weight is zero, and where
// zero times it is not (an infinity or NaN), the workgroup finds a non-finite
// output at its end and walks its keys again, with such values taken out.
#include "attn_masked.h"

#include <algorithm>

namespace gpa {
namespace {

template <bool F16> constexpr float kUp = F16 ? 15.0f : 64.0f;

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

struct FwdArgs {
  const uint16_t* q;
  uint16_t* o;
  float* lse;             // nullable
  int64_t q_sb, q_sh, q_sm, o_sb, o_sh, o_sm, lse_sb, lse_sh;
  const float* slopes;
  int64_t slopes_sb;
  float* part;            // partial outputs [splits][rows][HD]; null: none
  float* stat;            // their (offset, sum) [splits][rows][2]
  int64_t rows;           // B * Hk * M * G
  int32_t B, Hk, G, splits;
  MaskArgs mask;
  ScoreArgs score;
  FwdSet set[2];          // the own keys; the shared prefix (no blocks: none)
};

template <int HD>
struct Slot {
  uint16_t k[kMTile * HD];
  uint16_t v[kMTile * HD];
};

template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, 2) void attn_masked_kernel(FwdArgs p) {
  constexpr int KS = HD / 16, DB = HD / 32, CH = HD / 8;
  constexpr int DJ = kMTile * CH / kMThreads;  // 16-byte DMAs per wave, tile and tensor
  __shared__ __attribute__((aligned(16))) Slot<HD> r0, r1, r2, r3;
  __shared__ int range[2][kMWaves];

  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int item = blockIdx.x;
  const int own_items = p.set[0].blocks * p.set[0].problems * p.set[0].splits;
  const bool second = item >= own_items;
  const FwdSet& S = p.set[second ? 1 : 0];
  if (second) item -= own_items;
  const int qb = item % S.blocks, prob = item / S.blocks % S.problems,
            z = item / S.blocks / S.problems;

  // This lane's row.
  const int r = qb * kMRows + wave * 32 + l32;
  const bool live = r < S.R;
  const int rc = live ? r : S.R - 1;
  const int per = p.mask.M * p.G;
  const int kvh = S.folded ? prob : prob % p.Hk;
  const int b = S.folded ? rc / per : prob / p.Hk;
  const int rr = S.folded ? rc % per : rc;
  const int m_tok = rr / p.G, h = kvh * p.G + rr % p.G;
  RowSpan span = row_span(p.mask, b, m_tok);
  if (S.folded) span = RowSpan{0, S.N, span.at + S.N};
  float slope = 0.f;
  if constexpr (SLOPE) slope = p.slopes[b * p.slopes_sb + h] * kMLog2e;

  bf16x8 qf[KS];
  {
    const uint16_t* Q = p.q + b * p.q_sb + h * p.q_sh + m_tok * p.q_sm;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(Q + 16 * ks + 8 * hi);
  }

  // The keys that this wave's rows see, and that the workgroup's do.
  const bool any = live && span.hi > span.lo;
  int w_lo = any ? span.lo : 0x7fffffff, w_hi = any ? span.hi : 0;   // some row's
  int a_lo = live ? span.lo : 0, a_hi = live ? span.hi : 0x7fffffff;  // every row's
  if (live && !any) a_hi = 0;
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
  if (n_hi <= n_lo) n_lo = n_hi = 0;           // nothing seen: no tile, empty DMAs
  const int all_tiles = n_hi > n_lo ? (n_hi - n_lo + kMTile - 1) / kMTile : 0;
  const int t_begin = (int)((int64_t)all_tiles * z / S.splits);
  const int t_end = (int)((int64_t)all_tiles * (z + 1) / S.splits);

  const int64_t kb = S.folded ? 0 : prob / p.Hk;
  const uint16_t* K = S.k + kb * S.k_sb + kvh * S.k_sh;
  const uint16_t* V = S.v + kb * S.v_sb + kvh * S.v_sh;
  uint32_t k_voff[DJ], v_voff[DJ];
#pragma unroll
  for (int j = 0; j < DJ; ++j) {
    const int pos = (wave * DJ + j) * 64 + lane, key = pos / CH;
    const uint32_t ch = (uint32_t)((pos % CH) ^ tile_swz<HD>(key)) * 16u;
    k_voff[j] = key * (uint32_t)(S.k_sn * 2) + ch;
    v_voff[j] = key * (uint32_t)(S.v_sn * 2) + ch;
  }
  // Tiles past the split's end are issued too, empty: the waits count them.
  const int n_end = min(n_lo + t_end * kMTile, n_hi);
  auto issue = [&](int t, Slot<HD>& T) {
    const int n0 = n_lo + t * kMTile;
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc<HD>(K, S.k_sn, n0, n_end);
    const __amdgpu_buffer_rsrc_t vr = tile_rsrc<HD>(V, S.v_sn, n0, n_end);
#pragma unroll
    for (int j = 0; j < DJ; ++j) m_dma16(kr, &T.k[(wave * DJ + j) * 512], k_voff[j]);
#pragma unroll
    for (int j = 0; j < DJ; ++j) m_dma16(vr, &T.v[(wave * DJ + j) * 512], v_voff[j]);
  };

  f32x16 o_acc[DB];
  float m, l;

  // Tile t's scores, in log2 units, -inf where the row does not see the key.
  auto scores = [&](const Slot<HD>& T, int n0, bool edge, float (&x)[16]) {
    f32x16 sv{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      sv = mfma32x32x16_t<F16>(row_frag<HD>(T.k, ks, l32, hi), qf[ks], sv);
    const float dist = (float)(span.at - n0 - 4 * hi);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = CAP ? cap_tanh(sv[i], p.score.c) * p.score.capl : sv[i] * p.score.c;
      if constexpr (SLOPE) y = __builtin_fmaf(-slope, fabsf(dist - (float)mfma_row(i, 0)), y);
      x[i] = y;
    }
    if (edge) {
      const int from = span.lo - n0 - 4 * hi, to = span.hi - n0 - 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (mfma_row(i, 0) < from || mfma_row(i, 0) >= to) x[i] = -INFINITY;
    }
  };
  auto weigh = [&](float (&x)[16]) {           // x to weights; m, l and O move
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    mx = max_halves(mx);
    const bool move = mx > m + kUp<F16>;
    if (__builtin_amdgcn_ballot_w64(move)) {
      const float m_new = move ? mx : m;
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o_acc[db] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - m);
      l += x[i];
    }
  };
  auto restart = [&]() {
    m = -1.0e30f;                              // finite: -inf - m is -inf
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o_acc[db] = f32x16{};
  };

  auto iter = [&](int t, const Slot<HD>& cur, Slot<HD>& dst) {
    m_wait<4 * DJ>();                          // tile t landed (two more in flight)
    __syncthreads();                           // ... for every wave; `dst` is free
    issue(t + 3, dst);
    const int n0 = n_lo + t * kMTile;
    if (n0 >= w_hi || n0 + kMTile <= w_lo) return;
    float x[16];
    scores(cur, n0, n0 < a_lo || n0 + kMTile > a_hi, x);
    weigh(x);
    bf16x8 pb[2];
    pack_frags<F16>(x, pb);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        o_acc[db] = mfma32x32x16_t<F16>(tr_frag<HD>(cur.v, lane, db, s), pb[s], o_acc[db]);
  };
  restart();
  issue(t_begin, r0);
  issue(t_begin + 1, r1);
  issue(t_begin + 2, r2);
  for (int t = t_begin; t < t_end; t += 4) {
    iter(t, r0, r3);
    if (t + 1 >= t_end) break;
    iter(t + 1, r1, r0);
    if (t + 2 >= t_end) break;
    iter(t + 2, r2, r1);
    if (t + 3 >= t_end) break;
    iter(t + 3, r3, r2);
  }
  m_wait<0>();                                 // no DMA may land after the workgroup ends

  float total = sum_halves(l);
  bool odd = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd |= !(fabsf(o_acc[db][i]) < INFINITY);
  if (__syncthreads_or(odd && live)) {
    // Again, one tile at a time, without the values that a row does not see.
    restart();
    for (int t = t_begin; t < t_end; ++t) {
      __syncthreads();
      issue(t, r0);
      m_wait<0>();
      __syncthreads();
      const int n0 = n_lo + t * kMTile;
      float x[16], sx[16];
      scores(r0, n0, true, x);
      const int from = span.lo - n0 - 4 * hi, to = span.hi - n0 - 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sx[i] = mfma_row(i, 0) < from || mfma_row(i, 0) >= to ? 0.f : 1.f;
      weigh(x);
      bf16x8 pb[2], sb[2];
      pack_frags<F16>(x, pb);
      pack_frags<F16>(sx, sb);
#pragma unroll
      for (int db = 0; db < DB; ++db)
        o_acc[db] = careful_mfma<HD, F16>(r0.v, lane, db, pb, sb, o_acc[db]);
    }
    total = sum_halves(l);
  }
  if (!live) return;

  if (p.part) {
    const int64_t row = (((int64_t)b * p.Hk + kvh) * p.mask.M + m_tok) * p.G + (h - kvh * p.G);
    const int64_t at = (int64_t)(S.z0 + z) * p.rows + row;
    float* O = p.part + at * HD;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(O + db * 32 + 8 * g + 4 * hi) =
            f32x4{o_acc[db][4 * g], o_acc[db][4 * g + 1], o_acc[db][4 * g + 2], o_acc[db][4 * g + 3]};
    if (hi == 0) {
      p.stat[2 * at] = m;
      p.stat[2 * at + 1] = total;
    }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;   // no key seen: zeros
  uint16_t* O = p.o + b * p.o_sb + h * p.o_sh + m_tok * p.o_sm;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const bf16x2 lo = pack2<F16>(o_acc[db][4 * g + 0] * inv, o_acc[db][4 * g + 1] * inv);
      const bf16x2 up = pack2<F16>(o_acc[db][4 * g + 2] * inv, o_acc[db][4 * g + 3] * inv);
      *reinterpret_cast<u32x2*>(O + db * 32 + 8 * g + 4 * hi) =
          u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, up)};
    }
  if (p.lse && hi == 0)
    p.lse[b * p.lse_sb + h * p.lse_sh + m_tok] = total == 0.f ? -INFINITY : m + __log2f(total);
}

// One wave a row: the partial outputs of its splits put together.
template <int HD, bool F16>
__global__ __launch_bounds__(256) void attn_masked_join_kernel(FwdArgs p) {
  constexpr int E = HD / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int g = (int)(row % p.G);
  const int64_t t = row / p.G;
  const int m_tok = (int)(t % p.mask.M);
  const int64_t bh = t / p.mask.M, b = bh / p.Hk;
  const int h = (int)(bh % p.Hk) * p.G + g;

  // The splits' offsets and sums, one lane a split (64 at a time).
  float top = -INFINITY;
  for (int z = lane; z < p.splits; z += 64) top = fmaxf(top, p.stat[2 * (z * p.rows + row)]);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
  float total = 0.f, o[E] = {};
  for (int z0 = 0; z0 < p.splits; z0 += 64) {
    const int z = z0 + lane;
    float w = 0.f;
    if (z < p.splits) {
      const int64_t at = z * p.rows + row;
      w = __builtin_amdgcn_exp2f(p.stat[2 * at] - top);
      const float sum = p.stat[2 * at + 1];
      total = __builtin_fmaf(w, sum, total);
      if (sum == 0.f) w = 0.f;
    }
    const int n = min(64, p.splits - z0);
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl(w, i);
      const float* O = p.part + ((int64_t)(z0 + i) * p.rows + row) * HD;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(wi, O[lane * E + e], o[e]);
    }
  }
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) total += __shfl_xor(total, i);
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  uint16_t* O = p.o + b * p.o_sb + h * p.o_sh + m_tok * p.o_sm;
  if constexpr (E == 2) {
    const bf16x2 v = pack2<F16>(o[0] * inv, o[1] * inv);
    *reinterpret_cast<uint32_t*>(O + 2 * lane) = __builtin_bit_cast(uint32_t, v);
  } else {
    O[lane] = __builtin_bit_cast(uint16_t, f32_to_half<F16>(o[0] * inv));
  }
  if (p.lse && lane == 0)
    p.lse[b * p.lse_sb + h * p.lse_sh + m_tok] = total == 0.f ? -INFINITY : top + __log2f(total);
}

template <int HD, bool F16>
hipError_t launch(const FwdArgs& a, bool cap, hipStream_t s) {
  int64_t items = 0;
  for (const FwdSet& t : a.set) items += (int64_t)t.blocks * t.problems * t.splits;
  const dim3 grid((unsigned)items), block(kMThreads);
  if (cap && a.slopes) hipLaunchKernelGGL((attn_masked_kernel<HD, F16, true, true>), grid, block, 0, s, a);
  else if (cap) hipLaunchKernelGGL((attn_masked_kernel<HD, F16, true, false>), grid, block, 0, s, a);
  else if (a.slopes) hipLaunchKernelGGL((attn_masked_kernel<HD, F16, false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((attn_masked_kernel<HD, F16, false, false>), grid, block, 0, s, a);
  if (a.part) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_masked_join_kernel<HD, F16>), dim3((unsigned)((a.rows + 3) / 4)),
                       dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

// Splits of a set's key range.  A workgroup walks its keys alone, so few row
// blocks over many keys are bound by one workgroup's walk; kWant workgroups
// (two a CU) fill the chip.  A split has at least kLeast tiles: below that
// the join costs what the shorter walk saves.
constexpr int64_t kWant = 512, kLeast = 8;
int splits_of(int64_t items, int64_t keys) {
  const int64_t tiles = (keys + kMTile - 1) / kMTile;
  int64_t z = items > 0 ? kWant / items : 1;
  z = std::min(z, tiles / kLeast);
  return (int)std::max<int64_t>(z, 1);
}

struct Plan { int blocks, problems, splits, p_blocks, p_problems, p_splits; };
Plan plan(int64_t B, int64_t Hk, int64_t G, int64_t M, int64_t N, int64_t P) {
  Plan x{};
  x.blocks = (int)((M * G + kMRows - 1) / kMRows);
  x.problems = (int)(B * Hk);
  if (P > 0) {
    x.p_blocks = (int)((B * M * G + kMRows - 1) / kMRows);
    x.p_problems = (int)Hk;
    x.p_splits = splits_of((int64_t)x.p_blocks * Hk, P);
  }
  x.splits = splits_of((int64_t)x.blocks * x.problems, N);
  return x;
}

}  // namespace
}  // namespace gpa

using namespace gpa;

int gpa::masked_check(const char* fn, int dtype, const gpa_attn_masked_args* a, bool has_o) {
  if (!a) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  if (dtype != GPA_DTYPE_BF16 && dtype != GPA_DTYPE_F16) {
    gpa_set_error("%s: dtype %d is not bf16 or fp16", fn, dtype);
    return GPA_E_INVALID;
  }
  if (a->B < 0 || a->H < 0 || a->Hk < 0 || a->M < 0 || a->N < 0 || a->P < 0 || a->docs < 0) {
    gpa_set_error("%s: negative size", fn);
    return GPA_E_INVALID;
  }
  if (a->D != 64 && a->D != 128) {
    gpa_set_error("%s: head dim %lld unsupported (64, 128)", fn, (long long)a->D);
    return GPA_E_UNSUPPORTED;
  }
  if (a->H > 0 && (a->Hk == 0 || a->H % a->Hk != 0)) {
    gpa_set_error("%s: %lld query heads do not share %lld key heads evenly", fn, (long long)a->H,
                  (long long)a->Hk);
    return GPA_E_INVALID;
  }
  if (!(a->sm_scale > 0.f) || !isfinite(a->sm_scale) || !(a->cap >= 0.f) || !isfinite(a->cap)) {
    gpa_set_error("%s: sm_scale must be finite and > 0, cap finite and >= 0", fn);
    return GPA_E_INVALID;
  }
  if (a->docs < 1 || (a->docs > 1 && (!a->q_offsets || !a->k_offsets)) ||
      ((a->lens || a->P > 0) && (a->docs != 1 || a->q_offsets || a->k_offsets))) {
    gpa_set_error("%s: several documents need both offsets; lens and a shared prefix go with one "
                  "document and no offsets", fn);
    return GPA_E_INVALID;
  }
  if ((a->prefix || a->prefix_len != 0) && (!a->causal || a->prefix_len < 0)) {
    gpa_set_error("%s: a visible prefix goes with the causal mask and is not negative", fn);
    return GPA_E_INVALID;
  }
  // Row numbers are 32-bit, and a block's first row beyond the last is formed.
  const int64_t lim = (int64_t)1 << 30;
  if (a->M >= lim || a->N >= lim || a->P >= lim || a->B * a->M >= lim || a->docs >= lim ||
      (a->Hk && a->B * a->M * (a->H / a->Hk) >= lim)) {
    gpa_set_error("%s: too many tokens", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (a->B == 0 || a->H == 0 || a->M == 0) return GPA_OK;
  const bool keys = a->N > 0, pre = a->P > 0;
  if (!a->q || (has_o && !a->o) || (keys && (!a->k || !a->v)) || (pre && (!a->pk || !a->pv))) {
    gpa_set_error("%s: null pointer", fn);
    return GPA_E_INVALID;
  }
  const int64_t B = a->B, H = a->H, Hk = a->Hk;
  if (!rows_aligned(a->q, B, a->q_sb, H, a->q_sh, a->M, a->q_sm) ||
      (has_o && !rows_aligned(a->o, B, a->o_sb, H, a->o_sh, a->M, a->o_sm)) ||
      (keys && (!rows_aligned(a->k, B, a->k_sb, Hk, a->k_sh, a->N, a->k_sn) ||
                !rows_aligned(a->v, B, a->v_sb, Hk, a->v_sh, a->N, a->v_sn))) ||
      (pre && (!rows_aligned(a->pk, 1, 0, Hk, a->pk_sh, a->P, a->pk_sn) ||
               !rows_aligned(a->pv, 1, 0, Hk, a->pv_sh, a->P, a->pv_sn)))) {
    gpa_set_error("%s: rows must be 16-byte aligned", fn);
    return GPA_E_INVALID;
  }
  // A tile's 32 rows are addressed by 32-bit offsets from its first one.
  const int64_t row_lim = (int64_t)1 << 23;
  const bool many = a->N > 1, pre_many = a->P > 1;
  for (const int64_t s : {many ? a->k_sn : 0, many ? a->v_sn : 0, pre_many ? a->pk_sn : 0,
                          pre_many ? a->pv_sn : 0})
    if (s < 0 || s >= row_lim) {
      gpa_set_error("%s: key row stride %lld unsupported (0 to 2^23)", fn, (long long)s);
      return GPA_E_UNSUPPORTED;
    }
  return GPA_OK;
}

gpa_attn_masked_args gpa::masked_plain(const gpa_attn_masked_args* a) {
  gpa_attn_masked_args x = *a;
  if (a->B < 2) x.q_sb = x.k_sb = x.v_sb = x.o_sb = x.lse_sb = x.slopes_sb = x.qo_sb = x.ko_sb = x.prefix_sb = 0;
  if (a->H < 2) x.q_sh = x.o_sh = x.lse_sh = 0;
  if (a->Hk < 2) x.k_sh = x.v_sh = x.pk_sh = x.pv_sh = 0;
  if (a->M < 2) x.q_sm = x.o_sm = a->D;
  if (a->N < 2) x.k_sn = x.v_sn = a->D;
  if (a->P < 2) x.pk_sn = x.pv_sn = a->D;
  return x;
}

void gpa::masked_fill(const gpa_attn_masked_args* a, MaskArgs* m, ScoreArgs* s) {
  m->q_off = a->q_offsets;
  m->k_off = a->k_offsets;
  m->lens = a->lens;
  m->prefix = a->prefix;
  m->qo_sb = a->qo_sb; m->ko_sb = a->ko_sb; m->prefix_sb = a->prefix_sb;
  m->docs = (int32_t)a->docs;
  m->prefix_len = (int32_t)std::min<int64_t>(a->prefix_len, a->N);
  m->causal = a->causal != 0;
  m->M = (int32_t)a->M;
  m->N = (int32_t)a->N;
  s->c = a->cap > 0.f ? 2.0f * kMLog2e * a->sm_scale / a->cap : a->sm_scale * kMLog2e;
  s->capl = a->cap * kMLog2e;
}

extern "C" size_t gpa_attn_masked_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t M,
                                                  int64_t N, int64_t P, int64_t D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || M <= 0 || N < 0 || P < 0 || H % Hk) return 0;
  const Plan x = plan(B, Hk, H / Hk, M, N, P);
  const int z = x.splits + x.p_splits;
  return z > 1 ? (size_t)z * B * H * M * (D + 2) * sizeof(float) : 0;
}

extern "C" int gpa_attn_masked(int dtype, const gpa_attn_masked_args* args, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_attn_masked";
  gpa_clear_error();
  const int rc = masked_check(fn, dtype, args, true);
  if (rc != GPA_OK) return rc;
  const gpa_attn_masked_args plain_args = masked_plain(args), *a = &plain_args;
  if (a->B == 0 || a->H == 0 || a->M == 0) return GPA_OK;
  const int64_t G = a->H / a->Hk;
  const Plan x = plan(a->B, a->Hk, G, a->M, a->N, a->P);
  const int64_t items = (int64_t)x.blocks * x.problems * x.splits +
                        (int64_t)x.p_blocks * x.p_problems * x.p_splits;
  const size_t need = gpa_attn_masked_workspace_bytes(a->B, a->H, a->Hk, a->M, a->N, a->P, a->D);
  if (items > 0x7fffffff || a->B * a->H * a->M >= (int64_t)1 << 31) {
    gpa_set_error("%s: too many rows", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, need);
    return GPA_E_WORKSPACE;
  }
  FwdArgs f{};
  f.q = (const uint16_t*)a->q;
  f.o = (uint16_t*)a->o;
  f.lse = a->lse;
  f.q_sb = a->q_sb; f.q_sh = a->q_sh; f.q_sm = a->q_sm;
  f.o_sb = a->o_sb; f.o_sh = a->o_sh; f.o_sm = a->o_sm;
  f.lse_sb = a->lse_sb; f.lse_sh = a->lse_sh;
  f.slopes = a->slopes;
  f.slopes_sb = a->slopes_sb;
  f.rows = a->B * a->H * a->M;
  f.B = (int32_t)a->B; f.Hk = (int32_t)a->Hk; f.G = (int32_t)G;
  f.splits = x.splits + x.p_splits;
  masked_fill(a, &f.mask, &f.score);
  if (need > 0) {
    f.part = (float*)workspace;
    f.stat = f.part + (int64_t)f.splits * f.rows * a->D;
  }
  FwdSet& own = f.set[0];
  own.k = (const uint16_t*)a->k; own.v = (const uint16_t*)a->v;
  own.k_sb = a->k_sb; own.k_sh = a->k_sh; own.k_sn = a->k_sn;
  own.v_sb = a->v_sb; own.v_sh = a->v_sh; own.v_sn = a->v_sn;
  own.N = (int32_t)a->N;
  own.R = (int32_t)(a->M * G);
  own.blocks = x.blocks; own.problems = x.problems; own.splits = x.splits; own.z0 = 0;
  FwdSet& pre = f.set[1];
  pre.k = (const uint16_t*)a->pk; pre.v = (const uint16_t*)a->pv;
  pre.k_sh = a->pk_sh; pre.k_sn = a->pk_sn; pre.v_sh = a->pv_sh; pre.v_sn = a->pv_sn;
  pre.N = (int32_t)a->P;
  pre.R = (int32_t)(a->B * a->M * G);
  pre.blocks = x.p_blocks; pre.problems = x.p_problems; pre.splits = x.p_splits;
  pre.z0 = x.splits; pre.folded = 1;
  const bool f16 = dtype == GPA_DTYPE_F16, cap = a->cap > 0.f;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t e = a->D == 64 ? (f16 ? launch<64, true>(f, cap, s) : launch<64, false>(f, cap, s))
                                  : (f16 ? launch<128, true>(f, cap, s) : launch<128, false>(f, cap, s));
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
