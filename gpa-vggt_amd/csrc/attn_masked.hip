// Masked attention, forward: packed documents, causal and prefix masks,
// tanh-capped scores, a bias by distance, shared key heads, and a prefix of
// keys that a whole batch shares (attn_masked.h has the formulas and the
// ranges that the masks are).
//
// Scores are computed transposed, S^T = K . Q^T on v_mfma_f32_32x32x16, so that a
// lane owns one row and the softmax needs no exchange but one between lane
// halves; P^T is used in place as the B operand of O^T += V^T . P^T.  The softmax
// offset starts at the first tile's row max and moves only where a later one
// exceeds it by more than the format of P allows (64 for bf16, 15 for fp16, in log2
// units): the largest |q.k| of a tile, and what a slope below zero adds to it at the
// tile's largest distance, bound its scores (caps and slopes above zero only lower
// them), so a tile's exact maximum is formed only where the bound passes that.
// Sums are fp32; P is rounded to the operand format for the product with V,
// as the framework's other attention does (its relative error, 2^-9 or 2^-12,
// is that of the output's own rounding).
//
// attn_masked_kernel, many rows: a workgroup has 128 rows (32 a wave) of one
// problem and walks the keys that any of them sees, 32 a tile, through a
// four-slot LDS ring filled by DMA; S of the next tile is computed beside the
// softmax of this one.
//
// attn_masked_few_kernel, up to 32 rows (new tokens): all four waves have the same
// rows, and each walks every fourth tile through buffers of its own, K's free again
// after the scores and V's after the product, with no barrier in the loop; their
// results are added up in LDS.
//
// Few rows and many keys leave most of the chip without work: the key range
// of a block is then split over workgroups, whose unnormalised outputs, offsets
// and sums (fp32) attn_masked_join_kernel puts together.  A shared prefix
// is one more set of rows, those of all sequences, over its own keys, joined
// the same way.
//
// Many rows under a mask: blocks see between none and all of the keys, and a launch
// lasts as long as the longest ones and what starts last.  Two small kernels count
// each block's tiles, cut the longest and list the pieces by length, and
// attn_masked_piece_kernel takes them in that order (`deals`).
//
// Measured (us a kernel after 200 passes; the first ten of a process take a tenth to a
// fifth longer): many rows, 289 at 16 heads of 64 and 10,992 tokens of four documents,
// capped (590 TFLOP/s), 92 at 2 x 16 heads of 128 on 2 x 4, 4,096 tokens of four causal
// documents, capped (540).  Bound by vector issue at head dim 64: four fifths of a busy
// SIMD's time with a cap or slopes, 710 cycles a tile of 32 x 32, of which the matrix
// instructions run 256.  At 128 vector issue takes 48 %, matrix instructions run 27 %, and
// two waves a SIMD do not hide all of the rest.  Few rows, 16 for one token over 130,001
// keys of 2 x 64 (4.1 TB/s) and 5 for the join; bound by HBM and a launch's start and end.
//
// A masked key's value does not reach a row: its weight is zero, and where
// zero times it is not (an infinity or NaN), the workgroup (the wave, where it
// walks alone) finds a non-finite output at its end and walks its keys again,
// with such values taken out.  Weights of up to 2^64 can also take finite bf16
// values out of fp32's range: an output that is still not below kBig is formed
// once more, with weights that no sum of finite values passes it with.
#include "attn_masked_deal.h"
#include "attn_masked_rows.h"

#include <algorithm>

namespace gpa {
namespace {

// Block qb of a problem: `share(tiles)` says which of its tiles are this workgroup's
// (x, y), `part(row)` where a row's part of the outputs goes.
template <int HD, bool F16, bool CAP, bool SLOPE, class Share, class ToPart>
__device__ __forceinline__ void walk(const FwdArgs& p, const FwdSet& S, int prob, int qb, Share share, ToPart part) {
  constexpr int CH = HD / 8;
  constexpr int DJ = kMTile * CH / kMThreads;  // 16-byte DMAs per wave, tile and tensor
  __shared__ __attribute__((aligned(16))) Slot<HD> r0, r1, r2, r3;
  __shared__ int range[2][kMWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Row row = locate(p, S, prob, qb * kMRows + wave * 32 + (lane & 31));
  Rows<HD, F16, CAP, SLOPE> R(p, row, lane);

  if (lane == 0) {
    range[0][wave] = row.w_lo;
    range[1][wave] = row.w_hi;
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
  const int all_tiles = (n_hi - n_lo + kMTile - 1) / kMTile;
  const int2 mine = share(all_tiles);
  const int t_begin = mine.x, t_end = mine.y;

  const int64_t kb = S.folded ? 0 : prob / p.Hk;
  const uint16_t* K = S.k + kb * S.k_sb + row.kvh * S.k_sh;
  const uint16_t* V = S.v + kb * S.v_sb + row.kvh * S.v_sh;
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

  // Iteration t: tile t in `cur`, its products in s; tile t + 1 in `nxt`; tile t + 3
  // issued into `dst`, the slot of tile t - 1, free once every wave passed the barrier.
  f32x16 s;
  auto iter = [&](int t, const Slot<HD>& cur, const Slot<HD>& nxt, Slot<HD>& dst) {
    m_wait_barrier<2 * DJ>();                  // tile t + 1 landed (t + 2 in flight) for every wave
    issue(t + 3, dst);
    R.rd.fresh();
    const int n0 = n_lo + t * kMTile;
    const bool edge = n0 < row.a_lo || n0 + kMTile > row.a_hi;
    if (n0 < row.w_hi && n0 + kMTile > row.w_lo) {
      const bool poly = R.settle(s, n0, edge);
      float x[16];
      R.template scores<false>(s, n0, poly, R.m, x);
      const f32x16 next = R.products(nxt.k);   // beside the exponentials
      R.weigh(n0, edge, x);
      R.add(cur.v, x);
      s = next;
    } else {
      s = R.products(nxt.k);
    }
  };
  R.restart();
  issue(t_begin, r0);
  issue(t_begin + 1, r1);
  issue(t_begin + 2, r2);
  m_wait_barrier<4 * DJ>();
  s = R.products(r0.k);
  for (int t = t_begin; t < t_end; t += 4) {
    iter(t, r0, r1, r3);
    if (t + 1 >= t_end) break;
    iter(t + 1, r1, r2, r0);
    if (t + 2 >= t_end) break;
    iter(t + 2, r2, r3, r1);
    if (t + 3 >= t_end) break;
    iter(t + 3, r3, r0, r2);
  }
  m_wait<0>();                                 // no DMA may land after the workgroup ends

  for (float up = kUp<F16>; __syncthreads_or(R.odd() && row.live); up = kDown) {
    R.restart();
    for (int t = t_begin; t < t_end; ++t) {
      __syncthreads();
      issue(t, r0);
      m_wait<0>();
      __syncthreads();
      R.careful(r0.k, r0.v, n_lo + t * kMTile, up);
    }
    if (F16 || up < 0.f) break;                // fp16's values times its weights are finite
  }
  R.finish(p, row, part(row), sum_halves(R.l), sum_halves(R.n));
}

// A block, or split z of it.
template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, kPerCu<HD>) void attn_masked_kernel(FwdArgs p, int which) {
  const FwdSet& S = p.set[which];
  const int z = blockIdx.x / (S.blocks * S.problems);
  int qb, prob;
  item_of(blockIdx.x % (S.blocks * S.problems), S.blocks, S.problems, qb, prob);
  walk<HD, F16, CAP, SLOPE>(
      p, S, prob, S.blocks - 1 - qb,
      [&](int tiles) { return int2{share_of(tiles, z, S.splits), share_of(tiles, z + 1, S.splits)}; },
      [&](const Row& x) { return split_part<HD>(p, S, x, z); });
}

// A piece of a block.  The heads of a sequence take the same piece together, each on
// an XCD of its own where they are a multiple of the eight.
template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, kPerCu<HD>) void attn_masked_piece_kernel(FwdArgs p) {
  const FwdSet& S = p.set[0];
  const int kvh = blockIdx.x % p.Hk, at = blockIdx.x / p.Hk;
  if (at >= p.deal->pieces) return;
  const int4 x = same(p.deal->piece[at]);
  walk<HD, F16, CAP, SLOPE>(
      p, S, x.x / S.blocks * p.Hk + kvh, x.x % S.blocks,
      [&](int tiles) { return int2{share_of(tiles, x.y, x.z), share_of(tiles, x.y + 1, x.z)}; },
      [&](const Row&) {
        if (x.w < 0) return Part{};
        return part_at<HD>(p, ((int64_t)x.w * p.Hk + kvh) * kMRows + (threadIdx.x >> 6) * 32 + (threadIdx.x & 31));
      });
}

// The pieces of a block that was cut, put together, HD / 4 lanes a row.
template <int HD, bool F16>
__global__ __launch_bounds__(256) void attn_masked_piece_join_kernel(FwdArgs p) {
  constexpr int L = HD / 4;
  const int kvh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk, nb = p.set[0].blocks;
  if (c >= p.deal->cuts) return;
  const int4 s = p.deal->cut[c];
  const int local = blockIdx.y * (256 / L) + threadIdx.x / L, at = threadIdx.x % L;
  const int r = s.x % nb * kMRows + local;
  if (r >= p.set[0].R) return;
  auto slot = [&](int i) { return ((int64_t)(s.z + i) * p.Hk + kvh) * kMRows + local; };
  const float2* stat = reinterpret_cast<const float2*>(p.stat);
  float top = -INFINITY, total = 0.f;
  for (int i = 0; i < s.y; ++i) top = fmaxf(top, stat[slot(i)].x);
  f32x4 o{};
#pragma unroll 4
  for (int i = 0; i < s.y; ++i) {
    const float2 t = stat[slot(i)];
    const f32x4 v = reinterpret_cast<const f32x4*>(p.part)[slot(i) * L + at];
    const float a = t.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(t.x - top);
    total = __builtin_fmaf(a, t.y, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a, v[e], o[e]);
  }
  const int64_t b = s.x / nb, h = (int64_t)kvh * p.G + r % p.G, tok = r / p.G;
  emit<F16>(p, b, h, tok, at, o, total);
  if (p.lse && at == 0)
    p.lse[b * p.lse_sb + h * p.lse_sh + tok] = total == 0.f ? -INFINITY : top + __log2f(total);
}

template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, HD == 64 ? 3 : 2) void attn_masked_few_kernel(FwdArgs p, int which) {
  constexpr int CH = HD / 8, DB = HD / 32;
  constexpr int DJ = kMTile * CH / 64;         // 16-byte DMAs per tile and tensor: one wave's
  constexpr int ROW = 64 / CH;                 // rows of a DMA
  __shared__ __attribute__((aligned(16))) uint16_t kt[kMWaves][kMTile * HD];
  __shared__ __attribute__((aligned(16))) uint16_t vt[kMWaves][kMTile * HD];
  __shared__ float stat[kMWaves][2][32];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const FwdSet& S = p.set[which];
  const int prob = blockIdx.x % S.problems, z = blockIdx.x / S.problems;
  const Row row = locate(p, S, prob, lane & 31);
  Rows<HD, F16, CAP, SLOPE> R(p, row, lane);
  const int n_lo = row.w_hi > row.w_lo ? row.w_lo : 0, n_hi = row.w_hi > row.w_lo ? row.w_hi : 0;
  const int all_tiles = (n_hi - n_lo + kMTile - 1) / kMTile;
  const int t_begin = share_of(all_tiles, z, S.splits) + wave, t_end = share_of(all_tiles, z + 1, S.splits);

  const int64_t kb = S.folded ? 0 : prob / p.Hk;
  const uint16_t* K = S.k + kb * S.k_sb + row.kvh * S.k_sh;
  const uint16_t* V = S.v + kb * S.v_sb + row.kvh * S.v_sh;
  uint16_t *kw = kt[wave], *vw = vt[wave];
  // Tiles past the wave's last one are issued too, empty: the waits count them.
  auto issue = [&](const uint16_t* base, int64_t stride, int t, uint16_t* T) {
    const __amdgpu_buffer_rsrc_t r = tile_rsrc<HD>(base, stride, n_lo + t * kMTile, t < t_end ? n_hi : 0);
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int key = j * ROW + lane / CH;
      m_dma16(r, T + j * 512, key * (uint32_t)(stride * 2) + (uint32_t)((lane % CH) ^ tile_swz<HD>(key)) * 16u);
    }
  };
  R.restart();
  issue(K, S.k_sn, t_begin, kw);
  issue(V, S.v_sn, t_begin, vw);
  for (int t = t_begin; t < t_end; t += kMWaves) {
    const int n0 = n_lo + t * kMTile;
    m_wait<DJ>();                              // K landed, V in flight
    const f32x16 s = R.products(kw);
    __builtin_amdgcn_s_waitcnt(0xc07f);        // lgkmcnt(0): K is read, its buffer free
    issue(K, S.k_sn, t + kMWaves, kw);
    const bool edge = n0 < row.a_lo || n0 + kMTile > row.a_hi;
    float x[16];
    const bool poly = R.settle(s, n0, edge);
    R.template scores<false>(s, n0, poly, R.m, x);
    R.weigh(n0, edge, x);
    m_wait<DJ>();                              // V landed, the next K in flight
    R.add(vw, x);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    issue(V, S.v_sn, t + kMWaves, vw);
  }
  m_wait<0>();
  for (float up = kUp<F16>; __builtin_amdgcn_ballot_w64(R.odd() && row.live); up = kDown) {
    R.restart();
    for (int t = t_begin; t < t_end; t += kMWaves) {
      issue(K, S.k_sn, t, kw);
      issue(V, S.v_sn, t, vw);
      m_wait<0>();
      R.careful(kw, vw, n_lo + t * kMTile, up);
      __builtin_amdgcn_s_waitcnt(0xc07f);
    }
    if (F16 || up < 0.f) break;
  }

  // The four waves' results in wave 0, by way of K's buffers, all at one offset.
  float total = sum_halves(R.l);
  const float norm = sum_halves(R.n), even = norm == 0.f ? 0.f : total / norm;
  if (lane < 32) {
    stat[wave][0][lane] = R.m;
    stat[wave][1][lane] = total;
  }
  __syncthreads();
  float m = stat[0][0][lane & 31];
#pragma unroll
  for (int i = 1; i < kMWaves; ++i) m = fmaxf(m, stat[i][0][lane & 31]);
  total = 0.f;
#pragma unroll
  for (int i = 0; i < kMWaves; ++i)
    total = __builtin_fmaf(__builtin_amdgcn_exp2f(stat[i][0][lane & 31] - m), stat[i][1][lane & 31], total);
  const float alpha = __builtin_amdgcn_exp2f(R.m - m) * even;
#pragma unroll
  for (int db = 0; db < DB; ++db) R.o[db] *= alpha;
  R.m = m;
  f32x4* ex = reinterpret_cast<f32x4*>(&kt[0][0]) + lane;   // [2][DB * 4][64]
  auto give = [&](int at) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        ex[(at * DB * 4 + db * 4 + g) * 64] = f32x4{R.o[db][4 * g], R.o[db][4 * g + 1], R.o[db][4 * g + 2],
                                                   R.o[db][4 * g + 3]};
  };
  auto take = [&](int at) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = ex[(at * DB * 4 + db * 4 + g) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) R.o[db][4 * g + e] += v[e];
      }
  };
  if (wave >= 2) give(wave - 2);
  __syncthreads();
  if (wave < 2) take(wave);
  __syncthreads();
  if (wave == 1) give(0);
  __syncthreads();
  if (wave > 0) return;
  take(0);
  R.finish(p, row, split_part<HD>(p, S, row, z), total, total);
}

// The partial outputs of a row's splits put together, by WAVES waves.
constexpr int kMaxSplits = 512;
template <int HD, bool F16, int WAVES>
__global__ __launch_bounds__(256) void attn_masked_join_kernel(FwdArgs p) {
  constexpr int ROWS = 4 / WAVES, T = WAVES * 64, L = HD / 4, GR = T / L;   // L lanes have the row once
  constexpr int MAXZ = WAVES == 1 ? 16 : kMaxSplits;
  __shared__ float weight[ROWS][MAXZ];
  __shared__ float red[4];
  __shared__ f32x4 acc[4][L];
  const int slot = threadIdx.x / T, tid = threadIdx.x % T, lane = tid & 63, wave = threadIdx.x >> 6;
  const int64_t row = std::min((int64_t)blockIdx.x * ROWS + slot, p.rows - 1);
  auto over = [&](float v, auto op) {          // over the row's lanes
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) v = op(v, __shfl_xor(v, i));
    if constexpr (WAVES > 1) {
      __syncthreads();
      if (lane == 0) red[wave] = v;
      __syncthreads();
      v = op(op(red[0], red[1]), op(red[2], red[3]));
    }
    return v;
  };
  constexpr int PER = (MAXZ + T - 1) / T;
  float m[PER], l[PER], top = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int z = tid + i * T;
    m[i] = -INFINITY;
    l[i] = 0.f;
    if (z < p.splits) {
      const float2 s = reinterpret_cast<const float2*>(p.stat)[z * p.rows + row];
      m[i] = s.x;
      l[i] = s.y;
    }
    top = fmaxf(top, m[i]);
  }
  top = over(top, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int z = tid + i * T;
    const float w = l[i] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[i] - top);
    total = __builtin_fmaf(w, l[i], total);
    if (z < p.splits) weight[slot][z] = w;
  }
  total = over(total, [](float a, float b) { return a + b; });
  __syncthreads();
  const int at = tid % L, group = tid / L;
  f32x4 o{};
  const f32x4* P = reinterpret_cast<const f32x4*>(p.part) + row * L + at;
#pragma unroll 4
  for (int z = group; z < p.splits; z += GR) {
    const f32x4 v = P[(int64_t)z * p.rows * L];
    const float w = weight[slot][z];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
  }
#pragma unroll
  for (int i = L; i < 64; i <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], i);
  if constexpr (WAVES > 1) {
    if (lane < L) acc[wave][at] = o;
    __syncthreads();
    o = acc[0][at];
#pragma unroll
    for (int i = 1; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += acc[i][at][e];
  }
  if (tid >= L || (int64_t)blockIdx.x * ROWS + slot >= p.rows) return;
  const int g = (int)(row % p.G);
  const int64_t t = row / p.G, tok = t % p.mask.M, b = t / p.mask.M / p.Hk;
  const int64_t h = t / p.mask.M % p.Hk * p.G + g;
  emit<F16>(p, b, h, tok, at, o, total);
  if (p.lse && at == 0)
    p.lse[b * p.lse_sb + h * p.lse_sh + tok] = total == 0.f ? -INFINITY : top + __log2f(total);
}

template <int HD, bool F16, bool CAP, bool SLOPE>
hipError_t launch_sets(const FwdArgs& a, hipStream_t s) {
  if (a.deal) {
    const int spans = kCus * kPerCu<HD>, Hk = a.Hk;
    hipError_t e = deal_out(a.mask, a.B, Hk, a.G, {a.deal, a.set[0].blocks, spans}, {}, s);
    if (e != hipSuccess) return e;
    // A head has fewer cut blocks than spans / Hk, and at most that many pieces more than blocks.
    const unsigned most = (unsigned)(a.B * a.set[0].blocks + spans / Hk) * Hk, cuts = (unsigned)(spans / Hk) * Hk;
    hipLaunchKernelGGL((attn_masked_piece_kernel<HD, F16, CAP, SLOPE>), dim3(most), dim3(kMThreads), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess || cuts == 0) return e;
    hipLaunchKernelGGL((attn_masked_piece_join_kernel<HD, F16>), dim3(cuts, kMRows * HD / 4 / 256), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  for (int i = 1; i >= 0; --i) {               // the prefix, then the own keys
    const FwdSet& t = a.set[i];
    const unsigned items = (unsigned)t.blocks * t.problems * t.splits;
    if (items == 0) continue;
    if (t.R <= 32)
      hipLaunchKernelGGL((attn_masked_few_kernel<HD, F16, CAP, SLOPE>), dim3(items), dim3(kMThreads), 0, s, a, i);
    else
      hipLaunchKernelGGL((attn_masked_kernel<HD, F16, CAP, SLOPE>), dim3(items), dim3(kMThreads), 0, s, a, i);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int HD, bool F16>
hipError_t launch(const FwdArgs& a, bool cap, hipStream_t s) {
  const hipError_t e = cap ? (a.slopes ? launch_sets<HD, F16, true, true>(a, s) : launch_sets<HD, F16, true, false>(a, s))
                           : (a.slopes ? launch_sets<HD, F16, false, true>(a, s) : launch_sets<HD, F16, false, false>(a, s));
  if (e != hipSuccess || a.deal || !a.part) return e;
  // A wave a row reads a few splits, four waves many.
  if (a.splits <= 16)
    hipLaunchKernelGGL((attn_masked_join_kernel<HD, F16, 1>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attn_masked_join_kernel<HD, F16, 4>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

// Splits of a set's key range.  A workgroup walks its keys alone, so few row
// blocks over many keys are bound by one workgroup's walk; two workgroups a CU fill
// the chip, and three of 128 rows at head dim 64 (16 heads over 32,771 shared keys:
// 46 us on 512 workgroups, 38 on 768; the few-row kernel, whose waves walk alone,
// gains nothing from them).  A split has at least kLeast tiles: below that the join
// costs what the shorter walk saves.
int splits_of(int64_t items, int64_t rows, int64_t keys, int64_t D) {
  const int64_t tiles = (keys + kMTile - 1) / kMTile;
  const int64_t want = kCus * (rows > 32 && D == 64 ? kPerCu<64> : 2);
  const int64_t z = std::min({items > 0 ? want / items : 1, tiles / kLeast, (int64_t)kMaxSplits / 2});
  return (int)std::max<int64_t>(z, 1);
}

// Whether a launch's blocks are counted, cut and sorted first.  That takes two small
// kernels and a join, 10 to 15 us, and pays where the mask makes blocks unequal and their
// number is between what the splits above fill the chip with and what evens
// itself out.  Measured (us, without and with; bf16):
//   one causal document, 8 heads of 64, 4,096 tokens (256 blocks)     71    52
//   16 of 64, 4,096 tokens (512)                                      78    71
//   2 x 16 of 64, 4,096 tokens (1,024)                               100   111
//   8 of 128, 4,096 tokens (256)                                      85    66
//   16 of 128, 4,096 tokens (512)                                    102   106
//   four documents, 16 of 64, 10,992 tokens (1,376)                  417   330
//   three documents, 4 x 16 of 64, 4,096 tokens (2,048)              129   130
bool deals(Unequal u, int64_t P, int64_t rows, int64_t items, int64_t entries, int64_t N, int64_t spans) {
  const int64_t tiles = (N + kMTile - 1) / kMTile;
  if (u == Unequal::no || P > 0 || rows <= 32 || items < 128 || tiles < 64) return false;
  if (entries > kDealItems || N >= (int64_t)1 << 24) return false;   // the list's length; 32-bit sums
  return u == Unequal::documents ? items <= 2 * spans : 2 * items <= spans || (items < spans && tiles >= 128);
}

struct Plan {
  int blocks, problems, splits, p_blocks, p_problems, p_splits;
  bool deal;
  size_t parts, bytes;    // parts of a row of outputs, workspace
};
Plan plan(int64_t B, int64_t Hk, int64_t G, int64_t M, int64_t N, int64_t P, int64_t D, Unequal unequal) {
  Plan x{};
  x.blocks = (int)((M * G + kMRows - 1) / kMRows);
  x.problems = (int)(B * Hk);
  if (P > 0) {
    x.p_blocks = (int)((B * M * G + kMRows - 1) / kMRows);
    x.p_problems = (int)Hk;
    x.p_splits = splits_of((int64_t)x.p_blocks * Hk, B * M * G, P, D);
  }
  x.splits = splits_of((int64_t)x.blocks * x.problems, M * G, N, D);
  const int64_t items = (int64_t)x.blocks * x.problems, spans = kCus * (D == 64 ? kPerCu<64> : kPerCu<128>);
  x.deal = deals(unequal, P, M * G, items, B * x.blocks, N, spans);
  if (x.deal) x.splits = 1;
  const int z = x.splits + x.p_splits;
  x.parts = x.deal ? (size_t)(2 * spans * kMRows) : z > 1 ? (size_t)z * B * Hk * G * M : 0;
  x.bytes = x.parts * (D + 2) * sizeof(float) + (x.deal ? sizeof(Deal) : 0);
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
      (has_o && (!rows_aligned(a->o, B, a->o_sb, H, a->o_sh, a->M, a->o_sm) || (uintptr_t)a->o_rest % 16)) ||
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
  s->c1 = a->sm_scale * kMLog2e;
  if (a->cap > 0.f) {
    const double g = (double)a->sm_scale / a->cap, l2e = 1.4426950408889634;
    s->ce = (float)std::min(2.0 * l2e * g, 1e38);   // times a product of 0: 0
    s->capl = a->cap * kMLog2e;
    s->lim = (float)std::min(kPolyMax / g, 1e18);   // s^2 stays finite
    s->half = (float)(0.5 / (l2e * a->cap));
    double scale = a->sm_scale * l2e;
    for (int i = 0; i < 4; ++i, scale *= g * g) s->poly[i] = (float)(kPoly[i] * scale);
    if (!isfinite(s->poly[3])) s->lim = -1.f;   // a cap so small that no product but 0 would take them
  }
}

extern "C" size_t gpa_attn_masked_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t M,
                                                  int64_t N, int64_t P, int64_t D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || M <= 0 || N < 0 || P < 0 || H % Hk) return 0;
  size_t most = 0;                             // whatever the mask
  for (const Unequal u : {Unequal::no, Unequal::causal, Unequal::documents})
    most = std::max(most, plan(B, Hk, H / Hk, M, N, P, D, u).bytes);
  return most;
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
  const Plan x = plan(a->B, a->Hk, G, a->M, a->N, a->P, a->D, unequal_of(*a));
  const int64_t items = (int64_t)x.blocks * x.problems * x.splits +
                        (int64_t)x.p_blocks * x.p_problems * x.p_splits;
  const size_t need = x.bytes;
  // A launch has less than 2^32 threads; the join has a wave a row.
  const int64_t rows = a->B * a->H * a->M;
  if (items > kMostWgs || rows >= (int64_t)1 << 31 || (need > 0 && !x.deal && rows > kMostWgs * 4)) {
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
  f.rest = (uint16_t*)a->o_rest;
  f.lse = a->lse;
  f.q_sb = a->q_sb; f.q_sh = a->q_sh; f.q_sm = a->q_sm;
  f.o_sb = a->o_sb; f.o_sh = a->o_sh; f.o_sm = a->o_sm;
  f.lse_sb = a->lse_sb; f.lse_sh = a->lse_sh;
  f.slopes = a->slopes;
  f.slopes_sb = a->slopes_sb;
  f.rows = rows;
  f.B = (int32_t)a->B; f.Hk = (int32_t)a->Hk; f.G = (int32_t)G;
  f.splits = x.splits + x.p_splits;
  masked_fill(a, &f.mask, &f.score);
  if (need > 0) {
    f.part = (float*)workspace;
    f.stat = f.part + x.parts * a->D;
    if (x.deal) f.deal = (Deal*)(f.stat + x.parts * 2);
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
