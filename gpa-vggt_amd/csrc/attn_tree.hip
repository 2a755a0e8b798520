// Attention of drafted tokens over their sequence's cache and over each other, a tree
// of them for each sequence: the step that checks a draft.
//
//   s_ij = score(q_i . k_j) - slope_h |p_i - p_j|         (attn_masked.h: scale, cap, slopes)
//   o_i  = sum_j softmax_j(s_ij) v_j,  j: the cache's first `length` keys, and the
//          drafted tokens that i's row of bits names (its ancestors and itself)
//
// Positions: key j of the cache stands at j, a drafted token at length + depth, its depth
// being one less than its bits; so token i lies as far from a drafted token j that it sees
// as it sees tokens behind j, which the bits alone tell.  (Of a tree's bits, in which a row has its token's
// ancestors and itself.  Any others are taken as masks; by a slope they are weighed as if they were a tree's.)
//
// gpa_draft_tree makes the bits and the positions from the tokens' parents, once a step:
// a thread a token walks up its ancestors, whose numbers fall, so its words fill from the
// last to the first.
//
// The attention.  Rows are (token, head of the group) of one sequence and key head, as
// in the masked attention, whose row code this is (attn_masked_rows.h): S^T = K Q^T, 32-key
// tiles by DMA, 128 rows a workgroup through a ring of four slots or up to 32 rows with a
// buffer a wave.  A walk's tiles are the cache's, which need no mask but behind the last
// key, then the drafted keys', 32 to a word of bits, whose exact maximum is formed.
//
// Caches are of unequal length and known on the device alone.  Every workgroup adds
// up the sequences' tiles and finds its own piece of one of them: pieces of at most S tiles, S so
// that all together fill the chip once (piece_tiles); a sequence in one piece writes its outputs
// itself, the others' pieces are joined.  No list is made before, no order of arrival matters.
//
// What bounds it: up to about 128 rows a key head the cache's bytes (8 sequences of 8,192 keys, 8 key
// heads of 128, 128 rows of each: 67 us and 8 for the join, 4.0 TB/s), above them vector issue and products
// in turn (256 rows: 97 + 11 us, 1.2 us a tile of two workgroups and 18 us of starts and ends).
#include "attn_masked.h"
#include "attn_masked_rows.h"

#include <algorithm>

namespace gpa {
namespace {

constexpr int kTreeCus = 256;
constexpr int kLeastTiles = 8;           // of a piece
// Sequences are cut where the caches' buffer has more tiles than this: the host knows its size and not
// the lengths, so short sequences in a long buffer are cut and joined too.  A launch for the join is worth
// 30 tiles to up to 32 rows (22 tiles whole 10.1 us, cut 11.9; 63 whole 15.5, cut 12.0) and 12 to more
// (head dim 64, 10 tiles 13.3 and 15.4, 17 tiles 16.6 and 15.5).
constexpr int kSplitFew = 32, kSplitMany = 12;
constexpr int64_t kMaxDraft = 1024;

struct TreeArgs {
  FwdArgs f;              // set[0]: the cache, set[1]: the drafted keys
  const uint32_t* seen;   // [B][T][words]
  int64_t seen_sb, seen_st;
  const int32_t* lens;    // nullable: all of the cache
  int32_t T, words, R, blocks, target, most;
  int32_t* firsts;        // [B + 1]: a sequence's first piece, for the join (null: none)
};

struct Where { int b, z, count, first, tiles, len; };

__device__ __forceinline__ int cache_len(const TreeArgs& p, int b) {
  const int N = p.f.set[0].N;
  return p.lens ? clampi(p.lens[b], 0, N) : N;
}
__device__ __forceinline__ int seq_tiles(const TreeArgs& p, int b) {
  return (cache_len(p, b) + kMTile - 1) / kMTile + (p.T + kMTile - 1) / kMTile;
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) v += __shfl_xor(v, i);
  return __builtin_amdgcn_readfirstlane(v);
}
// Tiles of a piece at most.  With fewer sequences than `target` pieces to fill the chip with: the
// least that gives no more than these (a sequence's last piece rounds up, so one even share is
// seldom enough); otherwise the chip is full, and only sequences a quarter longer than the mean are
// cut.  No sequence has more than `most` pieces.
__device__ __forceinline__ int piece_tiles(const TreeArgs& p) {
  const int lane = threadIdx.x & 63;
  int all = 0, top = 0;
  for (int b = lane; b < p.f.B; b += 64) {
    const int t = seq_tiles(p, b);
    all += t;
    top = max(top, t);
  }
  all = wave_sum(all);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) top = max(top, __shfl_xor(top, i));
  top = __builtin_amdgcn_readfirstlane(top);
  int S = max(kLeastTiles, (top + p.most - 1) / p.most);
  if (p.f.B >= p.target) return max(S, (int)((5 * (int64_t)all / 4 + p.f.B - 1) / p.f.B));
  S = max(S, (all + p.target - 1) / p.target);
  while (S < top) {
    int n = 0;
    for (int b = lane; b < p.f.B; b += 64) n += (seq_tiles(p, b) + S - 1) / S;
    n = wave_sum(n);
    if (n <= p.target) break;
    S = max(S + 1, (int)((int64_t)S * n / p.target));
  }
  return S;
}
// Piece `at` of all sequences' (b = -1: there are not so many).  With `list` their firsts are written down.
__device__ __forceinline__ Where find_piece(const TreeArgs& p, int at, bool list) {
  const int lane = threadIdx.x & 63, S = piece_tiles(p);
  Where w{-1, 0, 0, 0, 0, 0};
  int before = 0;
  for (int base = 0; base < p.f.B && (list || w.b < 0); base += 64) {
    const int tiles = base + lane < p.f.B ? seq_tiles(p, base + lane) : 0, n = (tiles + S - 1) / S;
    int upto = n;                              // pieces up to this sequence's
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const int v = __shfl_up(upto, i);
      if (lane >= i) upto += v;
    }
    if (list && base + lane < p.f.B) p.firsts[base + lane + 1] = before + upto;
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > at);
    if (past && w.b < 0) {
      const int l = __builtin_ctzll(past);
      w.b = base + l;
      w.count = __builtin_amdgcn_readlane(n, l);
      w.first = before + __builtin_amdgcn_readlane(upto, l) - w.count;
      w.z = at - w.first;
      w.tiles = __builtin_amdgcn_readlane(tiles, l);
      w.len = __builtin_amdgcn_readfirstlane(cache_len(p, w.b));
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (list) p.firsts[0] = 0;
  return w;
}

// Row r; `blind`: it sees nothing, computes with a query of zeros, and its results are dropped (its
// keys are not masked, so that the others' tiles need no mask for it).
struct Drafted : Row { const uint32_t* bits; bool blind; };
__device__ __forceinline__ Drafted locate_drafted(const TreeArgs& p, const Where& w, int kvh, int r) {
  Drafted x;
  x.live = r < p.R;
  const int rc = x.live ? r : p.R - 1;
  x.kvh = kvh;
  x.b = w.b;
  x.tok = rc / p.f.G;
  x.h = kvh * p.f.G + rc % p.f.G;
  x.bits = p.seen + x.b * p.seen_sb + x.tok * p.seen_st;
  int n = 0;
  for (int i = 0; i < p.words; ++i) n += __popc(i == p.words - 1 ? x.bits[i] & (0xffffffffu >> (31 & (32 * p.words - p.T))) : x.bits[i]);
  x.blind = !x.live || n == 0;                 // a token that sees no drafted one sees nothing
  x.lo = x.w_lo = x.a_lo = 0;
  x.hi = x.a_hi = w.len;
  x.at = w.len + n - 1;
  x.w_hi = __builtin_amdgcn_ballot_w64(!x.blind) ? w.len : 0;
  return x;
}

template <int HD, bool F16, bool CAP, bool SLOPE>
struct TreeRows : Rows<HD, F16, CAP, SLOPE> {
  typedef Rows<HD, F16, CAP, SLOPE> Base;
  using Base::hi; using Base::m; using Base::l; using Base::n; using Base::o; using Base::rd; using Base::slope;
  using Base::end; using Base::at;
  const TreeArgs& p;
  const uint32_t* bits;
  bool live;
  __device__ __forceinline__ TreeRows(const TreeArgs& args, const Drafted& x, int lane)
      : Base(args.f, x, lane), p(args), bits(x.bits), live(!x.blind) {
    if (x.blind)
#pragma unroll
      for (int ks = 0; ks < Base::KS; ++ks) Base::qf[ks] = bf16x8{};
  }
  __device__ __forceinline__ bool lost() const { return live && Base::odd(); }
  __device__ __forceinline__ void drop_blind() {
    if (live) return;
    l = n = 0.f;
#pragma unroll
    for (int db = 0; db < Base::DB; ++db) o[db] = f32x16{};
  }

  // This lane's bits of tile t of the drafted keys, its own half's keys at the bits
  // mfma_row(i, 0), and how many seen tokens lie behind the tile.
  __device__ __forceinline__ uint32_t word_of(int t) const {
    const int left = p.T - kMTile * t;
    return live ? left < kMTile ? bits[t] & (0xffffffffu >> (kMTile - left)) : bits[t] : 0u;
  }
  // A tile of the drafted keys, or CAREFUL any tile (t < ct: the cache's), where a key or value
  // that a row does not see may hold infinities or NaN, or weights took finite values out of
  // range (`up`: as in settle).
  template <bool CAREFUL>
  __device__ __forceinline__ void slow(const uint16_t* k, const uint16_t* v, int t, int ct, float up) {
    const f32x16 s = Base::products(k);
    float x[16];
    Base::template scores<false, false>(s, 0, false, 0.f, x);
    uint32_t word;                             // this lane's row sees key mfma_row(i, 0) + 4 hi
    if (!CAREFUL || t >= ct) {
      word = word_of(t - ct);
      if constexpr (SLOPE) {
        int later = 0;
        for (int i = t - ct + 1; i < p.words; ++i) later += __popc(word_of(i));
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[i] = __builtin_fmaf(-slope, (float)(__popc((word >> (4 * hi + mfma_row(i, 0))) >> 1) + later), x[i]);
      }
    } else {
      const int left = end - t * kMTile;       // the row sees so many of the tile's keys
      word = left >= kMTile ? 0xffffffffu : left > 0 ? (1u << left) - 1 : 0u;
      if constexpr (SLOPE) {
        const float dist = (float)(at - t * kMTile - 4 * hi);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(-slope, fabsf(dist - (float)mfma_row(i, 0)), x[i]);
      }
    }
    word >>= 4 * hi;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = word >> mfma_row(i, 0) & 1 ? x[i] : -INFINITY;
      mx = fmaxf(mx, x[i]);
    }
    mx = max_halves(mx);
    const float m_new = mx > m + up ? mx - fminf(up, 0.f) : m, alpha = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    l *= alpha;
    n *= alpha;
#pragma unroll
    for (int db = 0; db < Base::DB; ++db) o[db] *= alpha;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - m);
      l += x[i];
    }
    if constexpr (!CAREFUL) {
      Base::add(v, x);
      return;
    }
    asm volatile("" : "+v"(word));             // its bits anew: not in 32 scalar registers since the scores
    float seen[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) seen[i] = (float)(word >> mfma_row(i, 0) & 1);
    bf16x8 pb[2], sb[2];
    pack_frags<F16>(x, pb);
    pack_frags<F16>(seen, sb);
#pragma unroll
    for (int e = 0; e < 2; ++e) n = sum_frag<F16>(pb[e], n);
#pragma unroll
    for (int db = 0; db < Base::DB; ++db) o[db] = careful_mfma<HD, F16>(rd, v, db, pb, sb, o[db]);
  }
};

// Where a row's part of the outputs goes (a sequence in one piece: to no part).
template <int HD>
__device__ __forceinline__ Part tree_part(const TreeArgs& p, const Where& w, int kvh, int r) {
  if (w.count == 1) return {};
  return part_at<HD>(p.f, ((int64_t)(w.first + w.z) * p.f.Hk + kvh) * p.R + r);
}

// Workgroup L's piece, key head and block of rows: blocks that read the same keys
// follow each other on one XCD (workgroups go round the eight of them).
struct Item { int piece, kvh, block; };
__device__ __forceinline__ Item tree_item(const TreeArgs& p, int L) {
  const int x = L & 7, y = L >> 3, i = y / p.blocks * 8 + x;
  return {i / p.f.Hk, i % p.f.Hk, y % p.blocks};
}

template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, kPerCu<HD>) void attn_tree_kernel(TreeArgs p) {
  constexpr int CH = HD / 8;
  constexpr int DJ = kMTile * CH / kMThreads;  // 16-byte DMAs per wave, tile and tensor
  __shared__ __attribute__((aligned(16))) Slot<HD> r0, r1, r2, r3;
  const Item it = tree_item(p, blockIdx.x);
  const Where w = find_piece(p, it.piece, p.firsts && blockIdx.x == 0);
  if (w.b < 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = it.block * kMRows + wave * 32 + (lane & 31);
  const Drafted row = locate_drafted(p, w, it.kvh, r);
  TreeRows<HD, F16, CAP, SLOPE> R(p, row, lane);
  const int t_begin = share_of(w.tiles, w.z, w.count), t_end = share_of(w.tiles, w.z + 1, w.count);
  const int ct = (w.len + kMTile - 1) / kMTile;      // the cache's tiles

  const FwdSet &C = p.f.set[0], &D = p.f.set[1];
  const uint16_t* K = C.k + w.b * C.k_sb + it.kvh * C.k_sh;
  const uint16_t* V = C.v + w.b * C.v_sb + it.kvh * C.v_sh;
  const uint16_t* DK = D.k + w.b * D.k_sb + it.kvh * D.k_sh;
  const uint16_t* DV = D.v + w.b * D.v_sb + it.kvh * D.v_sh;
  uint32_t k_voff[DJ], v_voff[DJ];
#pragma unroll
  for (int j = 0; j < DJ; ++j) {
    const int pos = (wave * DJ + j) * 64 + lane, key = pos / CH;
    const uint32_t ch = (uint32_t)((pos % CH) ^ tile_swz<HD>(key)) * 16u;
    k_voff[j] = key * (uint32_t)(C.k_sn * 2) + ch;
    v_voff[j] = key * (uint32_t)(C.v_sn * 2) + ch;
  }
  // The cache's tiles of this piece.  Tiles past them are issued too, empty: the waits count them.
  const int c_end = min(t_end, ct);
  auto issue = [&](int t, Slot<HD>& T) {
    const int n0 = t * kMTile, end = t < c_end ? w.len : 0;
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc<HD>(K, C.k_sn, n0, end);
    const __amdgpu_buffer_rsrc_t vr = tile_rsrc<HD>(V, C.v_sn, n0, end);
#pragma unroll
    for (int j = 0; j < DJ; ++j) m_dma16(kr, &T.k[(wave * DJ + j) * 512], k_voff[j]);
#pragma unroll
    for (int j = 0; j < DJ; ++j) m_dma16(vr, &T.v[(wave * DJ + j) * 512], v_voff[j]);
  };
  // A tile of the drafted keys.
  auto issue_drafted = [&](int t, Slot<HD>& T) {
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc<HD>(DK, D.k_sn, t * kMTile, p.T);
    const __amdgpu_buffer_rsrc_t vr = tile_rsrc<HD>(DV, D.v_sn, t * kMTile, p.T);
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int pos = (wave * DJ + j) * 64 + lane, key = pos / CH;
      const uint32_t ch = (uint32_t)((pos % CH) ^ tile_swz<HD>(key)) * 16u;
      m_dma16(kr, &T.k[(wave * DJ + j) * 512], key * (uint32_t)(D.k_sn * 2) + ch);
      m_dma16(vr, &T.v[(wave * DJ + j) * 512], key * (uint32_t)(D.v_sn * 2) + ch);
    }
  };

  // Iteration t: tile t in `cur`, its products in s; tile t + 1 in `nxt`; tile t + 3
  // issued into `dst`, the slot of tile t - 1, free once every wave passed the barrier.
  f32x16 s;
  auto iter = [&](int t, const Slot<HD>& cur, const Slot<HD>& nxt, Slot<HD>& dst) {
    m_wait_barrier<2 * DJ>();                  // tile t + 1 landed (t + 2 in flight) for every wave
    issue(t + 3, dst);
    R.rd.fresh();
    const int n0 = t * kMTile;
    if (n0 < row.w_hi) {
      const bool edge = n0 + kMTile > row.a_hi;
      const bool poly = R.settle(s, n0, edge);
      float x[16];
      R.template scores<false>(s, n0, poly, R.m, x);
      __builtin_amdgcn_s_setprio(1);
      const f32x16 next = R.products(nxt.k);     // beside the exponentials
      // Both blocks in this order: what is read from LDS, arithmetic while it comes, then a product at a
      // time; and a wave with products goes before one without (together 117 -> 113 us with a cap, 8
      // sequences of 8,192 keys, 32 + 8 heads of 128, 64 drafted tokens; 67 -> 65 with heads of 64).
      __builtin_amdgcn_sched_group_barrier(0x100, HD / 16, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, 16, 0);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 256 / HD, 0);
      }
      R.weigh(n0, edge, x);
      R.add(cur.v, x);
      __builtin_amdgcn_sched_group_barrier(0x100, HD / 8, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, 24, 0);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      s = next;
    } else {
      s = R.products(nxt.k);
    }
  };
  R.restart();
  if (t_begin < c_end) {
    issue(t_begin, r0);
    issue(t_begin + 1, r1);
    issue(t_begin + 2, r2);
    m_wait_barrier<4 * DJ>();
    s = R.products(r0.k);
    for (int t = t_begin; t < c_end; t += 4) {
      iter(t, r0, r1, r3);
      if (t + 1 >= c_end) break;
      iter(t + 1, r1, r2, r0);
      if (t + 2 >= c_end) break;
      iter(t + 2, r2, r3, r1);
      if (t + 3 >= c_end) break;
      iter(t + 3, r3, r0, r2);
    }
  }
  m_wait<0>();                                 // no DMA of the ring may land later

  for (int t = max(t_begin, ct); t < t_end; ++t) {
    __syncthreads();
    issue_drafted(t - ct, r0);
    m_wait<0>();
    __syncthreads();
    R.template slow<false>(r0.k, r0.v, t, ct, kUp<F16>);
  }
  for (float up = kUp<F16>; __syncthreads_or(R.lost()); up = kDown) {
    R.restart();
    for (int t = t_begin; t < t_end; ++t) {
      __syncthreads();
      if (t < ct) issue(t, r0);
      else issue_drafted(t - ct, r0);
      m_wait<0>();
      __syncthreads();
      R.template slow<true>(r0.k, r0.v, t, ct, up);
    }
    if (F16 || up < 0.f) break;                // fp16's values times its weights are finite
  }
  R.drop_blind();
  R.finish(p.f, row, tree_part<HD>(p, w, it.kvh, r), sum_halves(R.l), sum_halves(R.n));
}

// Up to 32 rows: all four waves have them, and each walks every fourth tile of the piece
// through buffers of its own, with no barrier.
template <int HD, bool F16, bool CAP, bool SLOPE>
__global__ __launch_bounds__(kMThreads, HD == 64 ? 3 : 2) void attn_tree_few_kernel(TreeArgs p) {
  constexpr int CH = HD / 8, DB = HD / 32;
  constexpr int DJ = kMTile * CH / 64;         // 16-byte DMAs per tile and tensor: one wave's
  constexpr int ROW = 64 / CH;                 // rows of a DMA
  __shared__ __attribute__((aligned(16))) uint16_t kt[kMWaves][kMTile * HD];
  __shared__ __attribute__((aligned(16))) uint16_t vt[kMWaves][kMTile * HD];
  __shared__ float stat[kMWaves][2][32];
  const int kvh = blockIdx.x % p.f.Hk;
  const Where w = find_piece(p, blockIdx.x / p.f.Hk, p.firsts && blockIdx.x == 0);
  if (w.b < 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Drafted row = locate_drafted(p, w, kvh, lane & 31);
  TreeRows<HD, F16, CAP, SLOPE> R(p, row, lane);
  const int t_begin = share_of(w.tiles, w.z, w.count) + wave, t_end = share_of(w.tiles, w.z + 1, w.count);
  const int ct = (w.len + kMTile - 1) / kMTile;

  const FwdSet &C = p.f.set[0], &D = p.f.set[1];
  const uint16_t* K = C.k + w.b * C.k_sb + kvh * C.k_sh;
  const uint16_t* V = C.v + w.b * C.v_sb + kvh * C.v_sh;
  const uint16_t* DK = D.k + w.b * D.k_sb + kvh * D.k_sh;
  const uint16_t* DV = D.v + w.b * D.v_sb + kvh * D.v_sh;
  uint16_t *kw = kt[wave], *vw = vt[wave];
  // Tiles past the wave's last one are issued too, empty: the waits count them.
  auto fetch = [&](const uint16_t* base, int64_t stride, int n0, int end, uint16_t* T) {
    const __amdgpu_buffer_rsrc_t r = tile_rsrc<HD>(base, stride, n0, end);
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int key = j * ROW + lane / CH;
      m_dma16(r, T + j * 512, key * (uint32_t)(stride * 2) + (uint32_t)((lane % CH) ^ tile_swz<HD>(key)) * 16u);
    }
  };
  const int c_end = min(t_end, ct);
  auto issue_k = [&](int t) { fetch(K, C.k_sn, t * kMTile, t < c_end ? w.len : 0, kw); };
  auto issue_v = [&](int t) { fetch(V, C.v_sn, t * kMTile, t < c_end ? w.len : 0, vw); };
  auto issue_drafted = [&](int t) {
    fetch(DK, D.k_sn, t * kMTile, p.T, kw);
    fetch(DV, D.v_sn, t * kMTile, p.T, vw);
  };
  R.restart();
  issue_k(t_begin);
  issue_v(t_begin);
  int t = t_begin;
  for (; t < c_end; t += kMWaves) {
    const int n0 = t * kMTile;
    m_wait<DJ>();                              // K landed, V in flight
    const f32x16 s = R.products(kw);
    __builtin_amdgcn_s_waitcnt(0xc07f);        // lgkmcnt(0): K is read, its buffer free
    issue_k(t + kMWaves);
    const bool edge = n0 + kMTile > row.a_hi;
    float x[16];
    const bool poly = R.settle(s, n0, edge);
    R.template scores<false>(s, n0, poly, R.m, x);
    R.weigh(n0, edge, x);
    m_wait<DJ>();                              // V landed, the next K in flight
    R.add(vw, x);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    issue_v(t + kMWaves);
  }
  m_wait<0>();                                 // the empty tiles too
  for (; t < t_end; t += kMWaves) {
    __builtin_amdgcn_s_waitcnt(0xc07f);
    issue_drafted(t - ct);
    m_wait<0>();
    R.template slow<false>(kw, vw, t, ct, kUp<F16>);
  }
  for (float up = kUp<F16>; __builtin_amdgcn_ballot_w64(R.lost()); up = kDown) {
    R.restart();
    for (t = t_begin; t < t_end; t += kMWaves) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      if (t < ct) {
        issue_k(t);
        issue_v(t);
      } else {
        issue_drafted(t - ct);
      }
      m_wait<0>();
      R.template slow<true>(kw, vw, t, ct, up);
    }
    if (F16 || up < 0.f) break;
  }

  R.drop_blind();

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
  R.finish(p.f, row, tree_part<HD>(p, w, kvh, lane & 31), total, total);
}

// The pieces of a sequence's rows put together, by WAVES waves a row.
constexpr int kMaxPieces = 768;
template <int HD, bool F16, int WAVES>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs p) {
  constexpr int T = WAVES * 64, L = HD / 4, GR = T / L;   // L lanes have the row once
  constexpr int MAXZ = WAVES == 1 ? 64 : kMaxPieces;
  __shared__ float weight[4 / WAVES][MAXZ];
  __shared__ float red[4];
  __shared__ f32x4 acc[4][L];
  const int slot = threadIdx.x / T, tid = threadIdx.x % T, lane = tid & 63, wave = threadIdx.x >> 6;
  const int per = (p.R + 4 / WAVES - 1) / (4 / WAVES);     // workgroups of a (sequence, key head)
  const int kvh = blockIdx.x / per % p.f.Hk, b = blockIdx.x / per / p.f.Hk;
  const int r = blockIdx.x % per * (4 / WAVES) + slot;
  const int first = p.firsts[b], count = p.firsts[b + 1] - first;
  if (count == 1) return;                      // the whole workgroup's
  const int rc = min(r, p.R - 1);
  auto at_piece = [&](int z) { return ((int64_t)(first + z) * p.f.Hk + kvh) * p.R + rc; };
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
  const float2* stat = reinterpret_cast<const float2*>(p.f.stat);
  constexpr int PER = (MAXZ + T - 1) / T;
  float m[PER], l[PER], top = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int z = tid + i * T;
    m[i] = -INFINITY;
    l[i] = 0.f;
    if (z < count) {
      const float2 s = stat[at_piece(z)];
      m[i] = s.x;
      l[i] = s.y;
    }
    top = fmaxf(top, m[i]);
  }
  top = over(top, [](float a, float c) { return fmaxf(a, c); });
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int z = tid + i * T;
    const float x = l[i] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[i] - top);
    total = __builtin_fmaf(x, l[i], total);
    if (z < count) weight[slot][z] = x;
  }
  total = over(total, [](float a, float c) { return a + c; });
  __syncthreads();
  const int at = tid % L, group = tid / L;
  f32x4 o{};
#pragma unroll 4
  for (int z = group; z < count; z += GR) {
    const f32x4 v = reinterpret_cast<const f32x4*>(p.f.part)[at_piece(z) * L + at];
    const float x = weight[slot][z];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x, v[e], o[e]);
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
  if (tid >= L || r >= p.R) return;
  const int64_t h = (int64_t)kvh * p.f.G + r % p.f.G, tok = r / p.f.G;
  emit<F16>(p.f, b, h, tok, at, o, total);
  if (p.f.lse && at == 0)
    p.f.lse[b * p.f.lse_sb + h * p.f.lse_sh + tok] = total == 0.f ? -INFINITY : top + __log2f(total);
}

struct DraftArgs {
  const int32_t *parents, *lens, *sizes;
  int64_t parents_sb;
  int32_t* positions;
  uint32_t* seen;
  int32_t T, words;
};

__global__ __launch_bounds__(256) void draft_tree_kernel(DraftArgs p) {
  __shared__ int up[kMaxDraft];
  const int64_t b = blockIdx.x;
  const int size = p.sizes ? clampi(p.sizes[b], 0, p.T) : p.T;
  for (int i = threadIdx.x; i < size; i += 256) {
    const int x = p.parents[b * p.parents_sb + i];
    up[i] = x >= 0 && x < i ? x : -1;          // a parent that is no earlier token: the cache's last
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T; i += 256) {
    int at = i < size ? i : -1, n = 0;
    for (int w = p.words - 1; w >= 0; --w) {
      uint32_t word = 0;
      while (at >= 32 * w) {                   // -1 is below
        word |= 1u << (at & 31);
        ++n;
        at = up[at];
      }
      p.seen[(b * p.T + i) * p.words + w] = word;
    }
    p.positions[b * p.T + i] = i < size ? p.lens[b] + n - 1 : 0;
  }
}

struct TreePlan { int blocks, target, most; bool few, join; int64_t pieces; size_t parts, bytes; };
TreePlan tree_plan(int64_t B, int64_t Hk, int64_t G, int64_t T, int64_t N, int64_t D) {
  TreePlan x{};
  const int64_t R = T * G, tiles = (N + kMTile - 1) / kMTile + (T + kMTile - 1) / kMTile;
  x.few = R <= 32;
  x.blocks = (int)((R + kMRows - 1) / kMRows);
  // Workgroups that a CU holds, of the many-row kernel at head dim 64 three (256, 512, 768 and 1,024 pieces
  // of all: 128 features 134, 110, 122, 124 us, 64 features 98, 68, 65, 74).
  const int64_t want = kTreeCus * (!x.few && D == 64 ? 3 : 2);
  x.target = (int)std::max<int64_t>(1, std::min<int64_t>(want / std::max<int64_t>(1, x.blocks * Hk), kMaxPieces));
  x.join = tiles > (x.few ? kSplitFew : kSplitMany) && (x.target > 1 || B > 1);
  x.most = !x.join ? 1 : x.target > 64 ? kMaxPieces : 64;   // as the join's two forms hold
  // (piece_tiles: all / S and one of each sequence's, S being 5 / 4 of the mean)
  x.pieces = !x.join ? B : B < x.target ? x.target : 2 * B;
  x.parts = x.join ? (size_t)(x.pieces * Hk * R) : 0;
  x.bytes = x.join ? x.parts * (D + 2) * sizeof(float) + (B + 1) * sizeof(int32_t) : 0;
  return x;
}

template <int HD, bool F16, bool CAP, bool SLOPE>
hipError_t tree_launch(const TreeArgs& a, const TreePlan& x, hipStream_t s) {
  const unsigned items = (unsigned)(x.pieces * a.f.Hk);
  if (x.few)
    hipLaunchKernelGGL((attn_tree_few_kernel<HD, F16, CAP, SLOPE>), dim3(items), dim3(kMThreads), 0, s, a);
  else
    hipLaunchKernelGGL((attn_tree_kernel<HD, F16, CAP, SLOPE>), dim3((items + 7) / 8 * 8 * x.blocks), dim3(kMThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !x.join) return e;
  const unsigned problems = (unsigned)(a.f.B * a.f.Hk);
  if (x.most > 64)
    hipLaunchKernelGGL((attn_tree_join_kernel<HD, F16, 4>), dim3(problems * a.R), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attn_tree_join_kernel<HD, F16, 1>), dim3(problems * ((a.R + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <int HD, bool F16>
hipError_t tree_go(const TreeArgs& a, const TreePlan& x, bool cap, hipStream_t s) {
  if (cap) return a.f.slopes ? tree_launch<HD, F16, true, true>(a, x, s) : tree_launch<HD, F16, true, false>(a, x, s);
  return a.f.slopes ? tree_launch<HD, F16, false, true>(a, x, s) : tree_launch<HD, F16, false, false>(a, x, s);
}

// The masked attention's arguments, for its checks: the cache as keys, the drafted ones as a
// prefix (whose rows and strides are then checked too).
gpa_attn_masked_args as_masked(const gpa_attn_tree_args* a) {
  gpa_attn_masked_args m{};
  m.q = a->q; m.k = a->cache_k; m.v = a->cache_v; m.o = a->o; m.lse = a->lse;
  m.B = a->B; m.H = a->H; m.Hk = a->Hk; m.M = a->T; m.N = a->N; m.D = a->D;
  m.q_sb = a->q_sb; m.q_sh = a->q_sh; m.q_sm = a->q_st;
  m.k_sb = a->ck_sb; m.k_sh = a->ck_sh; m.k_sn = a->ck_sn;
  m.v_sb = a->cv_sb; m.v_sh = a->cv_sh; m.v_sn = a->cv_sn;
  m.o_sb = a->o_sb; m.o_sh = a->o_sh; m.o_sm = a->o_st;
  m.lse_sb = a->lse_sb; m.lse_sh = a->lse_sh;
  m.slopes = a->slopes; m.slopes_sb = a->slopes_sb;
  m.lens = a->lengths; m.docs = 1; m.causal = 1;
  m.pk = a->k; m.pv = a->v; m.P = a->T;
  m.pk_sh = a->k_sh; m.pk_sn = a->k_st; m.pv_sh = a->v_sh; m.pv_sn = a->v_st;
  m.sm_scale = a->sm_scale; m.cap = a->cap;
  return m;
}

}  // namespace
}  // namespace gpa

using namespace gpa;

extern "C" int gpa_draft_tree(const int32_t* parents, int64_t parents_sb, const int32_t* lengths, const int32_t* sizes,
                              int64_t B, int64_t T, int32_t* positions, int32_t* seen, void* stream) {
  const char* fn = "gpa_draft_tree";
  gpa_clear_error();
  if (B < 0 || T < 0) {
    gpa_set_error("%s: negative size", fn);
    return GPA_E_INVALID;
  }
  if (T > kMaxDraft || B > 0x7fffff) {
    gpa_set_error("%s: %lld drafted tokens of %lld sequences (up to %lld, and 2^23)", fn, (long long)T, (long long)B,
                  (long long)kMaxDraft);
    return GPA_E_UNSUPPORTED;
  }
  if (B == 0 || T == 0) return GPA_OK;
  if (!parents || !lengths || !positions || !seen) {
    gpa_set_error("%s: null pointer", fn);
    return GPA_E_INVALID;
  }
  const DraftArgs a{parents, lengths, sizes, B > 1 ? parents_sb : 0, positions, (uint32_t*)seen, (int32_t)T, (int32_t)((T + 31) / 32)};
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}

extern "C" size_t gpa_attn_tree_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t T, int64_t N, int64_t D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || T <= 0 || N < 0 || H % Hk || (D != 64 && D != 128)) return 0;
  return tree_plan(B, Hk, H / Hk, T, N, D).bytes;
}

extern "C" int gpa_attn_tree(int dtype, const gpa_attn_tree_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gpa_attn_tree";
  gpa_clear_error();
  if (!args) {
    gpa_set_error("%s: null arguments", fn);
    return GPA_E_INVALID;
  }
  gpa_attn_masked_args m = as_masked(args);
  const int rc = masked_check(fn, dtype, &m, true);
  if (rc != GPA_OK) return rc;
  if (m.B == 0 || m.H == 0 || m.M == 0) return GPA_OK;
  if (args->T > kMaxDraft) {
    gpa_set_error("%s: %lld drafted tokens (up to %lld)", fn, (long long)args->T, (long long)kMaxDraft);
    return GPA_E_UNSUPPORTED;
  }
  if (!args->seen || (m.B > 1 && (args->k_sb % 8 || args->v_sb % 8))) {
    gpa_set_error("%s: no bits, or rows that are not 16-byte aligned", fn);
    return GPA_E_INVALID;
  }
  m = masked_plain(&m);
  const int64_t G = m.H / m.Hk, R = m.M * G, tiles = (m.N + m.M) / kMTile + 2;
  const TreePlan x = tree_plan(m.B, m.Hk, G, m.M, m.N, m.D);
  // A launch has less than 2^32 threads; tiles of all sequences are counted in 31 bits.
  if ((x.pieces * m.Hk + 8) * x.blocks > kMostWgs || m.B * m.Hk * R > kMostWgs || m.B > ((int64_t)1 << 30) / tiles ||
      x.pieces * m.Hk >= (int64_t)1 << 30) {
    gpa_set_error("%s: too many rows or sequences", fn);
    return GPA_E_UNSUPPORTED;
  }
  if (x.bytes > 0 && (!workspace || workspace_bytes < x.bytes || (uintptr_t)workspace % 16)) {
    gpa_set_error("%s: workspace of %zu bytes, 16-byte aligned, needed", fn, x.bytes);
    return GPA_E_WORKSPACE;
  }
  TreeArgs a{};
  FwdArgs& f = a.f;
  f.q = (const uint16_t*)m.q; f.o = (uint16_t*)m.o; f.lse = m.lse;
  f.q_sb = m.q_sb; f.q_sh = m.q_sh; f.q_sm = m.q_sm;
  f.o_sb = m.o_sb; f.o_sh = m.o_sh; f.o_sm = m.o_sm;
  f.lse_sb = m.lse_sb; f.lse_sh = m.lse_sh;
  f.slopes = m.slopes; f.slopes_sb = m.slopes_sb;
  f.B = (int32_t)m.B; f.Hk = (int32_t)m.Hk; f.G = (int32_t)G;
  masked_fill(&m, &f.mask, &f.score);
  if (x.bytes > 0) {
    f.part = (float*)workspace;
    f.stat = f.part + x.parts * m.D;
    a.firsts = (int32_t*)(f.stat + x.parts * 2);
  }
  FwdSet &c = f.set[0], &d = f.set[1];
  c.k = (const uint16_t*)m.k; c.v = (const uint16_t*)m.v; c.N = (int32_t)m.N;
  c.k_sb = m.k_sb; c.k_sh = m.k_sh; c.k_sn = m.k_sn; c.v_sb = m.v_sb; c.v_sh = m.v_sh; c.v_sn = m.v_sn;
  d.k = (const uint16_t*)m.pk; d.v = (const uint16_t*)m.pv; d.N = (int32_t)m.P;
  d.k_sb = m.B > 1 ? args->k_sb : 0; d.k_sh = m.pk_sh; d.k_sn = m.pk_sn;
  d.v_sb = m.B > 1 ? args->v_sb : 0; d.v_sh = m.pv_sh; d.v_sn = m.pv_sn;
  a.seen = (const uint32_t*)args->seen;
  a.T = (int32_t)m.M; a.words = (int32_t)((m.M + 31) / 32);
  a.seen_st = a.words; a.seen_sb = (int64_t)a.words * m.M;
  a.lens = m.lens;
  a.R = (int32_t)R; a.blocks = x.blocks; a.target = x.target; a.most = x.most;
  const bool f16 = dtype == GPA_DTYPE_F16, cap = m.cap > 0.f;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t e = m.D == 64 ? (f16 ? tree_go<64, true>(a, x, cap, s) : tree_go<64, false>(a, x, cap, s))
                                 : (f16 ? tree_go<128, true>(a, x, cap, s) : tree_go<128, false>(a, x, cap, s));
  if (e != hipSuccess) {
    gpa_set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return GPA_E_LAUNCH;
  }
  return GPA_OK;
}
