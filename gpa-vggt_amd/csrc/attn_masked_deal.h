// Blocks of unequal length: counted, cut and listed by length, before a kernel takes
// them in that order.
#pragma once
#include "attn_masked.h"

#include <algorithm>

namespace gpa {

constexpr int kCus = 256;
constexpr int kDealItems = 2048;               // (sequence, block) pairs of a list at most
constexpr int64_t kLeast = 8;                  // tiles of a piece at least

// The pieces of a problem's blocks, the same for every key head of a sequence.
struct Deal {
  int32_t pieces, cuts, pad[2];
  int4 piece[kDealItems + kCus * 3];           // sequence and block, number, of how many, first part (-1: whole)
  int4 cut[kCus * 3];                          // sequence and block, pieces, first part
  int32_t count[kDealItems];                   // tiles of a sequence's block
};
// A list to be made of `blocks` blocks a sequence, for `spans` resident workgroups.
struct DealOf {
  Deal* list;
  int32_t blocks, spans;
};

// What makes row blocks see key ranges of unequal length.
enum class Unequal { no, causal, documents };
inline Unequal unequal_of(const gpa_attn_masked_args& a) {
  return a.q_offsets || a.k_offsets || a.lens ? Unequal::documents : a.causal ? Unequal::causal : Unequal::no;
}

namespace {

// A value of memory that is the same for all lanes, in scalar registers: without it
// the buffer descriptors that follow from it are rebuilt in a loop over the lanes.
__device__ __forceinline__ int4 same(int4 x) {
  return {__builtin_amdgcn_readfirstlane(x.x), __builtin_amdgcn_readfirstlane(x.y), __builtin_amdgcn_readfirstlane(x.z),
          __builtin_amdgcn_readfirstlane(x.w)};
}

struct DealArgs {
  MaskArgs mask;
  int32_t B, Hk, G;
  DealOf rows, keys;
};

// The tiles of the blocks of 128 rows (a tile: 32 keys, counted from the first that the
// block sees), then of those of 64 keys (64 rows, from row 0): one workgroup each, at
// least one tile.
__global__ __launch_bounds__(kMRows) void attn_masked_count_kernel(DealArgs p) {
  __shared__ int range[2][kMRows / 64];
  const bool of_keys = (int)blockIdx.x >= p.B * p.rows.blocks;
  const DealOf& d = of_keys ? p.keys : p.rows;
  const int at = blockIdx.x - (of_keys ? p.B * p.rows.blocks : 0), b = at / d.blocks;
  int lo = 0, hi = 0;
  if (of_keys) {
    const int j = at % d.blocks * 64 + threadIdx.x;
    if (threadIdx.x < 64 && j < p.mask.N) {
      const KeySpan s = key_span(p.mask, b, j);
      lo = s.lo * p.G;
      hi = s.hi * p.G;
    }
  } else {
    const int r = at % d.blocks * kMRows + threadIdx.x;
    if (r < p.mask.M * p.G) {
      const RowSpan s = row_span(p.mask, b, r / p.G);
      lo = s.lo;
      hi = s.hi;
    }
  }
  if (hi <= lo) lo = 0x7fffffff, hi = 0;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    lo = min(lo, __shfl_xor(lo, i));
    hi = max(hi, __shfl_xor(hi, i));
  }
  if (threadIdx.x % 64 == 0) {
    range[0][threadIdx.x / 64] = lo;
    range[1][threadIdx.x / 64] = hi;
  }
  __syncthreads();
  if (threadIdx.x > 0) return;
  lo = min(range[0][0], range[0][1]);
  hi = max(range[1][0], range[1][1]);
  const int tiles = of_keys ? (hi + 63) / 64 - lo / 64 : (hi - lo + kMTile - 1) / kMTile;
  d.list->count[at] = hi > lo ? tiles : 1;
}

// The blocks' pieces, long ones first.  With T tiles in all for `spans` workgroups
// that are resident at once, a block of more than C = T / spans is cut into equal
// pieces of C at most, so no piece outlasts the rest.  With one causal document,
// whose lengths go from the shortest to the longest evenly, C is half as much
// again: fewer parts, 7 to 14 % less time on 128 to 512 blocks; where a block lies
// astride two documents and walks both, that C costs 15 % (16 heads, 10,992 tokens).
// The atomics order pieces of about one length among themselves, which changes no result.
__global__ __launch_bounds__(1024) void attn_masked_deal_kernel(DealArgs p) {
  constexpr int EACH = kDealItems / 1024, KINDS = 256;
  const DealOf& d = blockIdx.x == 0 ? p.rows : p.keys;
  Deal* D = d.list;
  if (d.blocks == 0) return;
  __shared__ int part[16];
  __shared__ int at[KINDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.B * d.blocks;
  // The sum of the threads before this one, and the total.
  auto scan = [&](int v, int& total) {
    auto upto = [&](int x, int width) {
#pragma unroll
      for (int i = 1; i < width; i <<= 1) {
        const int y = __shfl_up(x, i);
        x += lane >= i ? y : 0;
      }
      return x;
    };
    const int x = upto(v, 64);
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    const int s = upto(part[lane & 15], 16);
    total = __shfl(s, 15);
    const int before = __shfl(s, (wave - 1) & 15);
    return x - v + (wave > 0 ? before : 0);
  };
  int c[EACH], tiles = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    c[i] = tid * EACH + i < n ? D->count[tid * EACH + i] : 0;
    tiles += c[i];
  }
  if (tid < KINDS) at[tid] = 0;
  scan(tiles, all);
  const int64_t line = (int64_t)all * p.Hk * (p.mask.q_off || p.mask.k_off || p.mask.lens ? 2 : 3) / 2;
  const int most = (int)std::max<int64_t>((line + d.spans - 1) / d.spans, kLeast);
  int pieces[EACH], key[EACH], cut = 0, total;   // cut blocks, and 2^12 for each of their pieces
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    pieces[i] = (c[i] + most - 1) / most;
    const int len = pieces[i] > 1 ? (c[i] + pieces[i] - 1) / pieces[i] : c[i];
    key[i] = KINDS - 1 - (int)((int64_t)std::max(len - 1, 0) * KINDS / most);
    if (pieces[i] > 1) cut += (pieces[i] << 12) + 1;
    if (pieces[i] > 0) atomicAdd(&at[key[i]], pieces[i]);
  }
  cut = scan(cut, total);
  const int num = tid < KINDS ? at[tid] : 0;
  int listed;
  const int first = scan(num, listed);
  if (tid < KINDS) at[tid] = first;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = tid * EACH + i;
    const bool whole = pieces[i] < 2;
    if (pieces[i] == 0) continue;
    const int to = atomicAdd(&at[key[i]], pieces[i]), slot = cut >> 12;
    for (int k = 0; k < pieces[i]; ++k) D->piece[to + k] = int4{e, k, pieces[i], whole ? -1 : slot + k};
    if (whole) continue;
    D->cut[cut & 4095] = int4{e, pieces[i], slot, 0};
    cut += (pieces[i] << 12) + 1;
  }
  if (tid == 0) {
    D->pieces = listed;
    D->cuts = total & 4095;
  }
}

// Makes the lists (no blocks: none).
hipError_t deal_out(const MaskArgs& mask, int B, int Hk, int G, DealOf rows, DealOf keys, hipStream_t s) {
  const DealArgs a{mask, B, Hk, G, rows, keys};
  hipLaunchKernelGGL(attn_masked_count_kernel, dim3((unsigned)(B * (rows.blocks + keys.blocks))), dim3(kMRows), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(attn_masked_deal_kernel, dim3(keys.blocks ? 2 : 1), dim3(1024), 0, s, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace gpa
