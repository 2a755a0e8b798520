// The matrix product of linear_gate.hip and linear_gate_bwd.hip: out[i][j] = sum_k Q(i, k)
// P(j, k) of 16-bit operands in fp32, then what stands in Finish, element by element.
//
// An operand lies k-contiguous (rows of j or i) or "turned" (rows of k, the output's rows
// or columns contiguous).  Either way a stage of 32 k is fetched as it lies, by DMA, into a
// ring in LDS, each slot an array of its own (so that the compiler sees that reads of one
// and DMA into another do not touch); a turned operand's fragments come out by transposing reads.
// A workgroup has four waves, two by two, each with WI x WJ blocks of 16 x 16 in registers;
// the fragments of stage k + 1 are read and stage k + R is fetched beside the products of
// stage k.  A fragment read feeds WI or WJ products: with 8 x 8 blocks the LDS delivers
// half of what it can, with 4 x 8 three quarters, with 4 x 4 all.
//
// The sums go through LDS, strip by strip, to be finished and stored in rows of 16
// bytes a lane: out of the accumulators a lane would have 8 bytes of a row, and the
// code for an activation would be there once for each of them.
//
// What bounds it: the matrix instructions, by the power that they take.  8,192 x 4,096 x 4,096 in bf16:
// 210 to 221 us (1,240 to 1,310 TFLOP/s; 1,594 is what a product of 16,384^3 reaches in the vendor's
// library, which takes 218 to 222 us here), its turned forms 207 to 237 (the library 254 and 287);
// bias, tanh GELU, residual and the fp32 sums kept for the backward add 65 to 75 us of stores and arithmetic.
#pragma once

#include <type_traits>
#include <utility>

#include "linear_gate.h"

namespace gpa {
namespace {

struct Operand {
  const uint16_t* p;
  int64_t stride;         // of its rows, a multiple of 8
  int64_t rows, cols;     // cols: a multiple of 8 (k-contiguous: of k)
};

struct GemmArgs {
  Operand P, Q;           // columns j and rows i of the output
  int32_t nk;             // stages of 32 k
  int32_t ti, tj, splits; // tiles of i and j; parts that k is cut into
  Finish out;
};

template <int N>
__device__ __forceinline__ void wait_dma() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

constexpr uint32_t kNowhere = 0x40000000u;     // a DMA offset outside every descriptor: zeros

// One operand of a workgroup: BL blocks of 16 a wave, two waves' worth a tile.  Zeros past the last k:
// by last_ok, or turned by the descriptor's end, behind which the rows past the last one begin (so
// they may not lie over each other: stride >= cols).
template <int BL, bool TURNED>
struct Feed {
  static constexpr int T = 32 * BL;            // rows of i or j of a tile
  static constexpr int BYTES = T * 64;         // of a stage
  static constexpr int DMAS = BL / 2;          // a wave's, of a stage
  static constexpr int READS = TURNED ? 2 * BL : BL;
  const uint16_t* base;
  int64_t stride;
  int32_t left, tail, nk; // rows from the tile's first; k (or columns) that the last stage (tile) has
  uint32_t voff[DMAS];
  bool last_ok[DMAS];
  uint32_t at[TURNED ? BL : 1];

  // Turned: where row k's 32-byte piece s lies, s ^ piece(k): the 16 rows that a read
  // takes a piece of fall on all banks.
  static __device__ __forceinline__ int piece(int k) {
    if constexpr (T == 64) return (k >> 1 & 1) | (k >> 3 & 1) << 1;
    else if constexpr (T == 128) return (k & 3) | (k >> 3 & 1) << 2;
    else return (k & 3) | (k >> 3 & 3) << 2;
  }
  // k-contiguous: chunk c of row r lies at c ^ chunk(r).
  static __device__ __forceinline__ int chunk(int r) { return ((r >> 1) & 3) ^ (((r >> 3) & 1) * 3); }

  __device__ __forceinline__ Feed(const Operand& o, int64_t first, int stages, int wave, int lane, int half)
      : stride(o.stride), nk(stages) {
    const int quad = lane >> 4, l16 = lane & 15;
    if constexpr (!TURNED) {
      base = o.p + first * o.stride;
      left = (int)(o.rows - first < T ? o.rows - first : T);
      tail = (int)o.cols;                      // of a row
#pragma unroll
      for (int j = 0; j < DMAS; ++j) {
        const int row = (wave * DMAS + j) * 16 + (lane >> 2), c = (lane & 3) ^ chunk(row);
        voff[j] = (uint32_t)row * (uint32_t)(stride * 2) + c * 16;
        last_ok[j] = c * 8 < tail - 32 * (nk - 1);
      }
      at[0] = (half * BL * 16 + l16) * 64 + ((quad ^ chunk(l16)) << 4);
    } else {
      base = o.p + first;
      left = (int)(o.rows < 0x7fffffff ? o.rows : 0x7fffffff);
      tail = (int)(o.cols - first < T ? o.cols - first : T);
#pragma unroll
      for (int j = 0; j < DMAS; ++j) {
        constexpr int PER = 512 / T, CH = T / 8;   // rows of a DMA, chunks of a row
        const int row = (wave * DMAS + j) * PER + lane / CH, c = lane % CH;
        const int s = (c >> 1 ^ piece(row)) * 2 + (c & 1);
        voff[j] = s * 8 < tail ? (uint32_t)row * (uint32_t)(stride * 2) + s * 16 : kNowhere;
        last_ok[j] = true;
      }
      const int row = 8 * quad + (l16 >> 2);
#pragma unroll
      for (int b = 0; b < BL; ++b) at[b] = row * (2 * T) + (((half * BL + b) ^ piece(row)) << 5) + (l16 & 3) * 8;
    }
  }
  // Stage kc into a slot; past the last one nothing is read, and the waits count it.
  __device__ __forceinline__ void issue(int kc, uint8_t* slot, int wave) const {
    auto put = [&](__amdgpu_buffer_rsrc_t r, int j, uint32_t off) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(slot + (wave * DMAS + j) * 1024), 16, off, 0, 0, 0);
    };
    if constexpr (!TURNED) {
      // The base moves with k, so that a row's end is the descriptor's for the last row.
      const int cols = tail - 32 * kc;
      const uint32_t bytes = kc < nk ? (uint32_t)((left - 1) * stride + cols) * 2u : 0u;
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base + 32 * (int64_t)kc, bytes);
      const bool whole = cols >= 32;
#pragma unroll
      for (int j = 0; j < DMAS; ++j) put(r, j, whole || last_ok[j] ? voff[j] : kNowhere);
    } else {
      int n = left - 32 * kc;
      n = n > 32 ? 32 : n;
      const uint32_t bytes = kc < nk && n > 0 ? (uint32_t)((n - 1) * stride + tail) * 2u : 0u;
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base + 32 * (int64_t)kc * stride, bytes);
#pragma unroll
      for (int j = 0; j < DMAS; ++j) put(r, j, voff[j]);
    }
  }
  // A wave's fragments of a stage: lane (quad, l16) has row 16 b + l16, k 8 quad .. +7.
  __device__ __forceinline__ void read(const uint8_t* slot, bf16x8 (&f)[BL]) const {
    typedef __attribute__((address_space(3))) const char* lds_ptr;
#pragma unroll
    for (int b = 0; b < BL; ++b) {
      if constexpr (!TURNED) {
        f[b] = *reinterpret_cast<const bf16x8*>(slot + at[0] + b * 1024);
      } else {
        typedef short i16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) i16x4* tr_ptr;
        const lds_ptr p = (lds_ptr)slot + at[b];
        const bf16x4 lo = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)p));
        const bf16x4 up = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(p + 8 * T)));
        f[b] = bf16x8{lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
      }
    }
  }
};

// Products, LDS reads and DMA issues of a stage, spread evenly.
template <int PRODUCTS, int READS, int DMAS, int... E>
__device__ __forceinline__ void spread(std::integer_sequence<int, E...>) {
  constexpr int ALL = READS + DMAS;
  (([&] {
     constexpr int n = (E + 1) * PRODUCTS / ALL - E * PRODUCTS / ALL;
     if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x008, n, 0);
     constexpr bool dma = (E + 1) * DMAS / ALL > E * DMAS / ALL;
     __builtin_amdgcn_sched_group_barrier(dma ? 0x010 : 0x100, 1, 0);
   }()),
   ...);
}

// Which tile a workgroup has.  Workgroups go round the eight XCDs: each has a run of
// tiles, eight rows of them at a time column by column, so that what runs together on it
// shares rows and columns in its L2.
__device__ __forceinline__ bool tile_of(const GemmArgs& p, int L, int& i, int& j, int& split) {
  const int per = p.ti * p.tj, all = per * p.splits, chunk = (all + 7) / 8;
  const int t = (L & 7) * chunk + (L >> 3);
  if ((L >> 3) >= chunk || t >= all) return false;
  split = t / per;
  const int u = t - split * per, g = u / (8 * p.tj), in = u - g * 8 * p.tj;
  const int rows = p.ti - 8 * g < 8 ? p.ti - 8 * g : 8;
  i = 8 * g + in % rows;
  j = in / rows;
  return true;
}

template <int WI, int WJ, int R, int PER_CU, bool PT, bool QT, bool F16>
__global__ __launch_bounds__(256, PER_CU) void linear_gemm_kernel(GemmArgs a) {
  typedef Feed<WJ, PT> FP;
  typedef Feed<WI, QT> FQ;
  static_assert(R == 3 || R == 4, "slots of the ring");
  __shared__ __attribute__((aligned(16))) uint8_t p0[FP::BYTES], p1[FP::BYTES], p2[FP::BYTES], p3[R > 3 ? FP::BYTES : 16],
      q0[FQ::BYTES], q1[FQ::BYTES], q2[FQ::BYTES], q3[R > 3 ? FQ::BYTES : 16];
  uint8_t* const ps[4] = {p0, p1, p2, p3};
  uint8_t* const qs[4] = {q0, q1, q2, q3};

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave & 1, wj = wave >> 1;
  int ti, tj, split;
  if (!tile_of(a, blockIdx.x, ti, tj, split)) return;
  ti = __builtin_amdgcn_readfirstlane(ti);
  tj = __builtin_amdgcn_readfirstlane(tj);
  split = __builtin_amdgcn_readfirstlane(split);
  const int k0 = (int)((int64_t)a.nk * split / a.splits), k1 = (int)((int64_t)a.nk * (split + 1) / a.splits);
  const FP fp(a.P, (int64_t)tj * FP::T, a.nk, wave, lane, wj);
  const FQ fq(a.Q, (int64_t)ti * FQ::T, a.nk, wave, lane, wi);
  auto issue = [&](int kc, int slot) __attribute__((always_inline)) {
    const int k = kc < k1 ? kc : a.nk;         // past the part: nothing
    fp.issue(k, ps[slot], wave);
    fq.issue(k, qs[slot], wave);
  };
  constexpr int DMAS = FP::DMAS + FQ::DMAS;

  f32x4 acc[WI][WJ];
#pragma unroll
  for (int i = 0; i < WI; ++i)
#pragma unroll
    for (int j = 0; j < WJ; ++j) acc[i][j] = f32x4{};
  bf16x8 fp0[WJ], fq0[WI], fp1[WJ], fq1[WI];
  auto mma = [&](const bf16x8 (&p)[WJ], const bf16x8 (&q)[WI]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
      for (int j = 0; j < WJ; ++j) acc[i][j] = mfma16x16x32_t<F16>(p[j], q[i], acc[i][j]);
  };
  // Stage kc, in slot u % R, its fragments in set u % 2: wait for stage kc + 1 (those behind it
  // stay in flight); after the barrier every wave has stage kc's fragments, so its slot takes
  // stage kc + R.
  auto step = [&](int kc, auto which) __attribute__((always_inline)) {
    constexpr int u = decltype(which)::value, here = u % R, next = (u + 1) % R;
    __builtin_amdgcn_sched_barrier(0);
    wait_dma<DMAS * (R - 2)>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(kc + R, here);
    if constexpr (u % 2 == 0) {
      fp.read(ps[next], fp1);
      fq.read(qs[next], fq1);
      mma(fp0, fq0);
    } else {
      fp.read(ps[next], fp0);
      fq.read(qs[next], fq0);
      mma(fp1, fq1);
    }
    spread<WI * WJ, FP::READS + FQ::READS, DMAS>(std::make_integer_sequence<int, FP::READS + FQ::READS + DMAS>{});
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int s = 0; s < R; ++s) issue(k0 + s, s);
  wait_dma<DMAS * (R - 1)>();
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  fp.read(ps[0], fp0);
  fq.read(qs[0], fq0);
  constexpr int U = R % 2 ? 2 * R : R;         // steps after which slots and sets recur
  int kc = k0;
  for (; kc + U <= k1; kc += U) {
    step(kc, std::integral_constant<int, 0>{});
    step(kc + 1, std::integral_constant<int, 1>{});
    step(kc + 2, std::integral_constant<int, 2>{});
    step(kc + 3, std::integral_constant<int, 3>{});
    if constexpr (U == 6) {
      step(kc + 4, std::integral_constant<int, 4>{});
      step(kc + 5, std::integral_constant<int, 5>{});
    }
  }
  // What is left, fewer than U stages, one by one.  (Ways out between the steps above
  // would give the sums other registers on each of them, 200 to 1,200 of them in memory.)
#pragma unroll 1
  for (int slot = 0; kc < k1; ++kc) {
    wait_dma<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    uint8_t* const p = slot == 0 ? p0 : slot == 1 ? p1 : slot == 2 ? p2 : p3;
    uint8_t* const q = slot == 0 ? q0 : slot == 1 ? q1 : slot == 2 ? q2 : q3;
    fp.read(p, fp0);
    fq.read(q, fq0);
    if constexpr (U - 1 > R) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (kc + R < k1) {
        fp.issue(kc + R, p, wave);
        fq.issue(kc + R, q, wave);
      }
    }
    mma(fp0, fq0);
    slot = slot == R - 1 ? 0 : slot + 1;
  }
  wait_dma<0>();                               // no DMA may land in what follows
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // Two strips of 16 rows a round, of this wave's own: strip s at `to[s]`, its 16-byte chunks
  // XORed by the row.
  constexpr int CH = WJ * 4;                   // chunks of a strip's row
  typedef __attribute__((address_space(3))) uint8_t* lds8;
  typedef __attribute__((address_space(3))) f32x4* lds_f4;
  const bool own = R == 4 || wave < 3;         // with three slots the last wave takes those of Q
  const lds8 strip = own ? wave == 0 ? (lds8)p0 : wave == 1 ? (lds8)p1 : wave == 2 ? (lds8)p2 : (lds8)p3 : (lds8)q0;
  const lds8 to[2] = {strip, own || WI == WJ ? strip + WJ * 1024 : (lds8)q1};
  const int quad = lane >> 4, l16 = lane & 15;
  const int64_t i0 = (int64_t)ti * FQ::T + wi * WI * 16, j0 = (int64_t)tj * FP::T + wj * WJ * 16;
  // A lane has the same eight columns throughout, and row r0 + RP it of a round's 32.
  constexpr int RP = 32 / WJ, MASK = CH < 16 ? CH - 1 : 15;
  const int c8 = lane % (WJ * 2), r0 = lane / (WJ * 2);
  const int64_t j = j0 + c8 * 8;
  auto down = [&](int h) __attribute__((always_inline)) {   // strips h, h + 1 into LDS
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 0; b < WJ; ++b) *(lds_f4)(to[s] + (l16 * CH + ((4 * b + quad) ^ (l16 & MASK))) * 16) = acc[h + s][b];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  auto up = [&](int it, float (&v)[8]) __attribute__((always_inline)) {
    const int row = it * RP + r0, r = row & 15, x = r & MASK;
    const lds8 from = it * 2 / WJ ? to[1] : to[0];
    const f32x4 lo = *(lds_f4)(from + (r * CH + ((2 * c8) ^ x)) * 16), hi = *(lds_f4)(from + (r * CH + ((2 * c8 + 1) ^ x)) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lo[e];
      v[4 + e] = hi[e];
    }
  };
  if (a.splits > 1) {
#pragma unroll
    for (int h = 0; h < WI; h += 2) {
      down(h);
#pragma unroll 2
      for (int it = 0; it < WJ; ++it) {
        float v[8];
        up(it, v);
        part8(a.out, i0 + h * 16 + it * RP + r0, j, split, v);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    return;
  }
  // Columns that do not come in aligned groups of eight: a lane has one column of eight rows at a
  // time, so that what a wave loads and stores at once lies together.
  if (!a.out.wide) {
    constexpr int W = WJ * 16 < 64 ? WJ * 16 : 64, DOWN = 64 / W;   // columns and rows of 64 lanes
#pragma unroll
    for (int h = 0; h < WI; h += 2) {
      down(h);
#pragma unroll 1
      for (int it = 0; it < 32 / DOWN / 8 * (WJ * 16 / W); ++it) {
        const int c = it % (WJ * 16 / W) * W + lane % W, first = it / (WJ * 16 / W) * 8 * DOWN + lane / W;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = first + e * DOWN, r = row & 15;
          const lds8 from = row >> 4 ? to[1] : to[0];
          v[e] = *(__attribute__((address_space(3))) float*)(from + (r * CH + ((c >> 2) ^ (r & MASK))) * 16 + (c & 3) * 4);
        }
        finish_down<F16, DOWN>(a.out, i0 + h * 16 + first, j0 + c, v);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    return;
  }
  // Whole groups of eight columns: what a column has is loaded once, the residual a round ahead,
  // before the stores of the round between, which a wait for it would wait for too.
  const bool in = j < a.out.J;
  float bias[8], gate[8];
  if (a.out.bias && in) param8<F16>(a.out.bias, a.out.pf32, 1, j, 8, bias);
  if (a.out.gate && in) param8<F16>(a.out.gate, a.out.pf32, 1, j, 8, gate);
  auto rounds = [&](auto which) __attribute__((always_inline)) {
    constexpr int ACT = decltype(which)::value;
    constexpr int SETS = WI == 8 ? 2 : 1;      // two waves a SIMD hide each other's waits
    u32x4 res[SETS][WJ];
    auto ahead = [&](int h) __attribute__((always_inline)) {
      const int64_t i = i0 + h * 16 + r0;
#pragma unroll
      for (int it = 0; it < WJ; ++it)
        if (in && i + it * RP < a.out.I)
          res[h / 2 % SETS][it] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.out.residual) + (i + it * RP) * a.out.res_s + j);
    };
    if (SETS == 2 && a.out.residual) ahead(0);
#pragma unroll
    for (int h = 0; h < WI; h += 2) {
      const int64_t i = i0 + h * 16 + r0;
      if (a.out.residual && (SETS == 1 || h + 2 < WI)) ahead(SETS == 1 ? h : h + 2);
      down(h);
#pragma unroll
      for (int it = 0; it < WJ; ++it) {
        float v[8];
        up(it, v);
        if (!in || i + it * RP >= a.out.I) continue;
        if (a.out.unscale) {
          const float factor = a.out.unscale[i + it * RP];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= factor;
        }
        if (a.out.bias) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += bias[e];
        }
        if (a.out.z) keep8(a.out, (i + it * RP) * a.out.J + j, 8, v);
        act8<ACT>(v);
        if (a.out.gate) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= gate[e];
        }
        if (a.out.residual) {
          const bf16x8 x = __builtin_bit_cast(bf16x8, res[h / 2 % SETS][it]);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += half_to_f32<F16>(x[e]);
        }
        bf16x8 y;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const bf16x2 w = pack2<F16>(v[e], v[e + 1]);
          y[e] = w[0];
          y[e + 1] = w[1];
        }
        *reinterpret_cast<bf16x8*>(static_cast<uint16_t*>(a.out.out) + (i + it * RP) * a.out.out_s + j) = y;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
  if constexpr (PT) {                          // gradients: no activation
    rounds(std::integral_constant<int, kActNone>{});
  } else {
    switch (a.out.act) {
      case kActGelu: rounds(std::integral_constant<int, kActGelu>{}); break;
      case kActGeluTanh: rounds(std::integral_constant<int, kActGeluTanh>{}); break;
      case kActSilu: rounds(std::integral_constant<int, kActSilu>{}); break;
      case kActRelu: rounds(std::integral_constant<int, kActRelu>{}); break;
      default: rounds(std::integral_constant<int, kActNone>{});
    }
  }
}

// The parts of a product that was cut along k, in their order, finished.
template <bool F16>
__global__ __launch_bounds__(256) void linear_join_kernel(Finish f, int splits) {
  const int64_t per = (f.J + 7) / 8, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= per * f.I) return;
  const int64_t i = at / per, j = at % per * 8;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int z = 0; z < splits; ++z) {
    const f32x4* p = reinterpret_cast<const f32x4*>(f.part + ((int64_t)z * f.I + i) * per * 8 + j);
    const f32x4 lo = p[0], hi = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += lo[e];
      v[4 + e] += hi[e];
    }
  }
  finish8<F16>(f, i, j, v);
}

template <int WI, int WJ, int R, int PER_CU, bool PT, bool QT, bool F16>
hipError_t gemm_launch(const GemmArgs& a, hipStream_t s) {
  const int64_t all = (int64_t)a.ti * a.tj * a.splits;
  hipLaunchKernelGGL((linear_gemm_kernel<WI, WJ, R, PER_CU, PT, QT, F16>), dim3((unsigned)((all + 7) / 8 * 8)), dim3(256), 0, s, a);
  return hipGetLastError();
}

// out = sum_k Q P as planned, and the join where k is cut.
template <bool PT, bool QT, bool F16>
hipError_t gemm(GemmArgs a, const GemmPlan& x, hipStream_t s) {
  a.ti = (int32_t)x.ti; a.tj = (int32_t)x.tj; a.splits = (int32_t)x.splits;
  hipError_t e;
  if (x.tile == 0) e = gemm_launch<8, 8, 4, 1, PT, QT, F16>(a, s);
  else if (x.tile == 2) e = gemm_launch<4, 4, 3, 2, PT, QT, F16>(a, s);
  else if (x.tile == 3) e = gemm_launch<2, 2, 4, 4, PT, QT, F16>(a, s);
  else if constexpr (!PT) e = gemm_launch<4, 8, 3, 2, PT, QT, F16>(a, s);
  else return hipErrorInvalidValue;            // not planned for turned operands
  if (e != hipSuccess || x.splits == 1) return e;
  const int64_t threads = (a.out.J + 7) / 8 * a.out.I;
  hipLaunchKernelGGL((linear_join_kernel<F16>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a.out, (int)x.splits);
  return hipGetLastError();
}

}  // namespace
}  // namespace gpa
