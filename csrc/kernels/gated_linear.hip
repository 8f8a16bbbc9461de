// Gated linear layer in 16-bit types:  h = act(x Wg^T) * (x Wu^T), and its gradients
//
//   dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// with g = x Wg^T, u = x Wu^T in fp32.
//
// Many rows: bound by the matrix cores.  One kernel computes both products: a tile's column halves
// are rows of Wg and Wu for the same outputs, so a wave ends with g and u of the same outputs in
// its accumulators and h is formed in registers.  Operand tiles go global -> LDS by DMA into two
// stages, eight waves take a k tile in four phases with one half of them a barrier behind the other
// (see take_tiles).  Rows past the end and the ragged end of k read zeros through the buffer
// descriptor's range check.  bf16, x [m][k], f outputs: 8192 x 4096 x 12288 takes 1090-1180 us
// (1400-1510 TFLOP/s; a plain library product of this size 1081 us).
//
// Backward: one launch forms dg and du side by side, another computes the three products with the same
// loop.  Where an operand has the reduction as its rows (the weights in dx, everything in dWg
// and dWu), its tile goes to LDS as it lies in memory and the fragments are read across (see
// take_tiles), so nothing is transposed in memory.  Forward and backward of 4096 x 2048 x 6144 take
// 530-570 us, of which the products' work is 412 us at 1500 TFLOP/s (with transposed copies of
// dg, du, x and the weights it was 580-600, and the backward pass of 1000 x 4096 x 4096 181 instead of
// 146).
//
// Few rows (up to 16, and up to 64 where it is faster): bound by reading the weights.  The waves of
// a workgroup cut k; each loads whole 128-byte stretches of the rows of Wg, Wu and x, forms
// fragments through a small LDS image of its own, and the waves' sums meet in LDS in a fixed order.
// bf16: 1 x 2048 x 6144 10 us (5 TB/s of weights), 33 x 4096 x 10240 41 us (4.1 TB/s).
//
// Roundings: h once; for training, g and u are kept in fp32 (a 16-bit copy would add its own
// rounding to every gradient, 1.7 instead of 1.4 times the error of the result's own rounding);
// dg and du are rounded to the operands' type because the matrix cores multiply 16-bit numbers, or,
// where the caller asks for it, taken as sums of two such numbers, for twice the products.
// Copyright 2026 veles.simd_amd authors. Apache-2.0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>
#include <utility>

#include "csrc/kernels/device.h"
#include "csrc/kernels/number.h"
#include "csrc/runtime/runtime.h"
#include "simd/gpu.h"

namespace vs {
namespace glin {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

template <class N>
__device__ __forceinline__ floatx4 mma(const u32x4 &a, const u32x4 &b, floatx4 c) {
  if constexpr (std::is_same_v<N, num::BF16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// -------------------------------------------------------------- activations
// No tail is the rest of a subtraction: it is computed and the large side is what it leaves of 1, and the
// sigmoid's slope is e / (1 + e)^2, not s (1 - s).
//
// The normal distribution Phi(g) and E = exp(-g^2 / 2).  With z = |g|, Phi(-z) / E falls smoothly from 1/2 as
// 1 / (sqrt(2 pi) z): times z + 3 it is a polynomial of degree 8 in (z - 3) / (z + 3), fitted on 0 <= z <= 14 (E
// underflows at 13.2) to the least largest relative error, 5e-8; in fp32 3.4e-7.  (8192 x 1024, 8192 outputs, gelu:
// 267 us, 305 with the library's erfcf, 295 with 1 + erff, whose tail has no digits from -5 on.)
struct Normal {
  float phi, e;
};
__device__ __forceinline__ Normal normal(float g) {
  const float z = fabsf(g), e = __expf(-0.5f * z * z), r = __builtin_amdgcn_rcpf(z + 3.f), t = fmaf(-6.f, r, 1.f);
  float p = -2.6676857e-4f;
  p = fmaf(p, t, -9.0325432e-4f);
  p = fmaf(p, t, 1.0760390e-3f);
  p = fmaf(p, t, 6.9239237e-3f);
  p = fmaf(p, t, -1.0479936e-2f);
  p = fmaf(p, t, -4.7256101e-2f);
  p = fmaf(p, t, 0.23001935f);
  p = fmaf(p, t, -0.50933230f);
  p = fmaf(p, t, 0.72908366f);
  const float tail = p * r * e;
  return Normal{g < 0.f ? tail : 1.f - tail, e};
}
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}
__device__ __forceinline__ float act(int kind, float g) {
  switch (kind) {
    case VS_ACT_SILU: return g * sigmoid(g);
    case VS_ACT_GELU: return g * normal(g).phi;
    case VS_ACT_RELU: return g > 0.f ? g : g == g ? 0.f : g;
    default: return sigmoid(g);
  }
}
__device__ __forceinline__ float act_slope(int kind, float g) {
  switch (kind) {
    case VS_ACT_SILU: {
      const float s = sigmoid(g);
      return s * fmaf(g, 1.f - s, 1.f);
    }
    case VS_ACT_GELU: {
      const Normal n = normal(g);
      return fmaf(g * 0.39894228040143268f, n.e, n.phi);
    }
    case VS_ACT_RELU: return g > 0.f ? 1.f : 0.f;
    default: {
      const float e = __expf(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + e);
      return e * r * r;
    }
  }
}

// ------------------------------------------------------------------- tiles
struct Args {
  // Forward: a [m][k], b[0] and b[1] [n][k].  Backward: a [m][k] or, with `across`, [k][m]; b [k][n].  Every
  // `fold` rows of b are b[0] and b[1] in turn, `have` rows of each (zeros behind), up to four times; with
  // `across` every `fold` rows of a begin `next` columns further on, from the first row again.
  const uint16_t *a;
  const uint16_t *b[2];
  int64_t lda, ldb[2];
  int m, n, k;            // n: outputs (columns of h, or of c)
  int across, fold, have, next;
  uint16_t *c;            // [m][n], row stride n
  float2 *pre;            // [m][n] (g, u), or null
  int act;
  // k in `parts` parts of `k_part` (a multiple of 64) when `parts` > 1: part i's sums, fp32 (pairs of
  // the gated product), go to sums + i m n and the join kernel adds them
  int parts, k_part;
  float *sums;
};

// Up to three products in a launch: tiles up to end[0] belong to q[0], up to end[1] to q[1], ...
constexpr int kProducts = 3;
struct Work {
  Args q[kProducts];
  unsigned end[kProducts];
};

// A tile of 2 (rows) x 4 (columns) waves, each with 2 x 2 quadrants of 16 XH x 16 YH products.
// GATED: the column quadrants are Wg and Wu of the same outputs.
// SAVE: of the gated product, (g, u) are results too (or the only ones: parts of the sums).
template <int XH_, int YH_, bool GATED_, bool SAVE_ = false>
struct Cfg {
  static constexpr int XH = XH_, YH = YH_, BK = 64;
  static constexpr bool GATED = GATED_, SAVE = SAVE_;
  static constexpr int BM = 64 * XH, BN = 128 * YH;    // products
  static constexpr int BO = GATED ? BN / 2 : BN;       // output columns
  static constexpr int kThreads = 512;
  static constexpr int RB = 2 * BK;                    // bytes of an image row
  static constexpr int kHalfA = BM / 2 * RB, kHalfB = BN / 2 * RB;
  static constexpr int kBuf = 2 * (kHalfA + kHalfB);   // A0 A1 B0 B1
  static constexpr int PA = kHalfA / 8192, PB = kHalfB / 8192;  // 1 KiB pieces per wave
  static constexpr int kLds = 2 * kBuf;
  static_assert(kHalfA % 8192 == 0 && kHalfB % 8192 == 0, "whole pieces for every wave");
};

constexpr uint32_t kOut = 0x80000000u;  // past every descriptor's range: reads zeros

// 16-byte chunk c of image row r lies at chunk c ^ (r / 2 & 7): the 16 rows that a fragment read
// takes at one k hit 16 different bank groups.
__device__ __forceinline__ int swz(int row, int c) { return c ^ ((row >> 1) & 7); }

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t *dst, uint32_t voff,
                                      uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass rejects a size of 16
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)dst, 16, voff, soff, 0, 0);
#endif
}

// Rows from `row0` on of a [rows][k] operand, as a buffer whose range ends with the last row.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint16_t *p, int64_t ld, int row0,
                                                          int rows, int tile, int k) {
  const int have = rows - row0 < tile ? rows - row0 : tile;
  const int64_t bytes = have > 0 ? ((have - 1) * ld + k) * 2 : 0;
  return __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t *>(p + (have > 0 ? row0 * ld : 0)), 0, static_cast<uint32_t>(bytes),
      0x00020000);
}

// Rows [row0, row0 + rows) of a [.][n] operand from column c0 on, 64 of them at most.  (Rows hold
// whole 16-byte pieces.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t columns_of(const uint16_t *p, int64_t ld, int row0,
                                                             int rows, int c0, int n) {
  const int have = rows < 64 ? rows : 64;
  const uint32_t bytes = (static_cast<uint32_t>(have - 1) * static_cast<uint32_t>(ld) + (n + 7) / 8 * 8 - c0) * 2;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p + row0 * ld + c0), 0,
                                           have > 0 ? bytes : 0u, 0x00020000);  // (0: nothing is read)
}

// Where the 32 bytes of 16 columns lie in an image row of ROW bytes that is read across: piece p of
// row r at p ^ turn(r), so the 8 rows of two 16-lane groups are in different banks.
template <int ROW>
__device__ __forceinline__ int turn(int r) {
  return ROW == 256 ? (r & 3) | (r >> 1 & 4) : (r >> 1 & 1) | (r >> 2 & 2);
}

// A fragment, in one piece or as two reads bring it.
struct Halves {
  u32x2 lo, hi;
};
template <bool T>
using Frag = std::conditional_t<T, Halves, u32x4>;
__device__ __forceinline__ const u32x4 &whole(const u32x4 &f) { return f; }
__device__ __forceinline__ u32x4 whole(const Halves &f) {
  return __builtin_shufflevector(f.lo, f.hi, 0, 1, 2, 3);
}

// Fragment reads are inline asm: the compiler would wait for every DMA in flight before a read of
// LDS that it sees.  `settle` is the wait, and the registers pass through it, so no product can
// move above it.
template <int OFF>
__device__ __forceinline__ void read_frag(u32x4 &f, uint32_t at) {
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f) : "v"(at), "i"(OFF) : "memory");
}
template <int OFF, int ROW>
__device__ __forceinline__ void read_across(Halves &f, uint32_t at) {
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.lo) : "v"(at), "i"(OFF) : "memory");
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.hi) : "v"(at), "i"(OFF + 4 * ROW) : "memory");
}
template <int XH>
__device__ __forceinline__ void settle(u32x4 (&f)[XH][2]) {
  if constexpr (XH == 4)
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(f[0][0]), "+v"(f[1][0]), "+v"(f[2][0]), "+v"(f[3][0]), "+v"(f[0][1]),
                   "+v"(f[1][1]), "+v"(f[2][1]), "+v"(f[3][1])::"memory");
  else if constexpr (XH == 2)
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(f[0][0]), "+v"(f[1][0]), "+v"(f[0][1]), "+v"(f[1][1])::"memory");
  else
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0][0]), "+v"(f[0][1])::"memory");
}
template <int XH>
__device__ __forceinline__ void settle(Halves (&f)[XH][2]) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(f[0][0].lo), "+v"(f[0][0].hi), "+v"(f[0][1].lo), "+v"(f[0][1].hi)::"memory");
  if constexpr (XH > 1)  // (no instruction: nothing may move above the wait)
    asm volatile("" : "+v"(f[1][0].lo), "+v"(f[1][0].hi), "+v"(f[1][1].lo), "+v"(f[1][1].hi)::"memory");
  if constexpr (XH > 2) {
    asm volatile("" : "+v"(f[2][0].lo), "+v"(f[2][0].hi), "+v"(f[2][1].lo), "+v"(f[2][1].hi)::"memory");
    asm volatile("" : "+v"(f[3][0].lo), "+v"(f[3][0].hi), "+v"(f[3][1].lo), "+v"(f[3][1].hi)::"memory");
  }
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// The k loop.  A k tile of 64 is taken in four phases, one quadrant of every wave's products
// each.  With first / second the column halves 0 / 1 in even tiles and 1 / 0 in odd ones:
//
//   phase  reads into registers     multiplies          starts the DMA of (two tiles ahead)
//   0      A0                       A0 x first          first
//   1      second                   A0 x second         A0
//   2      A1                       A1 x second         second
//   3      first of the next tile   A1 x first          A1
//
// (the next tile's first half is this tile's second index, whose registers are free by then).
// A phase is: start the reads and the DMA, wait for the reads, barrier, products, barrier.  Waves
// 4-7 are one barrier behind waves 0-3, so of the two waves on a SIMD one multiplies while the
// other reads and issues.  The halves h_0, h_1, ... in this order are read in phase j - 1 and
// started in phase j - 8, right after the phase that read what they overwrite: a wave's reads
// have arrived before its first barrier of a phase, and no wave is further than that barrier
// behind a wave that starts the next phase.  Before that barrier a wave also waits until its
// pieces of the half that the next phase reads have landed; six halves stay in flight.  Tiles
// past the end of k are started out of range (zeros), so the counts hold to the end.
//
// A workgroup takes tiles blockIdx.x, + gridDim.x, ...; the next tile's first eight halves are
// started before the results of the last one are stored.
// TA, TB: the operand has k as its rows.  Its image halves are 64 k of neighbouring columns then, and
// fragments are read across: ds_read_b64_tr_b16 gives lane i of 16 the i-th of 16 columns of four
// rows, whose 8-byte pieces lanes 4 r .. 4 r + 3 point at.  Columns past the end read what lies there
// (inside the operand) and are not stored.  SPLIT: their rows begin again, at most three times (TA once).
template <class N, class C, bool TA, bool TB, bool SPLIT>
__device__ __forceinline__ void take_tiles(const Args &p, unsigned begin, unsigned end, uint8_t *lds) {
  constexpr int XH = C::XH, YH = C::YH;
  constexpr int RA = TA ? 64 * XH : C::RB, RT = TB ? 128 * YH : C::RB;  // bytes of an image row
  const unsigned tiles_m = (p.m + C::BM - 1) / C::BM, tiles_n = (p.n + C::BO - 1) / C::BO;
  const uint16_t *pa = p.a, *pb0 = p.b[0], *pb1 = p.b[1];
  const int64_t lda = p.lda, ldb = p.ldb[0];
  const int pm = p.m, pn = p.n, fold = p.fold, have = p.have, next = p.next;
  // Row of the operand that step `at` of k is, and how often the rows began again before it (`most` times at most).
  const auto unfold = [&](auto most, int at, int &row) {
    int turns = 0;
    row = at;
#pragma unroll
    for (int i = 0; i < decltype(most)::value; i++)
      if (row >= fold) {
        row -= fold;
        turns++;
      }
    return turns;
  };
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid / 4, wn = wid % 4;
  const int l16 = lane & 15, lq = lane >> 4;

  int m0, n0, part, k, ks0;  // of the tile: first row and column, part, length and start of k
  __amdgpu_buffer_rsrc_t ra, rb0, rb1;
  const auto place = [&](unsigned tile) {
    unsigned tm, tn;
    const unsigned at = dev::xcd_remap(tile - begin, tiles_m * tiles_n * p.parts);
    part = at / (tiles_m * tiles_n);
    dev::grouped_tile(at - part * (tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
    m0 = tm * C::BM;
    n0 = tn * C::BO;
    ks0 = part * p.k_part;
    k = p.k - ks0 < p.k_part ? p.k - ks0 : p.k_part;
    if constexpr (!TA) ra = rows_of(p.a + ks0, p.lda, m0, p.m, C::BM, k);
    if constexpr (!TB) {
      rb0 = rows_of(p.b[0] + ks0, p.ldb[0], n0, p.n, C::BO, k);
      rb1 = C::GATED ? rows_of(p.b[1] + ks0, p.ldb[1], n0, p.n, C::BO, k) : rb0;
    }
  };
  // Image row r of A half h is row 32 XH (r / 16 XH) + 16 XH h + r % 16 XH of the tile; of B half
  // h it is the same with YH and four waves (GATED: row r of operand h).  Piece i of a wave: image rows
  // 8 (P wid + i) + lane / 8, chunk lane % 8.
  // TA, TB: column c of half h is column (half the tile) h + c of the tile.  Piece i of a wave: bytes
  // 1024 (P wid + i) on, rows of RA (RT) bytes.
  uint32_t offa[2][C::PA], offb[2][C::PB];
  int ka[C::PA], kb[C::PB];
#pragma unroll
  for (int i = 0; i < C::PA; i++) {
    if constexpr (TA) {
      const int o = (wid * C::PA + i) * 1024 + lane * 16, r = o / RA, c = o % RA / 16;
#pragma unroll
      for (int h = 0; h < 2; h++)
        offa[h][i] = static_cast<uint32_t>((r * p.lda + h * (RA / 2) + 8 * (c ^ 2 * turn<RA>(r))) * 2);
      continue;
    }
    const int r = (wid * C::PA + i) * 8 + lane / 8;
    ka[i] = 8 * swz(r, lane % 8);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int row = r / (16 * XH) * (32 * XH) + 16 * XH * h + r % (16 * XH);
      offa[h][i] = static_cast<uint32_t>((row * p.lda + ka[i]) * 2);
    }
  }
#pragma unroll
  for (int i = 0; i < C::PB; i++) {
    if constexpr (TB) {
      const int o = (wid * C::PB + i) * 1024 + lane * 16, r = o / RT, c = o % RT / 16;
#pragma unroll
      for (int h = 0; h < 2; h++)  // both operands of a fold have one row stride
        offb[h][i] = static_cast<uint32_t>((r * p.ldb[0] + h * (RT / 2) + 8 * (c ^ 2 * turn<RT>(r))) * 2);
      continue;
    }
    const int r = (wid * C::PB + i) * 8 + lane / 8;
    kb[i] = 8 * swz(r, lane % 8);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int row = C::GATED ? r : r / (16 * YH) * (32 * YH) + 16 * YH * h + r % (16 * YH);
      offb[h][i] = static_cast<uint32_t>((row * p.ldb[C::GATED ? h : 0] + kb[i]) * 2);
    }
  }
  const auto start_a = [&](auto half, auto buf, int tile) {
    constexpr int h = decltype(half)::value;
    uint8_t *dst = lds + decltype(buf)::value * C::kBuf + h * C::kHalfA + wid * (C::PA * 1024);
    const int k0 = tile * C::BK, at = k0 < k ? 2 * k0 : 0;  // (at stays inside the range)
    if constexpr (TA) {
      int row;
      const int turns = unfold(std::integral_constant<int, SPLIT ? 1 : 0>{}, ks0 + k0, row);
      const int left = have - row < k - k0 ? have - row : k - k0;
      const auto r = columns_of(pa + turns * next, lda, row, left, m0, pm);
#pragma unroll
      for (int i = 0; i < C::PA; i++) dma16(r, dst + i * 1024, offa[h][i], 0);
      return;
    }
#pragma unroll
    for (int i = 0; i < C::PA; i++)
      dma16(ra, dst + i * 1024, ka[i] < k - k0 ? offa[h][i] : kOut, at);
  };
  const auto start_b = [&](auto half, auto buf, int tile) {
    constexpr int h = decltype(half)::value;
    uint8_t *dst = lds + decltype(buf)::value * C::kBuf + 2 * C::kHalfA + h * C::kHalfB +
                   wid * (C::PB * 1024);
    const int k0 = tile * C::BK, at = k0 < k ? 2 * k0 : 0;
    if constexpr (TB) {
      int row;
      const int turns = unfold(std::integral_constant<int, SPLIT ? 3 : 1>{}, ks0 + k0, row);
      const int left = have - row < k - k0 ? have - row : k - k0;
      const auto r = columns_of(turns & 1 ? pb1 : pb0, ldb, row, left, n0, pn);
#pragma unroll
      for (int i = 0; i < C::PB; i++) dma16(r, dst + i * 1024, offb[h][i], 0);
      return;
    }
#pragma unroll
    for (int i = 0; i < C::PB; i++)
      dma16(h ? rb1 : rb0, dst + i * 1024, kb[i] < k - k0 ? offb[h][i] : kOut, at);
  };
  // LDS addresses of this lane's fragments: [buffer][32-deep step], TA, TB: [buffer][16 columns]
  uint32_t ata[2][TA ? XH : 2], atb[2][TB ? YH : 2];
  {
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)lds));
    const int arow = wm * (16 * XH) + l16, brow = wn * (16 * YH) + l16;
    const int trow = 8 * lq + l16 / 4, tcol = 8 * (l16 % 4);
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
      for (int x = 0; x < (TA ? XH : 2); x++)
        ata[b][x] = base + b * C::kBuf +
                    (TA ? trow * RA + 32 * ((wm * XH + x) ^ turn<RA>(trow)) + tcol
                        : arow * C::RB + 16 * swz(arow, 4 * x + lq));
#pragma unroll
      for (int y = 0; y < (TB ? YH : 2); y++)
        atb[b][y] = base + b * C::kBuf + 2 * C::kHalfA +
                    (TB ? trow * RT + 32 * ((wn * YH + y) ^ turn<RT>(trow)) + tcol
                        : brow * C::RB + 16 * swz(brow, 4 * y + lq));
    }
  }
  Frag<TA> fa[XH][2];
  Frag<TB> fb[2][YH][2];
  const auto read_a = [&](auto half, auto buf) {
    constexpr int O = decltype(half)::value * C::kHalfA, b = decltype(buf)::value;
    if constexpr (TA) {
#pragma unroll
      for (int x = 0; x < XH; x++) {
        read_across<O, RA>(fa[x][0], ata[b][x]);
        read_across<O + 32 * RA, RA>(fa[x][1], ata[b][x]);
      }
      return;
    } else
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      read_frag<O>(fa[0][ks], ata[b][ks]);
      if constexpr (XH > 1) read_frag<O + 2048>(fa[1][ks], ata[b][ks]);
      if constexpr (XH > 2) read_frag<O + 4096>(fa[2][ks], ata[b][ks]);
      if constexpr (XH > 2) read_frag<O + 6144>(fa[3][ks], ata[b][ks]);
    }
  };
  const auto read_b = [&](auto half, auto buf) {
    constexpr int h = decltype(half)::value, O = h * C::kHalfB, b = decltype(buf)::value;
    if constexpr (TB) {
#pragma unroll
      for (int y = 0; y < YH; y++) {
        read_across<O, RT>(fb[h][y][0], atb[b][y]);
        read_across<O + 32 * RT, RT>(fb[h][y][1], atb[b][y]);
      }
      return;
    } else
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      read_frag<O>(fb[h][0][ks], atb[b][ks]);
      if constexpr (YH > 1) read_frag<O + 2048>(fb[h][1][ks], atb[b][ks]);
    }
  };
  // Weights are the matrix instruction's first operand, so a lane ends with four neighbouring
  // columns (4 lq + r of the 16) of one row (l16) of the result.  SAVE: they are the second, and a
  // lane ends with four rows of one column, since the pairs are most of what is written then and 16
  // neighbouring lanes' pairs are 128 neighbouring bytes.
  floatx4 acc[2][XH][2][YH];
  const auto multiply = [&](auto ih, auto jh) {
    constexpr int i = decltype(ih)::value, j = decltype(jh)::value;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int x = 0; x < XH; x++)
#pragma unroll
        for (int y = 0; y < YH; y++)
          acc[i][x][j][y] = C::SAVE ? mma<N>(whole(fa[x][ks]), whole(fb[j][y][ks]), acc[i][x][j][y])
                                    : mma<N>(whole(fb[j][y][ks]), whole(fa[x][ks]), acc[i][x][j][y]);
    __builtin_amdgcn_s_setprio(0);
  };
  constexpr std::integral_constant<int, 0> c0{};
  constexpr std::integral_constant<int, 1> c1{};
  constexpr int kFlight = 3 * (C::PA + C::PB);
  const auto phases = [&](auto first, auto second, auto buf, auto other, int t) {
    constexpr int S = decltype(second)::value;
    read_a(c0, buf);
    start_b(first, buf, t + 2);
    wait_vmcnt<kFlight>();
    settle(fa);
    meet();
    multiply(c0, first);
    meet();
    read_b(second, buf);
    start_a(c0, buf, t + 2);
    wait_vmcnt<kFlight>();
    settle(fb[S]);
    meet();
    multiply(c0, second);
    meet();
    read_a(c1, buf);
    start_b(second, buf, t + 2);
    wait_vmcnt<kFlight>();
    settle(fa);
    meet();
    multiply(c1, second);
    meet();
    read_b(second, other);  // the next tile's first half
    start_a(c1, buf, t + 2);
    wait_vmcnt<kFlight>();
    settle(fb[S]);
    meet();
    multiply(c1, first);
    meet();
  };
  const auto start_tile = [&] {
    start_b(c0, c0, 0);
    start_a(c0, c0, 0);
    start_b(c1, c0, 0);
    start_a(c1, c0, 0);
    start_b(c1, c1, 1);
    start_a(c0, c1, 1);
    start_b(c0, c1, 1);
    start_a(c1, c1, 1);
  };
  place(blockIdx.x);
  start_tile();
  for (unsigned tile = blockIdx.x;;) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int x = 0; x < XH; x++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int y = 0; y < YH; y++) acc[i][x][j][y] = floatx4{0.f, 0.f, 0.f, 0.f};
    wait_vmcnt<kFlight>();
    meet();
    read_b(c0, c0);
    settle(fb[0]);
    meet();
    if (wid >= 4) meet();
    for (int t = 0; t * C::BK < k; t += 2) {
      phases(c0, c1, c0, c1, t);
      phases(c1, c0, c1, c0, t + 1);
    }
    if (wid < 4) meet();
    wait_vmcnt<0>();  // the pieces started past the end of k have written their zeros
    meet();
    // first row of accumulator rows i, first column of column block b (of 2 YH; GATED: of YH)
    const int rm = m0 + wm * (TA ? 16 * XH : 32 * XH), rn = n0 + wn * (C::GATED || TB ? 16 * YH : 32 * YH);
    const auto row_of = [&](int i, int x) { return rm + i * (TA ? 32 * XH : 16 * XH) + 16 * x; };
    const auto col_of = [&](int b) { return rn + (TB ? b / YH * (64 * YH) + 16 * (b % YH) : 16 * b); };
    const int64_t skip = static_cast<int64_t>(part) * p.m * p.n;  // where the sums of this part begin
    tile += gridDim.x;
    if (tile < end) {
      place(tile);
      start_tile();
    }

    if constexpr (C::SAVE) {
      // Odd and even lanes exchange, so that a lane stores two columns of h: of rows r and r + 1 the
      // even lane takes the first.
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int x = 0; x < XH; x++)
#pragma unroll
          for (int b = 0; b < YH; b++) {
            const int row = row_of(i, x) + 4 * lq, col = col_of(b) + l16;
            const floatx4 g = acc[i][x][0][b], u = acc[i][x][1][b];
            float2 *pre = (p.parts > 1 ? reinterpret_cast<float2 *>(p.sums) + skip : p.pre) +
                          static_cast<int64_t>(row) * p.n + col;
            const int odd = lane & 1;
#pragma unroll
            for (int r = 0; r < 4; r++)
              if (row + r < p.m && col < p.n) pre[static_cast<int64_t>(r) * p.n] = make_float2(g[r], u[r]);
            if (p.parts > 1) continue;
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
              const uint32_t v0 = N::save(act(p.act, g[r]) * u[r]);
              const uint32_t v1 = N::save(act(p.act, g[r + 1]) * u[r + 1]);
              const uint32_t give = odd ? v0 : v1;
              const uint32_t take = __builtin_amdgcn_update_dpp(0u, give, 0xb1, 0xf, 0xf, true);
              const uint32_t w = odd ? take | v1 << 16 : v0 | take << 16;
              if (row + r + odd >= p.m) continue;
              uint16_t *out = p.c + static_cast<int64_t>(row + r + odd) * p.n + (col - odd);
              if (col - odd + 1 < p.n) __builtin_memcpy(out, &w, 4);
              else if (col - odd < p.n) *out = static_cast<uint16_t>(w);
            }
          }
      if (tile >= end) return;
      continue;
    }
    if constexpr (!C::GATED)
      if (p.parts > 1) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int x = 0; x < XH; x++)
#pragma unroll
            for (int b = 0; b < 2 * YH; b++) {
              const int row = row_of(i, x) + l16, col = col_of(b) + 4 * lq;
              float *dst = p.sums + skip + static_cast<int64_t>(row) * p.n + col;
              const floatx4 v = acc[i][x][b / YH][b % YH];
              if (row >= p.m) continue;
              if (col + 4 <= p.n) {
                __builtin_memcpy(dst, &v, 16);
              } else {
#pragma unroll
                for (int r = 0; r < 3; r++)
                  if (col + r < p.n) dst[r] = v[r];
              }
            }
        if (tile >= end) return;
        continue;
      }
    // Results: rows of 16-bit values, two neighbouring 16-column blocks exchanged between odd and
    // even lane groups where there are two, so a lane stores 16 bytes.
    constexpr int NB = C::GATED ? YH : 2 * YH;
    // (Rows of any alignment: the memory pipeline takes unaligned 16-byte stores.)
    const auto put = [&](uint16_t *out, int col, const auto &v) {
      constexpr int E = sizeof(v) / 2;
      if (col + E <= p.n) {
        __builtin_memcpy(out + col, &v, sizeof(v));
      } else {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (col + e < p.n) out[col + e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1)));
      }
    };
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int x = 0; x < XH; x++) {
        const int row = row_of(i, x) + l16;
        uint32_t w[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            if constexpr (C::GATED) v[r] = act(p.act, acc[i][x][0][b][r]) * acc[i][x][1][b][r];
            else v[r] = acc[i][x][b / YH][b % YH][r];
          }
          w[b][0] = N::save(v[0]) | static_cast<uint32_t>(N::save(v[1])) << 16;
          w[b][1] = N::save(v[2]) | static_cast<uint32_t>(N::save(v[3])) << 16;
        }
        if (row >= p.m) continue;
        uint16_t *out = p.c + static_cast<int64_t>(row) * p.n;
        if constexpr (NB % 2 == 0) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
          for (int b = 0; b + 1 < NB; b += 2) {
            const u32x2 lo = __builtin_amdgcn_permlane16_swap(w[b][0], w[b + 1][0], false, false);
            const u32x2 hi = __builtin_amdgcn_permlane16_swap(w[b][1], w[b + 1][1], false, false);
            put(out, (lq & 1 ? col_of(b + 1) : col_of(b)) + 8 * (lq >> 1), u32x4{lo.x, hi.x, lo.y, hi.y});
          }
#endif
        } else {
#pragma unroll
          for (int b = 0; b < NB; b++) put(out, col_of(b) + 4 * lq, u32x2{w[b][0], w[b][1]});
        }
      }
    if (tile >= end) return;
  }
}

// The forward product: workgroups walk its tiles.
template <class N, class C>
__global__ __launch_bounds__(512) void tile_kernel(Work w) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  take_tiles<N, C, false, false, false>(w.q[0], 0, w.end[0], lds);
}
// The backward products: a workgroup per tile.
template <class N, class C, bool SPLIT>
__global__ __launch_bounds__(512) void backward_kernel(Work w) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  int i = 0;
  while (blockIdx.x >= w.end[i]) i++;
  const unsigned begin = i ? w.end[i - 1] : 0;
  if (w.q[i].across) take_tiles<N, C, true, true, SPLIT>(w.q[i], begin, 0, lds);
  else take_tiles<N, C, false, true, SPLIT>(w.q[i], begin, 0, lds);
}

// Adds the parts of up to three products, in order.  One thread per four results.
struct Join {
  Args q[kProducts];
  int64_t fours[kProducts];
};
template <class N, bool GATED>
__global__ __launch_bounds__(256) void join_kernel(Join j) {
  for (int64_t at = blockIdx.x * 256ll + threadIdx.x; at < j.fours[0] + j.fours[1] + j.fours[2];
       at += gridDim.x * 256ll) {
    int64_t i = at;
    int w = 0;
    while (i >= j.fours[w]) i -= j.fours[w++];
    const Args &p = j.q[w];
    const int64_t size = static_cast<int64_t>(p.m) * p.n;
    i *= 4;
    constexpr int V = GATED ? 2 : 1;
    float sum[4 * V] = {};
    const int have = size - i < 4 ? static_cast<int>(size - i) : 4;
    const float *src = p.sums + V * i;
    for (int s = 0; s < p.parts; s++, src += V * size) {
      if (have == 4) {
        float v[4 * V];
        __builtin_memcpy(v, src, sizeof(v));
#pragma unroll
        for (int e = 0; e < 4 * V; e++) sum[e] += v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4 * V; e++)
          if (e < V * have) sum[e] += src[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (e >= have) continue;
      if constexpr (GATED) {
        p.c[i + e] = N::save(act(p.act, sum[2 * e]) * sum[2 * e + 1]);
        if (p.pre) p.pre[i + e] = make_float2(sum[2 * e], sum[2 * e + 1]);
      } else {
        p.c[i + e] = N::save(sum[e]);
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
constexpr int kFewWaves = 8;

// Eight values of a row from k0 on, zeros from k on.  The tensor ends at `end`: before it, what lies
// behind the row may be read (and is masked).
__device__ __forceinline__ u32x4 row_end(const uint16_t *row, int k0, int k, const uint16_t *end) {
  u32x4 v = {0, 0, 0, 0};
  if (k0 >= k) return v;
  if (row + k0 + 8 <= end) {
    __builtin_memcpy(&v, row + k0, 16);
#pragma unroll
    for (int i = 0; i < 4; i++)
      v[i] &= k0 + 2 * i + 1 < k ? 0xffffffffu : k0 + 2 * i < k ? 0xffffu : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (k0 + i < k) v[i / 2] |= static_cast<uint32_t>(row[k0 + i]) << (16 * (i & 1));
  }
  return v;
}

// RT row tiles of 16, CT column tiles of 16 outputs.  The rows are read once per workgroup (from
// the caches), the weights once.  A step is 64 k: the 128 bytes of a row are loaded by eight
// neighbouring lanes and fragments are formed through LDS, a 2 KB image of 16 rows each.  (Loads
// in fragment order, 16 rows in 16 neighbouring lanes, cost the cache four times the lookups:
// one CU took in 31 bytes a nanosecond that way.)  Two steps are in flight; their loads are
// issued unconditionally (past the end the last step again), since a load under a condition would
// make the compiler wait for all.
template <class N, int RT, int CT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(Args p) {
  constexpr int H = kFewWaves / 2, kImages = 2 * CT + RT;
  union Shared {
    u32x4 image[kFewWaves][kImages][128];
    float part[H][2 * CT * RT * 4][64];
  };
  __shared__ Shared lds;
  auto &part = lds.part;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int r8 = lane / 8, c8 = lane % 8;  // row (of 8) and 16-byte chunk that this lane loads
  const int n0 = blockIdx.x * (16 * CT);
  const uint16_t *row[kImages][2];  // Wg and Wu of each column tile, then the rows of x
#pragma unroll
  for (int h = 0; h < 2; h++) {
#pragma unroll
    for (int c = 0; c < CT; c++) {
      const int n = n0 + 16 * c + 8 * h + r8 < p.n ? n0 + 16 * c + 8 * h + r8 : p.n - 1;
#pragma unroll
      for (int i = 0; i < 2; i++) row[2 * c + i][h] = p.b[i] + n * p.ldb[i];
    }
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const int m = 16 * t + 8 * h + r8 < p.m ? 16 * t + 8 * h + r8 : p.m - 1;
      row[2 * CT + t][h] = p.a + m * p.lda;  // copies of the last row are not stored
    }
  }
  const int steps = (p.k + 63) / 64, per = (steps + kFewWaves - 1) / kFewWaves;
  const int first = wave * per, last = first + per < steps ? first + per : steps;
  const int whole = last * 64 <= p.k ? last : last - 1;  // steps that end inside their rows
  struct Step {
    u32x4 v[kImages][2];
  };
  const auto fetch = [&](Step &s, int st) {
#pragma unroll
    for (int j = 0; j < kImages; j++)
#pragma unroll
      for (int h = 0; h < 2; h++) __builtin_memcpy(&s.v[j][h], row[j][h] + st * 64 + 8 * c8, 16);
  };
  floatx4 acc[2][CT][RT];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
      for (int t = 0; t < RT; t++) acc[i][c][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  u32x4 *image = &lds.image[wave][0][0];
  const auto multiply = [&](const Step &s) {
    // LDS works in order within a wave: the reads see these writes, and the next step's writes
    // come after them
#pragma unroll
    for (int j = 0; j < kImages; j++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        image[128 * j + 8 * (8 * h + r8) + swz(8 * h + r8, c8)] = s.v[j][h];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int at = 8 * l16 + swz(l16, 4 * h + lq);
      u32x4 w[2 * CT], x[RT];
#pragma unroll
      for (int j = 0; j < 2 * CT; j++) w[j] = image[128 * j + at];
#pragma unroll
      for (int t = 0; t < RT; t++) x[t] = image[128 * (2 * CT + t) + at];
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int c = 0; c < CT; c++) acc[i][c][t] = mma<N>(x[t], w[2 * c + i], acc[i][c][t]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  if (first < whole) {
    Step v[2];
#pragma unroll
    for (int u = 0; u < 2; u++) fetch(v[u], first + u < whole ? first + u : whole - 1);
    int st = first;
    for (; st + 2 <= whole; st += 2)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        multiply(v[u]);
        fetch(v[u], st + u + 2 < whole ? st + u + 2 : whole - 1);
      }
    if (st < whole) multiply(v[0]);
  }
  if (first < last && whole < last) {  // the rows end inside the last step
    Step t;
    const int k0 = whole * 64 + 8 * c8;
    const uint16_t *end[3] = {p.b[0] + (p.n - 1) * p.ldb[0] + p.k, p.b[1] + (p.n - 1) * p.ldb[1] + p.k,
                              p.a + (p.m - 1) * p.lda + p.k};
#pragma unroll
    for (int j = 0; j < kImages; j++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        t.v[j][h] = row_end(row[j][h], k0, p.k, end[j < 2 * CT ? j % 2 : 2]);
    multiply(t);
  }
  __syncthreads();  // the images make room for the sums
  // waves 4..7 add to waves 0..3, and those four are added in order
  const auto slot = [&](int i, int c, int t, int r) { return ((i * CT + c) * RT + t) * 4 + r; };
#pragma unroll
  for (int half = 1; half >= 0; half--) {
    if (wave / H == half)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
          for (int t = 0; t < RT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              float *at = &part[wave % H][slot(i, c, t, r)][lane];
              *at = half ? acc[i][c][t][r] : *at + acc[i][c][t][r];
            }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < CT * RT * 256; e += 64 * kFewWaves) {
    const int c = e / (RT * 256), t = e / 256 % RT, r = e / 64 % 4, l = e % 64;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int v = 0; v < H; v++) {
      g += part[v][slot(0, c, t, r)][l];
      u += part[v][slot(1, c, t, r)][l];
    }
    const int m = 16 * t + 4 * (l / 16) + r, n = n0 + 16 * c + l % 16;
    if (m >= p.m || n >= p.n) continue;
    const int64_t at = static_cast<int64_t>(m) * p.n + n;
    p.c[at] = N::save(act(p.act, g) * u);
    if (p.pre) p.pre[at] = make_float2(g, u);
  }
}

// ------------------------------------------------- layout and element-wise
// Up to three matrices [rows][cols] (row stride ld) copied to rows of cols_p, zeros behind: rows that
// the DMA can read.  One thread per 16-byte piece, the matrices one after the other.
struct Pad {
  const uint16_t *src[3];
  int64_t ld[3], pieces[3];
  uint16_t *dst[3];
  int cols, cols_p;
};
__global__ __launch_bounds__(256) void pad_kernel(Pad p) {
  const int chunks = p.cols_p / 8;
  const int64_t all = p.pieces[0] + p.pieces[1] + p.pieces[2];
  for (int64_t at = blockIdx.x * 256ll + threadIdx.x; at < all; at += gridDim.x * 256ll) {
    int64_t i = at;
    int j = 0;
    while (i >= p.pieces[j]) i -= p.pieces[j++];
    const int64_t r = i / chunks;
    const int c = static_cast<int>(i - r * chunks) * 8;
    const uint16_t *s = p.src[j] + r * p.ld[j] + c;
    uint32_t e[4] = {0, 0, 0, 0};
    if (c + 8 <= p.cols) {
      __builtin_memcpy(e, s, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (c + k < p.cols) e[k / 2] |= static_cast<uint32_t>(s[k]) << (16 * (k & 1));
    }
    *reinterpret_cast<uint4 *>(p.dst[j] + r * p.cols_p + c) = uint4{e[0], e[1], e[2], e[3]};
  }
}

// The gradients of g and u as the backward products read them: [m][2 fp], dg's columns, then du's, zeros
// behind each.  With `split` every one is the sum of two 16-bit numbers (to 2^-16 of it in bf16, 2^-22 or 2^-25
// in fp16), and the rows are [4 fp], the second numbers in the same order behind the first.
struct Slopes {
  const uint16_t *dh;
  int64_t ld;
  const float2 *pre;
  int act, m, f, fp, split;
  uint16_t *rows;
};
// What the rounded value `hi` leaves of v; nothing where it is infinite or no number.
template <class N>
__device__ __forceinline__ uint16_t rest(float v, uint16_t hi) {
  const float r = v - N::load(hi);
  return N::save(fabsf(r) < __builtin_inff() ? r : 0.f);
}

// Four columns of a row a thread: 32 bytes of pairs, 8 of dh and of each result.
template <class N>
__global__ __launch_bounds__(256) void slope_kernel(Slopes p) {
  const int64_t all = static_cast<int64_t>(p.m) * (p.fp / 4);
  for (int64_t at = blockIdx.x * 256ll + threadIdx.x; at < all; at += gridDim.x * 256ll) {
    const int64_t r = at / (p.fp / 4);
    const int c = static_cast<int>(at - r * (p.fp / 4)) * 4;
    const float2 *s = p.pre + r * p.f + c;
    const uint16_t *q = p.dh + r * p.ld + c;
    float2 gu[4] = {};
    uint16_t d[4] = {};
    if (c + 4 <= p.f) {
      __builtin_memcpy(gu, s, 32);
      __builtin_memcpy(d, q, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (c + e < p.f) {
          gu[e] = s[e];
          d[e] = q[e];
        }
    }
    uint16_t dg[4], du[4];
    float vg[4], vu[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {  // 0 behind the row: d, g and u are
      const float v = N::load(d[e]);
      vg[e] = v * gu[e].y * act_slope(p.act, gu[e].x);
      vu[e] = v * act(p.act, gu[e].x);
      // one fp32 number each: the compiler would round a product to 16 bits by itself in one place and by way of
      // fp32 in the other, and rest() would be that of the number next to the one stored
      asm("" : "+v"(vg[e]), "+v"(vu[e]));
      dg[e] = N::save(vg[e]);
      du[e] = N::save(vu[e]);
    }
    uint16_t *dst = p.rows + r * (p.split ? 4 : 2) * p.fp + c;
    __builtin_memcpy(dst, dg, 8);
    __builtin_memcpy(dst + p.fp, du, 8);
    if (p.split) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        dg[e] = rest<N>(vg[e], dg[e]);
        du[e] = rest<N>(vu[e], du[e]);
      }
      __builtin_memcpy(dst + 2 * p.fp, dg, 8);
      __builtin_memcpy(dst + 3 * p.fp, du, 8);
    }
  }
}

// -------------------------------------------------------------------- host
constexpr int kFewRows = 64;
constexpr int64_t kMostLd = 1 << 21;  // 32-bit offsets over 256 rows
int up8(int64_t v) { return static_cast<int>((v + 7) / 8 * 8); }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Whether the DMA can read a [.][k] operand where it is: whole 16-byte chunks.
bool direct(const void *p, int64_t ld, int64_t k) {
  return k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

int k_tiles(const Args &p) { return (std::min(p.k, p.k_part) + 63) / 64; }

template <class C>
int64_t tiles_of(const Args &p) {
  return static_cast<int64_t>((p.m + C::BM - 1) / C::BM) * ((p.n + C::BO - 1) / C::BO) * p.parts;
}

// Tiles of one launch.  Backward a grid holds fewer than 2^32 threads; forward workgroups walk the tiles.
template <class C>
constexpr int64_t kMostTiles = C::GATED ? 1ll << 31 : 1ll << 23;

template <class N, class C, bool SPLIT>
vs_status launch_tile(const Args *q, int count, hipStream_t s) {
  constexpr auto kernel = [] {
    if constexpr (C::GATED) return &tile_kernel<N, C>;
    else return &backward_kernel<N, C, SPLIT>;
  }();
  static const hipError_t attr = hipFuncSetAttribute(
      reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds);
  VS_HIP(attr);
  Work w{};
  int64_t tiles = 0;
  for (int i = 0; i < kProducts; i++) {
    if (i < count) {
      w.q[i] = q[i];
      tiles += tiles_of<C>(q[i]);
    }
    VS_REQUIRE(tiles < kMostTiles<C>, "gated_linear: too many output tiles");
    w.end[i] = static_cast<unsigned>(tiles);
  }
  // forward: as many workgroups as fit the chip walk the tiles; backward: a workgroup per tile, the
  // longer products' first, so whichever CU is free takes the next
  const int64_t fit = static_cast<int64_t>(device_cu_count()) * (160 * 1024 / C::kLds);
  const unsigned grid = static_cast<unsigned>(C::GATED ? std::min(tiles, fit) : tiles);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(C::kThreads), C::kLds, s, w);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

constexpr double kNever = 1e30;  // the estimate of what does not fit a launch

// Estimated time, in units of 1 us at the sizes below, of `count` products with tiles of C.  A tile
// of nk k tiles takes `fixed` + `step` nk when the chip is full of them and `fixed` + `alone` nk
// when there are few (fewer share the caches and the power).  Measured at x [m][k], f outputs, both
// ways round: 1000 x 4096 x 4096 takes 83 us in 256 x 256 tiles and 60 in 128 x 256,
// 4096 x 4096 x 4096 192 and 233 (243 in 128 x 128), 256 x 2048 x 8192 43, 30 and 23.
template <class C>
double estimate(const Args *q, int count) {
  constexpr double fixed = C::XH == 4 ? 6.5 : C::YH == 2 ? 4.8 : 3.5;
  constexpr double step = C::XH == 4 ? 1.36 : C::YH == 2 ? 0.83 : 0.89;
  constexpr double alone = C::XH == 4 ? 0.92 : C::YH == 2 ? 0.59 : 0.42;
  const double slots = device_cu_count() * (160 * 1024 / C::kLds);
  double total = 0, longest = 0, t = 0;
  int64_t tiles = 0;
  for (int i = 0; i < count; i++) tiles += tiles_of<C>(q[i]);
  if (tiles >= kMostTiles<C>) return kNever;
  for (int i = 0; i < count; i++) {
    const double nk = k_tiles(q[i]), n = static_cast<double>(tiles_of<C>(q[i]));
    const int64_t rounds = static_cast<int64_t>(n / slots);
    const double rest = n - static_cast<double>(rounds) * slots;
    t = static_cast<double>(rounds) * (fixed + step * nk) +
        (rest > 0 ? fixed + std::max(alone, step * rest / slots) * nk : 0);
    total += n * (fixed + step * nk) / slots;
    longest = std::max(longest, fixed + alone * nk);
  }
  return count == 1 ? t : std::max(longest, total);
}

// Few tiles and a long k leave most of the chip idle: then k is cut, the parts' sums go through memory
// in fp32, and another launch adds them, which takes about 4 us and reads what was written at
// about 4 TB/s.  Parts are doubled for the products with the longest tiles as long as the
// estimate falls.  us in one part and as chosen, bf16: 300 x 8192 to 200 outputs 65 and 20, the backward pass of
// 64 x 2048 with 16384 outputs 333 and 95, of 8192 x 256 with 256 outputs 79 and 26.
size_t sums_bytes(const Args &p, bool gated) {
  return p.parts > 1 ? up256(static_cast<size_t>(gated ? 8 : 4) * p.parts * p.m * p.n) : 0;
}
template <class C>
double cut(Args *q, int count) {
  const auto cost = [&] {
    double bytes = 0, memory = 0;  // the parts' sums; the operands once
    for (int i = 0; i < count; i++) bytes += static_cast<double>(sums_bytes(q[i], C::GATED));
    for (int i = 0; i < count; i++) memory += 2.0 * q[i].k * (q[i].m + (C::GATED ? 2.0 : 1.0) * q[i].n) / 5e6;
    const double time = estimate<C>(q, count);
    return std::max(time, memory) + 0.01 * time + (bytes > 0 ? 4 + bytes / 2e6 : 0);
  };
  for (int i = 0; i < count; i++) q[i].parts = 1, q[i].k_part = std::max(q[i].k, 1);
  double best = cost();
  for (;;) {
    Args before[kProducts];
    int longest = 0;
    for (int i = 0; i < count; i++) {
      before[i] = q[i];
      longest = std::max(longest, k_tiles(q[i]));
    }
    if (longest < 8) return best;
    for (int i = 0; i < count; i++)
      if (k_tiles(q[i]) == longest && q[i].parts >= 32) return best;
    for (int i = 0; i < count; i++) {
      if (k_tiles(before[i]) < longest) continue;
      q[i].k_part = (longest + 1) / 2 * 64;
      q[i].parts = (q[i].k + q[i].k_part - 1) / q[i].k_part;
    }
    const double now = cost();
    if (now >= best) {
      std::copy(before, before + count, q);
      return best;
    }
    best = now;
  }
}

// Tile shape (0: 256 x 256, 1: 128 x 256, 2: 128 x 128; -1: too many tiles of every shape) and the parts of each
// product.
template <bool GATED>
int plan(Args *q, int count) {
  Args w[kProducts], s[kProducts];
  for (int i = 0; i < count; i++) w[i] = s[i] = q[i];
  const double large = cut<Cfg<4, 2, GATED>>(q, count), wide = cut<Cfg<2, 2, GATED>>(w, count),
               small = cut<Cfg<2, 1, GATED>>(s, count);
  if (std::min({large, wide, small}) >= kNever) return -1;
  if (large <= wide && large <= small) return 0;
  for (int i = 0; i < count; i++) q[i] = wide <= small ? w[i] : s[i];
  return wide <= small ? 1 : 2;
}

template <class N, bool GATED, bool SAVE, bool SPLIT>
vs_status launch_shape(int shape, const Args *q, int count, hipStream_t s) {
  if (shape == 0) return launch_tile<N, Cfg<4, 2, GATED, SAVE>, SPLIT>(q, count, s);
  if (shape == 1) return launch_tile<N, Cfg<2, 2, GATED, SAVE>, SPLIT>(q, count, s);
  return launch_tile<N, Cfg<2, 1, GATED, SAVE>, SPLIT>(q, count, s);
}

template <class N, bool GATED, bool SPLIT = false>
vs_status product(int shape, const Args *q, int count, hipStream_t s) {
  if constexpr (GATED) {
    if (q->pre || q->parts > 1) VS_TRY((launch_shape<N, true, true, false>(shape, q, count, s)));
    else VS_TRY((launch_shape<N, true, false, false>(shape, q, count, s)));
  } else {
    VS_TRY((launch_shape<N, false, false, SPLIT>(shape, q, count, s)));
  }
  Join j{};
  int n = 0;
  for (int i = 0; i < count; i++)
    if (q[i].parts > 1) {
      j.fours[n] = (static_cast<int64_t>(q[i].m) * q[i].n + 3) / 4;
      j.q[n++] = q[i];
    }
  if (const int64_t all = j.fours[0] + j.fours[1] + j.fours[2]) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((all + 255) / 256, 1 << 20));
    hipLaunchKernelGGL((join_kernel<N, GATED>), dim3(grid), dim3(256), 0, s, j);
    VS_HIP(hipGetLastError());
  }
  return VS_OK;
}

// Bump allocator over the caller's workspace or the library's pool.
struct Space {
  uint8_t *base = nullptr;
  size_t used = 0;
  uint16_t *take(size_t elems) {
    uint8_t *p = base + used;
    used += up256(2 * elems);
    return reinterpret_cast<uint16_t *>(p);
  }
  float *take_sums(size_t bytes) { return reinterpret_cast<float *>(take(bytes / 2)); }
};

vs_status open_space(Space &sp, DeviceBuffer &own, void *workspace, size_t bytes, size_t need,
                     hipStream_t s) {
  if (need == 0) return VS_OK;
  if (workspace) {
    VS_REQUIRE(bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "gated_linear: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    sp.base = static_cast<uint8_t *>(workspace);
  } else {
    VS_TRY(own.alloc(need, s));
    sp.base = own.as<uint8_t>();
  }
  return VS_OK;
}

// Copies of operands whose rows the DMA cannot read, to rows of whole 16-byte pieces.
struct Copies {
  Space &sp;
  Pad pd{};
  int n = 0;
  Copies(Space &space, int cols) : sp(space) {
    pd.cols = cols;
    pd.cols_p = up8(cols);
  }
  void add(const uint16_t *&src, int64_t &ld, int64_t rows) {
    pd.src[n] = src;
    pd.ld[n] = ld;
    pd.dst[n] = sp.take(static_cast<size_t>(rows) * pd.cols_p);
    pd.pieces[n] = rows * (pd.cols_p / 8);
    src = pd.dst[n++];
    ld = pd.cols_p;
  }
  vs_status launch(hipStream_t s) {
    if (const int64_t all = pd.pieces[0] + pd.pieces[1] + pd.pieces[2]) {
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>((all + 255) / 256, 1 << 20));
      hipLaunchKernelGGL(pad_kernel, dim3(grid), dim3(256), 0, s, pd);
      VS_HIP(hipGetLastError());
    }
    return VS_OK;
  }
};

vs_status check(const char *who, int dtype, int act, int64_t m, int64_t f, int64_t k) {
  VS_REQUIRE(dtype == VS_F16 || dtype == VS_BF16, "%s: unsupported dtype %d (fp16, bf16)", who, dtype);
  VS_REQUIRE(act >= VS_ACT_SILU && act <= VS_ACT_SIGMOID, "%s: unknown activation %d", who, act);
  VS_REQUIRE(m >= 0 && f >= 0 && k >= 0, "%s: negative dimension", who);
  // 32-bit offsets inside a tile of 256 rows; tile counts inside one grid
  VS_REQUIRE(m < (1ll << 31) - 256 && f <= (1 << 20) && k <= (1 << 20),
             "%s: dimension too large (rows < 2^31, features <= 2^20)", who);
  return VS_OK;
}

struct ForwardNeed {
  bool px, pg, pu;  // copies to rows that the DMA can read
  int shape;
  size_t sums, bytes;
};
// Sets p's parts as well.
ForwardNeed forward_need(Args &p, bool dx, bool dg, bool du) {
  ForwardNeed q{};
  q.px = !dx;
  q.pg = !dg;
  q.pu = !du;
  const size_t kp = up8(p.k);
  q.shape = plan<true>(&p, 1);
  q.sums = sums_bytes(p, true);
  const size_t m = p.m, n = p.n;
  q.bytes = q.sums + (q.px ? up256(2 * m * kp) : 0) + ((q.pg ? 1 : 0) + (q.pu ? 1 : 0)) * up256(2 * n * kp);
  return q;
}

template <class N, int RT, int CT>
void launch_few_as(const Args &p, hipStream_t s) {
  hipLaunchKernelGGL((few_kernel<N, RT, CT>), dim3(static_cast<unsigned>((p.n + 16 * CT - 1) / (16 * CT))),
                     dim3(64 * kFewWaves), 0, s, p);
}

// Column tiles of few_kernel for up to kFewRows rows; 0: the tile kernel is faster.  One CU takes in
// about 40 bytes a nanosecond of weights and rows this way and the chip about 5.5 TB/s of weights;
// workgroups of two column tiles run one at a time.  us at 48 rows with one tile, two tiles and the
// tile kernel: 8192 x 16384 114, 98, 125; 2048 x 6144 19, 17, 22; 4096 x 10240 46, 50, 42;
// 4096 x 4096 17, 23, 36.
int few_columns(const Args &p, bool all_direct) {
  const int rt = (p.m + 15) / 16;
  if (rt == 1) return 1;
  const double cu = device_cu_count(), memory = 4.0 * p.n * p.k / 5.5e6;
  const auto few = [&](int ct) {
    const double groups = (p.n + 16 * ct - 1) / (16 * ct) / cu;
    const double rounds = ct == 2 ? std::ceil(groups) : std::max(1.0, groups);
    return 3 + std::max(memory, rounds * (64.0 * ct + 32.0 * rt) * p.k / 40e3);
  };
  const double one = few(1), two = few(2);
  Args one_part = p;
  one_part.parts = 1;
  one_part.k_part = std::max(p.k, 1);
  const double tile = 5 + std::max(estimate<Cfg<2, 1, true>>(&one_part, 1), 4.0 * p.n * p.k / 4.6e6);
  if (all_direct && tile < std::min(one, two)) return 0;
  return one <= two ? 1 : 2;
}

template <class N>
void launch_few(const Args &p, int ct, hipStream_t s) {
  if (p.m <= 16) launch_few_as<N, 1, 1>(p, s);
  else if (p.m <= 32) ct == 2 ? launch_few_as<N, 2, 2>(p, s) : launch_few_as<N, 2, 1>(p, s);
  else if (p.m <= 48) ct == 2 ? launch_few_as<N, 3, 2>(p, s) : launch_few_as<N, 3, 1>(p, s);
  else ct == 2 ? launch_few_as<N, 4, 2>(p, s) : launch_few_as<N, 4, 1>(p, s);
}

template <class N>
vs_status forward(Args p, void *workspace, size_t bytes, hipStream_t s) {
  const bool da = direct(p.a, p.lda, p.k), dg = direct(p.b[0], p.ldb[0], p.k),
             du = direct(p.b[1], p.ldb[1], p.k);
  if (p.m <= kFewRows) {
    if (const int ct = few_columns(p, da && dg && du)) {
      launch_few<N>(p, ct, s);
      VS_HIP(hipGetLastError());
      return VS_OK;
    }
  }
  const ForwardNeed q = forward_need(p, da, dg, du);
  VS_REQUIRE(q.shape >= 0, "gated_linear: too many output tiles");
  DeviceBuffer own;
  Space sp;
  VS_TRY(open_space(sp, own, workspace, bytes, q.bytes, s));
  const int kp = up8(p.k);
  Copies copies(sp, p.k);
  if (q.px) copies.add(p.a, p.lda, p.m);
  if (q.pg) copies.add(p.b[0], p.ldb[0], p.n);
  if (q.pu) copies.add(p.b[1], p.ldb[1], p.n);
  VS_TRY(copies.launch(s));
  if (q.sums) p.sums = sp.take_sums(q.sums);
  p.k = kp;  // (the same where nothing was copied: a direct operand has whole pieces)
  if (p.parts == 1) p.k_part = kp;
  return product<N, true>(q.shape, &p, 1, s);
}

// The backward products, the longer k first: dx = [dg du] [Wg; Wu], dWg = dg^T x and dWu = du^T x.  `split`: k
// is twice as long, for the second numbers.
struct BackwardNeed {
  Args q[kProducts];
  int count, shape;
  int dx, dw[2];  // which of q each is, or -1
  size_t bytes;
};
BackwardNeed backward_need(int64_t m, int64_t f, int64_t k, bool dx, bool dwg, bool dwu, bool split, bool ax,
                           bool aw) {
  BackwardNeed b{};
  const int fp = static_cast<int>((f + 63) / 64 * 64), mp = static_cast<int>((m + 63) / 64 * 64);
  const auto add = [&](int64_t rows, int inner, int fold, int64_t have, int across) {
    Args &p = b.q[b.count];
    p.m = static_cast<int>(rows);
    p.n = static_cast<int>(k);
    p.k = inner;
    p.fold = fold;
    p.have = static_cast<int>(have);
    p.next = 2 * fp;
    p.across = across;
    return b.count++;
  };
  b.dx = b.dw[0] = b.dw[1] = -1;
  const bool first = 2 * fp >= m;
  const int s = split ? 2 : 1;
  if (dx && m && first) b.dx = add(m, 2 * s * fp, fp, f, 0);
  for (int i = 0; i < 2; i++)
    if ((i ? dwu : dwg) && f) b.dw[i] = add(f, split ? 2 * mp : static_cast<int>(m), mp, m, 1);
  if (dx && m && !first) b.dx = add(m, 2 * s * fp, fp, f, 0);
  const size_t kp = up8(k);
  b.bytes = up256(2 * m * s * 2 * fp) + ((dwg || dwu) && !ax ? up256(2 * m * kp) : 0) +
            (dx && !aw ? 2 * up256(2 * f * kp) : 0);
  if (b.count) b.shape = plan<false>(b.q, b.count);
  for (int i = 0; i < b.count; i++) b.bytes += sums_bytes(b.q[i], false);
  return b;
}

template <class N>
vs_status backward(const uint16_t *x, int64_t ldx, const uint16_t *wg, int64_t ldg,
                   const uint16_t *wu, int64_t ldu, const float2 *pre, const uint16_t *dh,
                   int64_t ldh, int act, bool split, int m, int f, int k, uint16_t *dx, uint16_t *const (&dw)[2],
                   void *workspace, size_t bytes, hipStream_t s) {
  DeviceBuffer own;
  Space sp;
  // read as they are: rows apart (what lies behind the last one has to be out of range), and both weights
  // with one row stride
  const bool ax = direct(x, ldx, k) && ldx >= k && ldx < kMostLd,
             aw = direct(wg, ldg, k) && direct(wu, ldu, k) && ldg == ldu && ldg >= k && ldg < kMostLd;
  BackwardNeed need = backward_need(m, f, k, dx, dw[0], dw[1], split, ax, aw);
  VS_REQUIRE(need.shape >= 0, "gated_linear_backward: too many output tiles");
  VS_TRY(open_space(sp, own, workspace, bytes, need.bytes, s));
  const int fp = (f + 63) / 64 * 64, ld = (split ? 4 : 2) * fp;
  Slopes sl{};
  sl.dh = dh;
  sl.ld = ldh;
  sl.pre = pre;
  sl.act = act;
  sl.m = m;
  sl.f = f;
  sl.fp = fp;
  sl.split = split;
  sl.rows = sp.take(static_cast<size_t>(m) * ld);
  if (const int64_t n = static_cast<int64_t>(m) * (fp / 4)) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 1 << 20));
    hipLaunchKernelGGL((slope_kernel<N>), dim3(grid), dim3(256), 0, s, sl);
    VS_HIP(hipGetLastError());
  }
  Copies copies(sp, k);
  if ((dw[0] || dw[1]) && !ax) copies.add(x, ldx, m);
  if (dx && !aw) {
    copies.add(wg, ldg, f);
    copies.add(wu, ldu, f);
  }
  VS_TRY(copies.launch(s));
  if (need.dx >= 0) {
    Args &p = need.q[need.dx];
    p.a = sl.rows;
    p.lda = ld;
    p.b[0] = wg;
    p.b[1] = wu;
    p.ldb[0] = ldg;
    p.c = dx;
  }
  for (int i = 0; i < 2; i++)
    if (need.dw[i] >= 0) {
      Args &p = need.q[need.dw[i]];
      p.a = sl.rows + i * fp;
      p.lda = ld;
      p.b[0] = p.b[1] = x;
      p.ldb[0] = ldx;
      p.c = dw[i];
    }
  for (int i = 0; i < need.count; i++)
    if (const size_t sums = sums_bytes(need.q[i], false)) need.q[i].sums = sp.take_sums(sums);
  if (!need.count) return VS_OK;
  return split ? product<N, false, true>(need.shape, need.q, need.count, s)
               : product<N, false>(need.shape, need.q, need.count, s);
}

vs_status check_gradients(int dtype, int act, bool split, int64_t m, int64_t f, int64_t k) {
  VS_TRY(check("gated_linear_backward", dtype, act, m, f, k));
  // twice the reduction, and rows of four numbers a feature, have to stay inside the same offsets
  VS_REQUIRE(!split || (m < (1ll << 30) - 256 && f <= (1 << 19)),
             "gated_linear_backward: dimension too large for split gradients (rows < 2^30, features <= 2^19)");
  return VS_OK;
}

}  // namespace
}  // namespace glin
}  // namespace vs

using namespace vs;

extern "C" {

size_t vs_gated_linear_workspace(int64_t m, int64_t f, int64_t k, int aligned) {
  if (glin::check("", VS_BF16, 0, m, f, k) != VS_OK || m == 0 || f == 0) return 0;
  glin::Args p{};
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(f);
  p.k = static_cast<int>(k);
  if (m <= glin::kFewRows && glin::few_columns(p, aligned != 0)) return 0;
  return glin::forward_need(p, aligned != 0, aligned != 0, aligned != 0).bytes;
}

vs_status vs_gated_linear(int dtype, int act, const void *x, int64_t ldx, const void *w_gate,
                          int64_t ld_gate, const void *w_up, int64_t ld_up, int64_t m, int64_t f,
                          int64_t k, void *h, float *pre, void *workspace, size_t workspace_bytes,
                          vs_stream_t stream) {
  clear_error();
  VS_TRY(glin::check("gated_linear", dtype, act, m, f, k));
  if (m == 0 || f == 0) return VS_OK;
  VS_REQUIRE(h && (k == 0 || (x && w_gate && w_up)), "gated_linear: null pointer");
  VS_REQUIRE((m == 1 || ldx >= k || ldx == 0) && (f == 1 || (ld_gate >= k && ld_up >= k)),
             "gated_linear: leading dimension too small");
  VS_REQUIRE(ldx < (1 << 21) && ld_gate < (1 << 21) && ld_up < (1 << 21),
             "gated_linear: leading dimension too large (2^21)");
  glin::Args p{};
  p.a = static_cast<const uint16_t *>(x);
  p.lda = ldx;
  p.b[0] = static_cast<const uint16_t *>(w_gate);
  p.ldb[0] = ld_gate;
  p.b[1] = static_cast<const uint16_t *>(w_up);
  p.ldb[1] = ld_up;
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(f);
  p.k = static_cast<int>(k);
  p.c = static_cast<uint16_t *>(h);
  p.pre = reinterpret_cast<float2 *>(pre);
  p.act = act;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == VS_BF16 ? glin::forward<num::BF16>(p, workspace, workspace_bytes, s)
                          : glin::forward<num::F16>(p, workspace, workspace_bytes, s);
}

size_t vs_gated_linear_gradients_workspace(int64_t m, int64_t f, int64_t k, int split, int want_dx,
                                           int want_dw_gate, int want_dw_up, int aligned) {
  if (glin::check_gradients(VS_BF16, 0, split != 0, m, f, k) != VS_OK || k == 0) return 0;
  const bool al = aligned != 0;
  return glin::backward_need(m, f, k, want_dx != 0, want_dw_gate != 0, want_dw_up != 0, split != 0, al, al).bytes;
}

vs_status vs_gated_linear_gradients(int dtype, int act, int split, const void *x, int64_t ldx,
                                    const void *w_gate, int64_t ld_gate, const void *w_up,
                                    int64_t ld_up, const float *pre, const void *dh, int64_t ld_dh,
                                    int64_t m, int64_t f, int64_t k, void *dx, void *dw_gate,
                                    void *dw_up, void *workspace, size_t workspace_bytes,
                                    vs_stream_t stream) {
  clear_error();
  VS_TRY(glin::check_gradients(dtype, act, split != 0, m, f, k));
  if (k == 0 || (!dx && !dw_gate && !dw_up)) return VS_OK;
  VS_REQUIRE((m == 0 || f == 0) || (x && w_gate && w_up && pre && dh),
             "gated_linear_backward: null pointer");
  VS_REQUIRE((m <= 1 || ((ldx >= k || ldx == 0) && (ld_dh >= f || ld_dh == 0))) &&
                 (f <= 1 || (ld_gate >= k && ld_up >= k)),
             "gated_linear_backward: leading dimension too small");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto u16 = [](const void *v) { return static_cast<const uint16_t *>(v); };
  uint16_t *const dw[2] = {static_cast<uint16_t *>(dw_gate), static_cast<uint16_t *>(dw_up)};
  const auto go = [&](auto tag) {
    using N = decltype(tag);
    return glin::backward<N>(u16(x), ldx, u16(w_gate), ld_gate, u16(w_up), ld_up,
                             reinterpret_cast<const float2 *>(pre), u16(dh), ld_dh, act, split != 0,
                             static_cast<int>(m), static_cast<int>(f), static_cast<int>(k),
                             static_cast<uint16_t *>(dx), dw, workspace, workspace_bytes, s);
  };
  return dtype == VS_BF16 ? go(num::BF16{}) : go(num::F16{});
}

size_t vs_gated_linear_backward_workspace(int64_t m, int64_t f, int64_t k, int want_dx, int want_dw,
                                          int aligned) {
  return vs_gated_linear_gradients_workspace(m, f, k, 0, want_dx, want_dw, want_dw, aligned);
}

vs_status vs_gated_linear_backward(int dtype, int act, const void *x, int64_t ldx,
                                   const void *w_gate, int64_t ld_gate, const void *w_up,
                                   int64_t ld_up, const float *pre, const void *dh, int64_t ld_dh,
                                   int64_t m, int64_t f, int64_t k, void *dx, void *dw,
                                   void *workspace, size_t workspace_bytes, vs_stream_t stream) {
  uint16_t *const gate = static_cast<uint16_t *>(dw);
  uint16_t *const up = gate && f > 0 && k > 0 ? gate + f * k : gate;
  return vs_gated_linear_gradients(dtype, act, 0, x, ldx, w_gate, ld_gate, w_up, ld_up, pre, dh,
                                   ld_dh, m, f, k, dx, gate, up, workspace, workspace_bytes, stream);
}

}  // extern "C"
