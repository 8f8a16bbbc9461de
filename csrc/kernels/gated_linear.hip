// Gated linear layer in 16-bit types:  h = act(x Wg^T) * (x Wu^T), and its gradients
//
//   dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// with g = x Wg^T, u = x Wu^T in fp32.
//
// Many rows: bound by the matrix cores.  One kernel computes both products: a tile's B image holds
// rows of Wg and Wu side by side, 32 and 32 for each wave, so a wave ends with g and u of the same
// outputs in its accumulators and h is formed in registers.  Operand tiles (256 x 64 or 128 x 64
// of each operand) go global -> LDS by DMA into two stages; the next tile's pieces are issued
// before the current tile's products, waves 4-7 a quarter of a tile later than waves 0-3, so one
// of the two waves of a SIMD multiplies while the other pays for issuing.  Rows past the end and
// the ragged end of k read zeros through the buffer descriptor's range check.  The backward
// products are the same kernel with one B operand: the gradients of g and u are written side by
// side, once as they are and once transposed, x and the weights are transposed, so every product
// has both operands contiguous in its reduction dimension.
//
// Few rows (up to 64): bound by reading the weights.  No LDS staging: a wave streams rows of Wg
// and Wu straight into matrix-core fragments, the waves of a workgroup cut k, and their sums meet
// in LDS in a fixed order.
//
// Roundings: h once; for training, g and u are kept in fp32 (a 16-bit copy would add its own
// rounding to every gradient, 1.7 instead of 1.4 times the error of the result's own rounding);
// dg and du are rounded to the operands' type because the matrix cores multiply 16-bit numbers.
// Copyright 2026 veles.simd_amd authors. Apache-2.0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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
typedef __attribute__((address_space(3))) void lds_void;

template <class N>
__device__ __forceinline__ floatx4 mma(const uint4 &a, const uint4 &b, floatx4 c) {
  if constexpr (std::is_same_v<N, num::BF16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// -------------------------------------------------------------- activations
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}
__device__ __forceinline__ float act(int kind, float g) {
  switch (kind) {
    case VS_ACT_SILU: return g * sigmoid(g);
    case VS_ACT_GELU: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
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
    case VS_ACT_GELU:
      return fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g),
                  0.5f * (1.f + erff(g * 0.70710678118654752f)));
    case VS_ACT_RELU: return g > 0.f ? 1.f : 0.f;
    default: {
      const float s = sigmoid(g);
      return s * (1.f - s);
    }
  }
}

// ------------------------------------------------------------------- tiles
struct Args {
  const uint16_t *a;      // [m][k], row stride lda
  const uint16_t *b[2];   // [n][k], row stride ldb[.]; b[1] only for the gated product
  int64_t lda, ldb[2];
  int m, n, k;            // n: outputs (columns of h, or of c)
  uint16_t *c;            // [m][n], row stride n
  float2 *pre;            // [m][n] (g, u), or null
  int act;
};

// BM x BN tile of products, WM x WN waves.  GATED: the BN product columns are BN / 2 outputs.
template <int BM_, int BN_, int WM_, int WN_, bool GATED_>
struct Cfg {
  static constexpr int BM = BM_, BN = BN_, BK = 64, WM = WM_, WN = WN_;
  static constexpr bool GATED = GATED_;
  static constexpr int BO = GATED ? BN / 2 : BN;  // output columns
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int XM = BM / WM / 16, XN = BN / WN / 16;
  static constexpr int RB = 2 * BK;               // bytes of an image row
  static constexpr int kImgA = BM * RB, kImgB = BN * RB, kStage = kImgA + kImgB;
  static constexpr int PA = kImgA / 1024 / kWaves, PB = kImgB / 1024 / kWaves;
  static constexpr int kLds = 2 * kStage;
  static_assert(BN / WN == 64, "a wave owns 64 product columns");
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

template <class N, class C>
__global__ __launch_bounds__(C::kThreads) void tile_kernel(Args p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  constexpr int XM = C::XM, XN = C::XN;
  const unsigned tiles_m = (p.m + C::BM - 1) / C::BM, tiles_n = (p.n + C::BO - 1) / C::BO;
  unsigned tm, tn;
  dev::grouped_tile(dev::xcd_remap(blockIdx.x, tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
  const int m0 = tm * C::BM, n0 = tn * C::BO;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid / C::WN, wn = wid % C::WN;
  const int l16 = lane & 15, lq = lane >> 4;

  const __amdgpu_buffer_rsrc_t ra = rows_of(p.a, p.lda, m0, p.m, C::BM, p.k);
  const __amdgpu_buffer_rsrc_t rb0 = rows_of(p.b[0], p.ldb[0], n0, p.n, C::BO, p.k);
  const __amdgpu_buffer_rsrc_t rb1 =
      C::GATED ? rows_of(p.b[1], p.ldb[1], n0, p.n, C::BO, p.k) : rb0;
  // piece i of this wave: image rows 8 (i of the wave's pieces) + lane / 8, chunk lane % 8
  uint32_t offa[C::PA], offb[C::PB];
  int ka, kb[C::PB];
  {
    const int r8 = lane / 8, pc = lane % 8;
#pragma unroll
    for (int i = 0; i < C::PA; i++) {
      const int row = (wid * C::PA + i) * 8 + r8;
      offa[i] = static_cast<uint32_t>((row * p.lda + 8 * swz(row, pc)) * 2);
    }
#pragma unroll
    for (int i = 0; i < C::PB; i++) {
      const int row = (wid * C::PB + i) * 8 + r8;  // image row
      // GATED: 64 image rows are 32 of Wg, then the same 32 of Wu
      const int src = C::GATED ? row / 64 * 32 + row % 32 : row;
      const bool up = C::GATED && (row & 32);
      offb[i] = static_cast<uint32_t>((src * p.ldb[up ? 1 : 0] + 8 * swz(row, pc)) * 2);
      kb[i] = 8 * swz(row, pc);
    }
    ka = pc;
  }
  const auto stage = [&](int buf, int k0) {
    uint8_t *base = lds + buf * C::kStage;
    const bool whole = k0 + C::BK <= p.k;
#pragma unroll
    for (int i = 0; i < C::PA; i++) {
      const int j = wid * C::PA + i, row = j * 8 + lane / 8;
      const uint32_t off = whole || k0 + 8 * swz(row, ka) < p.k ? offa[i] : kOut;
      dma16(ra, base + j * 1024, off, 2 * k0);
    }
#pragma unroll
    for (int i = 0; i < C::PB; i++) {
      const int j = wid * C::PB + i;
      const uint32_t off = whole || k0 + kb[i] < p.k ? offb[i] : kOut;
      const bool up = C::GATED && (j & 4);  // 8 rows a piece: rows 32..63 of each 64 are Wu's
      dma16(up ? rb1 : rb0, base + C::kImgA + j * 1024, off, 2 * k0);
    }
  };
  const auto frag = [&](const uint8_t *img, int row, int c) {
    return *reinterpret_cast<const uint4 *>(img + row * C::RB + swz(row, c) * 16);
  };

  floatx4 acc[XM][XN];
#pragma unroll
  for (int x = 0; x < XM; x++)
#pragma unroll
    for (int y = 0; y < XN; y++) acc[x][y] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int arow = wm * (C::BM / C::WM) + l16, brow = wn * 64 + l16;
  const int nk = (p.k + C::BK - 1) / C::BK;
  const bool late = C::kWaves == 8 && wid >= 4;
  if (nk > 0) stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int kt = 0; kt < nk; kt++) {
    const int cur = kt & 1;
    const uint8_t *ia = lds + cur * C::kStage, *ib = ia + C::kImgA;
    if (!late && kt + 1 < nk) stage(cur ^ 1, (kt + 1) * C::BK);
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      uint4 fa[XM], fb[XN];
#pragma unroll
      for (int x = 0; x < XM; x++) fa[x] = frag(ia, arow + 16 * x, 4 * ks + lq);
#pragma unroll
      for (int y = 0; y < XN; y++) fb[y] = frag(ib, brow + 16 * y, 4 * ks + lq);
#pragma unroll
      for (int x = 0; x < XM; x++) {
        if (ks == 0 && x == XM / 2 && late && kt + 1 < nk) stage(cur ^ 1, (kt + 1) * C::BK);
#pragma unroll
        for (int y = 0; y < XN; y++) acc[x][y] = mma<N>(fa[x], fb[y], acc[x][y]);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // Results leave through LDS: a 16 x 16 block leaves lane l with rows 4 (l / 16) + r of column
  // l % 16; from LDS a row of the tile is stored 16 bytes a lane.
  constexpr int YO = C::GATED ? XN / 2 : XN;  // 16-column blocks of outputs per wave
  constexpr int LD = C::BO + 8;               // elements of an LDS row
  constexpr int kRound = C::BM * LD * 2 > C::kLds ? 2 : 1;
  constexpr int XR = XM / kRound;
  uint16_t *img = reinterpret_cast<uint16_t *>(lds);
  const bool vec = p.n % 8 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0;
#pragma unroll
  for (int round = 0; round < kRound; round++) {
    if (round) __syncthreads();
#pragma unroll
    for (int x = 0; x < XR; x++)
#pragma unroll
      for (int y = 0; y < YO; y++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int xx = round * XR + x;
          const int lr = (wm * XR + x) * 16 + 4 * lq + r, lc = (wn * YO + y) * 16 + l16;
          float v;
          if constexpr (C::GATED) {
            const float g = acc[xx][y][r], u = acc[xx][y + YO][r];
            v = act(p.act, g) * u;
            const int row = m0 + wm * (C::BM / C::WM) + xx * 16 + 4 * lq + r, col = n0 + lc;
            if (p.pre && row < p.m && col < p.n)
              p.pre[static_cast<int64_t>(row) * p.n + col] = make_float2(g, u);
          } else {
            v = acc[xx][y][r];
          }
          img[lr * LD + lc] = N::save(v);
        }
    __syncthreads();
    constexpr int CH = C::BO / 8;  // 16-byte chunks of a row
    for (int i = threadIdx.x; i < C::BM / kRound * CH; i += C::kThreads) {
      const int lr = i / CH, lc = i % CH * 8;
      const int row = m0 + lr / (XR * 16) * (C::BM / C::WM) + round * XR * 16 + lr % (XR * 16);
      const int col = n0 + lc;
      if (row >= p.m || col >= p.n) continue;
      uint16_t *dst = p.c + static_cast<int64_t>(row) * p.n + col;
      if (vec) {
        *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(img + lr * LD + lc);
      } else {
        for (int e = 0; e < 8; e++)
          if (col + e < p.n) dst[e] = img[lr * LD + lc + e];
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
constexpr int kFewWaves = 8;

// RT row tiles of 16.  A workgroup owns 16 outputs; step: 64 k, a lane's two 16-byte loads of a
// weight row are neighbouring halves of a 128-byte line across the four 16-lane groups.
template <class N, int RT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(Args p) {
  __shared__ float part[kFewWaves][2][RT][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int n = n0 + l16 < p.n ? n0 + l16 : p.n - 1;
  const uint16_t *w[2] = {p.b[0] + n * p.ldb[0], p.b[1] + n * p.ldb[1]};
  const uint16_t *xr[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = 16 * t + l16 < p.m ? 16 * t + l16 : p.m - 1;  // copies of it are not stored
    xr[t] = p.a + row * p.lda;
  }
  const int steps = (p.k + 63) / 64, per = (steps + kFewWaves - 1) / kFewWaves;
  const int first = wave * per, last = first + per < steps ? first + per : steps;
  const auto load = [&](const uint16_t *row, int k0) {
    uint4 v = {0, 0, 0, 0};
    if (k0 + 8 <= p.k) {
      __builtin_memcpy(&v, row + k0, 16);
    } else {
      uint32_t e[4] = {0, 0, 0, 0};
      for (int i = 0; i < 8; i++)
        if (k0 + i < p.k) e[i / 2] |= static_cast<uint32_t>(row[k0 + i]) << (16 * (i & 1));
      v = uint4{e[0], e[1], e[2], e[3]};
    }
    return v;
  };
  floatx4 acc[2][RT];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int t = 0; t < RT; t++) acc[i][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  uint4 wv[2][2], nw[2][2];
  if (first < last)
    for (int h = 0; h < 2; h++)
      for (int i = 0; i < 2; i++) wv[h][i] = load(w[i], first * 64 + 32 * h + 8 * lq);
  for (int st = first; st < last; st++) {
    if (st + 1 < last)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < 2; i++) nw[h][i] = load(w[i], (st + 1) * 64 + 32 * h + 8 * lq);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const uint4 xv = load(xr[t], st * 64 + 32 * h + 8 * lq);
#pragma unroll
        for (int i = 0; i < 2; i++) acc[i][t] = mma<N>(xv, wv[h][i], acc[i][t]);
      }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < 2; i++) wv[h][i] = nw[h][i];
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) part[wave][i][t][r][lane] = acc[i][t][r];
  __syncthreads();
  for (int i = threadIdx.x; i < RT * 256; i += 64 * kFewWaves) {
    const int t = i / 256, r = i / 64 % 4, l = i % 64;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int v = 0; v < kFewWaves; v++) {
      g += part[v][0][t][r][l];
      u += part[v][1][t][r][l];
    }
    const int row = 16 * t + 4 * (l / 16) + r, col = n0 + l % 16;
    if (row >= p.m || col >= p.n) continue;
    const int64_t at = static_cast<int64_t>(row) * p.n + col;
    p.c[at] = N::save(act(p.act, g) * u);
    if (p.pre) p.pre[at] = make_float2(g, u);
  }
}

// ------------------------------------------------- layout and element-wise
// [rows][cols] (row stride ld) copied to rows of cols_p, zeros behind: rows that the DMA can read.
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t *__restrict__ src, int64_t ld,
                                                  int64_t rows, int cols, int cols_p,
                                                  uint16_t *__restrict__ dst) {
  const int chunks = cols_p / 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * chunks; i += gridDim.x * 256ll) {
    const int64_t r = i / chunks;
    const int c = static_cast<int>(i - r * chunks) * 8;
    const uint16_t *s = src + r * ld + c;
    uint32_t e[4] = {0, 0, 0, 0};
    if (c + 8 <= cols) {
      __builtin_memcpy(e, s, 16);
    } else {
      for (int j = 0; j < 8; j++)
        if (c + j < cols) e[j / 2] |= static_cast<uint32_t>(s[j]) << (16 * (j & 1));
    }
    *reinterpret_cast<uint4 *>(dst + r * cols_p + c) = uint4{e[0], e[1], e[2], e[3]};
  }
}

// dst[c][r] = src[r][c], rows of dst padded with zeros to ld_d (a multiple of 8): 64 x 64 tiles
// through LDS.  Tiles (x: columns of src, y: rows, folded into one grid dimension).
__global__ __launch_bounds__(256) void transpose_kernel(const uint16_t *__restrict__ src,
                                                        int64_t ld, int rows, int cols,
                                                        uint16_t *__restrict__ dst, int64_t ld_d,
                                                        int rows_p, int tiles_c) {
  __shared__ uint16_t tile[64][66];
  const int c0 = static_cast<int>(blockIdx.x % tiles_c) * 64;
  const int r0 = static_cast<int>(blockIdx.x / tiles_c) * 64;
  const int a = threadIdx.x >> 3, b = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = r0 + a + 32 * i;
    uint16_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r < rows) {
      const uint16_t *s = src + r * ld + c0 + b;
      if (c0 + b + 8 <= cols) {
        __builtin_memcpy(v, s, 16);
      } else {
        for (int j = 0; j < 8; j++)
          if (c0 + b + j < cols) v[j] = s[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) tile[a + 32 * i][b + j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int c = c0 + a + 32 * i, r = r0 + b;
    if (c >= cols || r >= rows_p) continue;
    uint32_t e[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      e[j] = tile[b + 2 * j][a + 32 * i] | (static_cast<uint32_t>(tile[b + 2 * j + 1][a + 32 * i]) << 16);
    *reinterpret_cast<uint4 *>(dst + c * ld_d + r) = uint4{e[0], e[1], e[2], e[3]};
  }
}

// (dh, g, u) -> dg, du as rows [m][2 fp] (dg, then du) and transposed [2 f][mp]; zeros in the
// padding of both.  Either output may be null.
template <class N>
__global__ __launch_bounds__(256) void slope_kernel(const uint16_t *__restrict__ dh, int64_t ld,
                                                    const float2 *__restrict__ pre, int kind, int m,
                                                    int f, int fp, int mp, int tiles_c,
                                                    uint16_t *__restrict__ rows,
                                                    uint16_t *__restrict__ cols) {
  __shared__ uint16_t tile[2][64][66];
  const int c0 = static_cast<int>(blockIdx.x % tiles_c) * 64;
  const int r0 = static_cast<int>(blockIdx.x / tiles_c) * 64;
  const int a = threadIdx.x >> 3, b = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = r0 + a + 32 * i;
    uint32_t eg[4] = {0, 0, 0, 0}, eu[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int c = c0 + b + j;
      uint16_t dg = 0, du = 0;
      if (r < m && c < f) {
        const float d = N::load(dh[r * ld + c]);
        const float2 gu = pre[static_cast<int64_t>(r) * f + c];
        dg = N::save(d * gu.y * act_slope(kind, gu.x));
        du = N::save(d * act(kind, gu.x));
      }
      eg[j / 2] |= static_cast<uint32_t>(dg) << (16 * (j & 1));
      eu[j / 2] |= static_cast<uint32_t>(du) << (16 * (j & 1));
      tile[0][a + 32 * i][b + j] = dg;
      tile[1][a + 32 * i][b + j] = du;
    }
    if (rows && r < m && c0 + b < fp) {
      uint16_t *dst = rows + static_cast<int64_t>(r) * (2 * fp) + c0 + b;
      *reinterpret_cast<uint4 *>(dst) = uint4{eg[0], eg[1], eg[2], eg[3]};
      *reinterpret_cast<uint4 *>(dst + fp) = uint4{eu[0], eu[1], eu[2], eu[3]};
    }
  }
  if (!cols) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int c = c0 + a + 32 * i, r = r0 + b;
      if (c >= f || r >= mp) continue;
      uint32_t e[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        e[j] = tile[k][b + 2 * j][a + 32 * i] |
               (static_cast<uint32_t>(tile[k][b + 2 * j + 1][a + 32 * i]) << 16);
      *reinterpret_cast<uint4 *>(cols + (static_cast<int64_t>(k) * f + c) * mp + r) =
          uint4{e[0], e[1], e[2], e[3]};
    }
}

// -------------------------------------------------------------------- host
constexpr int kFewRows = 64;
int up8(int64_t v) { return static_cast<int>((v + 7) / 8 * 8); }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Whether the DMA can read a [.][k] operand where it is: whole 16-byte chunks.
bool direct(const void *p, int64_t ld, int64_t k) {
  return k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

template <class N, class C>
vs_status launch_tile(const Args &p, hipStream_t s) {
  static const hipError_t attr =
      hipFuncSetAttribute(reinterpret_cast<const void *>(&tile_kernel<N, C>),
                          hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds);
  VS_HIP(attr);
  const int64_t tiles = static_cast<int64_t>((p.m + C::BM - 1) / C::BM) * ((p.n + C::BO - 1) / C::BO);
  VS_REQUIRE(tiles < (1ll << 23), "gated_linear: too many output tiles");
  hipLaunchKernelGGL((tile_kernel<N, C>), dim3(static_cast<unsigned>(tiles)), dim3(C::kThreads),
                     C::kLds, s, p);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

// Large tiles once they give every CU one, else 128 x 128.
template <class N, bool GATED>
vs_status product(const Args &p, hipStream_t s) {
  const int bo = GATED ? 128 : 256;
  const int64_t large = static_cast<int64_t>((p.m + 255) / 256) * ((p.n + bo - 1) / bo);
  if (large >= 256) return launch_tile<N, Cfg<256, 256, 2, 4, GATED>>(p, s);
  return launch_tile<N, Cfg<128, 128, 2, 2, GATED>>(p, s);
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

vs_status pad(const uint16_t *src, int64_t ld, int64_t rows, int cols, uint16_t *dst, hipStream_t s) {
  const int cp = up8(cols);
  const int64_t work = rows * (cp / 8);
  if (work == 0) return VS_OK;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((work + 255) / 256, 1 << 20));
  hipLaunchKernelGGL(pad_kernel, dim3(grid), dim3(256), 0, s, src, ld, rows, cols, cp, dst);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

vs_status transpose(const uint16_t *src, int64_t ld, int rows, int cols, uint16_t *dst, int64_t ld_d,
                    int rows_p, hipStream_t s) {
  const int tc = (cols + 63) / 64;
  const int64_t tiles = static_cast<int64_t>(tc) * ((rows_p + 63) / 64);
  if (tiles == 0) return VS_OK;
  hipLaunchKernelGGL(transpose_kernel, dim3(static_cast<unsigned>(tiles)), dim3(256), 0, s, src, ld,
                     rows, cols, dst, ld_d, rows_p, tc);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

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
  bool few, px, pg, pu;
  size_t bytes;
};
ForwardNeed forward_need(int64_t m, int64_t f, int64_t k, bool dx, bool dg, bool du) {
  ForwardNeed q{};
  q.few = m <= kFewRows;
  if (q.few) return q;
  q.px = !dx;
  q.pg = !dg;
  q.pu = !du;
  const size_t kp = up8(k);
  q.bytes = (q.px ? up256(2 * m * kp) : 0) + ((q.pg ? 1 : 0) + (q.pu ? 1 : 0)) * up256(2 * f * kp);
  return q;
}

template <class N>
vs_status forward(Args p, void *workspace, size_t bytes, hipStream_t s) {
  const ForwardNeed q = forward_need(p.m, p.n, p.k, direct(p.a, p.lda, p.k),
                                     direct(p.b[0], p.ldb[0], p.k), direct(p.b[1], p.ldb[1], p.k));
  if (q.few) {
    const dim3 grid(static_cast<unsigned>((p.n + 15) / 16)), block(64 * kFewWaves);
    if (p.m <= 16) hipLaunchKernelGGL((few_kernel<N, 1>), grid, block, 0, s, p);
    else if (p.m <= 32) hipLaunchKernelGGL((few_kernel<N, 2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((few_kernel<N, 4>), grid, block, 0, s, p);
    VS_HIP(hipGetLastError());
    return VS_OK;
  }
  DeviceBuffer own;
  Space sp;
  VS_TRY(open_space(sp, own, workspace, bytes, q.bytes, s));
  const int kp = up8(p.k);
  if (q.px) {
    uint16_t *d = sp.take(static_cast<size_t>(p.m) * kp);
    VS_TRY(pad(p.a, p.lda, p.m, p.k, d, s));
    p.a = d;
    p.lda = kp;
  }
  for (int i = 0; i < 2; i++)
    if (i ? q.pu : q.pg) {
      uint16_t *d = sp.take(static_cast<size_t>(p.n) * kp);
      VS_TRY(pad(p.b[i], p.ldb[i], p.n, p.k, d, s));
      p.b[i] = d;
      p.ldb[i] = kp;
    }
  p.k = kp;
  return product<N, true>(p, s);
}

size_t backward_need(int64_t m, int64_t f, int64_t k, bool dx, bool dw) {
  const size_t fp = up8(f), mp = up8(m);
  return (dx ? up256(2 * m * 2 * fp) + up256(2 * k * 2 * fp) : 0) +
         (dw ? up256(2 * 2 * f * mp) + up256(2 * k * mp) : 0);
}

template <class N>
vs_status backward(const uint16_t *x, int64_t ldx, const uint16_t *wg, int64_t ldg,
                   const uint16_t *wu, int64_t ldu, const float2 *pre, const uint16_t *dh,
                   int64_t ldh, int act, int m, int f, int k, uint16_t *dx, uint16_t *dw,
                   void *workspace, size_t bytes, hipStream_t s) {
  DeviceBuffer own;
  Space sp;
  VS_TRY(open_space(sp, own, workspace, bytes, backward_need(m, f, k, dx, dw), s));
  const int fp = up8(f), mp = up8(m);
  uint16_t *rows = dx ? sp.take(static_cast<size_t>(m) * 2 * fp) : nullptr;
  uint16_t *wt = dx ? sp.take(static_cast<size_t>(k) * 2 * fp) : nullptr;
  uint16_t *cols = dw ? sp.take(static_cast<size_t>(2) * f * mp) : nullptr;
  uint16_t *xt = dw ? sp.take(static_cast<size_t>(k) * mp) : nullptr;
  const int tc = (fp + 63) / 64;
  const int64_t tiles = static_cast<int64_t>(tc) * ((mp + 63) / 64);
  VS_REQUIRE(tiles < (1ll << 24), "gated_linear: too many tiles");
  if (tiles) {
    hipLaunchKernelGGL((slope_kernel<N>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, s, dh,
                       ldh, pre, act, m, f, fp, mp, tc, rows, cols);
    VS_HIP(hipGetLastError());
  }
  if (dx) {
    VS_TRY(transpose(wg, ldg, f, k, wt, 2 * fp, fp, s));
    VS_TRY(transpose(wu, ldu, f, k, wt + fp, 2 * fp, fp, s));
    Args p{};
    p.a = rows;
    p.b[0] = wt;
    p.lda = p.ldb[0] = 2 * fp;
    p.m = m;
    p.n = k;
    p.k = 2 * fp;
    p.c = dx;
    if (m && k) VS_TRY((product<N, false>(p, s)));
  }
  if (dw) {
    VS_TRY(transpose(x, ldx, m, k, xt, mp, mp, s));
    Args p{};
    p.a = cols;
    p.b[0] = xt;
    p.lda = p.ldb[0] = mp;
    p.m = 2 * f;
    p.n = k;
    p.k = mp;
    p.c = dw;
    if (f && k) VS_TRY((product<N, false>(p, s)));
  }
  return VS_OK;
}

}  // namespace
}  // namespace glin
}  // namespace vs

using namespace vs;

extern "C" {

size_t vs_gated_linear_workspace(int64_t m, int64_t f, int64_t k) {
  if (glin::check("", VS_BF16, 0, m, f, k) != VS_OK) return 0;
  return glin::forward_need(m, f, k, false, false, false).bytes;
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

size_t vs_gated_linear_backward_workspace(int64_t m, int64_t f, int64_t k, int want_dx, int want_dw) {
  if (glin::check("", VS_BF16, 0, m, f, k) != VS_OK) return 0;
  return glin::backward_need(m, f, k, want_dx != 0, want_dw != 0);
}

vs_status vs_gated_linear_backward(int dtype, int act, const void *x, int64_t ldx,
                                   const void *w_gate, int64_t ld_gate, const void *w_up,
                                   int64_t ld_up, const float *pre, const void *dh, int64_t ld_dh,
                                   int64_t m, int64_t f, int64_t k, void *dx, void *dw,
                                   void *workspace, size_t workspace_bytes, vs_stream_t stream) {
  clear_error();
  VS_TRY(glin::check("gated_linear_backward", dtype, act, m, f, k));
  if (k == 0 || (!dx && !dw)) return VS_OK;
  VS_REQUIRE((m == 0 || f == 0) || (x && w_gate && w_up && pre && dh),
             "gated_linear_backward: null pointer");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto u16 = [](const void *v) { return static_cast<const uint16_t *>(v); };
  const auto go = [&](auto tag) {
    using N = decltype(tag);
    return glin::backward<N>(u16(x), ldx, u16(w_gate), ld_gate, u16(w_up), ld_up,
                             reinterpret_cast<const float2 *>(pre), u16(dh), ld_dh, act,
                             static_cast<int>(m), static_cast<int>(f), static_cast<int>(k),
                             static_cast<uint16_t *>(dx), static_cast<uint16_t *>(dw), workspace,
                             workspace_bytes, s);
  };
  return dtype == VS_BF16 ? go(num::BF16{}) : go(num::F16{});
}

}  // extern "C"
