// Products of few rows with 4-bit weights:
//
//   y[m][n] = sum_k x[m][k] (q[n][k] - z[n][k / G]) s[n][k / G]
//
// q: two unsigned 4-bit numbers to a byte, row major, the even k in the low half; s in x's type,
// z an unsigned byte (8 where absent), one of each per row and group of G neighbouring k.
//
// Bound: the bandwidth of reading q (the rows of x and y are a few KB).  So the work per weight has
// to be small: unpacked to fp32 and multiplied on the vector units, three instructions a weight
// would take as long as reading it.  Here a weight costs one: the four bits are masked into the
// mantissa of a bf16 or fp16 number 1 (0x3f80 | q << 3 or 0x3c00 | q << 6), which is 1 + q / 16
// exactly, two to a register, and the matrix cores multiply (16 x 16 x 32, x as the A operand,
// rows it does not have are zero).  Per group and column the fp32 sums then become
//
//   s (sum x (1 + q / 16) - (16 + z) sum x / 16)
//
// where sum x / 16 comes from one more product, with sixteenths, in the layout it is needed in; the result is
// multiplied by 16 at the end.  Weights are never rounded.  What is rounded, to 2^-24 each time, are sums of
// |x| (16 + q) s and |x| (16 + z) s, not of |x (q - z)| s: weights near their zero point give a remainder of that
// size in the place of a smaller sum or of 0, and a group's sum of 2 |x| (of (1 + z / 16) |x| where z > 15) has
// to stay below fp32's largest number.
//
// A step is 128 k of 16 columns: 64 bytes of each row, which four neighbouring lanes load.  (16
// neighbouring lanes on 16 rows, the order the matrix instruction wants, cost the cache four times
// the lookups and ran at 2.8 TB/s however many loads were in flight.)  Through LDS a lane gets 16
// bytes of its column: 32 neighbouring k, of which an instruction takes 8 from each of the four
// 16-lane groups.  Two swaps of half and quarter waves transpose the four registers against the
// four groups, so that one instruction sees 32 neighbouring k and any group of 32 or more can be
// scaled.  The waves of a workgroup share its columns and cut k; their sums meet in LDS in a fixed
// order.  28000 x 8192 with groups of 64: 35 us for one row, 40 for 16 (3.6 and 3.1 TB/s).
// Copyright 2026 veles.simd_amd authors. Apache-2.0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "csrc/kernels/number.h"
#include "csrc/runtime/runtime.h"
#include "simd/gpu.h"

namespace vs {
namespace mv4 {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 128;  // k of one step: 16 bytes of q per lane
constexpr int kDepth = 2;

struct Args {
  const uint16_t *x;
  int64_t ldx;
  const uint8_t *q;
  int64_t ldq;
  const uint16_t *s;
  const uint8_t *z;  // or null: 8
  uint16_t *y;
  int m, n, k, groups, span;  // span: G in blocks of kBlock, for G > kBlock
};

struct Frag {
  uint32_t r[4];
};

template <class N>
__device__ __forceinline__ floatx4 mma(const Frag &a, const Frag &b, floatx4 c) {
  if constexpr (std::is_same_v<N, num::BF16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Eight 4-bit numbers as 1 + q / 16: pair p is (q_p, q_{p + 4}).  `base` holds 1 twice; it comes in a
// register, where the mask and it can be operands of one and-or.
template <class N>
__device__ __forceinline__ Frag unpack(uint32_t w, uint32_t base) {
  constexpr bool B = std::is_same_v<N, num::BF16>;
  constexpr uint32_t mask = B ? 0x00780078u : 0x03c003c0u;
  Frag f;
  f.r[0] = ((B ? w << 3 : w << 6) & mask) | base;
  f.r[1] = ((B ? w >> 1 : w << 2) & mask) | base;
  f.r[2] = ((B ? w >> 5 : w >> 2) & mask) | base;
  f.r[3] = ((B ? w >> 9 : w >> 6) & mask) | base;
  return f;
}

// Eight neighbouring values of x in the order that unpack() gives the weights.
__device__ __forceinline__ Frag pairs(const u32x4 &v) {
  Frag f;
  f.r[0] = __builtin_amdgcn_perm(v.z, v.x, 0x05040100);  // 0, 4
  f.r[1] = __builtin_amdgcn_perm(v.z, v.x, 0x07060302);  // 1, 5
  f.r[2] = __builtin_amdgcn_perm(v.w, v.y, 0x05040100);  // 2, 6
  f.r[3] = __builtin_amdgcn_perm(v.w, v.y, 0x07060302);  // 3, 7
  return f;
}

// (register j, 16-lane group l) -> (register l, group j)
__device__ __forceinline__ void transpose(uint32_t (&w)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int i = 0; i < 2; i++) {  // upper half of w[i] against lower half of w[i + 2]
    const u32x2 r = __builtin_amdgcn_permlane32_swap(w[i], w[i + 2], false, false);
    w[i] = r.x;
    w[i + 2] = r.y;
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {  // odd quarters of w[i] against even quarters of w[i + 1]
    const u32x2 r = __builtin_amdgcn_permlane16_swap(w[i], w[i + 1], false, false);
    w[i] = r.x;
    w[i + 1] = r.y;
  }
#endif
}

// CT: column tiles of 16 per workgroup; GS: MFMA steps of 32 per group (1, 2, 4; 4 covers larger
// groups through span); RV: accumulator rows in use, ceil(m / 4): row m of x is put where it
// comes out in accumulator register m / 4, so few rows scale few registers.
//
// kDepth steps of weights and x are in flight per wave.  Their loads are issued unconditionally (past
// the end the last step again): a load under a condition would make the compiler wait for all.
// Four neighbouring lanes load the 64 bytes of one row and the fragments are formed through LDS: a
// load in fragment order (16 rows in 16 neighbouring lanes) costs the cache four times the lookups.
// Two waves a SIMD have to fit (28000 x 8192 g32, 16 rows: 43 us, 55 where the compiler took more
// registers).  (Forming the next step's fragments while a step multiplies needs more registers
// than it hides: 36 us against 34 for one row of 28000 x 8192 g64, where the loads alone take 26.)
template <class N, int kWaves, int CT, int GS, int RV>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void matvec4_kernel(Args p) {
  constexpr int NG = 4 / GS;                 // groups in a step
  constexpr int kStage = 8;                  // steps whose scales a wave keeps in LDS
  constexpr int kCols = 16 * CT, kSlots = kStage * NG;
  constexpr int kShare = 64 / kCols;         // lanes that fetch scales for one column
  constexpr int kMine = kSlots / kShare;
  static_assert(kCols <= 64 && kSlots % kShare == 0, "a wave fetches the scales of its columns");
  // a wave's scales and zero points and one step of rows, then the waves' sums
  union Shared {
    struct {
      uint32_t sz[kWaves][kSlots][kCols];
      u32x4 turn[kWaves][CT + 4][64];
    };
    float part[kWaves][CT][RV][64];
  };
  __shared__ Shared lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int m0 = blockIdx.y * 16, n0 = blockIdx.x * kCols;
  const int r4 = lane / 4, c4 = lane % 4;    // row and 16-byte chunk that this lane loads
  const int row = m0 + r4 / 4 + 4 * (r4 % 4);  // A row r4
  const uint16_t *xr = p.x + (row < p.m ? row : 0) * p.ldx;  // copies of row 0 are not stored
  const uint8_t *qr[CT];
#pragma unroll
  for (int c = 0; c < CT; c++)
    qr[c] = p.q + (n0 + 16 * c + r4 < p.n ? n0 + 16 * c + r4 : p.n - 1) * p.ldq;
  // chunk c of row r lies at 4 r + (c ^ r / 4 % 4), which spreads both orders over the banks (16 rows of
  // 28000 x 8192: a fifth of the LDS cycles are conflicts)
  u32x4 *turn = &lds.turn[wave][0][0];
  const int put = 4 * r4 + (c4 ^ (r4 / 4 % 4)), get = 4 * l16 + (lq ^ (l16 / 4 % 4));
  const int blocks = (p.k + kBlock - 1) / kBlock, bytes = (p.k + 1) / 2;
  const int per = (blocks + kWaves - 1) / kWaves;
  const int first = wave * per, last = first + per < blocks ? first + per : blocks;
  const int whole = last * kBlock <= p.k ? last : last - 1;  // steps that end inside their row

  struct Step {
    u32x4 x[4], q[CT];
  };
  const auto fetch = [&](int kb, Step &v) {
#pragma unroll
    for (int j = 0; j < 4; j++) __builtin_memcpy(&v.x[j], xr + kb * kBlock + 32 * j + 8 * c4, 16);
#pragma unroll
    for (int c = 0; c < CT; c++) __builtin_memcpy(&v.q[c], qr[c] + kb * (kBlock / 2) + 16 * c4, 16);
  };
  // Scales (low half) and 16 + zero points (high half) of steps [kb, kb + kStage): this lane's
  // kMine neighbouring groups of one column.
  const int scol = lane % kCols, part = lane / kCols;
  const int64_t srow = static_cast<int64_t>(n0 + scol < p.n ? n0 + scol : p.n - 1) * p.groups;
  struct Scales {
    uint16_t s[kMine];
    uint8_t z[kMine];
  };
  const auto fetch_scales = [&](int kb, Scales &v) {
    const int g0 = NG > 1 ? kb * NG : kb / p.span;
    const int g = g0 + part * kMine;
    if (p.span == 1 && g0 + kSlots <= p.groups) {
      __builtin_memcpy(v.s, p.s + srow + g, sizeof(v.s));
      if (p.z) __builtin_memcpy(v.z, p.z + srow + g, sizeof(v.z));
    } else {
#pragma unroll
      for (int i = 0; i < kMine; i++) {
        int at = NG > 1 || p.span == 1 ? g + i : (kb + part * kMine + i) / p.span;
        at = at < p.groups ? at : p.groups - 1;
        v.s[i] = p.s[srow + at];
        if (p.z) v.z[i] = p.z[srow + at];
      }
    }
  };
  const auto keep_scales = [&](const Scales &v) {
#pragma unroll
    for (int i = 0; i < kMine; i++)
      lds.sz[wave][part * kMine + i][scol] =
          v.s[i] | static_cast<uint32_t>(p.z ? v.z[i] + 16 : 24) << 16;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };

  const Frag sixteenths = std::is_same_v<N, num::BF16>
                              ? Frag{{0x3d803d80u, 0x3d803d80u, 0x3d803d80u, 0x3d803d80u}}
                              : Frag{{0x2c002c00u, 0x2c002c00u, 0x2c002c00u, 0x2c002c00u}};
  uint32_t base = std::is_same_v<N, num::BF16> ? 0x3f803f80u : 0x3c003c00u;
  asm volatile("" : "+v"(base));
  float sum[CT][RV];
#pragma unroll
  for (int c = 0; c < CT; c++)
#pragma unroll
    for (int r = 0; r < RV; r++) sum[c][r] = 0.f;
  const auto multiply = [&](const Step &v, int slot) {
    // LDS works in order within a wave: the reads see these writes, and the next step's writes
    // come after them
#pragma unroll
    for (int j = 0; j < 4; j++) turn[64 * j + put] = v.x[j];
#pragma unroll
    for (int c = 0; c < CT; c++) turn[64 * (4 + c) + put] = v.q[c];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    u32x4 x[4];
    uint32_t q[CT][4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = turn[64 * j + get];
#pragma unroll
    for (int c = 0; c < CT; c++) {
      const u32x4 w = turn[64 * (4 + c) + get];
#pragma unroll
      for (int j = 0; j < 4; j++) q[c][j] = w[j];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < CT; c++) transpose(q[c]);
#pragma unroll
    for (int i = 0; i < NG; i++) {
      const floatx4 none = {0.f, 0.f, 0.f, 0.f};
      floatx4 sx = none, acc[CT];
#pragma unroll
      for (int c = 0; c < CT; c++) acc[c] = none;
#pragma unroll
      for (int j = i * GS; j < (i + 1) * GS; j++) {
        const Frag a = pairs(x[j]);
        sx = mma<N>(a, sixteenths, sx);
#pragma unroll
        for (int c = 0; c < CT; c++) acc[c] = mma<N>(a, unpack<N>(q[c][j], base), acc[c]);
      }
#pragma unroll
      for (int c = 0; c < CT; c++) {
        const uint32_t sz = lds.sz[wave][slot * NG + i][16 * c + l16];
        const float s = N::load(static_cast<uint16_t>(sz)), z = -static_cast<float>(sz >> 16);
#pragma unroll
        for (int r = 0; r < RV; r++) sum[c][r] = fmaf(s, fmaf(z, sx[r], acc[c][r]), sum[c][r]);
      }
    }
  };
  Scales sc;
  Step v[kDepth];
  if (first < last) fetch_scales(first, sc);
  if (first < whole)
#pragma unroll
    for (int u = 0; u < kDepth; u++) fetch(first + u < whole ? first + u : whole - 1, v[u]);
  for (int kb = first; kb < last; kb += kStage) {
    if (kb != first) {
      __builtin_amdgcn_wave_barrier();  // the last steps' reads of the image come first
      fetch_scales(kb, sc);
    }
    keep_scales(sc);
    const int end = kb + kStage < whole ? kb + kStage : whole;
    int i = kb;
    for (; i + kDepth <= end; i += kDepth)
#pragma unroll
      for (int u = 0; u < kDepth; u++) {
        multiply(v[u], i + u - kb);
        fetch(i + u + kDepth < whole ? i + u + kDepth : whole - 1, v[u]);
      }
#pragma unroll
    for (int u = 0; u < kDepth - 1; u++)  // the last steps of the wave
      if (i + u < end) multiply(v[u], i + u - kb);
    if (whole < last && last - kb <= kStage) {  // the row ends inside the last step
      // Bytes of q behind a row may be read where the tensor goes on (x is zero there).
      Step t;
      const int o = whole * (kBlock / 2) + 16 * c4;
      const uint8_t *qend = p.q + (p.n - 1) * p.ldq + bytes;
      const uint16_t *xend = p.x + (p.m - 1) * p.ldx + p.k;
#pragma unroll
      for (int c = 0; c < CT; c++) {
        t.q[c] = u32x4{0, 0, 0, 0};
        if (qr[c] + o + 16 <= qend) {
          __builtin_memcpy(&t.q[c], qr[c] + o, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (o + e < bytes) t.q[c][e / 4] |= static_cast<uint32_t>(qr[c][o + e]) << (8 * (e & 3));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int k0 = whole * kBlock + 32 * j + 8 * c4;
        t.x[j] = u32x4{0, 0, 0, 0};
        if (k0 >= p.k) continue;
        if (xr + k0 + 8 <= xend) {
          __builtin_memcpy(&t.x[j], xr + k0, 16);
#pragma unroll
          for (int e = 0; e < 4; e++)
            t.x[j][e] &= k0 + 2 * e + 1 < p.k ? 0xffffffffu : k0 + 2 * e < p.k ? 0xffffu : 0u;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (k0 + e < p.k) t.x[j][e / 2] |= static_cast<uint32_t>(xr[k0 + e]) << (16 * (e & 1));
        }
      }
      multiply(t, whole - kb);
    }
  }
  __syncthreads();  // the images make room for the sums
#pragma unroll
  for (int c = 0; c < CT; c++)
#pragma unroll
    for (int r = 0; r < RV; r++) lds.part[wave][c][r][lane] = sum[c][r];
  __syncthreads();
  for (int i = threadIdx.x; i < CT * RV * 64; i += 64 * kWaves) {
    const int c = i / (RV * 64), r = i / 64 % RV, l = i % 64;
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) total += lds.part[w][c][r][l];
    const int mm = m0 + l / 16 + 4 * r, nn = n0 + 16 * c + l % 16;
    if (mm < p.m && nn < p.n) p.y[static_cast<int64_t>(mm) * p.n + nn] = N::save(16.f * total);
  }
}

template <class N, int W, int CT, int GS>
void launch(const Args &p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.n + 16 * CT - 1) / (16 * CT)),
                  static_cast<unsigned>((p.m + 15) / 16));
  const dim3 block(64 * W);
  if (p.m <= 4) hipLaunchKernelGGL((matvec4_kernel<N, W, CT, GS, 1>), grid, block, 0, s, p);
  else if (p.m <= 8) hipLaunchKernelGGL((matvec4_kernel<N, W, CT, GS, 2>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((matvec4_kernel<N, W, CT, GS, 4>), grid, block, 0, s, p);
}

template <class N, int W, int CT>
void launch_group(const Args &p, int group, hipStream_t s) {
  if (group == 32) launch<N, W, CT, 1>(p, s);
  else if (group == 64) launch<N, W, CT, 2>(p, s);
  else launch<N, W, CT, 4>(p, s);
}

// Waves W and column tiles of a workgroup, by how many fall to a CU.  One workgroup of eight waves fits a CU, or two
// of four.  While one of them a CU is enough, eight waves with as many tiles as that takes; above, four
// waves with four tiles, which read and rearrange x once for 64 columns, unless two tiles spread so much
// more evenly that the fullest CU has less than 7/8 of the tiles.  (The rows do not count: a row gets the
// same bits in every batch.)  1 and 16 rows, us with (8 waves, 1 tile),
// (8, 2), (4, 2), (4, 4):
//   4096 x 4096 g128      6.0  7.1  7.4 10.3     6.4  7.7  7.7 11.2
//   8192 x 8192 g128     16.1 11.8 13.7 18.4    19.0 14.2 14.7 20.2
//   11008 x 4096 g64     18.2 17.1 11.4 12.3    19.4 19.5 13.3 13.3
//   24000 x 8192 g64     44.9 32.9 29.6 32.9    53.0 41.4 35.5 37.9   (96 columns a CU in pairs, 128 in fours)
//   27000 x 8192 g128    50.5 38.0 34.6 31.2    57.7 46.5 42.7 36.1   (128 both ways)
//   50000 x 4096 g64     73.0 57.0 32.0 33.1    77.7 67.7 40.0 37.8   (224, 256)
template <class N>
void launch_type(const Args &p, int group, hipStream_t s) {
  const int cus = device_cu_count();
  const auto groups = [&](int ct) { return (p.n + 16 * ct - 1) / (16 * ct); };
  const auto fullest = [&](int ct) { return (groups(ct) + cus - 1) / cus * ct; };
  if (groups(1) <= cus) launch_group<N, 8, 1>(p, group, s);
  else if (groups(2) <= cus) launch_group<N, 8, 2>(p, group, s);
  else if (groups(4) <= cus || 8 * fullest(2) < 7 * fullest(4)) launch_group<N, 4, 2>(p, group, s);
  else launch_group<N, 4, 4>(p, group, s);
}

}  // namespace
}  // namespace mv4
}  // namespace vs

using namespace vs;

extern "C" {

vs_status vs_matvec_int4(int dtype, const void *x, int64_t ldx, const uint8_t *qweight,
                         int64_t ldq, const void *scales, const uint8_t *zeros, int64_t group,
                         int64_t m, int64_t n, int64_t k, void *y, vs_stream_t stream) {
  clear_error();
  VS_REQUIRE(dtype == VS_F16 || dtype == VS_BF16, "matvec_int4: unsupported dtype %d (fp16, bf16)",
             dtype);
  VS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "matvec_int4: negative dimension");
  VS_REQUIRE(group == 32 || group == 64 || (group > 0 && group % 128 == 0),
             "matvec_int4: group of %lld (32, 64 or a multiple of 128)",
             static_cast<long long>(group));
  VS_REQUIRE(m < (1ll << 31) && n < (1ll << 30) && k < (1ll << 30) && group < (1ll << 30),
             "matvec_int4: dimension too large");
  if (m == 0 || n == 0) return VS_OK;
  VS_REQUIRE(y && (k == 0 || (x && qweight && scales)), "matvec_int4: null pointer");
  VS_REQUIRE(m == 1 || ldx >= k || ldx == 0, "matvec_int4: ldx < k");
  VS_REQUIRE(n == 1 || ldq >= (k + 1) / 2, "matvec_int4: ldq < (k + 1) / 2");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int64_t kRows = 16 * kMaxGridY;  // rows of one launch
  for (int64_t m0 = 0; m0 < m; m0 += kRows) {
    mv4::Args p{};
    p.x = static_cast<const uint16_t *>(x) + m0 * ldx;
    p.ldx = ldx;
    p.q = qweight;
    p.ldq = ldq;
    p.s = static_cast<const uint16_t *>(scales);
    p.z = zeros;
    p.y = static_cast<uint16_t *>(y) + m0 * n;
    p.m = static_cast<int>(std::min(kRows, m - m0));
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.groups = static_cast<int>((k + group - 1) / group);
    p.span = static_cast<int>(std::max<int64_t>(1, group / mv4::kBlock));
    if (dtype == VS_BF16) mv4::launch_type<num::BF16>(p, static_cast<int>(group), s);
    else mv4::launch_type<num::F16>(p, static_cast<int>(group), s);
    VS_HIP(hipGetLastError());
  }
  return VS_OK;
}

}  // extern "C"
