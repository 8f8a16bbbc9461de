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
// mantissa of a bf16 or fp16 number 16 (0x4180 | q << 3 or 0x4c00 | q << 6), which is 16 + q
// exactly, two to a register, and the matrix cores multiply (16 x 16 x 32, x as the A operand,
// rows it does not have are zero).  Per group and column the fp32 sums then become
//
//   s (sum x (16 + q) - (16 + z) sum x)
//
// where sum x comes from one more product, with ones, in the layout it is needed in.  The factor
// 16 costs at most 3 of fp32's 24 bits against the sum of |x (q - z)|; weights are never rounded.
//
// A lane loads 16 bytes of its column's row: 32 neighbouring k, of which a matrix instruction
// takes 8 from each of the four 16-lane groups.  Two swaps of half and quarter waves transpose
// the four registers against the four groups, so that one instruction sees 32 neighbouring k
// and any group of 32 or more can be scaled.  The waves of a workgroup share its columns and cut
// k; their sums meet in LDS in a fixed order.
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

constexpr int kWaves = 8;
constexpr int kBlock = 128;  // k of one step: 16 bytes of q per lane

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

// Eight 4-bit numbers as 16 + q: pair p is (q_p, q_{p + 4}).
template <class N>
__device__ __forceinline__ Frag unpack(uint32_t w) {
  constexpr bool B = std::is_same_v<N, num::BF16>;
  constexpr uint32_t mask = B ? 0x00780078u : 0x03c003c0u, one = B ? 0x41804180u : 0x4c004c00u;
  Frag f;
  f.r[0] = ((B ? w << 3 : w << 6) & mask) | one;
  f.r[1] = ((B ? w >> 1 : w << 2) & mask) | one;
  f.r[2] = ((B ? w >> 5 : w >> 2) & mask) | one;
  f.r[3] = ((B ? w >> 9 : w >> 6) & mask) | one;
  return f;
}

// Eight neighbouring values of x in the order that unpack() gives the weights.
__device__ __forceinline__ Frag pairs(const uint4 &v) {
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

// What one lane loads for one step.  CT column tiles of 16; NG groups in a step.
template <int CT, int NG>
struct Loaded {
  uint32_t q[CT][4];
  uint4 x[4];
  uint16_t s[CT][NG];
  uint8_t z[CT][NG];
};

// CT: column tiles of 16 per workgroup; GS: MFMA steps of 32 per group (1, 2, 4; 4 covers larger
// groups through span); RV: accumulator rows in use, ceil(m / 4): row m of x is put where it
// comes out in accumulator register m / 4, so few rows scale few registers.
template <class N, int CT, int GS, int RV>
__global__ __launch_bounds__(64 * kWaves) void matvec4_kernel(Args p) {
  constexpr int NG = 4 / GS;
  using L = Loaded<CT, NG>;
  __shared__ float part[kWaves][CT][RV][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int m0 = blockIdx.y * 16, n0 = blockIdx.x * (16 * CT);
  const int row = m0 + l16 / 4 + 4 * (l16 % 4);  // A row l16
  const bool has = row < p.m;
  const uint16_t *xr = p.x + (has ? row : 0) * p.ldx;
  const uint8_t *qr[CT];
  int64_t sr[CT];
#pragma unroll
  for (int c = 0; c < CT; c++) {
    const int64_t n = n0 + 16 * c + l16 < p.n ? n0 + 16 * c + l16 : p.n - 1;
    qr[c] = p.q + n * p.ldq;
    sr[c] = n * p.groups;
  }
  const int blocks = (p.k + kBlock - 1) / kBlock, bytes = (p.k + 1) / 2;
  const int per = (blocks + kWaves - 1) / kWaves;
  const int first = wave * per, last = first + per < blocks ? first + per : blocks;

  const auto fetch = [&](int kb, L &v) {
    const int qo = kb * (kBlock / 2) + 16 * lq;
    if ((kb + 1) * kBlock <= p.k) {
#pragma unroll
      for (int c = 0; c < CT; c++) __builtin_memcpy(v.q[c], qr[c] + qo, 16);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        v.x[j] = uint4{0, 0, 0, 0};
        if (has) __builtin_memcpy(&v.x[j], xr + kb * kBlock + 32 * j + 8 * lq, 16);
      }
    } else {  // the row ends inside
#pragma unroll
      for (int c = 0; c < CT; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          uint32_t w = 0;
          for (int b = 0; b < 4; b++)
            if (qo + 4 * j + b < bytes) w |= static_cast<uint32_t>(qr[c][qo + 4 * j + b]) << (8 * b);
          v.q[c][j] = w;
        }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t w[4] = {0, 0, 0, 0};
        const int k0 = kb * kBlock + 32 * j + 8 * lq;
        for (int e = 0; e < 8; e++)
          if (has && k0 + e < p.k) w[e / 2] |= static_cast<uint32_t>(xr[k0 + e]) << (16 * (e & 1));
        v.x[j] = uint4{w[0], w[1], w[2], w[3]};
      }
    }
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
      for (int i = 0; i < NG; i++) {
        int g = NG > 1 ? kb * NG + i : kb / p.span;
        g = g < p.groups ? g : p.groups - 1;
        v.s[c][i] = p.s[sr[c] + g];
        v.z[c][i] = p.z ? p.z[sr[c] + g] : 8;
      }
  };

  const Frag ones = std::is_same_v<N, num::BF16>
                        ? Frag{{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}}
                        : Frag{{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}};
  float sum[CT][RV];
#pragma unroll
  for (int c = 0; c < CT; c++)
#pragma unroll
    for (int r = 0; r < RV; r++) sum[c][r] = 0.f;
  L cur, next;
  if (first < last) fetch(first, cur);
  for (int kb = first; kb < last; kb++) {
    if (kb + 1 < last) fetch(kb + 1, next);
#pragma unroll
    for (int c = 0; c < CT; c++) transpose(cur.q[c]);
#pragma unroll
    for (int i = 0; i < NG; i++) {
      const floatx4 none = {0.f, 0.f, 0.f, 0.f};
      floatx4 sx = none, acc[CT];
#pragma unroll
      for (int c = 0; c < CT; c++) acc[c] = none;
#pragma unroll
      for (int j = i * GS; j < (i + 1) * GS; j++) {
        const Frag a = pairs(cur.x[j]);
        sx = mma<N>(a, ones, sx);
#pragma unroll
        for (int c = 0; c < CT; c++) acc[c] = mma<N>(a, unpack<N>(cur.q[c][j]), acc[c]);
      }
#pragma unroll
      for (int c = 0; c < CT; c++) {
        const float s = N::load(cur.s[c][i]), z = -16.f - static_cast<float>(cur.z[c][i]);
#pragma unroll
        for (int r = 0; r < RV; r++) sum[c][r] = fmaf(s, fmaf(z, sx[r], acc[c][r]), sum[c][r]);
      }
    }
    cur = next;
  }
#pragma unroll
  for (int c = 0; c < CT; c++)
#pragma unroll
    for (int r = 0; r < RV; r++) part[wave][c][r][lane] = sum[c][r];
  __syncthreads();
  for (int i = threadIdx.x; i < CT * RV * 64; i += 64 * kWaves) {
    const int c = i / (RV * 64), r = i / 64 % RV, l = i % 64;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) v += part[w][c][r][l];
    const int mm = m0 + l / 16 + 4 * r, nn = n0 + 16 * c + l % 16;
    if (mm < p.m && nn < p.n) p.y[static_cast<int64_t>(mm) * p.n + nn] = N::save(v);
  }
}

template <class N, int CT, int GS>
void launch(const Args &p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.n + 16 * CT - 1) / (16 * CT)),
                  static_cast<unsigned>((p.m + 15) / 16));
  const dim3 block(64 * kWaves);
  if (p.m <= 4) hipLaunchKernelGGL((matvec4_kernel<N, CT, GS, 1>), grid, block, 0, s, p);
  else if (p.m <= 8) hipLaunchKernelGGL((matvec4_kernel<N, CT, GS, 2>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((matvec4_kernel<N, CT, GS, 4>), grid, block, 0, s, p);
}

template <class N>
void launch_type(const Args &p, int group, hipStream_t s) {
  const bool wide = p.m > 4 && p.n >= 64 * 128;
  if (wide) {
    if (group == 32) launch<N, 4, 1>(p, s);
    else if (group == 64) launch<N, 4, 2>(p, s);
    else launch<N, 4, 4>(p, s);
  } else {
    if (group == 32) launch<N, 1, 1>(p, s);
    else if (group == 64) launch<N, 1, 2>(p, s);
    else launch<N, 1, 4>(p, s);
  }
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
  VS_REQUIRE(m <= (1 << 20) && n < (1ll << 30) && k < (1ll << 30) && group < (1ll << 30),
             "matvec_int4: dimension too large");
  if (m == 0 || n == 0) return VS_OK;
  VS_REQUIRE(y && (k == 0 || (x && qweight && scales)), "matvec_int4: null pointer");
  VS_REQUIRE(m == 1 || ldx >= k || ldx == 0, "matvec_int4: ldx < k");
  VS_REQUIRE(n == 1 || ldq >= (k + 1) / 2, "matvec_int4: ldq < (k + 1) / 2");
  mv4::Args p{};
  p.x = static_cast<const uint16_t *>(x);
  p.ldx = ldx;
  p.q = qweight;
  p.ldq = ldq;
  p.s = static_cast<const uint16_t *>(scales);
  p.z = zeros;
  p.y = static_cast<uint16_t *>(y);
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.groups = static_cast<int>((k + group - 1) / group);
  p.span = static_cast<int>(std::max<int64_t>(1, group / mv4::kBlock));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == VS_BF16) mv4::launch_type<num::BF16>(p, static_cast<int>(group), s);
  else mv4::launch_type<num::F16>(p, static_cast<int>(group), s);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

}  // extern "C"
