// The 16- and 32-bit floating types of the sequence operators: storage, conversion to and
// from the fp32 that every kernel computes in.
// Copyright 2026 veles.simd_amd authors. Apache-2.0.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vs {
namespace num {

struct F32 {
  using store = float;
  __device__ __forceinline__ static float load(float v) { return v; }
  __device__ __forceinline__ static float save(float v) { return v; }
};
struct BF16 {
  using store = uint16_t;
  __device__ __forceinline__ static float load(uint16_t v) {
    return __uint_as_float(static_cast<uint32_t>(v) << 16);
  }
  __device__ __forceinline__ static uint16_t save(float v) {
    const __bf16 h = static_cast<__bf16>(v);  // to nearest, ties to even
    return __builtin_bit_cast(uint16_t, h);
  }
};
struct F16 {
  using store = uint16_t;
  __device__ __forceinline__ static float load(uint16_t v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  __device__ __forceinline__ static uint16_t save(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  }
};

// One value, or two neighbouring 16-bit values in one register, as they lie in memory; set in order.
template <class N, int V>
struct Pack;
template <class N>
struct Pack<N, 1> {
  typename N::store v;
  __device__ __forceinline__ float operator[](int) const { return N::load(v); }
  __device__ __forceinline__ void set(int, float f) { v = N::save(f); }
};
template <class N>
struct Pack<N, 2> {
  uint32_t w;
  __device__ __forceinline__ float operator[](int i) const {
    return N::load(static_cast<uint16_t>(i ? w >> 16 : w));
  }
  __device__ __forceinline__ void set(int i, float f) {
    if (i == 0) w = N::save(f);
    else w |= static_cast<uint32_t>(N::save(f)) << 16;
  }
};

}  // namespace num
}  // namespace vs
