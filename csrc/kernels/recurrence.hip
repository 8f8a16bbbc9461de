// Gated linear recurrence: a first-order recursive filter whose coefficient is an input.
//
//   i_t = 1 / (1 + exp(g_t)),   h_t = h_{t-1} + i_t (x_t - h_{t-1}),   y_t = h_t
//
// for every channel of [batch][time][channel] arrays.  Backward, with m_t the gradient that step t
// receives from step t + 1 on:
//
//   l_t = dy_t + m_t,  dx_t = i_t l_t,  dg_t = i_t (1 - i_t) l_t (h_{t-1} - x_t),
//   m_{t-1} = (1 - i_t) l_t
//
// A step keeps the smaller of i and 1 - i, computed from the gate directly, and goes from the side of the
// larger: h + i (x - h) where the state is kept, i x + (1 - i) h where it is replaced.  So a small share is
// never the rest of a subtraction, a long memory is not multiplied by a rounded 1 - i, and a value that
// replaces a much larger state keeps its digits.  (Against h + i (x - h) alone: 1 x 65536 x 1024 fp32 150 us
// instead of 149, training pass 4 x 4096 x 4096 bf16 232 instead of 222, 16 x 1000 x 1536 fp16 35 instead
// of 31.  With x + (1 - i) (h - x) it would be 228 and 33, but an infinite x would give inf - inf.)
//
// Every step is an affine map s -> a s + b of the state (forward) or of m (backward), so a run
// of steps is one map too, and runs compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).
//
// Bound: bandwidth.  Forward reads x and g and writes y; backward reads x, g, dy and writes
// dx, dg.  The split that keeps it to one pass over the data: a workgroup works on a tile of W x L
// steps of 64 V channels, wave w on L of them.  A wave reduces its steps to one map per channel,
// the W maps meet in LDS, every wave composes them to its own initial state, and the steps run
// again from registers.  The state never leaves fp32.  Backward recomputes h from the state at the
// start of each tile, which the forward pass keeps (4 bytes per channel and tile, 1/64 of a read
// of y in 16 bits).
//
// Between tiles the maps pass through memory: a tile publishes its map as soon as it has it, and
// composes its initial state from the maps of the tiles before it in its run of kRun tiles and the
// state at the start of the run, which the last tile of the run before publishes.  What is composed
// with what does not depend on timing, so results are the same bits every time.  Measured against
// a workgroup that walks the tiles of its channels (forward, us): 1 x 65536 x 1024 fp32 152 against
// 2017 (295 with time cut into segments whose maps a first kernel computes, which reads x and g
// twice), 4 x 4096 x 4096 bf16 97 against 136, 8 x 2048 x 8192 bf16 169 against 186.  That is 5.3,
// 4.2 and 4.8 TB/s; a large copy reaches 5.1 to 5.3 on the same card.  Backward: 248, 150 and 275 us
// (5.4, 4.5 and 4.9 TB/s).
// Copyright 2026 veles.simd_amd authors. Apache-2.0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "csrc/kernels/number.h"
#include "csrc/runtime/runtime.h"
#include "simd/gpu.h"

namespace vs {
namespace rec {
namespace {

using num::Pack;

struct Args {
  const void *x, *g, *dy;            // dy may be null (zeros)
  int64_t xb, xt, gb, gt, yb, yt;    // strides in elements (channels are contiguous)
  const float *state;                // [batch][d] or null (zeros)
  const float *dfinal;               // [batch][d] or null (zeros)
  const void *lengths;               // [batch] or null
  int lengths64;
  void *y, *dx, *dg;                 // [batch][t][d]
  float *final, *dstate;             // [batch][d]
  float *starts;                     // [batch][tiles][d]: state at the start of each tile, or null
  uint64_t *maps;                    // [batch][tiles][d]: a tile's map (product low, sum high)
  uint32_t *heads;                   // [batch][runs][d]: what enters a run of tiles
  uint32_t *ticket;                  // a counter per group, or null where a sequence is one tile
  int spread;                        // words between two counters
  int64_t t, tiles;                  // steps, tiles
  int64_t group0;                    // first group (sequence and slab of 64 V channels) of this launch
  unsigned groups;                   // groups of this launch
  int d, slabs;
};

__device__ __forceinline__ int64_t steps_of(const Args &p, int64_t b) {
  if (!p.lengths) return p.t;
  const int64_t n = p.lengths64 ? static_cast<const int64_t *>(p.lengths)[b]
                                : static_cast<const int32_t *>(p.lengths)[b];
  return n < 0 ? 0 : n < p.t ? n : p.t;
}

// The smaller of a step's two shares, at most 1/2, with the gate's sign: that of the new value (i) where
// the gate is positive and the state is kept, that of the state (1 - i) where it is negative.
__device__ __forceinline__ float share(float g) {
  const float e = __expf(-fabsf(g));
  return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}
// q, to be used anew: the compiler would otherwise keep what it computed from the shares of all steps from
// one pass to the next, in 26 registers that cost a workgroup of three a CU.
__device__ __forceinline__ float anew(float q) {
  asm volatile("" : "+v"(q));
  return q;
}
__device__ __forceinline__ bool keeps(float q) { return __float_as_int(q) >= 0; }
__device__ __forceinline__ float advance(float q, float x, float h) {
  const float s = fabsf(q);
  return fmaf(s, keeps(q) ? x - h : h, keeps(q) ? h : (1.f - s) * x);
}
// (1 - i) v
__device__ __forceinline__ float kept(float q, float v) { return fmaf(-q, v, keeps(q) ? v : 0.f); }

template <class N, int V, int W, int L>
struct Shape {
  static constexpr int kTile = W * L, kLanes = 64 * V;
  using E = typename N::store;
  using P = Pack<N, V>;

  // The L steps of this wave from `t` on, at lane offset c: row addresses are the same for the
  // whole wave, so they live in scalar registers.  Steps in the padding load the last step that
  // is none (memory of the tensor; what comes of it is not used).
  __device__ __forceinline__ static void load(P (&r)[L], const void *base, int64_t off,
                                              int64_t stride, int c, int64_t t, int64_t len) {
    const E *row = static_cast<const E *>(base) + off;
    if (t + L <= len) {
      row += t * stride;
#pragma unroll
      for (int s = 0; s < L; s++) r[s] = *reinterpret_cast<const P *>(row + s * stride + c);
    } else {
#pragma unroll
      for (int s = 0; s < L; s++)
        r[s] = *reinterpret_cast<const P *>(row + (t + s < len ? t + s : len - 1) * stride + c);
    }
  }
  __device__ __forceinline__ static void store(void *base, int64_t row, int d, int c, const P &v) {
    *reinterpret_cast<P *>(static_cast<E *>(base) + row * d + c) = v;
  }
  __device__ __forceinline__ static P zero() {
    P z;
#pragma unroll
    for (int v = 0; v < V; v++) z.set(v, 0.f);
    return z;
  }

  // Shares of the wave's steps and their map: product a, end e from a zero state.  `on` steps are
  // none of padding; the others are left out (a share of 0 would turn an infinite state into NaN).
  __device__ __forceinline__ static void forward_map(const P (&x)[L], const P (&g)[L], int on,
                                                     float (&i)[L][V], float (&a)[V], float (&e)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
      a[v] = 1.f;
      e[v] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < L; s++)
#pragma unroll
      for (int v = 0; v < V; v++) i[s][v] = share(g[s][v]);
    steps(on, [&](int s, bool use) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float q = anew(i[s][v]), en = advance(q, x[s][v], e[v]), an = kept(q, a[v]);
        e[v] = use ? en : e[v];
        a[v] = use ? an : a[v];
      }
    });
  }
  // f(s, whether step s is none of padding) for s = 0 .. L - 1, or down from L - 1.
  template <bool DOWN = false, class F>
  __device__ __forceinline__ static void steps(int on, const F &f) {
    if (on >= L) {
#pragma unroll
      for (int s = 0; s < L; s++) f(DOWN ? L - 1 - s : s, true);
    } else {
#pragma unroll
      for (int s = 0; s < L; s++) f(DOWN ? L - 1 - s : s, (DOWN ? L - 1 - s : s) < on);
    }
  }
  // Runs the steps from state h and stores y.
  __device__ __forceinline__ static void forward_steps(const Args &p, int64_t b, int c, bool in, int64_t t,
                                                       int on, const P (&x)[L], const float (&i)[L][V],
                                                       float (&h)[V]) {
    steps(on, [&](int s, bool use) {
      P y;
#pragma unroll
      for (int v = 0; v < V; v++) {
        h[v] = advance(anew(i[s][v]), x[s][v], h[v]);
        y.set(v, h[v]);
      }
      if (in && (use || t + s < p.t)) store(p.y, b * p.t + t + s, p.d, c, use ? y : zero());
    });
  }
  // End q of the wave's steps backward from a zero m (the product is the forward one).
  __device__ __forceinline__ static void backward_map(const P (&dy)[L], int on, const float (&i)[L][V],
                                                      float (&q)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) q[v] = 0.f;
    steps<true>(on, [&](int s, bool use) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float l = q[v] + dy[s][v], qn = kept(i[s][v], l);
        q[v] = use ? qn : q[v];
      }
    });
  }
  // Runs the steps forward from state h, then backward from m, and stores dx and dg.
  __device__ __forceinline__ static void backward_steps(const Args &p, int64_t b, int c, bool in,
                                                        int64_t t, int on, const P (&x)[L],
                                                        const P (&dy)[L],
                                                        const float (&i)[L][V], float (&h)[V],
                                                        float (&m)[V]) {
    float before[L][V];  // h_{t-1} - x_t
#pragma unroll
    for (int s = 0; s < L; s++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        before[s][v] = h[v] - x[s][v];
        h[v] = advance(i[s][v], x[s][v], h[v]);
      }
    steps<true>(on, [&](int s, bool use) {
      P ox, og;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float l = m[v] + dy[s][v], q = i[s][v], small = fabsf(q) * l, large = fmaf(-fabsf(q), l, l);
        ox.set(v, keeps(q) ? small : large);
        og.set(v, fabsf(q) * large * before[s][v]);
        m[v] = use ? (keeps(q) ? large : small) : m[v];
      }
      if (in && (use || t + s < p.t)) {
        store(p.dx, b * p.t + t + s, p.d, c, use ? ox : zero());
        store(p.dg, b * p.t + t + s, p.d, c, use ? og : zero());
      }
    });
  }
  __device__ __forceinline__ static void zero_gradients(const Args &p, int64_t b, int c, bool in,
                                                        int64_t t) {
    if (in)
      for (int s = 0; s < L; s++)
        if (t + s < p.t) {
          store(p.dx, b * p.t + t + s, p.d, c, zero());
          store(p.dg, b * p.t + t + s, p.d, c, zero());
        }
  }
};

// ------------------------------------------------------------------ chain
// Workgroups take the tiles of a group (a sequence and a slab of channels) by a counter, position by
// position along time (from the end in the backward pass).  A tile waits for earlier positions of
// its group only, and a workgroup takes its position when it already runs: by induction over the
// positions every wait ends.  (One counter for all tiles costs about 15 ns a workgroup, one after
// the other: 16 x 1000 x 1536 fp16 47 us, 41 with a counter per group.)  Maps and
// states are published and polled as single relaxed atomics at device scope, 64 or 32 bits that are
// never all ones when they are valid (a NaN is stored as the canonical one), so no other memory has
// to be ordered with them.  The buffers are set to all ones before the launch.
constexpr int kRun = 8;  // 4 and 16 are slower where channels are few: 177 and 172 us at 1 x 65536 x 1024 fp32
constexpr uint32_t kNone = 0xffffffffu;
constexpr int kPolls = 1 << 20;  // about a second; then a NaN goes on in place of what did not come

__device__ __forceinline__ uint32_t bits(float f) {
  return f == f ? __float_as_uint(f) : 0x7fc00000u;
}

struct Map {
  float a, e;
};
__device__ __forceinline__ void publish(uint64_t *at, Map m) {
  __hip_atomic_store(at, bits(m.a) | static_cast<uint64_t>(bits(m.e)) << 32, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Map await(uint64_t *at) {
  for (int n = 0; n < kPolls; n++) {
    const uint64_t v = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (v != ~0ull) return Map{__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(v >> 32)};
    __builtin_amdgcn_s_sleep(1);
  }
  return Map{__builtin_nanf(""), __builtin_nanf("")};
}
__device__ __forceinline__ void publish(uint32_t *at, float s) {
  __hip_atomic_store(at, bits(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float await(uint32_t *at) {
  for (int n = 0; n < kPolls; n++) {
    const uint32_t v = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (v != kNone) return __uint_as_float(v);
    __builtin_amdgcn_s_sleep(1);
  }
  return __builtin_nanf("");
}

__global__ __launch_bounds__(256) void ones_kernel(uint4 *p, int64_t n) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
    p[i] = uint4{kNone, kNone, kNone, kNone};
}

template <int V, int W>
struct Chain {
  static constexpr int kLanes = 64 * V;
  float run[kRun - 1][2][kLanes];  // maps of the tiles before this one in its run
  float head[kLanes];              // what enters the run
  unsigned pos;
};

// This workgroup's position along the chain, its sequence and its slab of channels.  (Workgroups that
// stay and draw their next tile while they work were slower, 194 us against 164 at
// 1 x 65536 x 1024 fp32: the tiles behind wait for a position whose workgroup is not free yet.)
struct Place {
  int64_t pos, b;
  int slab;
};
template <int V, int W>
__device__ __forceinline__ Place take(const Args &p, Chain<V, W> &ch) {
  // A group moves on by one workgroup, so by one XCD, with every turn: if a slab stayed on its XCD,
  // its 256-byte pieces of rows a power of two apart would use a few of that cache's channels
  // (1 x 65536 x 2048 bf16: 208 us, 173 this way).
  const unsigned turn = blockIdx.x / p.groups;
  const int64_t group = p.group0 + (blockIdx.x + turn) % p.groups, b = group / p.slabs;
  unsigned pos = 0;
  if (p.ticket) {
    if (threadIdx.x == 0) ch.pos = atomicAdd(p.ticket + group * p.spread, 1u) + 1u;  // from all ones
    __syncthreads();
    pos = __builtin_amdgcn_readfirstlane(ch.pos);
  }
  return Place{pos, b, static_cast<int>(group - b * p.slabs)};
}

// Publishes this tile's map, and brings `s` to what enters the tile: `initial` at position 0.
// False: a tile of padding that nothing waits for beyond its map.
template <int V, int W>
__device__ __forceinline__ bool enter(const Args &p, Chain<V, W> &ch, int64_t b, int64_t pos, int c,
                                      bool in, int lane, int wave, bool live, const float *initial,
                                      const float (&ta)[V], const float (&te)[V], float (&s)[V]) {
  const int64_t runs = (p.tiles + kRun - 1) / kRun, q = pos / kRun;
  const int before = static_cast<int>(pos - q * kRun);
  const bool closes = before == kRun - 1 && pos + 1 < p.tiles, last = pos + 1 == p.tiles;
  uint64_t *maps = p.maps + (b * p.tiles + pos) * p.d + c;
  if (!closes && !last) {  // the state after those two goes on by itself
    if (wave == 0 && in)
#pragma unroll
      for (int v = 0; v < V; v++) publish(maps + v, Map{ta[v], te[v]});
    if (!live) return false;
  }
  for (int j = wave; j < before; j += W)
#pragma unroll
    for (int v = 0; v < V; v++) {
      Map m = {1.f, 0.f};
      if (in) m = await(maps + v - static_cast<int64_t>(before - j) * p.d);
      ch.run[j][0][lane * V + v] = m.a;
      ch.run[j][1][lane * V + v] = m.e;
    }
  if (wave == W - 1)
#pragma unroll
    for (int v = 0; v < V; v++) {
      float h = 0.f;
      if (q == 0) h = initial ? initial[b * p.d + c + v] : 0.f;
      else if (in) h = await(p.heads + (b * runs + q) * p.d + c + v);
      ch.head[lane * V + v] = h;
    }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; v++) s[v] = ch.head[lane * V + v];
  for (int j = 0; j < before; j++)
#pragma unroll
    for (int v = 0; v < V; v++)
      s[v] = fmaf(ch.run[j][0][lane * V + v], s[v], ch.run[j][1][lane * V + v]);
  if (closes && wave == 0 && in)
#pragma unroll
    for (int v = 0; v < V; v++)
      publish(p.heads + (b * runs + q + 1) * p.d + c + v, fmaf(ta[v], s[v], te[v]));
  return true;
}

template <class N, int V, int W, int L>
__global__ __launch_bounds__(64 * W) void forward_kernel(Args p) {
  using S = Shape<N, V, W, L>;
  using P = typename S::P;
  __shared__ float maps[2][W][S::kLanes];
  __shared__ Chain<V, W> ch;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [pos, b, slab] = take(p, ch);
  const int c0 = slab * S::kLanes + lane * V;
  const bool in = c0 < p.d;
  const int c = in ? c0 : 0;
  const int64_t len = steps_of(p, b), t0 = pos * S::kTile + wave * L;
  const bool live = pos * S::kTile < len;
  const int on = static_cast<int>(len - t0 < 0 ? 0 : len - t0 < L ? len - t0 : L);  // steps that are no padding
  P x[L], g[L];
  float i[L][V], ta[V], te[V], s[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    ta[v] = 1.f;
    te[v] = 0.f;
  }
  if (live) {
    float a[V], e[V];
    S::load(x, p.x, b * p.xb, p.xt, c, t0, len);
    S::load(g, p.g, b * p.gb, p.gt, c, t0, len);
    S::forward_map(x, g, on, i, a, e);
#pragma unroll
    for (int v = 0; v < V; v++) {
      maps[0][wave][lane * V + v] = a[v];
      maps[1][wave][lane * V + v] = e[v];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        te[v] = fmaf(maps[0][w][lane * V + v], te[v], maps[1][w][lane * V + v]);
        ta[v] *= maps[0][w][lane * V + v];
      }
  }
  if (!enter(p, ch, b, pos, c, in, lane, wave, live, p.state, ta, te, s)) {
    if (in)
      for (int k = 0; k < L; k++)
        if (t0 + k < p.t) S::store(p.y, b * p.t + t0 + k, p.d, c, S::zero());
    return;
  }
  if (wave == 0 && in)
#pragma unroll
    for (int v = 0; v < V; v++) {
      if (live && p.starts) p.starts[(b * p.tiles + pos) * p.d + c + v] = s[v];
      if (pos + 1 == p.tiles) p.final[b * p.d + c + v] = fmaf(ta[v], s[v], te[v]);
    }
  if (!live) {
    if (in)
      for (int k = 0; k < L; k++)
        if (t0 + k < p.t) S::store(p.y, b * p.t + t0 + k, p.d, c, S::zero());
    return;
  }
  for (int w = 0; w < wave; w++)
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = fmaf(maps[0][w][lane * V + v], s[v], maps[1][w][lane * V + v]);
  S::forward_steps(p, b, c, in, t0, on, x, i, s);
}

template <class N, int V, int W, int L>
__global__ __launch_bounds__(64 * W) void backward_kernel(Args p) {
  using S = Shape<N, V, W, L>;
  using P = typename S::P;
  __shared__ float maps[3][W][S::kLanes];
  __shared__ Chain<V, W> ch;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [pos, b, slab] = take(p, ch);
  const int64_t tile = p.tiles - 1 - pos;
  const int c0 = slab * S::kLanes + lane * V;
  const bool in = c0 < p.d;
  const int c = in ? c0 : 0;
  const int64_t len = steps_of(p, b), t0 = tile * S::kTile + wave * L;
  const bool live = tile * S::kTile < len;
  const int on = static_cast<int>(len - t0 < 0 ? 0 : len - t0 < L ? len - t0 : L);
  P x[L], g[L], dy[L];
  float i[L][V], h[V], ta[V], te[V], m[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    ta[v] = 1.f;
    te[v] = h[v] = 0.f;
  }
  if (live) {
    float a[V], e[V], q[V];
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = p.starts[(b * p.tiles + tile) * p.d + c + v];
    S::load(x, p.x, b * p.xb, p.xt, c, t0, len);
    S::load(g, p.g, b * p.gb, p.gt, c, t0, len);
    if (p.dy) {
      S::load(dy, p.dy, b * p.yb, p.yt, c, t0, len);
    } else {
#pragma unroll
      for (int k = 0; k < L; k++) dy[k] = S::zero();
    }
    S::forward_map(x, g, on, i, a, e);
    S::backward_map(dy, on, i, q);
#pragma unroll
    for (int v = 0; v < V; v++) {
      maps[0][wave][lane * V + v] = a[v];
      maps[1][wave][lane * V + v] = e[v];
      maps[2][wave][lane * V + v] = q[v];
    }
    __syncthreads();
#pragma unroll
    for (int w = W - 1; w >= 0; w--)
#pragma unroll
      for (int v = 0; v < V; v++) {
        te[v] = fmaf(maps[0][w][lane * V + v], te[v], maps[2][w][lane * V + v]);
        ta[v] *= maps[0][w][lane * V + v];
      }
  }
  if (!enter(p, ch, b, pos, c, in, lane, wave, live, p.dfinal, ta, te, m)) {
    S::zero_gradients(p, b, c, in, t0);
    return;
  }
  if (wave == 0 && in && pos + 1 == p.tiles && p.dstate)
#pragma unroll
    for (int v = 0; v < V; v++) p.dstate[b * p.d + c + v] = fmaf(ta[v], m[v], te[v]);
  if (!live) {
    S::zero_gradients(p, b, c, in, t0);
    return;
  }
  for (int w = 0; w < wave; w++)
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = fmaf(maps[0][w][lane * V + v], h[v], maps[1][w][lane * V + v]);
  for (int w = W - 1; w > wave; w--)
#pragma unroll
    for (int v = 0; v < V; v++) m[v] = fmaf(maps[0][w][lane * V + v], m[v], maps[2][w][lane * V + v]);
  S::backward_steps(p, b, c, in, t0, on, x, dy, i, h, m);
}

// ------------------------------------------------------------ single step
// One value per thread: a step of a decoding batch is a few hundred KB at most.
template <class N>
__global__ __launch_bounds__(256) void step_kernel(const typename N::store *__restrict__ x,
                                                   int64_t xb,
                                                   const typename N::store *__restrict__ g,
                                                   int64_t gb, float *__restrict__ state,
                                                   typename N::store *__restrict__ y,
                                                   int64_t n, int d) {
  for (int64_t at = blockIdx.x * 256ll + threadIdx.x; at < n; at += gridDim.x * 256ll) {
    const int64_t b = at / d, c = at - b * d;
    const float h0 = state[at];
    const float h = advance(share(N::load(g[b * gb + c])), N::load(x[b * xb + c]), h0);
    state[at] = h;
    y[at] = N::save(h);
  }
}

// ------------------------------------------------------------------- host
constexpr int kSteps = 16;  // steps of a wave in a tile

// Waves along time.  A short sequence would leave most of a tall tile empty.
int waves_of(int64_t t) { return t <= kSteps ? 1 : t <= 2 * kSteps ? 2 : 8; }
int64_t tiles_of(int64_t t) {
  const int tile = kSteps * waves_of(t);
  return (t + tile - 1) / tile;
}

// Workgroups of one launch: a grid holds fewer than 2^32 threads.
constexpr int64_t kMostTiles = 1 << 22;

struct Plan {
  int slabs;
  int64_t groups, at_once;             // groups, and those of one launch
  int spread;                          // words between two counters: lines of their own where they are few
  size_t tickets, maps, heads, bytes;  // sizes of the chain's buffers, and of the workspace
};

// Two 16-bit channels a lane where alignment allows it: a wave then reads 256 bytes of a step, as
// with one fp32 channel (4 x 4096 x 4096 bf16: 100 us against 125 when it was tried).
Plan plan(int64_t batch, int64_t t, int64_t d, bool pairs) {
  Plan q{};
  const int lanes = pairs ? 128 : 64;
  const int64_t tiles = std::max<int64_t>(1, tiles_of(t));
  q.slabs = static_cast<int>((d + lanes - 1) / lanes);
  q.groups = batch * q.slabs;
  q.at_once = std::max<int64_t>(1, std::min(q.groups, kMostTiles / tiles));
  if (tiles > 1) {
    q.spread = q.groups <= 4096 ? 64 : 1;
    q.tickets = static_cast<size_t>(q.groups * q.spread + 3) / 4 * 16;
    q.maps = static_cast<size_t>(batch) * tiles * d * sizeof(uint64_t);
    q.heads = static_cast<size_t>(batch) * ((tiles + kRun - 1) / kRun) * d * sizeof(uint32_t);
    q.bytes = (q.tickets + q.maps + q.heads + 15) / 16 * 16;
  }
  return q;
}

template <class N, int V, int W>
void launch(bool back, const Args &p, hipStream_t s) {
  const unsigned grid = p.groups * static_cast<unsigned>(p.tiles);
  if (back) hipLaunchKernelGGL((backward_kernel<N, V, W, kSteps>), dim3(grid), dim3(64 * W), 0, s, p);
  else hipLaunchKernelGGL((forward_kernel<N, V, W, kSteps>), dim3(grid), dim3(64 * W), 0, s, p);
}

template <class N, int V>
void launch_waves(bool back, const Args &p, hipStream_t s) {
  const int w = waves_of(p.t);
  if (w == 1) launch<N, V, 1>(back, p, s);
  else if (w == 2) launch<N, V, 2>(back, p, s);
  else launch<N, V, 8>(back, p, s);
}

template <class N>
void launch_type(bool back, bool pairs, const Args &p, hipStream_t s) {
  if constexpr (sizeof(typename N::store) == 2) {
    if (pairs) {
      launch_waves<N, 2>(back, p, s);
      return;
    }
  }
  launch_waves<N, 1>(back, p, s);
}

vs_status check(const char *who, int dtype, int64_t batch, int64_t t, int64_t d) {
  VS_REQUIRE(dtype == VS_F32 || dtype == VS_F16 || dtype == VS_BF16,
             "%s: unsupported dtype %d (fp32, fp16, bf16)", who, dtype);
  VS_REQUIRE(batch >= 0 && t >= 0 && d >= 0, "%s: negative dimension", who);
  VS_REQUIRE(d < (1ll << 28) && t < (1ll << 40) && batch < (1ll << 31),
             "%s: dimension too large", who);
  return VS_OK;
}

bool paired(const void *p, int64_t sb, int64_t st) {
  return reinterpret_cast<uintptr_t>(p) % 4 == 0 && sb % 2 == 0 && st % 2 == 0;
}

vs_status run(bool back, Args p, int dtype, int64_t batch, void *workspace, size_t bytes,
              hipStream_t s) {
  const bool pairs = dtype != VS_F32 && p.d % 2 == 0 && paired(p.x, p.xb, p.xt) &&
                     paired(p.g, p.gb, p.gt) && paired(p.dy, p.yb, p.yt) && paired(p.y, 0, 0) &&
                     paired(p.dx, 0, 0) && paired(p.dg, 0, 0);
  const Plan q = plan(batch, p.t, p.d, pairs);
  p.tiles = std::max<int64_t>(1, tiles_of(p.t));
  VS_REQUIRE(p.tiles <= kMostTiles, "gated_recurrence: sequence too long (%lld steps)",
             static_cast<long long>(p.t));
  p.slabs = q.slabs;
  DeviceBuffer own;
  if (q.bytes) {
    uint8_t *base = static_cast<uint8_t *>(workspace);
    if (workspace) {
      VS_REQUIRE(bytes >= q.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "gated_recurrence: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes,
                 q.bytes);
    } else {
      VS_TRY(own.alloc(q.bytes, s));
      base = own.as<uint8_t>();
    }
    p.ticket = reinterpret_cast<uint32_t *>(base);
    p.spread = q.spread;
    p.maps = reinterpret_cast<uint64_t *>(base + q.tickets);
    p.heads = reinterpret_cast<uint32_t *>(base + q.tickets + q.maps);
    const int64_t n = static_cast<int64_t>(q.bytes / 16);
    hipLaunchKernelGGL(ones_kernel, dim3(elementwise_grid(static_cast<size_t>(n), 256)), dim3(256), 0, s,
                       reinterpret_cast<uint4 *>(base), n);
    VS_HIP(hipGetLastError());
  }
  for (; p.group0 < q.groups; p.group0 += q.at_once) {
    p.groups = static_cast<unsigned>(std::min(q.at_once, q.groups - p.group0));
    if (dtype == VS_F32) launch_type<num::F32>(back, pairs, p, s);
    else if (dtype == VS_F16) launch_type<num::F16>(back, pairs, p, s);
    else launch_type<num::BF16>(back, pairs, p, s);
    VS_HIP(hipGetLastError());
  }
  return VS_OK;
}

}  // namespace
}  // namespace rec
}  // namespace vs

using namespace vs;

extern "C" {

int64_t vs_gated_recurrence_tiles(int64_t t) { return t > 0 ? rec::tiles_of(t) : 0; }

size_t vs_gated_recurrence_workspace(int64_t batch, int64_t t, int64_t d) {
  if (batch <= 0 || t <= 0 || d <= 0 || rec::check("", VS_F32, batch, t, d) != VS_OK) return 0;
  return std::max(rec::plan(batch, t, d, false).bytes, rec::plan(batch, t, d, true).bytes);
}

vs_status vs_gated_recurrence(int dtype, const void *x, int64_t x_batch, int64_t x_time,
                              const void *gate, int64_t gate_batch, int64_t gate_time,
                              const float *state, const void *lengths, int lengths64,
                              int64_t batch, int64_t t, int64_t d, void *y, float *final_state,
                              float *starts, void *workspace, size_t workspace_bytes,
                              vs_stream_t stream) {
  clear_error();
  VS_TRY(rec::check("gated_recurrence", dtype, batch, t, d));
  if (batch == 0 || d == 0) return VS_OK;
  VS_REQUIRE(final_state && (t == 0 || (x && gate && y)), "gated_recurrence: null pointer");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  rec::Args p{};
  p.x = x;
  p.xb = x_batch;
  p.xt = x_time;
  p.g = gate;
  p.gb = gate_batch;
  p.gt = gate_time;
  p.state = state;
  p.lengths = lengths;
  p.lengths64 = lengths64;
  p.y = y;
  p.final = final_state;
  p.starts = starts;
  p.t = t;
  p.d = static_cast<int>(d);
  return rec::run(false, p, dtype, batch, workspace, workspace_bytes, s);
}

vs_status vs_gated_recurrence_backward(int dtype, const void *x, int64_t x_batch, int64_t x_time,
                                       const void *gate, int64_t gate_batch, int64_t gate_time,
                                       const void *lengths, int lengths64, const float *starts,
                                       const void *dy, int64_t dy_batch, int64_t dy_time,
                                       const float *dfinal, int64_t batch, int64_t t, int64_t d,
                                       void *dx, void *dgate, float *dstate, void *workspace,
                                       size_t workspace_bytes, vs_stream_t stream) {
  clear_error();
  VS_TRY(rec::check("gated_recurrence_backward", dtype, batch, t, d));
  if (batch == 0 || d == 0) return VS_OK;
  VS_REQUIRE(t == 0 || (x && gate && starts && dx && dgate),
             "gated_recurrence_backward: null pointer");
  VS_REQUIRE(t > 0 || dstate, "gated_recurrence_backward: null pointer");
  rec::Args p{};
  p.x = x;
  p.xb = x_batch;
  p.xt = x_time;
  p.g = gate;
  p.gb = gate_batch;
  p.gt = gate_time;
  p.lengths = lengths;
  p.lengths64 = lengths64;
  p.starts = const_cast<float *>(starts);
  p.dy = dy;
  p.yb = dy_batch;
  p.yt = dy_time;
  p.dfinal = dfinal;
  p.dx = dx;
  p.dg = dgate;
  p.dstate = dstate;
  p.t = t;
  p.d = static_cast<int>(d);
  return rec::run(true, p, dtype, batch, workspace, workspace_bytes,
                  static_cast<hipStream_t>(stream));
}

vs_status vs_gated_recurrence_step(int dtype, const void *x, int64_t x_batch, const void *gate,
                                   int64_t gate_batch, float *state, int64_t batch, int64_t d,
                                   void *y, vs_stream_t stream) {
  clear_error();
  VS_TRY(rec::check("gated_recurrence_step", dtype, batch, 1, d));
  const int64_t n = batch * d;
  if (n == 0) return VS_OK;
  VS_REQUIRE(x && gate && state && y, "gated_recurrence_step: null pointer");
  const unsigned grid = elementwise_grid(static_cast<size_t>(n), 256);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int di = static_cast<int>(d);
  if (dtype == VS_F32)
    hipLaunchKernelGGL((rec::step_kernel<num::F32>), dim3(grid), dim3(256), 0, s,
                       static_cast<const float *>(x), x_batch, static_cast<const float *>(gate),
                       gate_batch, state, static_cast<float *>(y), n, di);
  else if (dtype == VS_F16)
    hipLaunchKernelGGL((rec::step_kernel<num::F16>), dim3(grid), dim3(256), 0, s,
                       static_cast<const uint16_t *>(x), x_batch,
                       static_cast<const uint16_t *>(gate), gate_batch, state,
                       static_cast<uint16_t *>(y), n, di);
  else
    hipLaunchKernelGGL((rec::step_kernel<num::BF16>), dim3(grid), dim3(256), 0, s,
                       static_cast<const uint16_t *>(x), x_batch,
                       static_cast<const uint16_t *>(gate), gate_batch, state,
                       static_cast<uint16_t *>(y), n, di);
  VS_HIP(hipGetLastError());
  return VS_OK;
}

}  // extern "C"
