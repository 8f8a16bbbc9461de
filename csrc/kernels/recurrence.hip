// Gated linear recurrence: a first-order recursive filter whose coefficient is an input.
//
//   i_t = 1 / (1 + exp(g_t)),   h_t = h_{t-1} + i_t (x_t - h_{t-1}),   y_t = h_t
//
// for every channel of [batch][time][channel] arrays.  i_t is the share of the new value and is
// computed from the gate directly (1 - sigmoid(g) would lose its digits where the memory is
// long), and the update in this form never multiplies the state by a rounded 1 - i_t.
//
// Backward, with m_t the gradient that step t receives from step t + 1 on:
//
//   l_t = dy_t + m_t,  dx_t = i_t l_t,  dg_t = i_t (1 - i_t) l_t (h_{t-1} - x_t),
//   m_{t-1} = l_t - i_t l_t
//
// Every step is an affine map s -> a s + b of the state (forward) or of m (backward), so a run
// of steps is one map too, and runs compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).
//
// Bound: bandwidth.  Forward reads x and g and writes y; backward reads x, g, dy and writes
// dx, dg.  The split that keeps it to one pass over the data: a workgroup owns 64 V channels of
// one sequence and walks time in tiles of W x L steps, wave w the L steps from w L on.  A wave
// reduces its steps to one map per channel, the W maps meet in LDS (one barrier a tile, two
// images in turn), every wave composes them to its own initial state, and the steps run again
// from registers.  The next tile's loads are issued before the tile is worked on.  The state
// never leaves fp32 registers.  Backward recomputes h from the state at the start of each tile,
// which the forward pass keeps (4 bytes per channel and tile, 1/32 to 1/64 of a read of y).
//
// Few sequences and channels leave most of the chip idle, so time is cut into segments then: a
// first kernel computes each segment's map (two of the three or five streams are read twice),
// and the second composes the maps before its own segment.
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
  float *maps;                       // [batch][segs][2][d]: the segments' maps
  int64_t t, tiles, seg_tiles;       // steps; tiles in all; tiles per segment
  int64_t b0;                        // first sequence of this launch
  int d, slabs, segs;
};

__device__ __forceinline__ int64_t steps_of(const Args &p, int64_t b) {
  if (!p.lengths) return p.t;
  const int64_t n = p.lengths64 ? static_cast<const int64_t *>(p.lengths)[b]
                                : static_cast<const int32_t *>(p.lengths)[b];
  return n < 0 ? 0 : n < p.t ? n : p.t;
}

__device__ __forceinline__ float share(float g) {
  return __builtin_amdgcn_rcpf(1.f + __expf(g));
}

template <class N, int V, int W, int L>
struct Shape {
  static constexpr int kTile = W * L, kLanes = 64 * V;
  using E = typename N::store;
  using P = Pack<N, V>;

  // The L steps of this wave from `t` on, at lane offset c: row addresses are the same for the
  // whole wave, so they live in scalar registers.  Steps in the padding load the last step that
  // is none (memory of the tensor; the value is replaced by blank() below).
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
  // Padding steps become `v`: a gate of +inf lets nothing in (share() is exactly 0), so they
  // keep the state and pass gradients through whatever the tensor holds there.
  __device__ __forceinline__ static void blank(P (&r)[L], int64_t t, int64_t len, float f) {
    P z;
#pragma unroll
    for (int v = 0; v < V; v++) z.set(v, f);
#pragma unroll
    for (int s = 0; s < L; s++)
      if (t + s >= len) r[s] = z;
  }
  __device__ __forceinline__ static P zero() {
    P z;
#pragma unroll
    for (int v = 0; v < V; v++) z.set(v, 0.f);
    return z;
  }
};

// Carries `s` through the maps of `count` segments from `from` on (step +1 or -1).  Each wave
// composes its share of them, eight loads in flight, and the W results meet in LDS.
template <int V, int W>
__device__ __forceinline__ void compose(const Args &p, int64_t b, int c, int lane, int wave, int from,
                                        int count, int step, float (&la)[W][64 * V],
                                        float (&le)[W][64 * V], float (&s)[V]) {
  const int per = (count + W - 1) / W;
  const int lo = wave * per, hi = lo + per < count ? lo + per : count;
  float a[V], e[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    a[v] = 1.f;
    e[v] = 0.f;
  }
#pragma unroll 8
  for (int j = lo; j < hi; j++) {
    const float *m = p.maps + (b * p.segs + from + step * j) * 2 * p.d + c;
#pragma unroll
    for (int v = 0; v < V; v++) {
      e[v] = fmaf(m[v], e[v], m[p.d + v]);
      a[v] *= m[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; v++) {
    la[wave][lane * V + v] = a[v];
    le[wave][lane * V + v] = e[v];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; w++)
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = fmaf(la[w][lane * V + v], s[v], le[w][lane * V + v]);
  __syncthreads();  // the images are free again
}

// ---------------------------------------------------------------- forward
// OUT: the whole pass; else only the segments' maps.
template <class N, int V, int W, int L, bool OUT>
__global__ __launch_bounds__(64 * W) void forward_kernel(Args p) {
  using S = Shape<N, V, W, L>;
  using P = typename S::P;
  __shared__ float maps[2][2][W][S::kLanes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x / p.slabs, b = p.b0 + row;
  const int slab = static_cast<int>(blockIdx.x - row * p.slabs);
  const int seg = blockIdx.y;
  const int c0 = slab * S::kLanes + lane * V;
  const bool in = c0 < p.d;
  const int c = in ? c0 : 0;
  const int64_t len = steps_of(p, b);
  const int64_t first = seg * p.seg_tiles;
  const int64_t last = first + p.seg_tiles < p.tiles ? first + p.seg_tiles : p.tiles;

  float ca[V], h0[V];  // the segment's map so far (not OUT) or the state (OUT)
#pragma unroll
  for (int v = 0; v < V; v++) {
    ca[v] = 1.f;
    h0[v] = OUT && p.state ? p.state[b * p.d + c + v] : 0.f;
  }
  if (OUT && p.segs > 1) compose<V, W>(p, b, c, lane, wave, 0, seg, 1, maps[0][0], maps[0][1], h0);

  P x[L], g[L], nx[L], ng[L];
  const int64_t mine = static_cast<int64_t>(wave) * L;
  if (first * S::kTile < len) {
    S::load(x, p.x, b * p.xb, p.xt, c, first * S::kTile + mine, len);
    S::load(g, p.g, b * p.gb, p.gt, c, first * S::kTile + mine, len);
  }
  for (int64_t tile = first; tile < last; tile++) {
    const int64_t t0 = tile * S::kTile + mine;
    if (tile * S::kTile >= len) {  // padding only (the same for the whole workgroup)
      if (OUT && in)
        for (int s = 0; s < L; s++)
          if (t0 + s < p.t) S::store(p.y, b * p.t + t0 + s, p.d, c, S::zero());
      continue;
    }
    if (tile + 1 < last && (tile + 1) * S::kTile < len) {
      S::load(nx, p.x, b * p.xb, p.xt, c, t0 + S::kTile, len);
      S::load(ng, p.g, b * p.gb, p.gt, c, t0 + S::kTile, len);
    }
    const bool full = t0 + L <= len;
    if (!full) {
      S::blank(x, t0, len, 0.f);
      S::blank(g, t0, len, __builtin_inff());
    }
    float i[L][V], a[V], e[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      a[v] = 1.f;
      e[v] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < L; s++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        i[s][v] = share(g[s][v]);
        e[v] = fmaf(i[s][v], x[s][v] - e[v], e[v]);
        a[v] = fmaf(-i[s][v], a[v], a[v]);
      }
    float (*m)[W][S::kLanes] = maps[tile & 1];
#pragma unroll
    for (int v = 0; v < V; v++) {
      m[0][wave][lane * V + v] = a[v];
      m[1][wave][lane * V + v] = e[v];
    }
    __syncthreads();
    float h[V];
    if (OUT && p.starts && wave == 0 && in)
#pragma unroll
      for (int v = 0; v < V; v++) p.starts[(b * p.tiles + tile) * p.d + c + v] = h0[v];
#pragma unroll
    for (int w = 0; w < W; w++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float ma = m[0][w][lane * V + v], me = m[1][w][lane * V + v];
        if (w == wave) h[v] = h0[v];
        h0[v] = fmaf(ma, h0[v], me);
        if (!OUT) ca[v] *= ma;
      }
    if (OUT) {
#pragma unroll
      for (int s = 0; s < L; s++) {
        P y;
#pragma unroll
        for (int v = 0; v < V; v++) {
          h[v] = fmaf(i[s][v], x[s][v] - h[v], h[v]);
          y.set(v, h[v]);
        }
        if (full ? in : in && t0 + s < p.t)
          S::store(p.y, b * p.t + t0 + s, p.d, c, full || t0 + s < len ? y : S::zero());
      }
    }
#pragma unroll
    for (int s = 0; s < L; s++) {
      x[s] = nx[s];
      g[s] = ng[s];
    }
  }
  if (wave != 0 || !in) return;
  if (OUT) {
    if (seg == p.segs - 1)
#pragma unroll
      for (int v = 0; v < V; v++) p.final[b * p.d + c + v] = h0[v];
  } else {
    float *m = p.maps + (b * p.segs + seg) * 2 * p.d + c;
#pragma unroll
    for (int v = 0; v < V; v++) {
      m[v] = ca[v];
      m[p.d + v] = h0[v];
    }
  }
}

// --------------------------------------------------------------- backward
template <class N, int V, int W, int L, bool OUT>
__global__ __launch_bounds__(64 * W) void backward_kernel(Args p) {
  using S = Shape<N, V, W, L>;
  using P = typename S::P;
  __shared__ float maps[2][3][W][S::kLanes];  // product; forward end from zero; backward end from zero
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x / p.slabs, b = p.b0 + row;
  const int slab = static_cast<int>(blockIdx.x - row * p.slabs);
  const int seg = blockIdx.y + (OUT ? 0 : 1);
  const int c0 = slab * S::kLanes + lane * V;
  const bool in = c0 < p.d;
  const int c = in ? c0 : 0;
  const int64_t len = steps_of(p, b);
  const int64_t first = seg * p.seg_tiles;
  const int64_t last = first + p.seg_tiles < p.tiles ? first + p.seg_tiles : p.tiles;

  float ca[V], m0[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    ca[v] = 1.f;
    m0[v] = OUT && p.dfinal ? p.dfinal[b * p.d + c + v] : 0.f;
  }
  if (OUT && p.segs > 1)
    compose<V, W>(p, b, c, lane, wave, p.segs - 1, p.segs - 1 - seg, -1, maps[0][0], maps[0][1], m0);

  P x[L], g[L], dy[L], nx[L], ng[L], ndy[L];
  float st[V], nst[V];
#pragma unroll
  for (int v = 0; v < V; v++) st[v] = nst[v] = 0.f;
  const int64_t mine = static_cast<int64_t>(wave) * L;
  const auto fetch = [&](int64_t tile, P (&fx)[L], P (&fg)[L], P (&fd)[L], float (&fs)[V]) {
    const int64_t t = tile * S::kTile + mine;
    if (OUT) {
      S::load(fx, p.x, b * p.xb, p.xt, c, t, len);
#pragma unroll
      for (int v = 0; v < V; v++) fs[v] = p.starts[(b * p.tiles + tile) * p.d + c + v];
    }
    S::load(fg, p.g, b * p.gb, p.gt, c, t, len);
    if (p.dy) S::load(fd, p.dy, b * p.yb, p.yt, c, t, len);
  };
  bool have = false;
  for (int64_t tile = last - 1; tile >= first; tile--) {
    const int64_t t0 = tile * S::kTile + mine;
    if (tile * S::kTile >= len) {
      if (OUT && in)
        for (int s = 0; s < L; s++)
          if (t0 + s < p.t) {
            S::store(p.dx, b * p.t + t0 + s, p.d, c, S::zero());
            S::store(p.dg, b * p.t + t0 + s, p.d, c, S::zero());
          }
      continue;
    }
    if (!have) {
      fetch(tile, x, g, dy, st);
      have = true;
    }
    if (tile > first) fetch(tile - 1, nx, ng, ndy, nst);
    const bool full = t0 + L <= len;
    if (!p.dy) S::blank(dy, 0, 0, 0.f);
    if (!full) {
      if (OUT) S::blank(x, t0, len, 0.f);
      S::blank(g, t0, len, __builtin_inff());
      S::blank(dy, t0, len, 0.f);
    }
    float i[L][V], a[V], e[V], q[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      a[v] = 1.f;
      e[v] = q[v] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < L; s++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        i[s][v] = share(g[s][v]);
        a[v] = fmaf(-i[s][v], a[v], a[v]);
        if (OUT) e[v] = fmaf(i[s][v], x[s][v] - e[v], e[v]);
      }
#pragma unroll
    for (int s = L - 1; s >= 0; s--)
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float l = q[v] + dy[s][v];
        q[v] = fmaf(-i[s][v], l, l);
      }
    float (*m)[W][S::kLanes] = maps[tile & 1];
#pragma unroll
    for (int v = 0; v < V; v++) {
      m[0][wave][lane * V + v] = a[v];
      m[1][wave][lane * V + v] = e[v];
      m[2][wave][lane * V + v] = q[v];
    }
    __syncthreads();
    float h[V], mm[V];
    if (OUT) {
#pragma unroll
      for (int w = 0; w < W; w++)
#pragma unroll
        for (int v = 0; v < V; v++) {
          if (w == wave) h[v] = st[v];
          st[v] = fmaf(m[0][w][lane * V + v], st[v], m[1][w][lane * V + v]);
        }
    }
#pragma unroll
    for (int w = W - 1; w >= 0; w--)
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float ma = m[0][w][lane * V + v];
        if (w == wave) mm[v] = m0[v];
        m0[v] = fmaf(ma, m0[v], m[2][w][lane * V + v]);
        if (!OUT) ca[v] *= ma;
      }
    if (OUT) {
      float before[L][V];  // h_{t-1} - x_t
#pragma unroll
      for (int s = 0; s < L; s++)
#pragma unroll
        for (int v = 0; v < V; v++) {
          before[s][v] = h[v] - x[s][v];
          h[v] = fmaf(-i[s][v], before[s][v], h[v]);
        }
#pragma unroll
      for (int s = L - 1; s >= 0; s--) {
        P ox, og;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const float l = mm[v] + dy[s][v];
          const float il = i[s][v] * l;
          mm[v] = l - il;
          ox.set(v, il);
          og.set(v, (1.f - i[s][v]) * il * before[s][v]);
        }
        if (full ? in : in && t0 + s < p.t) {
          const bool on = full || t0 + s < len;
          S::store(p.dx, b * p.t + t0 + s, p.d, c, on ? ox : S::zero());
          S::store(p.dg, b * p.t + t0 + s, p.d, c, on ? og : S::zero());
        }
      }
    }
#pragma unroll
    for (int s = 0; s < L; s++) {
      x[s] = nx[s];
      g[s] = ng[s];
      dy[s] = ndy[s];
    }
#pragma unroll
    for (int v = 0; v < V; v++) st[v] = nst[v];
  }
  if (wave != 0 || !in) return;
  if (OUT) {
    if (seg == 0 && p.dstate)
#pragma unroll
      for (int v = 0; v < V; v++) p.dstate[b * p.d + c + v] = m0[v];
  } else {
    float *m = p.maps + (b * p.segs + seg) * 2 * p.d + c;
#pragma unroll
    for (int v = 0; v < V; v++) {
      m[v] = ca[v];
      m[p.d + v] = m0[v];
    }
  }
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
    const float h = fmaf(share(N::load(g[b * gb + c])), N::load(x[b * xb + c]) - h0, h0);
    state[at] = h;
    y[at] = N::save(h);
  }
}

// ------------------------------------------------------------------- host
constexpr int kSteps = 16;  // steps of a wave in a tile

// Waves along time.  A short sequence would leave most of a tall tile empty.
int waves_of(int64_t t) { return t <= 2 * kSteps ? 1 : 8; }
int64_t tiles_of(int64_t t) {
  const int tile = kSteps * waves_of(t);
  return (t + tile - 1) / tile;
}

struct Plan {
  int lanes, slabs, segs;
  int64_t seg_tiles;
};

// Two 16-bit channels a lane where alignment allows it (a wave then reads 256 bytes of a step,
// as with one fp32 channel); time in segments until there are two workgroups for each CU.
Plan plan(int64_t batch, int64_t t, int d, bool pairs) {
  Plan q{};
  q.lanes = 64 * (pairs ? 2 : 1);
  q.slabs = (d + q.lanes - 1) / q.lanes;
  const int64_t tiles = tiles_of(t), groups = batch * q.slabs;
  const int64_t segs = std::max<int64_t>(1, std::min(tiles, 512 / groups));
  q.seg_tiles = (tiles + segs - 1) / segs;
  q.segs = q.seg_tiles ? static_cast<int>((tiles + q.seg_tiles - 1) / q.seg_tiles) : 1;
  return q;
}

template <class N, int V, int W>
void launch(bool back, const Args &p, int64_t groups, hipStream_t s) {
  const dim3 block(64 * W), all(static_cast<unsigned>(groups), static_cast<unsigned>(p.segs)),
      inner(static_cast<unsigned>(groups), static_cast<unsigned>(p.segs - 1));
  if (back) {
    if (p.segs > 1)
      hipLaunchKernelGGL((backward_kernel<N, V, W, kSteps, false>), inner, block, 0, s, p);
    hipLaunchKernelGGL((backward_kernel<N, V, W, kSteps, true>), all, block, 0, s, p);
  } else {
    if (p.segs > 1)
      hipLaunchKernelGGL((forward_kernel<N, V, W, kSteps, false>), inner, block, 0, s, p);
    hipLaunchKernelGGL((forward_kernel<N, V, W, kSteps, true>), all, block, 0, s, p);
  }
}

template <class N>
void launch_type(bool back, bool pairs, const Args &p, int64_t groups, hipStream_t s) {
  const bool tall = waves_of(p.t) > 1;
  if constexpr (sizeof(typename N::store) == 2) {
    if (pairs) {
      tall ? launch<N, 2, 8>(back, p, groups, s) : launch<N, 2, 1>(back, p, groups, s);
      return;
    }
  }
  tall ? launch<N, 1, 8>(back, p, groups, s) : launch<N, 1, 1>(back, p, groups, s);
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
  p.tiles = tiles_of(p.t);
  p.seg_tiles = q.seg_tiles;
  p.segs = q.segs;
  p.slabs = q.slabs;
  DeviceBuffer own;
  if (p.segs > 1) {
    const size_t need = static_cast<size_t>(batch) * p.segs * 2 * p.d * sizeof(float);
    if (workspace) {
      VS_REQUIRE(bytes >= need, "gated_recurrence: workspace of %zu bytes, %zu needed", bytes,
                 need);
      p.maps = static_cast<float *>(workspace);
    } else {
      VS_TRY(own.alloc(need, s));
      p.maps = own.as<float>();
    }
  }
  // a grid holds fewer than 2^32 threads
  const int64_t most = std::max<int64_t>(1, (1 << 22) / q.slabs);
  for (; p.b0 < batch; p.b0 += most) {
    const int64_t groups = std::min(most, batch - p.b0) * q.slabs;
    if (dtype == VS_F32) launch_type<num::F32>(back, pairs, p, groups, s);
    else if (dtype == VS_F16) launch_type<num::F16>(back, pairs, p, groups, s);
    else launch_type<num::BF16>(back, pairs, p, groups, s);
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
  size_t most = 0;
  for (const bool pairs : {false, true}) {
    const rec::Plan q = rec::plan(batch, t, static_cast<int>(d), pairs);
    if (q.segs > 1)
      most = std::max(most, static_cast<size_t>(batch) * q.segs * 2 * d * sizeof(float));
  }
  return most;
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
