// The step between two blocks of a residual network as one pass over its rows, and its backward pass as another:
//   n = norm(f) w2 + b2 (or f),   y = x + scale * sigmoid(gate) * n,   h = norm(y) w1 + b1
// with norm(v) = (v - mean v) / sqrt(var v + eps) (layer) or v / sqrt(mean v^2 + eps) (rms), each row by itself. gate: one per
// value, one per row, or none (1).
//
// Backward, with u2 = norm(f), u1 = norm(y), s = sigmoid(gate), r = the norms' factors, <.> a mean over the row:
//   G   = dy + r1 (dh w1 - <dh w1> - u1 <dh w1 u1>)          dx = G       (<dh w1> where the mean was taken off)
//   dn  = G scale s        dgate = G scale n s'(gate)         dscale = sum over rows of G s n
//   df  = r2 (dn w2 - <dn w2> - u2 <dn w2 u2>)                dw2 = sum dn u2, db2 = sum dn, dw1 = sum dh u1, db1 = sum dh
// y, the statistics and the normalised rows are computed again from x, f and gate: reading a row's statistics would save
// two of its reductions, reading y instead of x nothing.
//
// Both are bound by memory: a row is read once, held in registers (16 bytes of every matrix per lane; a part of a warp, a warp
// or up to 16 warps per row), and written once. A warp asks for its next row before it works on the one that it has: its
// chains of shuffles (up to nine sums of a row, one behind the other, for the layer norms' gradients) are longer than what
// the other warps of an SM cover. Parameters come out of L1 for every row; held in registers they cost a third of the warps.
// Statistics, products and sums are fp32 whatever the rows' type; y is rounded when it is stored, h is computed from it before.
// The sums over rows are kept per lane for the whole grid's pass, added up per block, and the blocks' sums are added in order
// by a second kernel: the same bits on every run.
#include "rows8.cuh"

namespace cxg {
namespace {

constexpr int kSums = 5;       // dscale, dw2, db2, dw1, db1
constexpr int kMostWarps = 16;
constexpr int kMostWidth = 4096;
constexpr int kBlock = 128;    // threads where a row takes a warp or less

struct ResArgs {
  cxg_residual_desc d;
  float inv_width;
  float *part;       // backward: [gridDim.x][kSums][width]
  int keep, groups;  // forward: rows in 8 bits of h
};

// Where a lane's values lie: Q vectors of N values, the lanes' first vectors side by side, then their second ones. Rows that are
// not whole 16-byte vectors are read value by value, as many per lane.
template <typename T, bool VEC, int VECTORS>
struct Place {
  static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  static constexpr int Q = VEC ? VECTORS : VECTORS * 16 / static_cast<int>(sizeof(T));
  static constexpr int V = N * Q;  // values
  using Element = T;
  static constexpr bool kVec = VEC;
};

// A lane's part of a row as it was loaded.
template <typename P>
struct Raw {
  using T = typename P::Element;
  typename Vec<T>::Raw v[P::kVec ? P::Q : 1];
  T e[P::kVec ? 1 : P::Q];
  __device__ __forceinline__ void load(const void *base, int64_t row, int width, int p, int lanes) {
    const T *src = static_cast<const T *>(base) + row * width;
#pragma unroll
    for (int q = 0; q < P::Q; ++q) {
      const int c = (q * lanes + p) * P::N;
      if constexpr (P::kVec) {
        v[q] = {};
        if (c < width) v[q] = Vec<T>::load(src + c);
      } else {
        e[q] = from_f32<T>(0.f);
        if (c < width) e[q] = __ldg(src + c);
      }
    }
  }
  __device__ __forceinline__ void get(float (&f)[P::V]) const {
#pragma unroll
    for (int q = 0; q < P::Q; ++q)
      if constexpr (P::kVec)
        Vec<T>::to_float(f + q * P::N, v[q]);
      else
        f[q] = to_f32(e[q]);
  }
};

template <typename P>
__device__ __forceinline__ void store_row(void *base, int64_t row, int width, int p, int lanes, const float (&v)[P::V]) {
  using T = typename P::Element;
  T *dst = static_cast<T *>(base) + row * width;
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
    if (c < width) {
      if constexpr (P::kVec)
        Vec<T>::store_stream(dst + c, Vec<T>::from_float(v + q * P::N));
      else
        dst[c] = from_f32<T>(v[q]);
    }
  }
}

// A parameter's values at the lane's columns (`other` where there is no parameter; anything behind the row).
template <typename P>
__device__ __forceinline__ void load_param(float (&v)[P::V], const float *w, float other, int width, int p, int lanes) {
#pragma unroll
  for (int i = 0; i < P::V; ++i) v[i] = other;
  if (w == nullptr) return;
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
    if (c >= width) continue;
    if constexpr (P::kVec) {
#pragma unroll
      for (int i = 0; i < P::N; i += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(w + c + i));
        v[q * P::N + i] = t.x, v[q * P::N + i + 1] = t.y, v[q * P::N + i + 2] = t.z, v[q * P::N + i + 3] = t.w;
      }
    } else {
      v[q] = __ldg(w + c);
    }
  }
}

// Sums over the lanes of a row; every lane gets them. Rows of several warps take turns between two places in shared memory, so
// that one barrier per sum is enough.
template <int LANES, int WARPS>
struct RowSum {
  float2 (*place)[WARPS];
  int turn = 0;
  __device__ explicit RowSum(float2 (*s)[WARPS]) : place(s) {}
  __device__ __forceinline__ float2 both(float a, float b) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, d);
      b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if constexpr (WARPS > 1) {
      if ((threadIdx.x & 31) == 0) place[turn][threadIdx.x >> 5] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 t = place[turn][w];
        a += t.x, b += t.y;
      }
      turn ^= 1;
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float one(float a) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
    if constexpr (WARPS > 1) {
      if ((threadIdx.x & 31) == 0) place[turn][threadIdx.x >> 5].x = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) a += place[turn][w].x;
      turn ^= 1;
    }
    return a;
  }
};

// v becomes norm(v); returns the factor. Values behind the row (zeros before) stay zeros.
template <typename P, typename Sum>
__device__ __forceinline__ float normalise(float (&v)[P::V], const ResArgs &a, Sum &sum, int p, int lanes) {
  if (a.d.layer) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < P::V; ++i) t += v[i];
    const float mean = sum.one(t) * a.inv_width;
#pragma unroll
    for (int q = 0; q < P::Q; ++q) {
      const float off = (q * lanes + p) * P::N < a.d.width ? mean : 0.f;
#pragma unroll
      for (int i = 0; i < P::N; ++i) v[q * P::N + i] -= off;
    }
  }
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < P::V; ++i) t = fmaf(v[i], v[i], t);
  const float r = __frsqrt_rn(fmaf(sum.one(t), a.inv_width, a.d.eps));
#pragma unroll
  for (int i = 0; i < P::V; ++i) v[i] *= r;
  return r;
}

// sigmoid and its derivative without cancellation: t = exp(-|g|), s = 1 / (1 + t) or t / (1 + t), s' = t / (1 + t)^2. The
// reciprocal of 1 .. 2 is the hardware's, off by an ulp.
__device__ __forceinline__ void sigmoid(float g, float *s, float *ds) {
  const float t = expf(-fabsf(g));
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + t));
  const float tq = t * q;
  *s = g >= 0.f ? q : tq;
  *ds = tq * q;
}

// Rows of the grid: `per` per block at a time; the lanes of a warp go through the loop together.
template <int LANES, int WARPS>
struct Rows {
  static constexpr int kPerBlock = WARPS > 1 ? 1 : kBlock / LANES;
  int64_t first, step;
  int sub;
  __device__ Rows() {
    const int slot = WARPS > 1 ? 0 : static_cast<int>(threadIdx.x) / 32 * (32 / LANES);
    first = blockIdx.x * static_cast<int64_t>(kPerBlock) + slot;
    step = gridDim.x * static_cast<int64_t>(kPerBlock);
    sub = WARPS > 1 ? 0 : (threadIdx.x & 31) / LANES;
  }
};

// h in 8 bits as it is stored, to row `row`; zeros where `in` is false.
template <typename P>
__device__ __forceinline__ void keep_row(const ResArgs &a, int64_t row, bool in, const float (&h)[P::V], int p, int lanes) {
  using T = typename P::Element;
  constexpr int kShare = rows8::kGroup / P::N;  // lanes that hold a group
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
    float v[P::N];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      v[i] = in && c < a.d.width ? to_f32(from_f32<T>(h[q * P::N + i])) : 0.f;
      top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int k = 1; k < kShare; k <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, k));
    const uint32_t e = rows8::scale_byte(top);
    uint32_t w[P::N / 4];
    rows8::codes_of<P::N>(w, v, e);
    if (row <= a.d.n && c < a.groups * rows8::kGroup) {
      uint8_t *out = static_cast<uint8_t *>(a.d.codes) + row * (static_cast<int64_t>(a.groups) * rows8::kGroup) + c;
      if constexpr (P::N == 4)
        *reinterpret_cast<uint32_t *>(out) = w[0];
      else
        *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[P::N / 4 - 1]);
      if (c % rows8::kGroup == 0)
        static_cast<uint8_t *>(a.d.scales)[row * a.groups + c / rows8::kGroup] = static_cast<uint8_t>(e);
    }
  }
}

// Warps per SM: 64 registers a thread forward, 128 backward, 168 where eight values per lane meet five sums of each (with 128
// registers these spill 250 bytes a lane).
constexpr int forward_warps(int values, bool gated) { return values > 4 && gated ? 24 : 32; }
constexpr int backward_warps(int values, bool biases) { return values > 4 && biases ? 12 : 16; }

// Blocks per SM of `threads` threads with that many warps.
constexpr int blocks_of(int warps, int threads) { return warps * 32 / threads > 0 ? warps * 32 / threads : 1; }

// GATED: a gate per value.
template <typename T, int LANES, int WARPS, bool VEC, int VECTORS, bool GATED>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock,
                                  blocks_of(forward_warps(Place<T, VEC, VECTORS>::V, GATED), WARPS > 1 ? 32 * WARPS : kBlock))
    residual_forward(const __grid_constant__ ResArgs a) {
  using P = Place<T, VEC, VECTORS>;
  constexpr int kLanes = LANES * WARPS;
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = threadIdx.x & (kLanes - 1), width = d.width;
  const bool with_f = d.f != nullptr, row_gate = d.gate_mode == CXG_GATE_ROW;
  dependency_wait();
  const Rows<LANES, WARPS> rows;
  Raw<P> rx, rf, rg;
  T rr = from_f32<T>(0.f);
  auto load = [&](int64_t row) {
    const int64_t at = row < d.n ? row : d.n - 1;
    rx.load(d.x, at, width, p, kLanes);
    if (with_f) rf.load(d.f, at, width, p, kLanes);
    if (GATED) rg.load(d.gate, at, width, p, kLanes);
    if (row_gate) rr = __ldg(static_cast<const T *>(d.gate) + at);
  };
  const int64_t n_end = d.n + a.keep;
  if (rows.first < n_end) load(rows.first + rows.sub);
  for (int64_t row0 = rows.first; row0 < n_end; row0 += rows.step) {
    const int64_t row = row0 + rows.sub;
    const bool in = row < d.n;
    float y[P::V], n[P::V], s[P::V], one = 1.f, ds;
    rx.get(y);
    if (with_f) rf.get(n);
    if (GATED) rg.get(s);
    const float g_row = to_f32(rr);
    if (row0 + rows.step < n_end) load(row + rows.step);
    if (with_f) {
      if (d.post) {
        normalise<P>(n, a, sum, p, kLanes);
        float w[P::V], b[P::V];
        load_param<P>(w, d.post_weight, 1.f, width, p, kLanes);
        if (d.post_bias != nullptr) {
          load_param<P>(b, d.post_bias, 0.f, width, p, kLanes);
#pragma unroll
          for (int i = 0; i < P::V; ++i) n[i] = fmaf(n[i], w[i], b[i]);
        } else {
#pragma unroll
          for (int i = 0; i < P::V; ++i) n[i] *= w[i];
        }
      }
      if (row_gate) sigmoid(g_row, &one, &ds);
      if (GATED) {
#pragma unroll
        for (int i = 0; i < P::V; ++i) sigmoid(s[i], &s[i], &ds);
      }
      float scale[P::V];
      load_param<P>(scale, d.scale, 1.f, width, p, kLanes);
#pragma unroll
      for (int i = 0; i < P::V; ++i) y[i] = fmaf(scale[i] * (GATED ? s[i] : one), n[i], y[i]);
      if (d.y != nullptr && in) store_row<P>(d.y, row, width, p, kLanes, y);
    }
    if (d.next) {
      normalise<P>(y, a, sum, p, kLanes);
      float w[P::V], b[P::V];
      load_param<P>(w, d.next_weight, 1.f, width, p, kLanes);
      load_param<P>(b, d.next_bias, 0.f, width, p, kLanes);
#pragma unroll
      for (int i = 0; i < P::V; ++i) y[i] = fmaf(y[i], w[i], b[i]);
      if (in) store_row<P>(d.h, row, width, p, kLanes, y);
      if constexpr (VEC) {
        if (a.keep) keep_row<P>(a, row, in, y, p, kLanes);
      }
    }
  }
}

// g becomes r (g - <g> - u <g u>) (without <g> where no mean was taken off)
template <int V, typename Sum>
__device__ __forceinline__ void back_through_norm(float (&g)[V], const float (&u)[V], float r, const ResArgs &a, Sum &sum) {
  float t0 = 0.f, t1 = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) t0 += g[i], t1 = fmaf(g[i], u[i], t1);
  float mean = 0.f, dot;
  if (a.d.layer) {
    const float2 t = sum.both(t0, t1);
    mean = t.x * a.inv_width, dot = t.y * a.inv_width;
  } else {
    dot = sum.one(t1) * a.inv_width;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) g[i] = r * (fmaf(-u[i], dot, g[i]) - mean);
}

// BIASES: sums for them too.
template <typename T, int LANES, int WARPS, bool VEC, int VECTORS, bool GATED, bool BIASES>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock,
                                  blocks_of(backward_warps(Place<T, VEC, VECTORS>::V, BIASES), WARPS > 1 ? 32 * WARPS : kBlock))
    residual_backward(const __grid_constant__ ResArgs a) {
  using P = Place<T, VEC, VECTORS>;
  constexpr int kLanes = LANES * WARPS;
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = threadIdx.x & (kLanes - 1), width = d.width;
  const bool with_f = d.f != nullptr, row_gate = d.gate_mode == CXG_GATE_ROW, next = d.next && d.dh != nullptr;
  dependency_wait();
  float acc[kSums][P::V];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < P::V; ++i) acc[k][i] = 0.f;
  const Rows<LANES, WARPS> rows;
  Raw<P> rx, rf, rg, ry, rh;
  T rr = from_f32<T>(0.f);
  auto load = [&](int64_t row) {
    const int64_t at = row < d.n ? row : d.n - 1;
    rx.load(d.x, at, width, p, kLanes);
    if (with_f) rf.load(d.f, at, width, p, kLanes);
    if (GATED) rg.load(d.gate, at, width, p, kLanes);
    if (row_gate) rr = __ldg(static_cast<const T *>(d.gate) + at);
    if (d.dy != nullptr) ry.load(d.dy, at, width, p, kLanes);
    if (next) rh.load(d.dh, at, width, p, kLanes);
  };
  if (rows.first < d.n) load(rows.first + rows.sub);
  for (int64_t row0 = rows.first; row0 < d.n; row0 += rows.step) {
    const int64_t row = row0 + rows.sub;
    const bool in = row < d.n;  // lanes without a row go through it with gradients of zero
    float y[P::V], n[P::V], s[GATED ? P::V : 1], ds[GATED ? P::V : 1], g[P::V], dh[P::V];
    rx.get(y);
    if (with_f) rf.get(n);
    if constexpr (GATED) rg.get(s);
    const float g_row = to_f32(rr);
#pragma unroll
    for (int i = 0; i < P::V; ++i) g[i] = dh[i] = 0.f;
    if (in && d.dy != nullptr) ry.get(g);
    if (in && next) rh.get(dh);
    if (row0 + rows.step < d.n) load(row + rows.step);
    float r2 = 0.f, scale[P::V];
    if constexpr (!GATED) {
      s[0] = 1.f, ds[0] = 0.f;
      if (row_gate) sigmoid(g_row, &s[0], &ds[0]);
    }
    if (with_f) {
      load_param<P>(scale, d.scale, 1.f, width, p, kLanes);
      if constexpr (GATED) {
#pragma unroll
        for (int i = 0; i < P::V; ++i) sigmoid(s[i], &s[i], &ds[i]);
      }
      if (d.post) {
        r2 = normalise<P>(n, a, sum, p, kLanes);  // n is u2 from here on
        float w2[P::V], b2[P::V];
        load_param<P>(w2, d.post_weight, 1.f, width, p, kLanes);
        load_param<P>(b2, d.post_bias, 0.f, width, p, kLanes);
#pragma unroll
        for (int i = 0; i < P::V; ++i) y[i] = fmaf(scale[i] * s[GATED ? i : 0], fmaf(n[i], w2[i], b2[i]), y[i]);
      } else {
#pragma unroll
        for (int i = 0; i < P::V; ++i) y[i] = fmaf(scale[i] * s[GATED ? i : 0], n[i], y[i]);
      }
    }
    if (next) {
      const float r1 = normalise<P>(y, a, sum, p, kLanes);  // y is u1 from here on
      float t[P::V];
      load_param<P>(t, d.next_weight, 1.f, width, p, kLanes);
#pragma unroll
      for (int i = 0; i < P::V; ++i) {
        acc[3][i] = fmaf(dh[i], y[i], acc[3][i]);
        if (BIASES) acc[4][i] += dh[i];
        t[i] *= dh[i];
      }
      back_through_norm(t, y, r1, a, sum);
#pragma unroll
      for (int i = 0; i < P::V; ++i) g[i] += t[i];
#pragma unroll
      for (int i = 0; i < P::V; ++i)
        if (((i / P::N) * kLanes + p) * P::N >= width) g[i] = 0.f;
    }
    if (in && d.dx != nullptr) store_row<P>(d.dx, row, width, p, kLanes, g);
    if (with_f) {
      float w2[P::V], dg[P::V];
#pragma unroll
      for (int i = 0; i < P::V; ++i) dg[i] = n[i];
      if (d.post) {
        float b2[P::V];
        load_param<P>(w2, d.post_weight, 1.f, width, p, kLanes);
        load_param<P>(b2, d.post_bias, 0.f, width, p, kLanes);
#pragma unroll
        for (int i = 0; i < P::V; ++i) dg[i] = fmaf(n[i], w2[i], b2[i]);
      }
      load_param<P>(scale, d.scale, 1.f, width, p, kLanes);
#pragma unroll
      for (int i = 0; i < P::V; ++i) {
        acc[0][i] = fmaf(g[i] * s[GATED ? i : 0], dg[i], acc[0][i]);
        g[i] *= scale[i];
        dg[i] *= g[i] * ds[GATED ? i : 0];
        g[i] *= s[GATED ? i : 0];  // dn
      }
      if constexpr (GATED) {
        if (in && d.dgate != nullptr) store_row<P>(d.dgate, row, width, p, kLanes, dg);
      } else if (row_gate) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < P::V; ++i) t += dg[i];
        t = sum.one(t);
        if (in && p == 0 && d.dgate != nullptr) static_cast<T *>(d.dgate)[row] = from_f32<T>(t);
      }
      if (d.post) {
#pragma unroll
        for (int i = 0; i < P::V; ++i) {
          acc[1][i] = fmaf(g[i], n[i], acc[1][i]);
          if (BIASES) acc[2][i] += g[i];
          g[i] *= w2[i];
        }
        back_through_norm(g, n, r2, a, sum);
      }
      if (in && d.df != nullptr) store_row<P>(d.df, row, width, p, kLanes, g);
    }
  }
  // the block's sums: lanes of a warp that hold the same columns, then the warps in order
  float *part = a.part + static_cast<int64_t>(blockIdx.x) * kSums * width;
  if constexpr (WARPS == 1) {
    __shared__ float side[kBlock / 32][LANES * P::V];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (!BIASES && (k == 2 || k == 4)) {
        for (int c = threadIdx.x; c < width; c += kBlock) part[k * width + c] = 0.f;
        continue;
      }
#pragma unroll
      for (int i = 0; i < P::V; ++i)
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) acc[k][i] += __shfl_xor_sync(0xffffffffu, acc[k][i], o);
      if ((threadIdx.x & 31) < LANES) {
#pragma unroll
        for (int i = 0; i < P::V; ++i) side[warp][((i / P::N) * kLanes + p) * P::N + i % P::N] = acc[k][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < width; c += kBlock) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kBlock / 32; ++w) t += side[w][c];
        part[k * width + c] = t;
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int i = 0; i < P::V; ++i) {
        const int c = ((i / P::N) * kLanes + p) * P::N + i % P::N;
        if (c < width) part[k * width + c] = acc[k][i];
      }
  }
}

// Lanes of a row: the smallest power of two, from 8 on, that holds it (16 bytes a lane; 32 where 16 warps are not enough).
int values_of(int dtype) { return dtype == CXG_F32 ? 4 : 8; }
int lanes_of(int width, int dtype) {
  int lanes = 8;
  while (lanes < 32 * kMostWarps && lanes * values_of(dtype) < width) lanes *= 2;
  return lanes;
}
int rows_per_block(int lanes) { return lanes > 32 ? 1 : kBlock / lanes; }
int backward_blocks(int64_t n, int lanes) {
  const int64_t most = kNumSM * blocks_of(16, lanes > 32 ? lanes : kBlock);
  const int64_t want = (n + rows_per_block(lanes) - 1) / rows_per_block(lanes);
  return static_cast<int>(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, bool VEC, bool GATED, typename Go>
cudaError_t by_width(int width, int dtype, Go go) {
  switch (lanes_of(width, dtype)) {
    case 8: return go.template run<T, 8, 1, VEC, 1, GATED>();
    case 16: return go.template run<T, 16, 1, VEC, 1, GATED>();
    case 32: return go.template run<T, 32, 1, VEC, 1, GATED>();
    case 64: return go.template run<T, 32, 2, VEC, 1, GATED>();
    case 128: return go.template run<T, 32, 4, VEC, 1, GATED>();
    case 256: return go.template run<T, 32, 8, VEC, 1, GATED>();
    default: break;
  }
  if constexpr (sizeof(T) == 4)
    if (width > 32 * kMostWarps * 4) return go.template run<T, 32, kMostWarps, VEC, 2, GATED>();
  return go.template run<T, 32, kMostWarps, VEC, 1, GATED>();
}
template <typename T, typename Go>
cudaError_t by_kind(const cxg_residual_desc &d, bool vec, Go go) {
  const bool gated = d.gate_mode == CXG_GATE_VALUE;
  if (vec) return gated ? by_width<T, true, true>(d.width, d.dtype, go) : by_width<T, true, false>(d.width, d.dtype, go);
  return gated ? by_width<T, false, true>(d.width, d.dtype, go) : by_width<T, false, false>(d.width, d.dtype, go);
}
template <typename Go>
cudaError_t by_type(const cxg_residual_desc &d, bool vec, Go go) {
  return d.dtype == CXG_F32 ? by_kind<float>(d, vec, go) : by_kind<__nv_bfloat16>(d, vec, go);
}

struct Forward {
  const ResArgs &a;
  cudaStream_t st;
  template <typename T, int LANES, int WARPS, bool VEC, int VECTORS, bool GATED>
  cudaError_t run() const {
    const int per = rows_per_block(LANES * WARPS);
    constexpr int kThreads = WARPS > 1 ? 32 * WARPS : kBlock;
    const int64_t want = (a.d.n + a.keep + per - 1) / per, most = kNumSM * blocks_of(forward_warps(Place<T, VEC, VECTORS>::V, GATED), kThreads);
    return launch_dependent(residual_forward<T, LANES, WARPS, VEC, VECTORS, GATED>, static_cast<unsigned>(want < most ? want : most),
                            kThreads, 0, st, a);
  }
};
struct Backward {
  const ResArgs &a;
  cudaStream_t st;
  int *blocks;
  template <typename T, int LANES, int WARPS, bool VEC, int VECTORS, bool GATED, bool BIASES>
  cudaError_t go() const {
    constexpr int kThreads = WARPS > 1 ? 32 * WARPS : kBlock;
    const int most = kNumSM * blocks_of(backward_warps(Place<T, VEC, VECTORS>::V, BIASES), kThreads);
    if (*blocks > most) *blocks = most;
    return launch_dependent(residual_backward<T, LANES, WARPS, VEC, VECTORS, GATED, BIASES>, static_cast<unsigned>(*blocks), kThreads, 0,
                            st, a);
  }
  template <typename T, int LANES, int WARPS, bool VEC, int VECTORS, bool GATED>
  cudaError_t run() const {
    return a.d.post_bias != nullptr || a.d.next_bias != nullptr ? go<T, LANES, WARPS, VEC, VECTORS, GATED, true>()
                                                                : go<T, LANES, WARPS, VEC, VECTORS, GATED, false>();
  }
};

// Rows of whole 16-byte vectors: all matrices, and the parameters, which are fp32.
bool whole_vectors(const cxg_residual_desc &d) {
  uint64_t bits = static_cast<uint64_t>(d.width) * (d.dtype == CXG_F32 ? 4 : 2);
  const void *rows[] = {d.x, d.f, d.y, d.h, d.dy, d.dh, d.dx, d.df, d.scale, d.post_weight, d.post_bias, d.next_weight, d.next_bias};
  for (const void *p : rows) bits |= reinterpret_cast<uintptr_t>(p);
  if (d.gate_mode == CXG_GATE_VALUE) bits |= reinterpret_cast<uintptr_t>(d.gate) | reinterpret_cast<uintptr_t>(d.dgate);
  return bits % 16 == 0;
}

int check_desc(const cxg_residual_desc *d, const char *who) {
  CXG_REQUIRE(d != nullptr, CXG_ENULL, "%s: desc is NULL", who);
  CXG_REQUIRE(d->n >= 0 && d->width > 0 && (d->dtype == CXG_F32 || d->dtype == CXG_BF16), CXG_EINVAL, "%s: bad sizes or type", who);
  CXG_REQUIRE(d->width <= kMostWidth, CXG_EUNSUPPORTED, "%s: rows of %d values, at most %d", who, d->width, kMostWidth);
  CXG_REQUIRE(d->gate_mode == CXG_GATE_NONE || d->gate_mode == CXG_GATE_VALUE || d->gate_mode == CXG_GATE_ROW, CXG_EINVAL,
              "%s: gate_mode %d", who, d->gate_mode);
  CXG_REQUIRE(d->eps >= 0.f, CXG_EINVAL, "%s: eps %g", who, static_cast<double>(d->eps));
  CXG_REQUIRE(d->f != nullptr || (d->gate_mode == CXG_GATE_NONE && !d->post && d->next) || d->n == 0, CXG_EINVAL,
              "%s: without f there is the second norm alone", who);
  CXG_REQUIRE(d->n == 0 || (d->x != nullptr && (d->gate_mode == CXG_GATE_NONE || d->gate != nullptr)), CXG_ENULL, "%s: NULL argument", who);
  return CXG_OK;
}

}  // namespace
}  // namespace cxg

using namespace cxg;

extern "C" int cxg_residual_norm_max_width(void) { return kMostWidth; }

extern "C" int cxg_residual_norm_keeps(const cxg_residual_desc *d) { return d != nullptr && whole_vectors(*d) ? 1 : 0; }

extern "C" int cxg_residual_norm_forward(const cxg_residual_desc *d, void *stream) {
  const int rc = check_desc(d, "cxg_residual_norm_forward");
  if (rc != CXG_OK) return rc;
  const bool keep = d->codes != nullptr;
  CXG_REQUIRE(d->n == 0 || !d->next || d->h != nullptr, CXG_ENULL, "cxg_residual_norm_forward: h is NULL");
  CXG_REQUIRE(!keep || (d->next && d->scales != nullptr && whole_vectors(*d) && reinterpret_cast<uintptr_t>(d->codes) % 16 == 0),
              CXG_EINVAL, "cxg_residual_norm_forward: rows in 8 bits are kept of h, in whole 16-byte vectors");
  if (d->n == 0 && !keep) return CXG_OK;
  CXG_REQUIRE(d->n > 0, CXG_EINVAL, "cxg_residual_norm_forward: no rows to keep");
  ResArgs a = {};
  a.d = *d;
  a.inv_width = 1.f / static_cast<float>(d->width);
  a.keep = keep ? 1 : 0;
  a.groups = rows8::groups_of(d->width);
  const cudaError_t e = by_type(*d, whole_vectors(*d), Forward{a, as_stream(stream)});
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_residual_norm_forward: %s", cudaGetErrorString(e));
  count_launches(1);
  return check_launch("cxg_residual_norm_forward");
}

extern "C" int cxg_residual_norm_backward_workspace_size(int64_t n, int width, int dtype, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_residual_norm_backward_workspace_size: bytes is NULL");
  CXG_REQUIRE(n >= 0 && width > 0 && (dtype == CXG_F32 || dtype == CXG_BF16), CXG_EINVAL,
              "cxg_residual_norm_backward_workspace_size: bad sizes or type");
  CXG_REQUIRE(width <= kMostWidth, CXG_EUNSUPPORTED, "cxg_residual_norm: rows of %d values, at most %d", width, kMostWidth);
  *bytes = static_cast<size_t>(backward_blocks(n, lanes_of(width, dtype))) * kSums * width * sizeof(float);
  return CXG_OK;
}

extern "C" int cxg_residual_norm_backward(const cxg_residual_desc *d, float *sums, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = check_desc(d, "cxg_residual_norm_backward");
  if (rc != CXG_OK) return rc;
  CXG_REQUIRE(sums != nullptr, CXG_ENULL, "cxg_residual_norm_backward: sums is NULL");
  cudaStream_t st = as_stream(stream);
  if (d->n == 0) {
    if (cudaMemsetAsync(sums, 0, sizeof(float) * kSums * d->width, st) != cudaSuccess)
      return check_launch("cxg_residual_norm_backward: memset");
    return CXG_OK;
  }
  size_t need = 0;
  cxg_residual_norm_backward_workspace_size(d->n, d->width, d->dtype, &need);
  CXG_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, CXG_EWORKSPACE,
              "cxg_residual_norm_backward: workspace %zu bytes, need %zu", workspace_bytes, need);
  ResArgs a = {};
  a.d = *d;
  a.inv_width = 1.f / static_cast<float>(d->width);
  a.part = static_cast<float *>(workspace);
  int blocks = backward_blocks(d->n, lanes_of(d->width, d->dtype));
  const cudaError_t e = by_type(*d, whole_vectors(*d), Backward{a, st, &blocks});
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_residual_norm_backward: %s", cudaGetErrorString(e));
  column_sum_join(a.part, sums, blocks, kSums * d->width, st);
  count_launches(2);
  return check_launch("cxg_residual_norm_backward");
}
