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
// Both are bound by memory: a row is read once, held in registers (8 values per lane; a part of a warp, a warp or up to
// 16 warps per row), and written once. Statistics, products and sums are fp32 whatever the rows' type; y is rounded when it is
// stored, h is computed from it before. The sums over rows are kept per lane for the whole grid's pass, added up per block,
// and the blocks' sums are added in order by a second kernel: the same bits on every run.
#include "rows8.cuh"

namespace cxg {
namespace {

constexpr int kValues = 8;     // of a row per lane
constexpr int kSums = 5;       // dscale, dw2, db2, dw1, db1
constexpr int kMostWarps = 16;
constexpr int kMostWidth = kMostWarps * 32 * kValues;
constexpr int kBlock = 256;    // threads where a row takes a warp or less

struct ResArgs {
  cxg_residual_desc d;
  float inv_width;
  float *part;       // backward: [gridDim.x][kSums][width]
  int keep, groups;  // forward: rows in 8 bits of h
};

// Where a lane's values lie: vectors of N values, the lanes' first vectors side by side, then their second ones.
template <typename T, bool VEC>
struct Place {
  static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  static constexpr int Q = kValues / N;
};

template <typename T, bool VEC>
__device__ __forceinline__ void load_row(float (&v)[kValues], const void *base, int64_t row, int width, int p, int lanes) {
  using P = Place<T, VEC>;
  const T *src = static_cast<const T *>(base) + row * width;
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
    if constexpr (VEC) {
      if (c < width) Vec<T>::to_float(v + q * P::N, Vec<T>::load(src + c));
      else
#pragma unroll
        for (int i = 0; i < P::N; ++i) v[q * P::N + i] = 0.f;
    } else {
      v[q] = c < width ? to_f32(__ldg(src + c)) : 0.f;
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row(void *base, int64_t row, int width, int p, int lanes, const float (&v)[kValues]) {
  using P = Place<T, VEC>;
  T *dst = static_cast<T *>(base) + row * width;
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
    if (c < width) {
      if constexpr (VEC)
        Vec<T>::store_stream(dst + c, Vec<T>::from_float(v + q * P::N));
      else
        dst[c] = from_f32<T>(v[q]);
    }
  }
}

// A parameter's values at the lane's columns (`other` where there is no parameter, zeros behind the row).
template <typename T, bool VEC>
__device__ __forceinline__ void load_param(float (&v)[kValues], const float *w, float other, int width, int p, int lanes) {
  using P = Place<T, VEC>;
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = (q * lanes + p) * P::N;
#pragma unroll
    for (int i = 0; i < P::N; i += VEC ? 4 : 1) {
      if (w == nullptr || c + i >= width) {
#pragma unroll
        for (int k = 0; k < (VEC ? 4 : 1); ++k) v[q * P::N + i + k] = c + i < width ? other : 0.f;
      } else if constexpr (VEC) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(w + c + i));
        v[q * P::N + i] = t.x, v[q * P::N + i + 1] = t.y, v[q * P::N + i + 2] = t.z, v[q * P::N + i + 3] = t.w;
      } else {
        v[q] = __ldg(w + c);
      }
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

// v becomes norm(v); returns the factor. Values behind the row (column >= width) become zeros.
template <typename T, bool VEC, typename Sum>
__device__ __forceinline__ float normalise(float (&v)[kValues], const ResArgs &a, Sum &sum, int p, int lanes) {
  using P = Place<T, VEC>;
  if (a.d.layer) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kValues; ++i) t += v[i];
    const float mean = sum.one(t) * a.inv_width;
#pragma unroll
    for (int i = 0; i < kValues; ++i) v[i] = ((i / P::N) * lanes + p) * P::N + i % P::N < a.d.width ? v[i] - mean : 0.f;
  }
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kValues; ++i) t = fmaf(v[i], v[i], t);
  const float r = __frsqrt_rn(fmaf(sum.one(t), a.inv_width, a.d.eps));
#pragma unroll
  for (int i = 0; i < kValues; ++i) v[i] *= r;
  return r;
}

// sigmoid and its derivative without cancellation: t = exp(-|g|), s = 1 / (1 + t) or t / (1 + t), s' = t / (1 + t)^2
__device__ __forceinline__ void sigmoid(float g, float *s, float *ds) {
  const float t = expf(-fabsf(g)), q = __frcp_rn(1.f + t);
  *s = g >= 0.f ? q : t * q;
  *ds = t * q * q;
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

template <typename T, int LANES, int WARPS, bool VEC>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock) residual_forward(const __grid_constant__ ResArgs a) {
  using P = Place<T, VEC>;
  constexpr int kLanes = LANES * WARPS;
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = threadIdx.x & (kLanes - 1), width = d.width;
  dependency_wait();
  float scale[kValues], w2[kValues], b2[kValues], w1[kValues], b1[kValues];
  load_param<T, VEC>(scale, d.scale, 1.f, width, p, kLanes);
  load_param<T, VEC>(w2, d.post_weight, 1.f, width, p, kLanes);
  load_param<T, VEC>(b2, d.post_bias, 0.f, width, p, kLanes);
  load_param<T, VEC>(w1, d.next_weight, 1.f, width, p, kLanes);
  load_param<T, VEC>(b1, d.next_bias, 0.f, width, p, kLanes);
  const Rows<LANES, WARPS> rows;
  for (int64_t row0 = rows.first; row0 < d.n + a.keep; row0 += rows.step) {
    const int64_t row = row0 + rows.sub, at = row < d.n ? row : 0;
    const bool in = row < d.n;
    float y[kValues];
    if (in || WARPS == 1)
      load_row<T, VEC>(y, d.x, at, width, p, kLanes);
    else
#pragma unroll
      for (int i = 0; i < kValues; ++i) y[i] = 0.f;
    if (d.f != nullptr) {
      float n[kValues], g[kValues];
      float g_row = 0.f;
      if (in || WARPS == 1) {
        load_row<T, VEC>(n, d.f, at, width, p, kLanes);
        if (d.gate_mode == CXG_GATE_VALUE) load_row<T, VEC>(g, d.gate, at, width, p, kLanes);
        if (d.gate_mode == CXG_GATE_ROW) g_row = to_f32(__ldg(static_cast<const T *>(d.gate) + at));
      } else {
#pragma unroll
        for (int i = 0; i < kValues; ++i) n[i] = 0.f, g[i] = 0.f;
      }
      if (d.post) {
        normalise<T, VEC>(n, a, sum, p, kLanes);
#pragma unroll
        for (int i = 0; i < kValues; ++i) n[i] = fmaf(n[i], w2[i], b2[i]);
      }
      float s = 1.f, ds;
      if (d.gate_mode == CXG_GATE_ROW) sigmoid(g_row, &s, &ds);
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
        if (d.gate_mode == CXG_GATE_VALUE) sigmoid(g[i], &s, &ds);
        y[i] = fmaf(scale[i] * s, n[i], y[i]);
      }
      if (d.y != nullptr && in) store_row<T, VEC>(d.y, row, width, p, kLanes, y);
    }
    if (d.next) {
      normalise<T, VEC>(y, a, sum, p, kLanes);
#pragma unroll
      for (int i = 0; i < kValues; ++i) y[i] = fmaf(y[i], w1[i], b1[i]);
      if (in) store_row<T, VEC>(d.h, row, width, p, kLanes, y);
      if constexpr (VEC) {
        if (a.keep) {  // the rows in 8 bits of h as it is stored, and the row of zeros behind them
          constexpr int kShare = rows8::kGroup / P::N;  // lanes that hold a group
#pragma unroll
          for (int q = 0; q < P::Q; ++q) {
            const int c = (q * kLanes + p) * P::N;
            float v[P::N];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < P::N; ++i) {
              v[i] = in ? to_f32(from_f32<T>(y[q * P::N + i])) : 0.f;
              top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            }
#pragma unroll
            for (int k = 1; k < kShare; k <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, k));
            const uint32_t e = rows8::scale_byte(top);
            const float inv = e == rows8::kNotFinite ? 0.f : rows8::inverse_scale(e);
            uint32_t w[P::N / 4];
#pragma unroll
            for (int i = 0; i < P::N / 4; ++i)
              w[i] = e == rows8::kNotFinite
                         ? 0u
                         : rows8::pack_codes(rows8::code_bits(v[4 * i], inv), rows8::code_bits(v[4 * i + 1], inv),
                                             rows8::code_bits(v[4 * i + 2], inv), rows8::code_bits(v[4 * i + 3], inv));
            if (row <= d.n && c < a.groups * rows8::kGroup) {
              uint8_t *out = static_cast<uint8_t *>(d.codes) + row * (static_cast<int64_t>(a.groups) * rows8::kGroup) + c;
              if constexpr (P::N == 4)
                *reinterpret_cast<uint32_t *>(out) = w[0];
              else
                *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[P::N / 4 - 1]);
              if (c % rows8::kGroup == 0)
                static_cast<uint8_t *>(d.scales)[row * a.groups + c / rows8::kGroup] = static_cast<uint8_t>(e);
            }
          }
        }
      }
    }
  }
}

// g becomes r (g - <g> - u <g u>) (without <g> where no mean was taken off)
template <typename Sum>
__device__ __forceinline__ void back_through_norm(float (&g)[kValues], const float (&u)[kValues], float r, const ResArgs &a, Sum &sum) {
  float t0 = 0.f, t1 = 0.f;
#pragma unroll
  for (int i = 0; i < kValues; ++i) t0 += g[i], t1 = fmaf(g[i], u[i], t1);
  float mean = 0.f, dot;
  if (a.d.layer) {
    const float2 t = sum.both(t0, t1);
    mean = t.x * a.inv_width, dot = t.y * a.inv_width;
  } else {
    dot = sum.one(t1) * a.inv_width;
  }
#pragma unroll
  for (int i = 0; i < kValues; ++i) g[i] = r * (fmaf(-u[i], dot, g[i]) - mean);
}

template <typename T, int LANES, int WARPS, bool VEC>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock, WARPS > 1 ? kMostWarps / WARPS : 2)
    residual_backward(const __grid_constant__ ResArgs a) {
  using P = Place<T, VEC>;
  constexpr int kLanes = LANES * WARPS;
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = threadIdx.x & (kLanes - 1), width = d.width;
  dependency_wait();
  float acc[kSums][kValues];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < kValues; ++i) acc[k][i] = 0.f;
  const Rows<LANES, WARPS> rows;
  for (int64_t row0 = rows.first; row0 < d.n; row0 += rows.step) {
    const int64_t row = row0 + rows.sub, at = row < d.n ? row : 0;
    const bool in = row < d.n;
    float y[kValues], n[kValues], s[kValues], ds[kValues], g[kValues], dh[kValues];
    load_row<T, VEC>(y, d.x, at, width, p, kLanes);
    if (d.f != nullptr) load_row<T, VEC>(n, d.f, at, width, p, kLanes);
    if (d.gate_mode == CXG_GATE_VALUE) load_row<T, VEC>(s, d.gate, at, width, p, kLanes);
    if (d.gate_mode == CXG_GATE_ROW) s[0] = to_f32(__ldg(static_cast<const T *>(d.gate) + at));
    if (d.dy != nullptr)
      load_row<T, VEC>(g, d.dy, at, width, p, kLanes);
    else
#pragma unroll
      for (int i = 0; i < kValues; ++i) g[i] = 0.f;
    const bool next = d.next && d.dh != nullptr;
    if (next) load_row<T, VEC>(dh, d.dh, at, width, p, kLanes);
    if (!in) {  // lanes without a row go through it with gradients of zero
#pragma unroll
      for (int i = 0; i < kValues; ++i) g[i] = dh[i] = 0.f;
    }
    float r2 = 0.f, scale[kValues];
    if (d.f != nullptr) {
      load_param<T, VEC>(scale, d.scale, 1.f, width, p, kLanes);
      if (d.gate_mode == CXG_GATE_ROW) {
        float s0, ds0;
        sigmoid(s[0], &s0, &ds0);
#pragma unroll
        for (int i = 0; i < kValues; ++i) s[i] = s0, ds[i] = ds0;
      } else if (d.gate_mode == CXG_GATE_VALUE) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) sigmoid(s[i], &s[i], &ds[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kValues; ++i) s[i] = 1.f, ds[i] = 0.f;
      }
      if (d.post) {
        r2 = normalise<T, VEC>(n, a, sum, p, kLanes);  // n is u2 from here on
        float w2[kValues], b2[kValues];
        load_param<T, VEC>(w2, d.post_weight, 1.f, width, p, kLanes);
        load_param<T, VEC>(b2, d.post_bias, 0.f, width, p, kLanes);
#pragma unroll
        for (int i = 0; i < kValues; ++i) y[i] = fmaf(scale[i] * s[i], fmaf(n[i], w2[i], b2[i]), y[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kValues; ++i) y[i] = fmaf(scale[i] * s[i], n[i], y[i]);
      }
    }
    if (next) {
      const float r1 = normalise<T, VEC>(y, a, sum, p, kLanes);  // y is u1 from here on
      float t[kValues];
      load_param<T, VEC>(t, d.next_weight, 1.f, width, p, kLanes);
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
        acc[3][i] = fmaf(dh[i], y[i], acc[3][i]);
        acc[4][i] += dh[i];
        t[i] *= dh[i];
      }
      back_through_norm(t, y, r1, a, sum);
#pragma unroll
      for (int i = 0; i < kValues; ++i) g[i] += t[i];
    }
    if (in && d.dx != nullptr) store_row<T, VEC>(d.dx, row, width, p, kLanes, g);
    if (d.f != nullptr) {
      float w2[kValues], b2[kValues], dg[kValues];
      if (d.post) {
        load_param<T, VEC>(w2, d.post_weight, 1.f, width, p, kLanes);
        load_param<T, VEC>(b2, d.post_bias, 0.f, width, p, kLanes);
      }
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
        const float v = d.post ? fmaf(n[i], w2[i], b2[i]) : n[i];
        acc[0][i] = fmaf(g[i] * s[i], v, acc[0][i]);
        g[i] *= scale[i];
        dg[i] = g[i] * v * ds[i];
        g[i] *= s[i];  // dn
      }
      if (d.gate_mode == CXG_GATE_VALUE) {
        if (in && d.dgate != nullptr) store_row<T, VEC>(d.dgate, row, width, p, kLanes, dg);
      } else if (d.gate_mode == CXG_GATE_ROW) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kValues; ++i) t += dg[i];
        t = sum.one(t);
        if (in && p == 0 && d.dgate != nullptr) static_cast<T *>(d.dgate)[row] = from_f32<T>(t);
      }
      if (d.post) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
          acc[1][i] = fmaf(g[i], n[i], acc[1][i]);
          acc[2][i] += g[i];
          g[i] *= w2[i];
        }
        back_through_norm(g, n, r2, a, sum);
      }
      if (in && d.df != nullptr) store_row<T, VEC>(d.df, row, width, p, kLanes, g);
    }
  }
  // the block's sums: lanes of a warp that hold the same columns, then the warps in order
  float *part = a.part + static_cast<int64_t>(blockIdx.x) * kSums * width;
  if constexpr (WARPS == 1) {
    __shared__ float side[kBlock / 32][LANES * kValues];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
#pragma unroll
      for (int i = 0; i < kValues; ++i)
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) acc[k][i] += __shfl_xor_sync(0xffffffffu, acc[k][i], o);
      if ((threadIdx.x & 31) < LANES) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) side[warp][((i / P::N) * kLanes + p) * P::N + i % P::N] = acc[k][i];
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
      for (int i = 0; i < kValues; ++i) {
        const int c = ((i / P::N) * kLanes + p) * P::N + i % P::N;
        if (c < width) part[k * width + c] = acc[k][i];
      }
  }
}

// Lanes of a row: the smallest power of two, from 8 on, that holds it.
int lanes_of(int width) {
  int lanes = 8;
  while (lanes * kValues < width) lanes *= 2;
  return lanes;
}
int rows_per_block(int width) { return lanes_of(width) > 32 ? 1 : kBlock / lanes_of(width); }
int backward_blocks(int64_t n, int width) {
  const int lanes = lanes_of(width), per_sm = lanes > 32 ? kMostWarps * 32 / lanes : 2;
  const int64_t want = (n + rows_per_block(width) - 1) / rows_per_block(width);
  return static_cast<int>(want < 1 ? 1 : want < kNumSM * per_sm ? want : kNumSM * per_sm);
}

template <typename T, bool VEC, typename Go>
cudaError_t by_width(int width, Go go) {
  switch (lanes_of(width)) {
    case 8: return go.template run<T, 8, 1, VEC>();
    case 16: return go.template run<T, 16, 1, VEC>();
    case 32: return go.template run<T, 32, 1, VEC>();
    case 64: return go.template run<T, 32, 2, VEC>();
    case 128: return go.template run<T, 32, 4, VEC>();
    case 256: return go.template run<T, 32, 8, VEC>();
    default: return go.template run<T, 32, 16, VEC>();
  }
}
template <typename Go>
cudaError_t by_type(const cxg_residual_desc &d, bool vec, Go go) {
  if (d.dtype == CXG_F32) return vec ? by_width<float, true>(d.width, go) : by_width<float, false>(d.width, go);
  return vec ? by_width<__nv_bfloat16, true>(d.width, go) : by_width<__nv_bfloat16, false>(d.width, go);
}

struct Forward {
  const ResArgs &a;
  cudaStream_t st;
  template <typename T, int LANES, int WARPS, bool VEC>
  cudaError_t run() const {
    const int per = rows_per_block(a.d.width);
    const int64_t want = (a.d.n + a.keep + per - 1) / per, most = static_cast<int64_t>(kNumSM) * (WARPS > 1 ? 64 / WARPS : 8);
    return launch_dependent(residual_forward<T, LANES, WARPS, VEC>, static_cast<unsigned>(want < most ? want : most),
                            WARPS > 1 ? 32 * WARPS : kBlock, 0, st, a);
  }
};
struct Backward {
  const ResArgs &a;
  cudaStream_t st;
  int blocks;
  template <typename T, int LANES, int WARPS, bool VEC>
  cudaError_t run() const {
    return launch_dependent(residual_backward<T, LANES, WARPS, VEC>, static_cast<unsigned>(blocks), WARPS > 1 ? 32 * WARPS : kBlock, 0,
                            st, a);
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

extern "C" int cxg_residual_norm_backward_workspace_size(int64_t n, int width, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_residual_norm_backward_workspace_size: bytes is NULL");
  CXG_REQUIRE(n >= 0 && width > 0, CXG_EINVAL, "cxg_residual_norm_backward_workspace_size: bad sizes");
  CXG_REQUIRE(width <= kMostWidth, CXG_EUNSUPPORTED, "cxg_residual_norm: rows of %d values, at most %d", width, kMostWidth);
  *bytes = static_cast<size_t>(backward_blocks(n, width)) * kSums * width * sizeof(float);
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
  cxg_residual_norm_backward_workspace_size(d->n, d->width, &need);
  CXG_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, CXG_EWORKSPACE,
              "cxg_residual_norm_backward: workspace %zu bytes, need %zu", workspace_bytes, need);
  ResArgs a = {};
  a.d = *d;
  a.inv_width = 1.f / static_cast<float>(d->width);
  a.part = static_cast<float *>(workspace);
  const int blocks = backward_blocks(d->n, d->width);
  const cudaError_t e = by_type(*d, whole_vectors(*d), Backward{a, st, blocks});
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_residual_norm_backward: %s", cudaGetErrorString(e));
  column_sum_join(a.part, sums, blocks, kSums * d->width, st);
  count_launches(2);
  return check_launch("cxg_residual_norm_backward");
}
