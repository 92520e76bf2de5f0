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
// Both would be bound by memory, but the arithmetic of a value is what it takes some care to hide behind it. A lane holds 8
// values of a row (a part of a warp, a warp or up to 16 warps per row: what a row costs by itself, the chains of shuffles of
// its sums above all, is shared by many values) as pairs for packed fp32 instructions; the next row is on its way into
// shared memory meanwhile (16-byte asynchronous copies, each lane its own, so there is nothing to wait for but they).
// Statistics, products and sums are fp32 whatever the rows' type; y is rounded when it is stored, h is computed from it before.
// The sums over rows are kept per lane for the whole grid's pass, added up per block, and the blocks' sums are added in order
// by a second kernel: the same bits on every run.
//
// Measured: 169,343 rows of 256 bf16, rms, a gate per value: forward 78 us (5.6 TB/s), backward 137 (5.1 TB/s, 493 instructions a
// row and warp at 2.4 per cycle: what bounds it); 250,000 rows of 128 fp32, layer norm, a gate per row, both 227 us (5.6 TB/s).
#include <initializer_list>

#include "rows8.cuh"

namespace cxg {
namespace {

constexpr int kValues = 8;     // of a row per lane
constexpr int kPairs = kValues / 2;
constexpr int kSums = 5;       // dscale, dw2, db2, dw1, db1
constexpr int kMostWarps = 16;
constexpr int kMostWidth = kMostWarps * 32 * kValues;
constexpr int kBlock = 128;    // threads where a row takes a warp or less

struct ResArgs {
  cxg_residual_desc d;  // scale and weights are there: missing ones point at ones
  float inv_width;
  float *part;       // backward: [gridDim.x][kSums][width]
  int keep, groups;  // forward: rows in 8 bits of h
};

// Stands for a scale or weight that is not given.
struct alignas(16) Ones {
  float v[kMostWidth];
  constexpr Ones() : v() {
    for (int i = 0; i < kMostWidth; ++i) v[i] = 1.f;
  }
};
__device__ const Ones residual_ones{};

// Where a lane's values lie: Q vectors of N values (VB bytes: the widest that rows are whole in), the lanes' first vectors side by
// side, then their second ones, and so on.
// FULL: rows that fill their lanes, so that nothing asks where they end.
template <typename T, int VB, int LANES, bool FULL = false>
struct Place {
  static constexpr int N = VB / static_cast<int>(sizeof(T));
  static constexpr int Q = kValues / N;
  static constexpr int kBytes = VB;
  static constexpr int kLanes = LANES;
  using Element = T;
  static constexpr bool kStaged = VB >= 4;  // there are asynchronous copies of that many bytes
  __device__ __forceinline__ static int column(int p, int i) { return (i / N * LANES + p) * N + i % N; }
  __device__ __forceinline__ static bool has(int column, int width) { return FULL || column < width; }
  __device__ __forceinline__ static int width_of(int width) { return FULL ? LANES * kValues : width; }
};

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ Pair widened(uint32_t two) { return pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u)); }

// Rows on their way: per thread `tensors` x Q slots of VB bytes for each of two rows.
template <typename P>
struct Stage {
  uint32_t base, step;  // this thread's first slot; from a slot to the next
  int tensors;
  __device__ Stage(const void *smem, int n) : base(shared_address(smem) + threadIdx.x * P::kBytes), step(blockDim.x * P::kBytes), tensors(n) {}
  __device__ __forceinline__ uint32_t slot(int turn, int tensor, int q) const {
    return base + ((turn * tensors + tensor) * P::Q + q) * step;
  }
  // a row's offset in bytes, the lane's part included
  __device__ __forceinline__ void request(int turn, int tensor, const void *matrix, int64_t offset, int p, int width) const {
#pragma unroll
    for (int q = 0; q < P::Q; ++q) {
      const bool on = P::has(P::column(p, q * P::N), width);
      const uint8_t *src = on ? static_cast<const uint8_t *>(matrix) + offset + q * (P::kLanes * P::kBytes) : static_cast<const uint8_t *>(matrix);
      if constexpr (P::kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot(turn, tensor, q)), "l"(src), "r"(on ? 16 : 0) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(slot(turn, tensor, q)), "l"(src), "r"(on ? P::kBytes : 0),
                     "n"(P::kBytes)
                     : "memory");
    }
  }
  __device__ __forceinline__ void take(int turn, int tensor, Pair (&v)[kPairs]) const {
    constexpr int kWords = P::kBytes / 4;
    uint32_t w[P::Q * kWords];
#pragma unroll
    for (int q = 0; q < P::Q; ++q) {
      uint32_t *d = w + q * kWords;
      if constexpr (kWords == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "r"(slot(turn, tensor, q))
                     : "memory");
      else if constexpr (kWords == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(slot(turn, tensor, q)) : "memory");
      else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(d[0]) : "r"(slot(turn, tensor, q)) : "memory");
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if constexpr (sizeof(typename P::Element) == 4)
        v[i] = pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else
        v[i] = widened(w[i]);
    }
  }
};

// Rows of an odd number of bf16 values, straight from memory.
template <typename P>
__device__ __forceinline__ void read_row(Pair (&v)[kPairs], const void *matrix, int64_t row, int p, int width) {
  using T = typename P::Element;
  const T *src = static_cast<const T *>(matrix) + row * width;
  float f[kValues];
#pragma unroll
  for (int i = 0; i < kValues; ++i) f[i] = P::has(P::column(p, i), width) ? to_f32(__ldg(src + P::column(p, i))) : 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = pair(f[2 * i], f[2 * i + 1]);
}

template <typename P>
__device__ __forceinline__ void store_row(void *matrix, int64_t row, int p, int width, const Pair (&v)[kPairs]) {
  using T = typename P::Element;
  T *dst = static_cast<T *>(matrix) + row * width;
  float f[kValues];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 t = halves(v[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = P::column(p, q * P::N);
    if (!P::has(c, width)) continue;
    const float *g = f + q * P::N;
    if constexpr (P::kBytes == 16) {
      Vec<T>::store_stream(dst + c, Vec<T>::from_float(g));
    } else if constexpr (P::N == 1) {
      dst[c] = from_f32<T>(g[0]);
    } else if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float2 *>(dst + c), make_float2(g[0], g[1]));
    } else {
      uint32_t w[P::N / 2];
#pragma unroll
      for (int i = 0; i < P::N / 2; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(g[2 * i], g[2 * i + 1]);
        __builtin_memcpy(&w[i], &t, 4);
      }
      if constexpr (P::N == 4)
        __stcs(reinterpret_cast<uint2 *>(dst + c), make_uint2(w[0], w[1]));
      else
        __stcs(reinterpret_cast<unsigned *>(dst + c), w[0]);
    }
  }
}

// A parameter's values at the lane's columns (anything behind the row).
template <typename P>
__device__ __forceinline__ void load_param(Pair (&v)[kPairs], const float *w, int p, int width) {
#pragma unroll
  for (int i = 0; i < kPairs; i += P::N >= 4 ? 2 : 1) {
    const int c = P::column(p, 2 * i);
    if constexpr (P::N >= 4) {
      const ulonglong2 t = __ldg(reinterpret_cast<const ulonglong2 *>(w + (P::has(c, width) ? c : 0)));
      v[i] = t.x, v[i + 1] = t.y;
    } else if constexpr (P::N == 2) {
      v[i] = __ldg(reinterpret_cast<const unsigned long long *>(w + (P::has(c, width) ? c : 0)));
    } else {
      const int e = P::column(p, 2 * i + 1);
      v[i] = pair(__ldg(w + (P::has(c, width) ? c : 0)), __ldg(w + (P::has(e, width) ? e : 0)));
    }
  }
}

// Zeros behind the row.
template <typename P>
__device__ __forceinline__ void clear_behind(Pair (&v)[kPairs], int p, int width) {
  if (P::has(P::kLanes * kValues - 1, width)) return;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if (P::N > 1) {
      if (P::column(p, 2 * i) >= width) v[i] = 0;
    } else {
      const float2 t = halves(v[i]);
      v[i] = pair(P::column(p, 2 * i) < width ? t.x : 0.f, P::column(p, 2 * i + 1) < width ? t.y : 0.f);
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

// v becomes norm(v); returns the factor. Values behind the row are and stay zeros.
template <typename P, typename Sum>
__device__ __forceinline__ float normalise(Pair (&v)[kPairs], const ResArgs &a, Sum &sum, int p) {
  if (a.d.layer) {
    const float mean = sum.one(sum2(add2(add2(v[0], v[1]), add2(v[2], v[3])))) * a.inv_width;
    const Pair off = pair(-mean, -mean);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) v[i] = add2(v[i], off);
    clear_behind<P>(v, p, a.d.width);
  }
  const Pair t = add2(fma2(v[0], v[0], mul2(v[1], v[1])), fma2(v[2], v[2], mul2(v[3], v[3])));
  const float r = __frsqrt_rn(fmaf(sum.one(sum2(t)), a.inv_width, a.d.eps));
  const Pair rr = pair(r, r);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = mul2(v[i], rr);
  return r;
}

// sigmoid and its derivative without cancellation: t = exp(-|g|), s = 1 / (1 + t) or t / (1 + t), s' = t / (1 + t)^2; the
// reciprocal of 1 .. 2 is the hardware's, off by an ulp. (s (1 - s) for s' loses half its bits at g = 10 and all from 17 on.) For
// bf16 rows t is the hardware's 2^x of a product rounded once, off by 2^-22 + |g| 2^-24 of it (1.2e-6 at |g| = 16), where the rows
// round by 2^-9; where s alone is asked for it is 1 / (1 + exp(-g)), which loses nothing, two instructions less.
template <typename T>
__device__ __forceinline__ void sigmoid(float g, float *s, float *ds) {
  float t, q;
  if (sizeof(T) == 2 && ds == nullptr) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(g * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(*s) : "f"(1.f + t));
    return;
  }
  if constexpr (sizeof(T) == 2)
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fabsf(g) * -1.44269504f));
  else
    t = expf(-fabsf(g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + t));
  const float tq = t * q;
  *s = g >= 0.f ? q : tq;
  if (ds != nullptr) *ds = tq * q;
}
// The gate's values become sigmoids, and their derivatives where there is room for them.
template <typename T>
__device__ __forceinline__ void sigmoids(Pair (&s)[kPairs], Pair *ds) {
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 g = halves(s[i]);
    float a, b, da, db;
    sigmoid<T>(g.x, &a, ds != nullptr ? &da : nullptr);
    sigmoid<T>(g.y, &b, ds != nullptr ? &db : nullptr);
    s[i] = pair(a, b);
    if (ds != nullptr) ds[i] = pair(da, db);
  }
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
__device__ __forceinline__ void keep_row(const ResArgs &a, int64_t row, bool in, const Pair (&h)[kPairs], int p) {
  using T = typename P::Element;
  constexpr int kShare = rows8::kGroup / P::N;  // lanes that hold a group
#pragma unroll
  for (int q = 0; q < P::Q; ++q) {
    const int c = P::column(p, q * P::N);
    float v[P::N];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      const float2 t = halves(h[(q * P::N + i) / 2]);
      v[i] = in && P::has(c, a.d.width) ? to_f32(from_f32<T>(i & 1 ? t.y : t.x)) : 0.f;
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

// Warps per SM, by the registers a thread gets (80 forward, 128 backward), and blocks of `threads` threads with that many warps.
constexpr int kForwardWarps = 24, kBackwardWarps = 16;
constexpr int blocks_of(int warps, int threads) { return warps * 32 / threads > 0 ? warps * 32 / threads : 1; }
// Shared memory of a block for two rows of so many matrices.
template <typename P>
constexpr int stage_bytes(int tensors, int threads) { return P::kStaged ? 2 * tensors * P::Q * P::kBytes * threads : 0; }
constexpr int kForwardTensors = 3, kBackwardTensors = 5;

// GATED: a gate per value.
template <typename T, int LANES, int WARPS, int VB, bool GATED, bool FULL>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock, blocks_of(kForwardWarps, WARPS > 1 ? 32 * WARPS : kBlock))
    residual_forward(const __grid_constant__ ResArgs a) {
  constexpr int kLanes = LANES * WARPS;
  using P = Place<T, VB, kLanes, FULL>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = WARPS > 1 ? threadIdx.x : threadIdx.x & (LANES - 1), width = P::width_of(d.width);
  const bool with_f = d.f != nullptr, row_gate = d.gate_mode == CXG_GATE_ROW;
  dependency_wait();
  const Rows<LANES, WARPS> rows;
  const Stage<P> stage(smem, kForwardTensors);
  T rr = from_f32<T>(0.f);
  auto request = [&](int turn, int64_t row) {
    const int64_t at = row < d.n ? row : d.n - 1;
    if constexpr (P::kStaged) {
      const int64_t offset = at * width * static_cast<int64_t>(sizeof(T)) + p * VB;
      stage.request(turn, 0, d.x, offset, p, width);
      if (with_f) stage.request(turn, 1, d.f, offset, p, width);
      if (GATED) stage.request(turn, 2, d.gate, offset, p, width);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (row_gate) rr = __ldg(static_cast<const T *>(d.gate) + at);
  };
  const int64_t n_end = d.n + a.keep;
  int turn = 0;
  if (rows.first < n_end) request(0, rows.first + rows.sub);
  for (int64_t row0 = rows.first; row0 < n_end; row0 += rows.step, turn ^= 1) {
    const int64_t row = row0 + rows.sub, at = row < d.n ? row : d.n - 1;
    const bool in = row < d.n;
    const float g_row = to_f32(rr);
    Pair y[kPairs], n[kPairs], s[kPairs];
    if constexpr (P::kStaged) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (row0 + rows.step < n_end) request(turn ^ 1, row + rows.step);
    auto take = [&](Pair(&v)[kPairs], int tensor, const void *matrix) {
      if constexpr (P::kStaged)
        stage.take(turn, tensor, v);
      else
        read_row<P>(v, matrix, at, p, width);
    };
    take(y, 0, d.x);
    if (with_f) {
      take(n, 1, d.f);
      Pair w[kPairs], b[kPairs];
      if (d.post) {
        normalise<P>(n, a, sum, p);
        load_param<P>(w, d.post_weight, p, width);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) n[i] = mul2(n[i], w[i]);
        if (d.post_bias != nullptr) {
          load_param<P>(b, d.post_bias, p, width);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) n[i] = add2(n[i], b[i]);
        }
      }
      load_param<P>(w, d.scale, p, width);
      if (GATED) {
        take(s, 2, d.gate);
        sigmoids<T>(s, nullptr);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) w[i] = mul2(w[i], s[i]);
      } else if (row_gate) {
        float one;
        sigmoid<T>(g_row, &one, nullptr);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) w[i] = mul2(w[i], pair(one, one));
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) y[i] = fma2(w[i], n[i], y[i]);
      clear_behind<P>(y, p, width);
      if (d.y != nullptr && in) store_row<P>(d.y, row, p, width, y);
    }
    if (d.next) {
      normalise<P>(y, a, sum, p);
      Pair w[kPairs];
      load_param<P>(w, d.next_weight, p, width);
      if (d.next_bias != nullptr) {
        Pair b[kPairs];
        load_param<P>(b, d.next_bias, p, width);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) y[i] = fma2(y[i], w[i], b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) y[i] = mul2(y[i], w[i]);
      }
      if (in) store_row<P>(d.h, row, p, width, y);
      if constexpr (VB == 16 && P::kLanes * P::N >= rows8::kGroup) {  // the lanes' first vectors hold whole groups
        if (a.keep) keep_row<P>(a, row, in, y, p);
      }
    }
  }
}

// g becomes r (g - <g> - u <g u>) (without <g> where no mean was taken off); zeros behind the row
template <typename P, typename Sum>
__device__ __forceinline__ void back_through_norm(Pair (&g)[kPairs], const Pair (&u)[kPairs], float r, const ResArgs &a, Sum &sum, int p) {
  const Pair t = add2(fma2(g[0], u[0], mul2(g[1], u[1])), fma2(g[2], u[2], mul2(g[3], u[3])));
  float mean = 0.f, dot;
  if (a.d.layer) {
    const float2 m = sum.both(sum2(add2(add2(g[0], g[1]), add2(g[2], g[3]))), sum2(t));
    mean = m.x * a.inv_width, dot = m.y * a.inv_width;
  } else {
    dot = sum.one(sum2(t)) * a.inv_width;
  }
  const Pair rr = pair(r, r), dots = pair(-dot, -dot), means = pair(-mean, -mean);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    Pair v = fma2(u[i], dots, g[i]);
    if (a.d.layer) v = add2(v, means);
    g[i] = mul2(v, rr);
  }
  clear_behind<P>(g, p, a.d.width);
}

// BIASES: sums for them too.
template <typename T, int LANES, int WARPS, int VB, bool GATED, bool BIASES, bool FULL>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : kBlock, blocks_of(kBackwardWarps, WARPS > 1 ? 32 * WARPS : kBlock))
    residual_backward(const __grid_constant__ ResArgs a) {
  constexpr int kLanes = LANES * WARPS;
  using P = Place<T, VB, kLanes, FULL>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 place[2][WARPS];
  RowSum<LANES, WARPS> sum(place);
  const cxg_residual_desc &d = a.d;
  const int p = WARPS > 1 ? threadIdx.x : threadIdx.x & (LANES - 1), width = P::width_of(d.width);
  const bool with_f = d.f != nullptr, row_gate = d.gate_mode == CXG_GATE_ROW, next = d.next && d.dh != nullptr;
  dependency_wait();
  Pair acc[kSums][kPairs];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < kPairs; ++i) acc[k][i] = 0;
  const Rows<LANES, WARPS> rows;
  const Stage<P> stage(smem, kBackwardTensors);
  T rr = from_f32<T>(0.f);
  auto request = [&](int turn, int64_t row) {
    const int64_t at = row < d.n ? row : d.n - 1;
    if constexpr (P::kStaged) {
      const int64_t offset = at * width * static_cast<int64_t>(sizeof(T)) + p * VB;
      stage.request(turn, 0, d.x, offset, p, width);
      if (with_f) stage.request(turn, 1, d.f, offset, p, width);
      if (GATED) stage.request(turn, 2, d.gate, offset, p, width);
      if (d.dy != nullptr) stage.request(turn, 3, d.dy, offset, p, width);
      if (next) stage.request(turn, 4, d.dh, offset, p, width);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (row_gate) rr = __ldg(static_cast<const T *>(d.gate) + at);
  };
  int turn = 0;
  if (rows.first < d.n) request(0, rows.first + rows.sub);
  for (int64_t row0 = rows.first; row0 < d.n; row0 += rows.step, turn ^= 1) {
    const int64_t row = row0 + rows.sub;
    const bool in = kLanes >= 32 || row < d.n;  // lanes without a row go through the last one and add nothing
    const int64_t at = in ? row : d.n - 1;
    const float g_row = to_f32(rr);
    if constexpr (P::kStaged) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (row0 + rows.step < d.n) request(turn ^ 1, row + rows.step);
    auto take = [&](Pair(&v)[kPairs], int tensor, const void *matrix) {
      if constexpr (P::kStaged)
        stage.take(turn, tensor, v);
      else
        read_row<P>(v, matrix, at, p, width);
    };
    Pair y[kPairs], n[kPairs], s[GATED ? kPairs : 1], ds[GATED ? kPairs : 1], g[kPairs], w[kPairs];
    take(y, 0, d.x);
    float r2 = 0.f;
    if constexpr (!GATED) {
      float s0 = 1.f, ds0 = 0.f;
      if (row_gate) sigmoid<T>(g_row, &s0, &ds0);
      s[0] = pair(s0, s0), ds[0] = pair(ds0, ds0);
    }
    if (with_f) {
      take(n, 1, d.f);
      if constexpr (GATED) {
        take(s, 2, d.gate);
        sigmoids<T>(s, ds);
      }
      Pair t[kPairs];
      if (d.post) {
        r2 = normalise<P>(n, a, sum, p);  // n is u2 from here on
        load_param<P>(w, d.post_weight, p, width);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) t[i] = mul2(n[i], w[i]);
        if (BIASES && d.post_bias != nullptr) {
          load_param<P>(w, d.post_bias, p, width);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) t[i] = add2(t[i], w[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) t[i] = n[i];
      }
      load_param<P>(w, d.scale, p, width);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) y[i] = fma2(mul2(w[i], s[GATED ? i : 0]), t[i], y[i]);
      clear_behind<P>(y, p, width);
    }
    if (in && d.dy != nullptr)
      take(g, 3, d.dy);
    else
#pragma unroll
      for (int i = 0; i < kPairs; ++i) g[i] = 0;
    if (next) {
      Pair dh[kPairs], t[kPairs];
      if (in)
        take(dh, 4, d.dh);
      else
#pragma unroll
        for (int i = 0; i < kPairs; ++i) dh[i] = 0;
      load_param<P>(w, d.next_weight, p, width);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) t[i] = mul2(dh[i], w[i]);
      // the norm's factor and what goes back through it in one round of sums: <t u1> = r1 <t y>
      float mean_t = 0.f;
      if (d.layer) {
        const float2 m = sum.both(sum2(add2(add2(y[0], y[1]), add2(y[2], y[3]))), sum2(add2(add2(t[0], t[1]), add2(t[2], t[3]))));
        const Pair off = pair(-m.x * a.inv_width, -m.x * a.inv_width);
        mean_t = m.y * a.inv_width;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) y[i] = add2(y[i], off);
        clear_behind<P>(y, p, width);
      }
      const Pair yy = add2(fma2(y[0], y[0], mul2(y[1], y[1])), fma2(y[2], y[2], mul2(y[3], y[3])));
      const Pair ty = add2(fma2(t[0], y[0], mul2(t[1], y[1])), fma2(t[2], y[2], mul2(t[3], y[3])));
      const float2 q = sum.both(sum2(yy), sum2(ty));
      const float r1 = __frsqrt_rn(fmaf(q.x, a.inv_width, d.eps)), dot = q.y * r1 * a.inv_width;
      const Pair rr1 = pair(r1, r1), dots = pair(-dot, -dot), means = pair(-mean_t, -mean_t);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        y[i] = mul2(y[i], rr1);  // u1
        if (in) acc[3][i] = fma2(dh[i], y[i], acc[3][i]);
        if (BIASES && in) acc[4][i] = add2(acc[4][i], dh[i]);
        Pair v = fma2(y[i], dots, t[i]);
        if (d.layer) v = add2(v, means);
        t[i] = mul2(v, rr1);
      }
      if (d.layer) clear_behind<P>(t, p, width);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) g[i] = add2(g[i], t[i]);
    }
    if (in && d.dx != nullptr) store_row<P>(d.dx, row, p, width, g);
    if (with_f) {
      Pair w2[kPairs], t[kPairs];
      if (d.post) {
        load_param<P>(w2, d.post_weight, p, width);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) t[i] = mul2(n[i], w2[i]);
        if (BIASES && d.post_bias != nullptr) {
          load_param<P>(w, d.post_bias, p, width);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) t[i] = add2(t[i], w[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) t[i] = n[i];
      }
      load_param<P>(w, d.scale, p, width);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        if (in) acc[0][i] = fma2(mul2(g[i], s[GATED ? i : 0]), t[i], acc[0][i]);
        g[i] = mul2(g[i], w[i]);
        t[i] = mul2(mul2(t[i], g[i]), ds[GATED ? i : 0]);  // dgate
        g[i] = mul2(g[i], s[GATED ? i : 0]);               // dn
      }
      if constexpr (GATED) {
        if (in && d.dgate != nullptr) store_row<P>(d.dgate, row, p, width, t);
      } else if (row_gate) {
        clear_behind<P>(t, p, width);
        const float dg = sum.one(sum2(add2(add2(t[0], t[1]), add2(t[2], t[3]))));
        if (in && p == 0 && d.dgate != nullptr) static_cast<T *>(d.dgate)[row] = from_f32<T>(dg);
      }
      if (d.post) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          if (in) acc[1][i] = fma2(g[i], n[i], acc[1][i]);
          if (BIASES && in) acc[2][i] = add2(acc[2][i], g[i]);
          g[i] = mul2(g[i], w2[i]);
        }
        back_through_norm<P>(g, n, r2, a, sum, p);
      }
      if (in && d.df != nullptr) store_row<P>(d.df, row, p, width, g);
    }
  }
  // the block's sums: lanes of a warp that hold the same columns, then the warps in order
  float *part = a.part + static_cast<int64_t>(blockIdx.x) * kSums * width;
  [[maybe_unused]] __shared__ float side[WARPS == 1 ? kBlock / 32 : 1][WARPS == 1 ? LANES * kValues : 1];
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    float f[kValues];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 t = halves(acc[k][i]);
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
    if constexpr (WARPS == 1) {
      if (!BIASES && (k == 2 || k == 4)) {
        for (int c = threadIdx.x; c < width; c += kBlock) part[k * width + c] = 0.f;
        continue;
      }
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) f[i] += __shfl_xor_sync(0xffffffffu, f[i], o);
        if ((threadIdx.x & 31) < LANES) side[threadIdx.x >> 5][P::column(p, i)] = f[i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < width; c += kBlock) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kBlock / 32; ++w) t += side[w][c];
        part[k * width + c] = t;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < kValues; ++i)
        if (P::column(p, i) < width) part[k * width + P::column(p, i)] = f[i];
    }
  }
}

// Lanes of a row: the smallest power of two, from 2 on, that holds it, or three warps, six or twelve. (Eight and more alone: 937500
// rows of 32 bf16 values, forward and backward, 399 us instead of 189, 20 of them 409 instead of 216. Powers of two alone: 78,125 of
// 768 bf16 597 us instead of 470, 46,875 of 1280 793 instead of 623.)
int lanes_of(int width) {
  int lanes = 2;
  while (lanes * kValues < width) lanes *= 2;
  return lanes >= 128 && lanes / 4 * 3 * kValues >= width ? lanes / 4 * 3 : lanes;
}
int rows_per_block(int lanes) { return lanes > 32 ? 1 : kBlock / lanes; }
int blocks_for(int64_t n, int lanes, int warps) {
  const int64_t most = kNumSM * blocks_of(warps, lanes > 32 ? lanes : kBlock);
  const int64_t want = (n + rows_per_block(lanes) - 1) / rows_per_block(lanes);
  return static_cast<int>(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, int VB, bool GATED, typename Go>
cudaError_t by_width(int width, Go go) {
  switch (lanes_of(width)) {
    case 2: return go.template run<T, 2, 1, VB, GATED>();
    case 4: return go.template run<T, 4, 1, VB, GATED>();
    case 8: return go.template run<T, 8, 1, VB, GATED>();
    case 16: return go.template run<T, 16, 1, VB, GATED>();
    case 32: return go.template run<T, 32, 1, VB, GATED>();
    case 64: return go.template run<T, 32, 2, VB, GATED>();
    case 96: return go.template run<T, 32, 3, VB, GATED>();
    case 128: return go.template run<T, 32, 4, VB, GATED>();
    case 192: return go.template run<T, 32, 6, VB, GATED>();
    case 256: return go.template run<T, 32, 8, VB, GATED>();
    case 384: return go.template run<T, 32, 12, VB, GATED>();
    default: return go.template run<T, 32, 16, VB, GATED>();
  }
}
template <typename T, int VB, typename Go>
cudaError_t by_gate(const cxg_residual_desc &d, Go go) {
  return d.gate_mode == CXG_GATE_VALUE ? by_width<T, VB, true>(d.width, go) : by_width<T, VB, false>(d.width, go);
}
template <typename Go>
cudaError_t by_type(const cxg_residual_desc &d, int vb, Go go) {
  using bf16 = __nv_bfloat16;
  if (d.dtype == CXG_F32)
    return vb == 16 ? by_gate<float, 16>(d, go) : vb == 8 ? by_gate<float, 8>(d, go) : by_gate<float, 4>(d, go);
  return vb == 16  ? by_gate<bf16, 16>(d, go)
         : vb == 8 ? by_gate<bf16, 8>(d, go)
         : vb == 4 ? by_gate<bf16, 4>(d, go)
                   : by_gate<bf16, 2>(d, go);
}

template <typename P, typename Kernel>
cudaError_t launch(Kernel kernel, int tensors, int threads, int blocks, const ResArgs &a, cudaStream_t st) {
  const int smem = stage_bytes<P>(tensors, threads);
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(kernel, static_cast<unsigned>(blocks), threads, static_cast<size_t>(smem), st, a);
}

struct Forward {
  const ResArgs &a;
  cudaStream_t st;
  template <typename T, int LANES, int WARPS, int VB, bool GATED, bool FULL>
  cudaError_t go() const {
    return launch<Place<T, VB, LANES * WARPS>>(residual_forward<T, LANES, WARPS, VB, GATED, FULL>, kForwardTensors,
                                                WARPS > 1 ? 32 * WARPS : kBlock,
                                                blocks_for(a.d.n + a.keep, LANES * WARPS, kForwardWarps), a, st);
  }
  template <typename T, int LANES, int WARPS, int VB, bool GATED>
  cudaError_t run() const {
    if constexpr (VB == 16) {
      if (a.d.width == LANES * WARPS * kValues) return go<T, LANES, WARPS, VB, GATED, true>();
    }
    return go<T, LANES, WARPS, VB, GATED, false>();
  }
};
struct Backward {
  const ResArgs &a;
  cudaStream_t st;
  int blocks;
  template <typename T, int LANES, int WARPS, int VB, bool GATED, bool BIASES, bool FULL>
  cudaError_t go() const {
    return launch<Place<T, VB, LANES * WARPS>>(residual_backward<T, LANES, WARPS, VB, GATED, BIASES, FULL>, kBackwardTensors,
                                                WARPS > 1 ? 32 * WARPS : kBlock, blocks, a, st);
  }
  template <typename T, int LANES, int WARPS, int VB, bool GATED>
  cudaError_t run() const {
    if constexpr (VB == 16) {
      const bool biases = a.d.post_bias != nullptr || a.d.next_bias != nullptr;
      if (a.d.width == LANES * WARPS * kValues)
        return biases ? go<T, LANES, WARPS, VB, GATED, true, true>() : go<T, LANES, WARPS, VB, GATED, false, true>();
      if (!biases) return go<T, LANES, WARPS, VB, GATED, false, false>();
    }
    return go<T, LANES, WARPS, VB, GATED, true, false>();
  }
};

// The launch's arguments: missing scales and weights are ones.
cudaError_t arguments(const cxg_residual_desc &d, ResArgs *a) {
  *a = {};
  a->d = d;
  a->inv_width = 1.f / static_cast<float>(d.width);
  a->groups = rows8::groups_of(d.width);
  if (d.scale != nullptr && d.post_weight != nullptr && d.next_weight != nullptr) return cudaSuccess;
  void *ones = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&ones, residual_ones);
  for (const float **w : {&a->d.scale, &a->d.post_weight, &a->d.next_weight})
    if (*w == nullptr) *w = static_cast<const float *>(ones);
  return e;
}

// Bytes of the widest vectors that all matrices' rows are whole in; a lane reads as many values of the fp32 parameters, up to
// four, at once.
int vector_bytes(const cxg_residual_desc &d) {
  const int elem = d.dtype == CXG_F32 ? 4 : 2;
  uint64_t bits = static_cast<uint64_t>(d.width) * elem, params = 0;
  for (const void *p : {d.x, d.f, static_cast<const void *>(d.y), static_cast<const void *>(d.h), d.dy, d.dh, static_cast<const void *>(d.dx),
                        static_cast<const void *>(d.df)})
    bits |= reinterpret_cast<uintptr_t>(p);
  if (d.gate_mode == CXG_GATE_VALUE) bits |= reinterpret_cast<uintptr_t>(d.gate) | reinterpret_cast<uintptr_t>(d.dgate);
  for (const float *p : {d.scale, d.post_weight, d.post_bias, d.next_weight, d.next_bias}) params |= reinterpret_cast<uintptr_t>(p);
  int vb = 16;
  while (vb > elem && (bits % vb != 0 || params % (vb / elem < 4 ? vb / elem * 4 : 16) != 0)) vb /= 2;
  return vb;
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

extern "C" int cxg_residual_norm_keeps(const cxg_residual_desc *d) {
  return d != nullptr && vector_bytes(*d) == 16 && lanes_of(d->width) * (d->dtype == CXG_F32 ? 4 : 8) >= rows8::kGroup ? 1 : 0;
}

extern "C" int cxg_residual_norm_forward(const cxg_residual_desc *d, void *stream) {
  const int rc = check_desc(d, "cxg_residual_norm_forward");
  if (rc != CXG_OK) return rc;
  const bool keep = d->codes != nullptr;
  CXG_REQUIRE(d->n == 0 || !d->next || d->h != nullptr, CXG_ENULL, "cxg_residual_norm_forward: h is NULL");
  CXG_REQUIRE(!keep || (d->next && d->scales != nullptr && cxg_residual_norm_keeps(d) == 1 && reinterpret_cast<uintptr_t>(d->codes) % 16 == 0),
              CXG_EINVAL, "cxg_residual_norm_forward: rows in 8 bits are kept of h where cxg_residual_norm_keeps says 1");
  if (d->n == 0 && !keep) return CXG_OK;
  CXG_REQUIRE(d->n > 0, CXG_EINVAL, "cxg_residual_norm_forward: no rows to keep");
  ResArgs a;
  cudaError_t e = arguments(*d, &a);
  a.keep = keep ? 1 : 0;
  if (e == cudaSuccess) e = by_type(*d, vector_bytes(*d), Forward{a, as_stream(stream)});
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_residual_norm_forward: %s", cudaGetErrorString(e));
  count_launches(1);
  return check_launch("cxg_residual_norm_forward");
}

extern "C" int cxg_residual_norm_backward_workspace_size(int64_t n, int width, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_residual_norm_backward_workspace_size: bytes is NULL");
  CXG_REQUIRE(n >= 0 && width > 0, CXG_EINVAL, "cxg_residual_norm_backward_workspace_size: bad sizes");
  CXG_REQUIRE(width <= kMostWidth, CXG_EUNSUPPORTED, "cxg_residual_norm: rows of %d values, at most %d", width, kMostWidth);
  *bytes = static_cast<size_t>(blocks_for(n, lanes_of(width), kBackwardWarps)) * kSums * width * sizeof(float);
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
  ResArgs a;
  cudaError_t e = arguments(*d, &a);
  a.part = static_cast<float *>(workspace);
  const int blocks = blocks_for(d->n, lanes_of(d->width), kBackwardWarps);
  if (e == cudaSuccess) e = by_type(*d, vector_bytes(*d), Backward{a, st, blocks});
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_residual_norm_backward: %s", cudaGetErrorString(e));
  column_sum_join(a.part, sums, blocks, kSums * d->width, st);
  count_launches(2);
  return check_launch("cxg_residual_norm_backward");
}
