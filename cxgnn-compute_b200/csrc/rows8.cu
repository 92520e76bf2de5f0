// Writing and reading rows in 8 bits (rows8.cuh has the format): activations that a backward pass needs again, and caches of
// features or of hidden states that are written and read by node id.
//
// Both directions are bound by memory as long as they spend few instructions and have enough of it on the way: a lane writes
// from 32 bytes of values (8 fp32, 16 bf16: four or two lanes share a group of 32 and find its largest value in two shuffles
// or one) and reads 16 codes, and what an item costs by itself (its row and place, the row's target, the address) is spread
// over these. Lanes go along rows without regard to where these end, so that none is idle for a width that is no power of two;
// items are counted in 32 bits, larger matrices go in pieces. (4 fp32 values a lane, 64-bit counts and a limit on every code were
// 140 instructions an item and twice the time of memory.) Measured: 169,343 rows of 256 fp32 written 35 us (6.2 TB/s); 1.2 M rows
// of 128 bf16 to random rows of 2.4 M and 2 M random rows back 268 us (4.7 TB/s: rows are single
// lines, their four bytes of scales sectors of their own).
#include "rows8.cuh"

namespace cxg {
namespace {

using namespace rows8;

constexpr int kThreads = 256;
template <typename T>
constexpr int kWritten = 32 / static_cast<int>(sizeof(T));  // values of an item that is written
template <typename T>
constexpr int kSharing = kGroup / kWritten<T>;              // lanes of a group
constexpr int kRead = 16;                                   // codes of an item that is read
constexpr int kItems = 4;                                   // per thread
constexpr uint32_t kMostItems = 1u << 31;    // per launch

// Items of rows that have `per` each. The quotient by floor(2^32 / per) is at most one too small.
struct Items {
  uint32_t total, per, inverse;
  __device__ __forceinline__ void place(uint32_t i, uint32_t *row, uint32_t *chunk) const {
    uint32_t q = per > 1 ? __umulhi(i, inverse) : i, r = i - q * per;
    if (r >= per) ++q, r -= per;
    *row = q, *chunk = r;
  }
};

// How the wide side is accessed: in 32-byte vectors, in 16-byte ones, or, where rows are neither, read in the 16-byte vectors that
// hold the values and shifted (written value by value, or by rows8_read_flat). One access per value is a pass of the load path
// per four lanes: 303,000 rows of 99 bf16 written and 606,000 read took 360 us, now 110; of 99 fp32 296, now 145.
enum Access { kShifted, kVector, kWide };

__device__ __forceinline__ void load32(uint32_t (&w)[8], const void *p) {
  asm("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
      : "l"(p));
}
__device__ __forceinline__ void store32(void *p, const uint32_t *w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The larger of two absolute values, NaN where either is.
__device__ __forceinline__ float top_of(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// The values of a row from column c on as they were loaded; zeros behind the row.
template <typename T, Access A>
struct Loaded {
  static constexpr int V = kWritten<T>;
  static constexpr int kWords = A == kShifted ? 12 : 8;
  uint32_t w[kWords];
  int at;     // kShifted: bytes in front of the first value, number of values
  int count;
  // [from, to): the matrix, beyond which nothing is read
  __device__ __forceinline__ void load(const T *row, uint32_t c, uint32_t width, bool in, const T *from, const T *to) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    at = 0, count = 0;
    if (!in) return;
    if constexpr (A == kWide) {
      if (c < width) load32(w, row + c);
    } else if constexpr (A == kVector) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (c + i * (V / 2) < width) {
          const uint4 t = __ldg(reinterpret_cast<const uint4 *>(row + c + i * (V / 2)));
          w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        }
    } else {
      if (c >= width) return;
      count = static_cast<int>(min(width - c, static_cast<uint32_t>(V)));
      const uint8_t *first = reinterpret_cast<const uint8_t *>(row + c);
      at = static_cast<int>(reinterpret_cast<uintptr_t>(first) & 15);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const uint8_t *p = first - at + 16 * i;
        if (16 * i >= at + count * static_cast<int>(sizeof(T))) break;
        if (p >= reinterpret_cast<const uint8_t *>(from) && p + 16 <= reinterpret_cast<const uint8_t *>(to)) {
          const uint4 t = __ldg(reinterpret_cast<const uint4 *>(p));
          w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        } else {  // the vector at the matrix' start or end, value by value
#pragma unroll
          for (int j = 0; j < 16 / static_cast<int>(sizeof(T)); ++j) {
            const T *q = reinterpret_cast<const T *>(p) + j;
            if (q < from || q >= to) continue;
            if constexpr (sizeof(T) == 4)
              w[4 * i + j] = __ldg(reinterpret_cast<const uint32_t *>(q));
            else
              w[4 * i + j / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t *>(q))) << (16 * (j & 1));
          }
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) {
    if constexpr (A == kShifted) {
      if (at & 8) {
#pragma unroll
        for (int i = 0; i < 10; ++i) w[i] = w[i + 2];
      }
      if (at & 4) {
#pragma unroll
        for (int i = 0; i < 9; ++i) w[i] = w[i + 1];
      }
      if constexpr (sizeof(T) == 2) {
        if (at & 2) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if constexpr (sizeof(T) == 4)
        v[i] = __uint_as_float(w[i]);
      else
        v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    if (A == kShifted && count < V) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i >= count) v[i] = 0.f;
    }
  }
};

// The positions of a call that name rows: the last one of a row counts. Each enters itself in the row's word (position + 1, the
// largest stays); who is still there when all have done so writes the row, and sets the word's top bit, which makes it negative:
// less than what any later call enters. Positions are compared without that bit, so it does not matter who of a row's lanes sees it
// already. A call touches the words of its own rows alone: calls that write other rows may run beside it, in any number.
struct Claims {
  const int64_t *index;  // null: row i is row i
  int32_t *words;
  int64_t rows;
};
constexpr uint32_t kDone = 0x80000000u;
constexpr int kClaims = 4;  // per thread (1.2 M of them 11.5 us; one per thread 21)
__global__ void __launch_bounds__(kThreads) rows8_claim(const Claims c, int64_t n) {
  dependency_wait();
  const int64_t first = blockIdx.x * static_cast<int64_t>(kThreads * kClaims) + threadIdx.x;
  int64_t r[kClaims];
#pragma unroll
  for (int k = 0; k < kClaims; ++k) r[k] = first + k * kThreads < n ? __ldg(c.index + first + k * kThreads) : -1;
#pragma unroll
  for (int k = 0; k < kClaims; ++k)
    if (r[k] >= 0 && r[k] < c.rows) atomicMax(c.words + r[k], static_cast<int32_t>(first + k * kThreads + 1));
}

// Rows [0, n) of x to themselves, or to the rows that they claimed, in which they are row `before` and on; rows from n on are written as
// zeros.
template <typename T, Access A>
__global__ void __launch_bounds__(kThreads) rows8_write(const T *x, int64_t ld, uint32_t n, uint32_t width, Items items, uint8_t *codes,
                                                        uint8_t *scales, const Claims claims, uint32_t before) {
  constexpr int V = kWritten<T>, L = kSharing<T>;
  dependency_wait();
  const uint32_t groups = items.per / L, first = blockIdx.x * (kThreads * kItems) + threadIdx.x;
  const T *x_end = x + (n > 0 ? (n - 1) * ld + width : 0);
  Loaded<T, A> in[kItems];
  int64_t dst[kItems];
  uint32_t chunk[kItems], at[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const uint32_t i = first + k * kThreads;
    items.place(i, &at[k], &chunk[k]);
    const bool have = i < items.total, of_x = have && at[k] < n;
    dst[k] = have ? static_cast<int64_t>(at[k]) : int64_t{-1};
    if (claims.index != nullptr && of_x) dst[k] = __ldg(claims.index + at[k]);
    in[k].load(x + (of_x ? at[k] : 0) * ld, chunk[k] * V, width, of_x, x, x_end);
  }
  if (claims.index != nullptr) {
    uint32_t last[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (static_cast<uint64_t>(dst[k]) >= static_cast<uint64_t>(claims.rows)) dst[k] = -1;
      last[k] = dst[k] >= 0 ? static_cast<uint32_t>(__ldcg(claims.words + dst[k])) : 0u;
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      if ((last[k] & ~kDone) != before + at[k] + 1) dst[k] = -1;
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    float v[V];
    in[k].get(v);
    float top = top_of(v[0], v[1]);
#pragma unroll
    for (int j = 2; j < V; j += 2) top = top_of(top, top_of(v[j], v[j + 1]));
#pragma unroll
    for (int d = 1; d < L; d <<= 1) top = top_of(top, __shfl_xor_sync(0xffffffffu, top, d));
    const uint32_t e = scale_byte(__float_as_uint(top));
    uint32_t w[V / 4];
    codes_of<V>(w, v, e);
    if (dst[k] >= 0) {
      const int64_t group = dst[k] * groups + (chunk[k] / L);
      uint8_t *out = codes + group * kGroup + (chunk[k] % L) * V;
      if constexpr (V == 8)
        *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
      else
        *reinterpret_cast<uint4 *>(out) = make_uint4(w[0], w[1], w[V / 4 - 2], w[V / 4 - 1]);
      if (chunk[k] % L == 0) scales[group] = static_cast<uint8_t>(e);
      if (claims.index != nullptr && chunk[k] == 0) __stcg(claims.words + dst[k], static_cast<int32_t>(kDone | (before + at[k] + 1)));
    }
  }
}

// out[i] = the values of row index[i] (of row i without an index; ids outside the rows read as zeros).
template <typename T, Access A>
__global__ void __launch_bounds__(kThreads) rows8_read(const uint8_t *codes, const uint8_t *scales, int64_t n_rows, uint32_t width,
                                                       uint32_t groups, const int64_t *index, Items items, T *out, int64_t ld) {
  dependency_wait();
  const uint32_t first = blockIdx.x * (kThreads * kItems) + threadIdx.x;
  int64_t src[kItems];
  uint32_t row[kItems], chunk[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const uint32_t i = first + k * kThreads;
    items.place(i, &row[k], &chunk[k]);
    src[k] = n_rows;  // the row of zeros
    if (i < items.total) {
      const int64_t r = index != nullptr ? __ldg(index + row[k]) : static_cast<int64_t>(row[k]);
      if (static_cast<uint64_t>(r) < static_cast<uint64_t>(n_rows)) src[k] = r;
    }
  }
  uint4 w[kItems];
  uint32_t e[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t group = src[k] * groups + chunk[k] / (kGroup / kRead);
    w[k] = __ldg(reinterpret_cast<const uint4 *>(codes + group * kGroup + (chunk[k] % (kGroup / kRead)) * kRead));
    e[k] = __ldg(scales + group);
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    if (first + k * kThreads >= items.total) break;
    const float s = scale_of(e[k]);
    float f[kRead];
    code_values(f, w[k].x);
    code_values(f + 4, w[k].y);
    code_values(f + 8, w[k].z);
    code_values(f + 12, w[k].w);
#pragma unroll
    for (int j = 0; j < kRead; ++j) f[j] *= s;
    const uint32_t c = chunk[k] * kRead;
    T *o = out + row[k] * ld + c;
    if constexpr (A == kWide) {
      constexpr int V = kWritten<T>;  // values of 32 bytes
#pragma unroll
      for (int j = 0; j < kRead; j += V)
        if (c + j < width) {
          uint32_t v[8];
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(f[j + i]);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 t = Vec<T>::from_float(f + j + 8 * i);
              v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
            }
          }
          store32(o + j, v);
        }
    } else if constexpr (A == kVector) {
#pragma unroll
      for (int j = 0; j < kRead; j += Vec<T>::kElems)
        if (c + j < width) Vec<T>::store_stream(o + j, Vec<T>::from_float(f + j));
    } else {
#pragma unroll
      for (int j = 0; j < kRead; ++j)
        if (c + j < width) o[j] = from_f32<T>(f[j]);
    }
  }
}

// The same for rows that are not whole vectors and lie one behind the other: a lane writes a 16-byte vector of `out`, whose values
// may be of two rows. (Narrow rows, of which they would be of several, are better off value by value: 1.9 M of 7 bf16 are read
// in half the time.)
template <typename T>
__global__ void __launch_bounds__(kThreads) rows8_read_flat(const uint8_t *codes, const uint8_t *scales, int64_t n_rows, uint32_t groups,
                                                            const int64_t *index, Items values, T *out) {
  constexpr int N = Vec<T>::kElems, kVectors = 2;
  dependency_wait();
  const uint32_t width = values.per;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    const uint32_t first = ((blockIdx.x * kVectors + k) * kThreads + threadIdx.x) * N;
    if (first >= values.total) return;
    uint32_t row, c;
    values.place(first, &row, &c);
    auto source = [&](uint32_t i) {
      const int64_t r = index != nullptr ? __ldg(index + i) : static_cast<int64_t>(i);
      return static_cast<uint64_t>(r) < static_cast<uint64_t>(n_rows) ? r : n_rows;
    };
    int64_t src = source(row);
    uint32_t code[N], e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (c == width) {
        c = 0;
        ++row;
        if (first + i < values.total) src = source(row);
      }
      code[i] = __ldg(codes + src * (groups * kGroup) + c);
      e[i] = __ldg(scales + src * groups + c / kGroup);
      ++c;
    }
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = code_value<0>(code[i]) * scale_of(e[i]);
    if (first + N <= values.total) {
      Vec<T>::store_stream(out + first, Vec<T>::from_float(f));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (first + i < values.total) out[first + i] = from_f32<T>(f[i]);
    }
  }
}

template <typename T>
Access access_of(const void *p, int64_t ld, int width) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(p) | (static_cast<uint64_t>(ld) * sizeof(T)) | (static_cast<uint64_t>(width) * sizeof(T));
  return bits % 32 == 0 ? kWide : bits % 16 == 0 ? kVector : kShifted;
}

// go(first row, rows, items, blocks) for pieces of n rows with `per` items each.
template <typename Go>
void in_pieces(int64_t n, uint32_t per, Go go) {
  const int64_t most = kMostItems / per;
  for (int64_t r = 0; r < n; r += most) {
    const int64_t rows = n - r < most ? n - r : most;
    const Items items{static_cast<uint32_t>(rows * per), per, static_cast<uint32_t>((1ull << 32) / per)};
    go(r, rows, items, (items.total + kThreads * kItems - 1) / (kThreads * kItems));
    count_launches(1);
  }
}

template <typename T>
void launch_write(const void *x_, int64_t ld, int64_t n, int64_t n_end, int width, void *codes, void *scales, const Claims &claims,
                  cudaStream_t st) {
  const int groups = groups_of(width);
  const T *x = static_cast<const T *>(x_);
  in_pieces(n_end, static_cast<uint32_t>(groups * kSharing<T>), [&](int64_t r, int64_t rows, const Items &items, unsigned blocks) {
    const int64_t have = n - r < rows ? n - r : rows, at = claims.index != nullptr ? 0 : r;
    Claims mine = claims;
    if (mine.index != nullptr) mine.index += r;
    auto go = [&](auto kernel) {
      launch_dependent(kernel, blocks, kThreads, 0, st, x + (have > 0 ? r * ld : 0), ld, static_cast<uint32_t>(have > 0 ? have : 0),
                       static_cast<uint32_t>(width), items, static_cast<uint8_t *>(codes) + at * groups * kGroup,
                       static_cast<uint8_t *>(scales) + at * groups, mine, static_cast<uint32_t>(r));
    };
    const Access a = access_of<T>(x + (have > 0 ? r * ld : 0), ld, width);
    a == kWide ? go(rows8_write<T, kWide>) : a == kVector ? go(rows8_write<T, kVector>) : go(rows8_write<T, kShifted>);
  });
}

template <typename T>
void launch_read(const void *codes, const void *scales, int64_t n_rows, int width, const int64_t *index, int64_t n, void *out_,
                 int64_t ld, cudaStream_t st) {
  const int groups = groups_of(width);
  T *out = static_cast<T *>(out_);
  if (access_of<T>(out, ld, width) == kShifted && ld == width && width >= 16 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    // pieces of a multiple of 16 rows start on whole vectors
    const int64_t most = kMostItems / width / 16 * 16;
    for (int64_t r = 0; r < n; r += most) {
      const int64_t rows = n - r < most ? n - r : most, at = index != nullptr ? 0 : r;
      const Items values{static_cast<uint32_t>(rows * width), static_cast<uint32_t>(width), static_cast<uint32_t>((1ull << 32) / width)};
      constexpr uint32_t kBlock = kThreads * 2 * Vec<T>::kElems;
      launch_dependent(rows8_read_flat<T>, (values.total + kBlock - 1) / kBlock, kThreads, 0, st,
                       static_cast<const uint8_t *>(codes) + at * groups * kGroup, static_cast<const uint8_t *>(scales) + at * groups,
                       n_rows - at, static_cast<uint32_t>(groups), index != nullptr ? index + r : nullptr, values, out + r * width);
      count_launches(1);
    }
    return;
  }
  in_pieces(n, static_cast<uint32_t>((width + kRead - 1) / kRead), [&](int64_t r, int64_t rows, const Items &items, unsigned blocks) {
    const int64_t at = index != nullptr ? 0 : r;
    auto go = [&](auto kernel) {
      launch_dependent(kernel, blocks, kThreads, 0, st, static_cast<const uint8_t *>(codes) + at * groups * kGroup,
                       static_cast<const uint8_t *>(scales) + at * groups, n_rows - at, static_cast<uint32_t>(width),
                       static_cast<uint32_t>(groups), index != nullptr ? index + r : nullptr, items, out + r * ld, ld);
    };
    const Access a = access_of<T>(out + r * ld, ld, width);
    a == kWide ? go(rows8_read<T, kWide>) : a == kVector ? go(rows8_read<T, kVector>) : go(rows8_read<T, kShifted>);
  });
}

// What every entry point asks of a matrix of `width` columns.
bool bad_matrix(int dtype, int64_t ld, int64_t n, int width) {
  return n < 0 || width <= 0 || width > (1 << 20) || ld < width || (dtype != CXG_F32 && dtype != CXG_BF16);
}

}  // namespace
}  // namespace cxg

using namespace cxg;

extern "C" int cxg_rows8_pitch(int width) { return rows8::groups_of(width) * rows8::kGroup; }

extern "C" int cxg_rows8_write(const void *x, int dtype, int64_t ld, int64_t n, int width, void *codes, void *scales, int zero_row,
                               void *stream) {
  CXG_REQUIRE(!bad_matrix(dtype, ld, n, width), CXG_EINVAL, "cxg_rows8_write: bad sizes or type");
  const int64_t n_end = n + (zero_row ? 1 : 0);
  if (n_end == 0) return CXG_OK;
  CXG_REQUIRE(codes && scales && (x || n == 0), CXG_ENULL, "cxg_rows8_write: NULL argument");
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, CXG_EINVAL, "cxg_rows8_write: codes must be 16-byte aligned");
  if (dtype == CXG_F32)
    launch_write<float>(x, ld, n, n_end, width, codes, scales, Claims{}, as_stream(stream));
  else
    launch_write<__nv_bfloat16>(x, ld, n, n_end, width, codes, scales, Claims{}, as_stream(stream));
  return check_launch("cxg_rows8_write");
}

extern "C" int cxg_rows8_write_at(const void *x, int dtype, int64_t ld, int64_t n, int width, const int64_t *index, void *codes,
                                  void *scales, int64_t rows, void *claims, void *stream) {
  CXG_REQUIRE(!bad_matrix(dtype, ld, n, width) && rows >= 0, CXG_EINVAL, "cxg_rows8_write_at: bad sizes or type");
  if (n == 0) return CXG_OK;
  CXG_REQUIRE(x && index && codes && scales && claims, CXG_ENULL, "cxg_rows8_write_at: NULL argument");
  CXG_REQUIRE(n <= INT32_MAX, CXG_ELIMIT, "cxg_rows8_write_at: %lld rows, at most 2^31 - 1", static_cast<long long>(n));
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(claims) % 8 == 0, CXG_EINVAL,
              "cxg_rows8_write_at: codes must be 16-byte aligned, claims 8-byte");
  cudaStream_t st = as_stream(stream);
  const Claims c{index, static_cast<int32_t *>(claims), rows};
  const unsigned grid = static_cast<unsigned>((n + kThreads * kClaims - 1) / (kThreads * kClaims));
  const cudaError_t e = launch_dependent(rows8_claim, grid, kThreads, 0, st, c, n);
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_write_at: %s", cudaGetErrorString(e));
  if (dtype == CXG_F32)
    launch_write<float>(x, ld, n, n, width, codes, scales, c, st);
  else
    launch_write<__nv_bfloat16>(x, ld, n, n, width, codes, scales, c, st);
  count_launches(1);
  return check_launch("cxg_rows8_write_at");
}

extern "C" int cxg_rows8_read(const void *codes, const void *scales, int64_t rows, int width, const int64_t *index, int64_t n,
                              void *out, int dtype, int64_t ld, void *stream) {
  CXG_REQUIRE(!bad_matrix(dtype, ld, n, width) && rows >= 0, CXG_EINVAL, "cxg_rows8_read: bad sizes or type");
  CXG_REQUIRE(index != nullptr || n <= rows, CXG_EINVAL, "cxg_rows8_read: %lld rows of %lld", static_cast<long long>(n),
              static_cast<long long>(rows));
  if (n == 0) return CXG_OK;
  CXG_REQUIRE(codes && scales && out, CXG_ENULL, "cxg_rows8_read: NULL argument");
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, CXG_EINVAL, "cxg_rows8_read: codes must be 16-byte aligned");
  if (dtype == CXG_F32)
    launch_read<float>(codes, scales, rows, width, index, n, out, ld, as_stream(stream));
  else
    launch_read<__nv_bfloat16>(codes, scales, rows, width, index, n, out, ld, as_stream(stream));
  return check_launch("cxg_rows8_read");
}
