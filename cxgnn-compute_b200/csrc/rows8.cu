// Writing and reading rows in 8 bits (rows8.cuh has the format): activations that a backward pass needs again, and caches of
// features or of hidden states that are written and read by node id.
//
// Both directions are bound by memory. A lane takes the 16 bytes of one access on the side of the wide type: 4 fp32 or 8 bf16
// values, so 8 or 4 lanes share a group of 32 and find its largest value in 3 or 2 shuffles. Lanes go along rows without
// regard to where these end (the row of an item comes from a multiplication), so that no lane of a warp is idle for a width
// that is no power of two, and every lane has several items in flight.
#include "rows8.cuh"

namespace cxg {
namespace {

using namespace rows8;

constexpr int kThreads = 256;

template <typename T>
struct Pack {
  static constexpr int kN = 16 / static_cast<int>(sizeof(T));  // values per lane
  static constexpr int kLanes = kGroup / kN;                   // lanes per group
};

// Up to kN values of a row from column c on; zeros behind the row.
template <typename T, bool VEC>
__device__ __forceinline__ void load_values(float *f, const T *row, int c, int width) {
  constexpr int N = Pack<T>::kN;
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = 0.f;
  if (VEC) {
    if (c < width) Vec<T>::to_float(f, Vec<T>::load(row + c));  // width is a multiple of N
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < width) f[i] = to_f32(__ldg(row + c + i));
  }
}

// Rows [0, n) of x to the rows `to` names (itself without it; negative: nowhere); rows [n, n_end) are written as zeros.
// owner: the row's entry is given back (write_at).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) rows8_write(const T *x, int64_t ld, int64_t n, int64_t n_end, int width, Rows rows,
                                                        uint8_t *codes, uint8_t *scales, const int64_t *to, int32_t *owner) {
  constexpr int N = Pack<T>::kN, L = Pack<T>::kLanes;
  constexpr int kItems = 4;
  dependency_wait();
  const int groups = static_cast<int>(rows.per) / L;
  const uint64_t total = static_cast<uint64_t>(n_end) * rows.per;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kThreads;
  for (uint64_t i0 = blockIdx.x * static_cast<uint64_t>(kThreads) + (threadIdx.x & ~31u); i0 < total; i0 += kItems * step) {
    float f[kItems][N];
    int64_t row[kItems], dst[kItems];
    int chunk[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const uint64_t i = i0 + k * step + (threadIdx.x & 31);
      row[k] = i < total ? rows.row(i) : n_end;
      chunk[k] = static_cast<int>(i - static_cast<uint64_t>(row[k]) * rows.per);
      dst[k] = row[k] < n_end ? row[k] : -1;
      if (to != nullptr && row[k] < n) dst[k] = __ldg(to + row[k]);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      load_values<T, VEC>(f[k], x + (row[k] < n ? row[k] : 0) * ld, row[k] < n ? chunk[k] * N : width, width);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) top = max(top, __float_as_uint(f[k][j]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < L; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const uint32_t e = scale_byte(top);
      const float inv = e == kNotFinite ? 0.f : inverse_scale(e);
      uint32_t w[N / 4];
#pragma unroll
      for (int j = 0; j < N / 4; ++j)
        w[j] = e == kNotFinite ? 0u : pack_codes(code_bits(f[k][4 * j], inv), code_bits(f[k][4 * j + 1], inv),
                                                 code_bits(f[k][4 * j + 2], inv), code_bits(f[k][4 * j + 3], inv));
      if (dst[k] < 0) continue;
      uint8_t *out = codes + dst[k] * (static_cast<int64_t>(groups) * kGroup) + chunk[k] * N;
      if constexpr (N == 4)
        *reinterpret_cast<uint32_t *>(out) = w[0];
      else
        *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[N / 4 - 1]);
      if (chunk[k] % L == 0) scales[dst[k] * groups + chunk[k] / L] = static_cast<uint8_t>(e);
      if (owner != nullptr && chunk[k] == 0) owner[dst[k]] = -1;
    }
  }
}

// Of the positions that name the same row the last one counts: each enters itself in the row's word, then looks whether it is
// still there. The words are -1 between calls (rows8_write puts them back).
__global__ void __launch_bounds__(kThreads) rows8_claim(const int64_t *index, int64_t n, int64_t rows, int32_t *owner) {
  dependency_wait();
  const int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  if (i >= n) return;
  const int64_t r = index[i];
  if (r >= 0 && r < rows) atomicMax(owner + r, static_cast<int32_t>(i));
}
__global__ void __launch_bounds__(kThreads) rows8_settle(const int64_t *index, int64_t n, int64_t rows, const int32_t *owner,
                                                         int64_t *to) {
  dependency_wait();
  const int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  if (i >= n) return;
  const int64_t r = index[i];
  to[i] = r >= 0 && r < rows && owner[r] == static_cast<int32_t>(i) ? r : -1;
}

// out[i] = the values of row index[i] (of row i without an index; ids outside the rows read as zeros).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) rows8_read(const uint8_t *codes, const uint8_t *scales, int64_t n_rows, int width,
                                                       int groups, const int64_t *index, int64_t n, Rows rows, T *out, int64_t ld) {
  constexpr int N = Pack<T>::kN, L = Pack<T>::kLanes;
  constexpr int kItems = 4;
  dependency_wait();
  const uint64_t total = static_cast<uint64_t>(n) * rows.per;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kThreads;
  for (uint64_t i0 = blockIdx.x * static_cast<uint64_t>(kThreads) + threadIdx.x; i0 < total; i0 += kItems * step) {
    int64_t row[kItems], src[kItems];
    int chunk[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const uint64_t i = i0 + k * step;
      row[k] = i < total ? rows.row(i) : -1;
      chunk[k] = row[k] < 0 ? 0 : static_cast<int>(i - static_cast<uint64_t>(row[k]) * rows.per);
      src[k] = row[k] < 0 ? n_rows : index != nullptr ? __ldg(index + row[k]) : row[k];
      if (static_cast<uint64_t>(src[k]) > static_cast<uint64_t>(n_rows)) src[k] = n_rows;  // the row of zeros
    }
    uint32_t w[kItems][N / 4], e[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const uint8_t *p = codes + src[k] * (static_cast<int64_t>(groups) * kGroup) + chunk[k] * N;
      if constexpr (N == 4) {
        w[k][0] = __ldg(reinterpret_cast<const uint32_t *>(p));
      } else {
        const uint2 t = __ldg(reinterpret_cast<const uint2 *>(p));
        w[k][0] = t.x, w[k][N / 4 - 1] = t.y;
      }
      e[k] = __ldg(scales + src[k] * groups + chunk[k] / L);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (row[k] < 0) continue;
      const float s = scale_of(e[k]);
      float f[N];
#pragma unroll
      for (int j = 0; j < N / 4; ++j) code_values(f + 4 * j, w[k][j]);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= s;
      T *o = out + row[k] * ld + chunk[k] * N;
      const int left = width - chunk[k] * N;
      if (VEC) {
        if (left > 0) Vec<T>::store_stream(o, Vec<T>::from_float(f));
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < left) o[j] = from_f32<T>(f[j]);
      }
    }
  }
}

unsigned grid_of(uint64_t items, int per_thread) {
  const uint64_t want = (items + kThreads * per_thread - 1) / (kThreads * per_thread);
  const uint64_t most = static_cast<uint64_t>(kNumSM) * 8;
  return static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
}

template <typename T>
bool whole_vectors(const void *p, int64_t ld, int width) {
  return (reinterpret_cast<uintptr_t>(p) | (static_cast<uint64_t>(ld) * sizeof(T)) | (static_cast<uint64_t>(width) * sizeof(T))) % 16 == 0;
}

template <typename T>
void launch_write(const void *x, int64_t ld, int64_t n, int64_t n_end, int width, void *codes, void *scales, const int64_t *to,
                  int32_t *owner, cudaStream_t st) {
  const Rows rows(static_cast<uint32_t>(groups_of(width) * Pack<T>::kLanes));
  const unsigned grid = grid_of(static_cast<uint64_t>(n_end) * rows.per, 4);
  auto go = [&](auto kernel) {
    launch_dependent(kernel, grid, kThreads, 0, st, static_cast<const T *>(x), ld, n, n_end, width, rows,
                     static_cast<uint8_t *>(codes), static_cast<uint8_t *>(scales), to, owner);
  };
  whole_vectors<T>(x, ld, width) ? go(rows8_write<T, true>) : go(rows8_write<T, false>);
}

template <typename T>
void launch_read(const void *codes, const void *scales, int64_t n_rows, int width, const int64_t *index, int64_t n, void *out,
                 int64_t ld, cudaStream_t st) {
  const Rows rows(static_cast<uint32_t>((width + Pack<T>::kN - 1) / Pack<T>::kN));
  const unsigned grid = grid_of(static_cast<uint64_t>(n) * rows.per, 4);
  auto go = [&](auto kernel) {
    launch_dependent(kernel, grid, kThreads, 0, st, static_cast<const uint8_t *>(codes), static_cast<const uint8_t *>(scales),
                     n_rows, width, groups_of(width), index, n, rows, static_cast<T *>(out), ld);
  };
  whole_vectors<T>(out, ld, width) ? go(rows8_read<T, true>) : go(rows8_read<T, false>);
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
    launch_write<float>(x, ld, n, n_end, width, codes, scales, nullptr, nullptr, as_stream(stream));
  else
    launch_write<__nv_bfloat16>(x, ld, n, n_end, width, codes, scales, nullptr, nullptr, as_stream(stream));
  count_launches(1);
  return check_launch("cxg_rows8_write");
}

extern "C" int cxg_rows8_write_at_workspace_size(int64_t n, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_rows8_write_at_workspace_size: bytes is NULL");
  CXG_REQUIRE(n >= 0, CXG_EINVAL, "cxg_rows8_write_at_workspace_size: bad size");
  *bytes = static_cast<size_t>(n) * sizeof(int64_t);
  return CXG_OK;
}

extern "C" int cxg_rows8_write_at(const void *x, int dtype, int64_t ld, int64_t n, int width, const int64_t *index, void *codes,
                                  void *scales, int64_t rows, int32_t *owner, void *workspace, size_t workspace_bytes,
                                  void *stream) {
  CXG_REQUIRE(!bad_matrix(dtype, ld, n, width) && rows >= 0, CXG_EINVAL, "cxg_rows8_write_at: bad sizes or type");
  if (n == 0) return CXG_OK;
  CXG_REQUIRE(x && index && codes && scales && owner, CXG_ENULL, "cxg_rows8_write_at: NULL argument");
  CXG_REQUIRE(n <= INT32_MAX, CXG_ELIMIT, "cxg_rows8_write_at: %lld rows, at most 2^31 - 1", static_cast<long long>(n));
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, CXG_EINVAL, "cxg_rows8_write_at: codes must be 16-byte aligned");
  CXG_REQUIRE(workspace != nullptr && workspace_bytes >= n * sizeof(int64_t) && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
              CXG_EWORKSPACE, "cxg_rows8_write_at: workspace %zu bytes, need %zu", workspace_bytes, n * sizeof(int64_t));
  cudaStream_t st = as_stream(stream);
  int64_t *to = static_cast<int64_t *>(workspace);
  const unsigned grid = static_cast<unsigned>((n + kThreads - 1) / kThreads);
  launch_dependent(rows8_claim, grid, kThreads, 0, st, index, n, rows, owner);
  launch_dependent(rows8_settle, grid, kThreads, 0, st, index, n, rows, owner, to);
  if (dtype == CXG_F32)
    launch_write<float>(x, ld, n, n, width, codes, scales, to, owner, st);
  else
    launch_write<__nv_bfloat16>(x, ld, n, n, width, codes, scales, to, owner, st);
  count_launches(3);
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
  count_launches(1);
  return check_launch("cxg_rows8_read");
}
