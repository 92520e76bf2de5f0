// Aggregation over rows in 8 bits: y[d, :] = red over the edges e of row d of v[e] * codes[s(e), :] * scale[s(e), group].
//
// The walk of spmm_walk_impl.cuh with rows of a quarter of the bytes: tiles of edges from the same plan, a group of G lanes per
// tile, 32 / G tiles side by side in a warp, U edges in flight per lane, sums in edge order in one fp32 accumulator per
// column, partials of rows that cross tiles added by the same fix-up. Same bits on every run.
//
// A lane holds VB codes of a row, which lie in one group of 32 and share a scale. A code becomes fp32 by a byte permutation
// and an addition (rows8.cuh); code * scale is exact, and so is scale * v (a power of two) but where it falls below the normal
// numbers, so each edge rounds once, in the addition. Tiles with an edge value that could take scale * v out of range are walked
// once more, edge by edge, if it does (walk_carefully). (Two codes cost 2 permutations, a packed addition and a packed
// multiplication-addition; converting with the conversion instruction would cost a quarter-rate instruction per code.)
//
// Measured: 169,343 rows of 128, 2.3 M edges, mean, bf16 99 us (gathered: 3.1 TB/s); 1.94 M rows of 100, 21 M edges with values, fp32
// 773 us (3.6 TB/s). Bound by instructions and latency together: an edge of 128 columns takes 18 warp instructions, 10 of them
// to unpack it, a row's end about 80; with codes taken as they are the two graphs take 83 and 676 us.
#include <type_traits>

#include "rows8.cuh"
#include "spmm_walk_impl.cuh"

namespace cxg {
namespace {

using namespace rows8;
using walk::kFar;
using walk::kThreads;

struct Rows8Args {
  WalkArgs w;  // ptr, idx, y, edge_val, plan and partials; width: columns, row_bytes: pitch of the codes
  const uint8_t *codes, *scales;
  int64_t n_src;  // rows; ids outside stand for the row of zeros behind the last
  int groups;
  int whole;  // 2: rows of y are whole 16-byte vectors, 1: 8-byte ones
  bool staged;   // STAGED
  uint2 *marks;  // SPARSE: per edge that is the first of its row, that row and its end
};

// For graphs of mostly empty rows: y is zeroed here, and the walk goes from a row to the next one that has edges.
template <typename T>
__global__ void __launch_bounds__(256) rows8_mark(const __grid_constant__ Rows8Args r) {
  const WalkArgs &a = r.w;
  dependency_wait();
  const int64_t i0 = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll;
  const uint32_t e_total = static_cast<uint32_t>(edge_total(a));
  for (int64_t i = i0; i < a.n_dst; i += step) {
    const int row = static_cast<int>(i);
    const uint32_t b = walk::load_ptr_low(a.ptr, row, a.ptr_bytes), e = walk::load_ptr_low(a.ptr, row + 1, a.ptr_bytes);
    if (b < e && b < e_total) r.marks[b] = make_uint2(static_cast<uint32_t>(i), e);
  }
  const int64_t values = a.n_dst * a.width;
  constexpr int N = Vec<T>::kElems;
  T *y = static_cast<T *>(a.y);
  const int64_t vectors = reinterpret_cast<uintptr_t>(y) % 16 == 0 ? values / N : 0;
  for (int64_t i = i0; i < vectors; i += step) *reinterpret_cast<uint4 *>(y + i * N) = make_uint4(0, 0, 0, 0);
  for (int64_t i = vectors * N + i0; i < values; i += step) y[i] = from_f32<T>(0.f);
}

template <int VB>
struct Codes {
  static constexpr int W = VB / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const uint8_t *p) {
    if constexpr (VB == 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (VB == 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    }
  }
};

// acc[2i], acc[2i + 1] += codes * s
template <int VB>
__device__ __forceinline__ void add_codes(unsigned long long *acc, const Codes<VB> &c, float s) {
  unsigned long long ss, bias;
  asm("mov.b64 %0, {%1,%1};" : "=l"(ss) : "f"(s));
  asm("mov.b64 %0, {%1,%1};" : "=l"(bias) : "f"(-8388736.f));
#pragma unroll
  for (int i = 0; i < VB / 4; ++i) {
    const uint32_t w = c.w[i];
    const uint32_t a = __byte_perm(w, 0x4b000000u, 0x7440), b = __byte_perm(w, 0x4b000000u, 0x7441),
                   d = __byte_perm(w, 0x4b000000u, 0x7442), e = __byte_perm(w, 0x4b000000u, 0x7443);
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1,%2};\n\tadd.rn.f32x2 t, t, %3;\n\tfma.rn.f32x2 %0, t, %4, %0;\n\t}"
        : "+l"(acc[2 * i])
        : "r"(a), "r"(b), "l"(bias), "l"(ss));
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1,%2};\n\tadd.rn.f32x2 t, t, %3;\n\tfma.rn.f32x2 %0, t, %4, %0;\n\t}"
        : "+l"(acc[2 * i + 1])
        : "r"(d), "r"(e), "l"(bias), "l"(ss));
  }
}

__device__ __forceinline__ int end_in_tile(uint32_t raw, uint32_t begin) {
  return raw - begin > static_cast<uint32_t>(kFar) ? kFar : static_cast<int>(raw - begin);
}

// Whether a finite value takes one of the finite scales of a word out of range.
__device__ __forceinline__ bool out_of_range(uint32_t bytes, float v) {
  bytes &= ~__vcmpeq4(bytes, 0xffffffffu);
  const uint32_t top = max(max(bytes & 255u, (bytes >> 8) & 255u), max((bytes >> 16) & 255u, bytes >> 24));
  return fabsf(v) < __uint_as_float(0x7f800000u) && __float_as_uint(scale_of(top) * fabsf(v)) == 0x7f800000u;
}

// A tile of rows8_walk with edge values of kSafeValue or more: looks (unless SEEN: where the walk has) whether one of them takes a
// scale of its row out of range, a lane per edge, and if so walks the tile once more: the same lanes, sums in the same order, but
// with keep_zeros at every edge. (A function of its own, which leaves the walk its registers: the walk takes up to 3 % longer for
// it, with a test per step inside it took 3 to 14 %, with a second walk inside the kernel 2 to 8 %, with a test of the sums for NaN
// 6 %. Where all values are that large, looking takes 10 to 15 %, in the walk itself 2 %.)
template <typename T, int VB, int G, int NV, bool SPARSE, bool SEEN>
__device__ __noinline__ void walk_carefully(const Rows8Args &r, int t, int n_tiles) {
  const WalkArgs &a = r.w;
  const int lg = static_cast<int>(threadIdx.x) & (G - 1), n_dst = static_cast<int>(a.n_dst);
  const uint64_t pitch = static_cast<uint32_t>(a.row_bytes), groups = static_cast<uint32_t>(r.groups);
  WalkTile here = {};
  int len = 0;
  if (t < n_tiles) {
    here = load_tile(a, t);
    len = static_cast<int>(load_tile(a, t + 1).begin - here.begin);
  }
  const uint32_t begin = here.begin;
  auto row_of = [&](uint32_t edge) -> uint64_t {
    const int64_t id = a.idx_bytes == 8 ? __ldg(static_cast<const int64_t *>(a.idx) + edge)
                                        : static_cast<int64_t>(__ldg(static_cast<const int32_t *>(a.idx) + edge));
    return static_cast<uint64_t>(id) < static_cast<uint64_t>(r.n_src) ? id : r.n_src;
  };
  if constexpr (!SEEN) {
    bool out = false;
    constexpr int kDeep = 4;  // edges of a lane at once
    for (int first = lg; first < len; first += kDeep * G) {
      float v[kDeep];
      uint64_t id[kDeep];
      uint32_t top[kDeep] = {};  // the largest bytes of finite groups
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const bool on = first + u * G < len;
        v[u] = on ? __ldg(a.edge_val + begin + first + u * G) : 0.f;
        id[u] = on ? row_of(begin + first + u * G) : static_cast<uint64_t>(r.n_src);
        if (fabsf(v[u]) < kSafeValue) id[u] = static_cast<uint64_t>(r.n_src);
      }
      auto take = [&](int u, uint32_t bytes) { top[u] = __vmaxu4(top[u], bytes & ~__vcmpeq4(bytes, 0xffffffffu)); };
      if (groups % 4 == 0) {
        for (uint32_t g = 0; g < groups; g += 4)
#pragma unroll
          for (int u = 0; u < kDeep; ++u) take(u, __ldg(reinterpret_cast<const uint32_t *>(r.scales + id[u] * groups + g)));
      } else {
        for (uint32_t g = 0; g < groups; ++g)
#pragma unroll
          for (int u = 0; u < kDeep; ++u) take(u, __ldg(r.scales + id[u] * groups + g));
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) out = out || out_of_range(top[u], v[u]);
    }
    if (!__any_sync(0xffffffffu, out)) return;
  }
  __syncwarp();  // what this warp has stored of the tile is replaced
  int row = static_cast<int>(here.row), rend = row < n_dst ? end_in_tile(here.row_end, begin) : kFar;
  bool whole = here.row_begin >= begin;  // the row began in this tile
  unsigned long long acc[NV][VB / 2] = {};
  for (int pos = 0; pos < len; ++pos) {
    const uint64_t id = row_of(begin + pos);
    const float v = __ldg(a.edge_val + begin + pos);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int at = min((lg + q * G) * VB, a.row_bytes - VB);
      Codes<VB> c;
      c.load(r.codes + id * pitch + at);
      const uint32_t e = keep_zeros<VB / 4>(c.w, __ldg(r.scales + id * groups + at / kGroup), v);
      add_codes<VB>(acc[q], c, scale_of(e) * v);
    }
    const bool row_done = pos + 1 == rend;
    if (!row_done && pos + 1 < len) continue;
    T *y = static_cast<T *>(a.y) + static_cast<int64_t>(row) * a.width;
    float *p = a.partials + (static_cast<int64_t>(t) * 2 + (whole ? 1 : 0)) * a.part_stride;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < VB / 2; ++i) {
        const float2 f = halves(acc[q][i]);
        acc[q][i] = 0;
        const int col = (lg + q * G) * VB + 2 * i;
        if (row_done && whole) {
          if (col < a.width) y[col] = from_f32<T>(f.x);
          if (col + 1 < a.width) y[col + 1] = from_f32<T>(f.y);
        } else if (row < n_dst && col < a.part_stride) {
          *reinterpret_cast<float2 *>(p + col) = f;
        }
      }
    if (!row_done || pos + 1 == len) continue;
    whole = true;
    if constexpr (SPARSE) {
      const uint2 mark = __ldg(r.marks + begin + rend);
      row = static_cast<int>(min(mark.x, static_cast<uint32_t>(n_dst)));
      rend = row < n_dst ? end_in_tile(mark.y, begin) : kFar;
    } else {
      do {  // rows without edges have been written
        ++row;
        rend = row < n_dst ? end_in_tile(walk::load_ptr_low(a.ptr, row + 1, a.ptr_bytes), begin) : kFar;
      } while (rend == pos + 1);
    }
  }
}

// VALMODE: 0 sum, 1 a value per edge, 3 mean. WORDS: the (up to four) scales of an edge's row as one word, fetched with the ids by
// one lane per edge; otherwise every lane fetches its own with the codes.
// SPARSE: rows without edges have been written, the next one with edges is in r.marks. STAGED: bf16 rows that are no whole vectors
// go through shared memory, so that lanes write words side by side. (Value by value / staged, us: 278,000 rows with 1.6 M edges,
// width 99 190 / 146, 149 273 / 187, 301 550 / 269; 663,000 rows with 9.9 M edges 99 399 / 478, 149 607 / 677, 301 1130 / 1076: for
// graphs of few edges per row. Rows of up to 64, in vectors of 4 or 8 codes, have nothing to gain.)
template <typename T, int VB, int G, int NV, int U, int VALMODE, int MINB, bool WORDS, bool SPARSE, bool STAGED>
__global__ void __launch_bounds__(kThreads, MINB) rows8_walk(const __grid_constant__ Rows8Args r) {
  const WalkArgs &a = r.w;
  constexpr int NG = 32 / G;
  const int lane = threadIdx.x & 31;
  const int lg = lane & (G - 1);
  dependency_wait();
  const uint32_t e_total = static_cast<uint32_t>(edge_total(a));
  const int n_dst = static_cast<int>(a.n_dst);
  const int n_tiles = static_cast<int>((e_total + static_cast<int64_t>(a.tile) - 1) / a.tile);
  const int step = static_cast<int>(gridDim.x) * (kThreads / 32) * NG;  // tiles that are walked at the same time
  const uint32_t pitch = static_cast<uint32_t>(a.row_bytes), groups = static_cast<uint32_t>(r.groups);
  // codes [(lg + q * G) * VB, +VB) of a row; a lane behind the row reads its neighbours' line again and stores nothing
  const uint8_t *cq[NV], *sq[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int c = (lg + q * G) * VB, at = c < static_cast<int>(pitch) ? c : static_cast<int>(pitch) - VB;
    cq[q] = r.codes + at, sq[q] = r.scales + at / kGroup;
  }
  auto col = [&](int q) { return (lg + q * G) * VB; };

  [[maybe_unused]] __shared__ __align__(16) T out_stage[STAGED ? kThreads * VB : 1];
  [[maybe_unused]] T *const my_out = out_stage + (STAGED ? threadIdx.x / G * (G * VB) : 0);
  const unsigned members = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1) << (lane / G * G);
  // the group's row of bf16, column c from value(c), in whole words
  [[maybe_unused]] auto write_words = [&](T *y, auto value) {
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(y) >> 1) & 1;
    for (int c = 2 * lg - odd; c < a.width; c += 2 * G) {
      const bool lower = c >= 0, upper = c + 1 < a.width;
      const T first = value(lower ? c : 0), second = value(upper ? c + 1 : 0);
      if (lower && upper)
        *reinterpret_cast<uint32_t *>(y + c) =
            static_cast<uint32_t>(__bfloat16_as_ushort(first)) | static_cast<uint32_t>(__bfloat16_as_ushort(second)) << 16;
      else if (lower)
        y[c] = first;
      else if (upper)
        y[c + 1] = second;
    }
  };
  auto store = [&](int row, float (&f)[NV][VB]) {
    T *y = static_cast<T *>(a.y) + static_cast<int64_t>(row) * a.width;
    if constexpr (STAGED) {
      __syncwarp(members);  // the row before has been read
#pragma unroll
      for (int i = 0; i < VB; i += 2) *reinterpret_cast<__nv_bfloat162 *>(my_out + lg * VB + i) = __floats2bfloat162_rn(f[0][i], f[0][i + 1]);
      __syncwarp(members);
      write_words(y, [&](int c) { return my_out[c]; });
      return;
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      auto vectors = [&](auto bytes) {  // VB values in vectors of so many bytes, or the whole of them where they are fewer
        constexpr int kAll = VB * static_cast<int>(sizeof(T)), kBytes = decltype(bytes)::value < kAll ? decltype(bytes)::value : kAll;
        constexpr int N = kBytes / static_cast<int>(sizeof(T));
#pragma unroll
        for (int i = 0; i < VB; i += N)
          if (col(q) + i < a.width) walk::store_row_bytes<T, kBytes>(reinterpret_cast<uint8_t *>(y + col(q) + i), f[q] + i);
      };
      if (r.whole == 2) {
        vectors(std::integral_constant<int, 16>());
      } else if (r.whole == 1) {
        vectors(std::integral_constant<int, 8>());
      } else {
#pragma unroll
        for (int i = 0; i < VB; ++i)
          if (col(q) + i < a.width) y[col(q) + i] = from_f32<T>(f[q][i]);
      }
    }
  };
  auto zero_row = [&](int row) {
    if constexpr (STAGED) {
      write_words(static_cast<T *>(a.y) + static_cast<int64_t>(row) * a.width, [](int) { return from_f32<T>(0.f); });
      return;
    }
    float z[NV][VB];
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < VB; ++i) z[q][i] = 0.f;
    store(row, z);
  };
  const int t_first = static_cast<int>((blockIdx.x * static_cast<unsigned>(kThreads) + threadIdx.x) / G);
  if (e_total == 0) {  // no edge at all: every row is empty
    if constexpr (SPARSE) return;
    for (int row = t_first; row < n_dst; row += step) zero_row(row);
    return;
  }

  // ids and edge values of a batch of 32 edges per group (as in spmm_walk)
  constexpr int kBatch = 36;
  constexpr bool kWords = WORDS;
  static_assert(!WORDS || (G == 8 && NV == 1), "rows of up to 128 codes");
  __shared__ __align__(16) uint32_t scale_stage[kWords ? kThreads / 32 : 1][kWords ? NG * kBatch : 4];
  uint32_t *my_scales = kWords ? scale_stage[threadIdx.x >> 5] + lane / G * kBatch : nullptr;
  const int to_exponent = (23 - 8 * (lg * VB / kGroup)) & 31;  // rotation that takes the lane's scale to the exponent's place
  auto scale_word = [&](uint32_t id) -> uint32_t {
    if constexpr (VB == 4) return __ldg(r.scales + id);
    if constexpr (VB == 8) return __ldg(reinterpret_cast<const uint16_t *>(r.scales) + id);
    if (groups == 4) return __ldg(reinterpret_cast<const uint32_t *>(r.scales) + id);
    const uint8_t *p = r.scales + static_cast<uint64_t>(id) * groups;
    return __ldg(p) | __ldg(p + 1) << 8 | __ldg(p + 2) << 16;
  };
  __shared__ __align__(16) uint32_t id_stage[kThreads / 32][NG * kBatch];
  __shared__ __align__(16) float val_stage[VALMODE == 1 ? kThreads / 32 : 1][VALMODE == 1 ? NG * kBatch : 4];
  uint32_t *my_ids = id_stage[threadIdx.x >> 5] + lane / G * kBatch;
  float *my_vals = VALMODE == 1 ? val_stage[threadIdx.x >> 5] + lane / G * kBatch : nullptr;
  int t_next = 0;
  for (int t = t_first; t - lane / G < n_tiles; t = t_next) {
    t_next = n_tiles;
    if (step < n_tiles) {
      if (lane == 0) t_next = step + atomicAdd(a.hdr + kWalkHdrNext, NG);
    }
    uint32_t begin = 0, row_begin = 0, row_end = 0;
    int row = 0, len = 0;
    if (t < n_tiles) {
      const WalkTile here = load_tile(a, t);
      begin = here.begin, row_begin = here.row_begin, row_end = here.row_end;
      row = static_cast<int>(here.row);
      len = static_cast<int>(load_tile(a, t + 1).begin - begin);
    }

    constexpr int IB = 32 / G;
    uint32_t id_nxt[IB];
    float val_nxt[IB];
    auto load_batch = [&](int first) {
#pragma unroll
      for (int j = 0; j < IB; ++j) {
        const int pos = first + j * G + lg;
        id_nxt[j] = static_cast<uint32_t>(r.n_src);
        val_nxt[j] = 0.f;
        if (pos < len) {
          const uint32_t e = begin + pos;
          const uint64_t id = a.idx_bytes == 8
                                  ? static_cast<uint64_t>(walk::load_id_stream(static_cast<const int64_t *>(a.idx) + e))
                                  : static_cast<uint64_t>(static_cast<int64_t>(walk::load_id_stream(static_cast<const int32_t *>(a.idx) + e)));
          if (id < static_cast<uint64_t>(r.n_src)) id_nxt[j] = static_cast<uint32_t>(id);
          if (VALMODE == 1) val_nxt[j] = __ldg(a.edge_val + e);
        }
      }
    };

    auto end_raw = [&](int i) { return walk::load_ptr_low(a.ptr, min(i + 1, n_dst), a.ptr_bytes); };
    auto end_rel = [&](int i, uint32_t raw) -> int {
      const uint32_t v = raw - begin;
      return i >= n_dst || v > static_cast<uint32_t>(kFar) ? kFar : static_cast<int>(v);
    };
    int rend = kFar, rstart = 0, stop = kFar;
    uint32_t next_raw = 0;
    [[maybe_unused]] uint2 next_mark = make_uint2(0, 0);
    auto fetch_mark = [&]() {
      if (rend < len) next_mark = __ldg(r.marks + begin + rend);
    };
    if (len > 0) {
      if (t == 0 && !SPARSE)
        for (int i = 0; i < row; ++i) zero_row(i);  // leading rows without edges
      rstart = row_begin < begin ? -1 : 0;
      rend = end_rel(row, row_end);
      if constexpr (SPARSE)
        fetch_mark();
      else
        next_raw = end_raw(row + 1);
      stop = min(rend, len);
    }
    unsigned long long acc[NV][VB / 2];
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < VB / 2; ++i) acc[q][i] = 0ull;

    // the walk stands at a row end, at the end of the tile, or at both
    auto event = [&](int pos) {
      const bool row_done = pos == rend;
      float f[NV][VB];
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) {
          asm("mov.b64 {%0,%1}, %2;" : "=f"(f[q][2 * i]), "=f"(f[q][2 * i + 1]) : "l"(acc[q][i]));
          acc[q][i] = 0ull;
        }
      if (row_done && rstart >= 0) {
        if (VALMODE == 3) {
          // fp32: the quotient as f hi + f lo, hi + lo = 1 / count to 2^-44, which is the correctly rounded one for counts below 2^19
          // (no quotient by d is closer than 2^-25 / d to the middle of two neighbours) and sums above 2^-100. hi is a little below
          // the reciprocal, so that lo is positive and infinities stay what they are. (A division: 115 us in place of 99.) bf16, which
          // rounds to 8 bits next: by the correctly rounded reciprocal, which moves one value in 2^15 to its other neighbour (hi and
          // lo there too: 104 us).
          const float d = static_cast<float>(rend - rstart), r1 = __frcp_rn(d);
          const float hi = __uint_as_float(__float_as_uint(r1) - 1), lo = fmaf(-d, hi, 1.f) * r1;
#pragma unroll
          for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VB; ++i) f[q][i] = sizeof(T) == 4 ? fmaf(f[q][i], hi, f[q][i] * lo) : f[q][i] * r1;
        }
        store(row, f);
      } else if (row < n_dst) {
        // the row began in an earlier tile, or goes on in the next one
        float *p = a.partials + (static_cast<int64_t>(t) * 2 + (rstart < 0 ? 0 : 1)) * a.part_stride;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            if (col(q) + i < a.part_stride)
              *reinterpret_cast<float4 *>(p + col(q) + i) = make_float4(f[q][i], f[q][i + 1], f[q][i + 2], f[q][i + 3]);
      }
      if (row_done) {
        rstart = pos;
        if constexpr (SPARSE) {
          row = static_cast<int>(min(next_mark.x, static_cast<uint32_t>(n_dst)));
          rend = pos < len ? end_rel(row, next_mark.y) : kFar;
          fetch_mark();
        } else {
          for (;;) {
            ++row;
            rend = end_rel(row, next_raw);
            next_raw = end_raw(row + 1);
            if (rend != pos) break;
            zero_row(row);  // a row without edges
          }
        }
      }
      stop = pos == len ? kFar : min(rend, len);
    };

    const int longest = G == 32 ? len : __reduce_max_sync(0xffffffffu, len);
    load_batch(0);
    [[maybe_unused]] uint32_t words[IB];
    [[maybe_unused]] bool large = false;  // edge values with which scale * value is (WORDS) or may be out of range
    for (int p = 0; p < longest; p += U) {
      const int in_batch = p & 31;
      if (in_batch == 0) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < IB; ++j) {
          my_ids[j * G + lg] = id_nxt[j];
          if (VALMODE == 1) {
            my_vals[j * G + lg] = val_nxt[j];
            if (!kWords) large = large || !(fabsf(val_nxt[j]) < kSafeValue);
          }
        }
        __syncwarp();
        if constexpr (kWords) {
#pragma unroll
          for (int j = 0; j < IB; ++j) words[j] = scale_word(id_nxt[j]);
        }
        load_batch(p + 32);
      }
      Codes<VB> c[U][NV];
      uint32_t s[U][NV];
      constexpr int W4 = U < 4 ? U : 4;
      uint32_t ids[W4];
      float vals[W4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u % W4 == 0) walk::load_ids(ids, my_ids + in_batch + u);
        const uint64_t id = ids[u % W4];
#pragma unroll
        for (int q = 0; q < NV; ++q) {
          c[u][q].load(cq[q] + id * pitch);
          if constexpr (!kWords) s[u][q] = __ldg(sq[q] + id * groups);
        }
      }
      if constexpr (kWords) {
        if (in_batch == 0) {  // the words have been on their way together with the codes
#pragma unroll
          for (int j = 0; j < IB; ++j) my_scales[j * G + lg] = words[j];
          if constexpr (VALMODE == 1) {
#pragma unroll
            for (int j = 0; j < IB; ++j) {
              const float v = my_vals[j * G + lg];
              if (!(fabsf(v) < kSafeValue)) large = large || out_of_range(words[j], v);
            }
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (VALMODE == 1 && u % W4 == 0) walk::load_ids(vals, my_vals + in_batch + u);
        if constexpr (kWords) {
          if (u % W4 == 0) walk::load_ids(ids, my_scales + in_batch + u);
          s[u][0] = __funnelshift_l(ids[u % W4], ids[u % W4], to_exponent) & 0x7f800000u;
        } else {
#pragma unroll
          for (int q = 0; q < NV; ++q) s[u][q] <<= 23;
        }
#pragma unroll
        for (int q = 0; q < NV; ++q)
          add_codes<VB>(acc[q], c[u][q], VALMODE == 1 ? __uint_as_float(s[u][q]) * vals[u % W4] : __uint_as_float(s[u][q]));
        if (p + u + 1 == stop) event(p + u + 1);
      }
    }
    if constexpr (VALMODE == 1) {
      if (__any_sync(0xffffffffu, large)) walk_carefully<T, VB, G, NV, SPARSE, kWords>(r, t, n_tiles);
    }
    t_next = __shfl_sync(0xffffffffu, t_next, 0) + lane / G;
  }
}

// Lane layouts by the pitch of the codes. With resident set nothing is launched: it receives the tiles walked at the same time.
template <typename T, int VALMODE>
bool launch_pitch(const Rows8Args &r, cudaStream_t st, int *resident) {
  auto go = [&](auto kernel, int g, int ctas) {
    const int per_cta = kThreads / g;
    if (resident != nullptr) {
      *resident = kNumSM * ctas * per_cta;
      return true;
    }
    int64_t grid = (r.w.max_tiles + per_cta - 1) / per_cta;
    const int64_t most = kNumSM * ctas;
    if (grid > most) grid = most;
    return launch_dependent(kernel, static_cast<unsigned>(grid < 1 ? 1 : grid), kThreads, 0, st, r) == cudaSuccess;
  };
  constexpr bool kHalf = sizeof(T) == 2;
#define CXG_ROWS8_WALK(VB, G, NV, U, CTAS, WORDS)                                                                               \
  if (r.w.row_bytes <= VB * G * NV)                                                                                             \
  return r.marks != nullptr ? go(rows8_walk<T, VB, G, NV, U, VALMODE, CTAS, false, true, false>, G, CTAS)                       \
         : r.staged         ? go(rows8_walk<T, VB, G, NV, U, VALMODE, CTAS, WORDS, false, kHalf && VB == 16 && NV == 1>, G, CTAS) \
                            : go(rows8_walk<T, VB, G, NV, U, VALMODE, CTAS, WORDS, false, false>, G, CTAS)
  // Scales as words: 10.7 M edges, 32 columns bf16 214 -> 205 us, 100 fp32 with values 429 -> 405; 128 columns bf16 without values
  // 364 -> 374.
  CXG_ROWS8_WALK(4, 8, 1, 8, 8, true);
  CXG_ROWS8_WALK(8, 8, 1, 8, 8, true);
  CXG_ROWS8_WALK(16, 8, 1, 4, 8, VALMODE == 1);
  CXG_ROWS8_WALK(16, 16, 1, 4, 8, false);
  CXG_ROWS8_WALK(16, 32, 1, 4, 8, false);
  CXG_ROWS8_WALK(16, 32, 2, 2, 5, false);
  CXG_ROWS8_WALK(16, 32, 4, 2, 3, false);
#undef CXG_ROWS8_WALK
  return false;
}

bool dispatch(const Rows8Args &r, int out_dtype, cudaStream_t st, int *resident) {
  const int valmode = r.w.edge_val != nullptr ? 1 : r.w.reduce == CXG_MEAN ? 3 : 0;
  if (out_dtype == CXG_F32)
    return valmode == 0   ? launch_pitch<float, 0>(r, st, resident)
           : valmode == 1 ? launch_pitch<float, 1>(r, st, resident)
                          : launch_pitch<float, 3>(r, st, resident);
  return valmode == 0   ? launch_pitch<__nv_bfloat16, 0>(r, st, resident)
         : valmode == 1 ? launch_pitch<__nv_bfloat16, 1>(r, st, resident)
                        : launch_pitch<__nv_bfloat16, 3>(r, st, resident);
}

constexpr int kMostWidth = 2048;
// Graphs for one launch of clusters: one / three launches (us), mean, fp32: 13,264 edges, 33 columns 18.4 / 31.6, 256 20.4 / 31.7;
// 40,000 edges, 128 24.6 / 37.9, 256 30.7 / 37.9; 60,000, 128 28.6 / 37.9, 256 36.8 / 35.9; 84,000, 64 34.8 / 33.9. Against the
// launches for sparse graphs below: 100 columns bf16, 8192 rows and 2000 edges 22.6 / 23.3, 300 edges 67.6 / 21.6.
constexpr int64_t kSmallEdges = 65536, kSmallBytes = 12 << 20, kSmallRowsPerEdge = 4;

int tile_edges(const Rows8Args &r, int64_t nnz, int split_edges) {
  if (split_edges > 0) return split_edges;
  int resident = kNumSM * 32;
  dispatch(r, CXG_F32, nullptr, &resident);
  return walk_tile_of_waves(nnz, resident);
}

// Graphs with more rows than edges: most rows are empty, and a walk that looks at each of a tile's rows takes 0.2 us for each. (All
// rows / those with edges, us: 1.9 M rows and 1000 edges, 100 columns bf16 33,100 / 99; 300,000 and 100,000 122 / 47; 300,000
// and 300,000 77 / 63, 128 columns fp32 83 / 88; 500,000 edges 79 / 105.) With more edges than kMostMarked the tiles of one
// wave have few rows each. In small tiles, as a row's end is what takes time (64 edges: 59 us where 16 take 32); small graphs gain
// from them up to four edges per row (40,000 rows and 72,000 edges, 128 columns bf16 50 / 32; 243 columns fp32 63 / 81).
constexpr int64_t kMostMarked = 1 << 19;
bool is_sparse(int64_t n_dst, int64_t nnz, int width) {
  return (nnz <= kMostMarked && n_dst > nnz) || (nnz <= (1 << 17) && n_dst > nnz / 4 && width <= 128);
}
int sparse_tile(int64_t nnz, int width, int split_edges) {
  return split_edges > 0 ? split_edges : width > 512 ? 64 : nnz <= (1 << 18) ? 16 : 32;
}

}  // namespace
}  // namespace cxg

using namespace cxg;

extern "C" int cxg_rows8_aggregate_workspace_size(int64_t nnz, int width, int split_edges, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_rows8_aggregate_workspace_size: bytes is NULL");
  CXG_REQUIRE(nnz >= 0 && width > 0 && split_edges >= 0, CXG_EINVAL, "cxg_rows8_aggregate_workspace_size: bad sizes");
  CXG_REQUIRE(width <= kMostWidth, CXG_EUNSUPPORTED, "cxg_rows8_aggregate: rows of %d values, at most %d", width, kMostWidth);
  Rows8Args r = {};
  r.w.row_bytes = rows8::groups_of(width) * rows8::kGroup;
  WalkLayout L;
  int rc = walk_layout(nnz, walk_part_stride(width), tile_edges(r, nnz, split_edges), &L);
  if (rc != CXG_OK) return set_error(rc, "cxg_rows8_aggregate: graph too large for 32-bit tile ids");
  *bytes = L.total;
  if (nnz <= kMostMarked) {  // how many rows there are is not known here
    rc = walk_layout(nnz, walk_part_stride(width), sparse_tile(nnz, width, split_edges), &L);
    const size_t need = L.total + static_cast<size_t>(nnz) * sizeof(uint2);
    if (rc == CXG_OK && need > *bytes) *bytes = need;
  }
  return CXG_OK;
}

extern "C" int cxg_rows8_aggregate(const void *codes, const void *scales, int64_t n_src, int width, const void *ptr, int ptr_bytes,
                                   const void *idx, int idx_bytes, const float *edge_val, int64_t n_dst, int64_t nnz, int reduce,
                                   int split_edges, void *y, int y_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  CXG_REQUIRE(n_src >= 0 && width > 0 && n_dst >= 0 && nnz >= 0 && split_edges >= 0, CXG_EINVAL, "cxg_rows8_aggregate: bad sizes");
  CXG_REQUIRE((ptr_bytes == 4 || ptr_bytes == 8) && (idx_bytes == 4 || idx_bytes == 8), CXG_EINVAL,
              "cxg_rows8_aggregate: ptr and idx are of 4 or 8 bytes");
  CXG_REQUIRE(y_dtype == CXG_F32 || y_dtype == CXG_BF16, CXG_EINVAL, "cxg_rows8_aggregate: dtype %d", y_dtype);
  CXG_REQUIRE(reduce == CXG_SUM || (reduce == CXG_MEAN && edge_val == nullptr), CXG_EINVAL,
              "cxg_rows8_aggregate: a sum, or a mean without edge values");
  CXG_REQUIRE(width <= kMostWidth, CXG_EUNSUPPORTED, "cxg_rows8_aggregate: rows of %d values, at most %d", width, kMostWidth);
  constexpr int64_t most = INT32_MAX - (1 << 20);
  CXG_REQUIRE(n_dst <= most && nnz <= most && n_src < UINT32_MAX, CXG_ELIMIT,
              "cxg_rows8_aggregate: rows and edges are counted in 32 bits");
  if (n_dst == 0) return CXG_OK;
  CXG_REQUIRE(codes && scales && ptr && y && (idx || nnz == 0), CXG_ENULL, "cxg_rows8_aggregate: NULL argument");
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0, CXG_EINVAL,
              "cxg_rows8_aggregate: codes must be 16-byte aligned, scales 4-byte");
  Rows8Args r = {};
  WalkArgs &a = r.w;
  a.ptr = ptr, a.idx = idx, a.y = y, a.edge_val = edge_val;
  a.n_dst = n_dst, a.nnz = nnz, a.feat = a.width = width, a.heads = 1;
  a.row_bytes = a.x_pitch = rows8::groups_of(width) * rows8::kGroup;
  a.ptr_bytes = ptr_bytes, a.idx_bytes = idx_bytes, a.reduce = reduce;
  r.codes = static_cast<const uint8_t *>(codes), r.scales = static_cast<const uint8_t *>(scales);
  r.n_src = n_src, r.groups = rows8::groups_of(width);
  const uint64_t bits = static_cast<uint64_t>(width) * (y_dtype == CXG_F32 ? 4 : 2) | reinterpret_cast<uintptr_t>(y);
  r.whole = bits % 16 == 0 ? 2 : bits % 8 == 0 ? 1 : 0;
  r.staged = r.whole == 0 && nnz < 10 * n_dst;
  const bool marked = is_sparse(n_dst, nnz, width);
  a.tile = marked ? sparse_tile(nnz, width, split_edges) : tile_edges(r, nnz, split_edges);
  a.part_stride = static_cast<int>(walk_part_stride(width));
  WalkLayout L;
  const int rc = walk_layout(nnz, a.part_stride, a.tile, &L);
  if (rc != CXG_OK) return set_error(rc, "cxg_rows8_aggregate: graph too large for 32-bit tile ids");
  const size_t need = L.total + (marked ? static_cast<size_t>(nnz) * sizeof(uint2) : 0);
  CXG_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, CXG_EWORKSPACE,
              "cxg_rows8_aggregate: workspace %zu bytes, need %zu", workspace_bytes, need);
  char *ws = static_cast<char *>(workspace);
  a.hdr = reinterpret_cast<int32_t *>(ws + L.hdr);
  a.tiles = ws + L.tiles;
  a.count = reinterpret_cast<int32_t *>(ws + L.count);
  a.partials = reinterpret_cast<float *>(ws + L.partials);
  a.max_tiles = L.max_tiles;
  cudaStream_t st = as_stream(stream);
  // small graphs, as those of cxg_spmm_csr, in one launch of clusters
  if (nnz <= kSmallEdges && nnz * a.x_pitch <= kSmallBytes && n_dst <= small_most_rows() && n_dst <= kSmallRowsPerEdge * nnz + 64 &&
      width <= 256 && (split_edges == 0 || split_edges == 64)) {
    WalkArgs small = a;
    small.tile = 64;
    small.x = codes, small.x_rows = scales, small.rel_stride = n_src;
    if (small_launch_rows8(small, y_dtype, st)) {
      count_launches(1);
      return check_launch("cxg_rows8_aggregate (small)");
    }
  }
  if (marked) {
    r.marks = reinterpret_cast<uint2 *>(ws + L.total);
    const int64_t blocks = (n_dst + 255) / 256;
    const unsigned grid = static_cast<unsigned>(blocks < kNumSM * 8 ? blocks : kNumSM * 8);
    const cudaError_t e = y_dtype == CXG_F32 ? launch_dependent(rows8_mark<float>, grid, 256, 0, st, r)
                                             : launch_dependent(rows8_mark<__nv_bfloat16>, grid, 256, 0, st, r);
    if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_aggregate: %s", cudaGetErrorString(e));
    count_launches(1);
  }
  walk_plan_run(a, st);
  if (!dispatch(r, y_dtype, st, nullptr)) return set_error(CXG_ECUDA, "cxg_rows8_aggregate: %s", cudaGetErrorString(cudaGetLastError()));
  const cudaError_t e = walk_fix_run(a, y_dtype, st);
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_aggregate: %s", cudaGetErrorString(e));
  count_launches(3);
  return check_launch("cxg_rows8_aggregate");
}
