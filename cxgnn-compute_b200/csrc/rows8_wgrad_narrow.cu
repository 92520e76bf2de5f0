// Weight gradient from rows in 8 bits for a dy of few columns (output layers of few classes, gates with one value per row):
//   dW[o][i] = sum over the rows r of dy[r][o] * codes[r][i] * scale[r][i / 32],   db[o] = sum over the rows of dy[r][o]
//
// The tensor cores' kernel (rows8_wgrad.cu) makes operands of 64 columns of dy whatever there are. Here a lane holds four columns
// of the input and all (up to 16) of dy, as pairs of fp32 sums along the input: two packed multiply-adds per row and column of
// dy, and 20 or so instructions to get there, which is what bounds it. A chunk of each matrix is one piece of memory and comes
// by asynchronous copies, three chunks ahead; dy becomes pairs (g, g) of fp32 in rows of N one chunk ahead, from where all lanes
// of a row read the same vectors. c * s is exact in fp32, so each term rounds once, in the addition. A block owns a contiguous
// range of rows; lane groups, warps and then blocks (rows8_wgrad_join) are added in order: the same bits on every run.
#include "rows8.cuh"

namespace cxg {
namespace {

using namespace rows8;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kStages = 4;  // chunks in shared memory
constexpr int blocks_per_sm(int n) { return n == 16 ? 2 : n == 8 ? 3 : 4; }
constexpr int lanes_of(int pitch) { return pitch == 32 ? 8 : pitch == 64 ? 16 : 32; }  // of a row
constexpr int rows_of(int pitch, int n) { return (pitch == 32 && n == 16 ? 4 : 8) * (kThreads / lanes_of(pitch)); }  // of a chunk

// 16 bytes of a matrix, zeros behind its last `left` bytes
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t *from, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// N: columns of dy, rounded up to 4, 8 or 16.
template <typename T, int N, int PITCH>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(N)) wgrad_narrow(const __grid_constant__ Rows8Narrow a) {
  constexpr int LANES = lanes_of(PITCH), kGroups = kThreads / LANES, kRows = rows_of(PITCH, N), kPer = kRows / kGroups;
  constexpr int kScales = PITCH / kGroup, kCols = LANES * 4;
  constexpr int kMine = kRows * N / kThreads;  // values of dy per thread and chunk
  static_assert(kMine >= 1 && kRows % 16 == 0, "");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float db_side[kWarps][N];
  const int tid = threadIdx.x, p = tid & (LANES - 1), g = tid / LANES, warp = tid >> 5, lane = tid & 31;
  const bool x_in = p * 4 < PITCH;
  const uint32_t n = static_cast<uint32_t>(a.n);
  // a stage: codes, scales, dy of a chunk as they lie in memory; in front of the stages two chunks of dy as pairs
  constexpr int kCodeBytes = kRows * PITCH, kScaleBytes = kRows * kScales;
  const int dy_bytes = kRows * a.n * static_cast<int>(sizeof(T)), stage_bytes = kCodeBytes + kScaleBytes + dy_bytes;
  Pair(*side)[kRows][N] = reinterpret_cast<Pair(*)[kRows][N]>(smem);
  uint8_t *const stages = smem + 2 * kRows * N * sizeof(Pair);
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  for (int i = tid; i < 2 * kRows * N; i += kThreads) (&side[0][0][0])[i] = 0;
  dependency_wait();
  const int64_t chunks = (a.m + kRows - 1) / kRows;
  const int64_t lo = chunks * blockIdx.x / gridDim.x;
  const int count = static_cast<int>(chunks * (blockIdx.x + 1) / gridDim.x - lo);
  auto request = [&](int c) {
    if (c < count) {
      const int64_t chunk = lo + c;
      const uint32_t to = base + static_cast<uint32_t>(c % kStages) * stage_bytes;
      const uint8_t *codes = a.codes + chunk * kCodeBytes, *scales = a.scales + chunk * kScaleBytes;
      const uint8_t *dy = static_cast<const uint8_t *>(a.dy) + chunk * dy_bytes;
      const int64_t rows = a.m - chunk * kRows;
      if (rows >= kRows) {
#pragma unroll
        for (int i = 0; i < kCodeBytes; i += kThreads * 16)
          if (i + tid * 16 < kCodeBytes) copy16(to + i + tid * 16, codes + i + tid * 16, 16);
        if (tid * 16 < kScaleBytes) copy16(to + kCodeBytes + tid * 16, scales + tid * 16, 16);
        for (int i = tid * 16; i < dy_bytes; i += kThreads * 16) copy16(to + kCodeBytes + kScaleBytes + i, dy + i, 16);
      } else {
        auto part = [&](uint32_t at, const uint8_t *from, int bytes, int have) {
          for (int i = tid * 16; i < bytes; i += kThreads * 16)
            copy16(at + i, i < have ? from + i : from, static_cast<uint32_t>(min(max(have - i, 0), 16)));
        };
        const int have = static_cast<int>(rows);
        part(to, codes, kCodeBytes, have * PITCH);
        part(to + kCodeBytes, scales, kScaleBytes, have * kScales);
        part(to + kCodeBytes + kScaleBytes, dy, dy_bytes, have * a.n * static_cast<int>(sizeof(T)));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto widen = [&](int c) {
    const T *d = reinterpret_cast<const T *>(stages + (c % kStages) * stage_bytes + kCodeBytes + kScaleBytes);
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const uint32_t i = static_cast<uint32_t>(tid + q * kThreads);
      if (i >= kRows * n) break;
      uint32_t row = n > 1 ? __umulhi(i, a.inverse) : i, at = i - row * n;
      if (at >= n) ++row, at -= n;
      const float v = to_f32(d[i]);
      side[c & 1][row][at] = pair(v, v);
    }
  };

  Pair acc[N][2];
#pragma unroll
  for (int o = 0; o < N; ++o) acc[o][0] = acc[o][1] = 0;
  float db = 0.f;  // of column tid % N
#pragma unroll
  for (int c = 0; c < kStages - 1; ++c) request(c);
  asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
  __syncthreads();
  widen(0);
  for (int c = 0; c < count; ++c) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 3) : "memory");
    __syncthreads();  // dy of this chunk is widened, the next one is there, the one before has been read
    request(c + kStages - 1);
    if (c + 1 < count) widen(c + 1);
    const uint8_t *stage = stages + (c % kStages) * stage_bytes;
    const uint8_t *codes = stage + g * PITCH + (x_in ? p * 4 : 0), *scales = stage + kCodeBytes + g * kScales + (x_in ? p * 4 / kGroup : 0);
    const Pair *d = side[c & 1][g];
#pragma unroll 4
    for (int j = 0; j < kPer; ++j) {
      const uint32_t word = *reinterpret_cast<const uint32_t *>(codes + j * kGroups * PITCH);
      const float s = scale_of(scales[j * kGroups * kScales]);
      const Pair ss = pair(s, s), off = pair(-8388736.f, -8388736.f);
      auto as_float = [&](uint32_t b) { return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 | b)); };
      // rows behind the last: codes and scales of 0, so -128 * 0 times a dy of 0
      const Pair v0 = mul2(add2(pair(as_float(0), as_float(1)), off), ss), v1 = mul2(add2(pair(as_float(2), as_float(3)), off), ss);
#pragma unroll
      for (int o = 0; o < N; o += 2) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(d + j * kGroups * N + o);
        acc[o][0] = fma2(v0, t.x, acc[o][0]);
        acc[o][1] = fma2(v1, t.x, acc[o][1]);
        acc[o + 1][0] = fma2(v0, t.y, acc[o + 1][0]);
        acc[o + 1][1] = fma2(v1, t.y, acc[o + 1][1]);
      }
    }
    if (a.partial_db != nullptr) {
#pragma unroll
      for (int q = 0; q < kMine; ++q) db += halves((&side[c & 1][0][0])[tid + q * kThreads]).x;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float(*sums)[kCols] = reinterpret_cast<float(*)[kCols]>(smem);  // [N]

  // lane groups of a warp, then the warps in order
  float f[N][4];
#pragma unroll
  for (int o = 0; o < N; ++o) {
    const float2 t0 = halves(acc[o][0]), t1 = halves(acc[o][1]);
    f[o][0] = t0.x, f[o][1] = t0.y, f[o][2] = t1.x, f[o][3] = t1.y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = LANES; d < 32; d <<= 1) f[o][i] += __shfl_xor_sync(0xffffffffu, f[o][i], d);
  }
#pragma unroll
  for (int d = N; d < 32; d <<= 1) db += __shfl_xor_sync(0xffffffffu, db, d);
  if (lane < N) db_side[warp][lane] = db;
  for (int w = 0; w < kWarps; ++w) {
    if (warp == w && lane < LANES) {
#pragma unroll
      for (int o = 0; o < N; ++o) {
        float4 *s = reinterpret_cast<float4 *>(&sums[o][p * 4]);
        float4 t = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *s;
        t.x += f[o][0], t.y += f[o][1], t.z += f[o][2], t.w += f[o][3];
        *s = t;
      }
    }
    __syncthreads();
  }
  float *out = a.partial + static_cast<int64_t>(blockIdx.x) * (N * 128);
  for (int i = tid; i < a.n * kCols; i += kThreads) out[i / kCols * 128 + i % kCols] = sums[i / kCols][i % kCols];
  if (a.partial_db != nullptr && tid < a.n) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += db_side[w][tid];
    a.partial_db[static_cast<int64_t>(blockIdx.x) * a.n + tid] = t;
  }
}

int padded(int n) { return n <= 4 ? 4 : n <= 8 ? 8 : 16; }
// A million rows, us, here / on the tensor cores, which take as long for any width up to 128: fp32 100 to 105, bf16 70 to 73, 97 to
// 114 with an odd number of columns. k = 16: n = 1 35, 4 39, 8 45, 16 66. 50: 4 49, 8 59, 16 90. 128: 4 72, 8 98, 16 153.
int most_columns(int k) { return k <= 32 ? 16 : k <= 64 ? 8 : 4; }

}  // namespace

Rows8NarrowPlan rows8_narrow_plan(int64_t m, int k, int n) {
  Rows8NarrowPlan plan = {};
  if (k > 128 || n > most_columns(k) || m == 0) return plan;
  plan.columns = padded(n);
  const int rows = rows_of(groups_of(k) * kGroup, plan.columns);
  // a block per SM until each has four chunks: what the blocks leave is added in a chain
  const int64_t chunks = (m + rows - 1) / rows, most = kNumSM * blocks_per_sm(plan.columns);
  const int64_t want = chunks / 4 > kNumSM ? chunks / 4 : kNumSM;
  plan.parts = static_cast<int>(chunks < want ? chunks : want < most ? want : most);
  return plan;
}

cudaError_t rows8_narrow_run(const Rows8Narrow &args, const Rows8NarrowPlan &plan, int dtype, cudaStream_t st) {
  Rows8Narrow a = args;
  a.inverse = static_cast<uint32_t>((1ull << 32) / a.n);
  const int pitch = groups_of(a.k) * kGroup, rows = rows_of(pitch, plan.columns);
  const int smem = rows * (2 * plan.columns * static_cast<int>(sizeof(Pair)) + kStages * (pitch + pitch / kGroup + a.n * (dtype == CXG_F32 ? 4 : 2)));
  auto go = [&](auto kernel) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return e != cudaSuccess ? e : launch_dependent(kernel, static_cast<unsigned>(plan.parts), kThreads, smem, st, a);
  };
  auto by_columns = [&](auto t) {
    using T = decltype(t);
    if (plan.columns == 16) return go(wgrad_narrow<T, 16, 32>);
    if (plan.columns == 8) return pitch == 32 ? go(wgrad_narrow<T, 8, 32>) : go(wgrad_narrow<T, 8, 64>);
    return pitch == 32   ? go(wgrad_narrow<T, 4, 32>)
           : pitch == 64 ? go(wgrad_narrow<T, 4, 64>)
           : pitch == 96 ? go(wgrad_narrow<T, 4, 96>)
                         : go(wgrad_narrow<T, 4, 128>);
  };
  return dtype == CXG_F32 ? by_columns(float{}) : by_columns(__nv_bfloat16{});
}

}  // namespace cxg
