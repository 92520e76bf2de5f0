// Weight gradient from a layer's input held in 8 bits, on the 5th-generation tensor cores:
//   dW[o][i] = sum over the rows r of dy[r][o] * codes[r][i] * scale[r][i / 32],   db[o] = sum over the rows of dy[r][o]
//
// codes * scale has 7 bits and is an exact bf16 operand; fp32 dy is cut into three bf16 parts of 8 bits each, which hold all 24
// of its bits: dy = hi + mid + lo exactly (from 2^-110 on; below, the last bits of lo are under bf16's smallest number, 2^-133). So
// every product is exact and a sum of m rows takes three bf16 instructions' worth
// of tensor core time (one for bf16 dy), where compensated TF32 would take three of half the rate and lose bits.
//
// The contraction runs over rows, so both operands are "MN-major": a stage holds 64 rows of the input (A: 128 columns, two
// spans of 128 bytes per row in a 128-byte swizzle) and of dy (B: hi, then mid, then lo spans). Both are made in registers:
// producer warps load 16 or 32 bytes at a time two stages ahead, convert, and write the operands where the tensor core reads
// them. One instruction multiplies A by [hi | mid], another adds A by lo to mid's accumulator. An accumulator takes `chunk`
// stages, as the tensor core's additions cut off what an fp32 addition rounds (its error grows with the number of additions);
// the epilogue warps, each lane a column of the input, add the chunks up in shared memory.
//
// Measured: 2.4 M rows of 100 x 128 fp32 384 us (4.1 TB/s), 400,000 77. What bounds it is shared memory: per stage 64 KB of
// operands written and 80 read by the tensor core, besides the loads. Of the 400,000 rows' time with older loads (84), without MMA 75
// remain, without loads 58, without conversion 75, with neither of the last two 50.
//
// A block owns a contiguous range of rows of one pair of 128-column blocks; its sums go to a partial of its own and a second
// kernel adds the partials in order: the same bits on every run. Every wait is bounded (see tensor_core.cuh).
#include "rows8.cuh"
#include "tensor_core.cuh"

namespace cxg {
namespace {

using namespace tc;
using rows8::kGroup;

constexpr int kPos = 64;           // rows per stage
constexpr int kSpan = kPos * 128;  // bytes of a span: 64 columns of bf16, one row behind the other
constexpr int kProdWarps = 16, kEpiWarps = 8;
constexpr int kMmaWarp = kEpiWarps, kFirstProd = kMmaWarp + 4;  // roles in whole groups of four warps, which share out registers
constexpr int kThreads = 32 * (kFirstProd + kProdWarps);
// Registers per thread: 72 at the launch (896 threads take 64,512). The producers, which hold two stages of loads, take 24 more
// each from the others: 256 * 40 + 128 * 24 + 512 * 96 = 62,464. (One stage of loads in 72 registers: 85 us for 400,000 rows of
// 100 x 128 fp32, 25 of them waiting for loads; eight warps with two stages in 128 registers left the chip idle between their
// dependent instructions: 115 us; with 96 registers for all of them, loads were spilled, which waits for each: 202 us.)
constexpr int kIssuerRegs = 24, kEpilogueRegs = 40, kProducerRegs = 96;
constexpr int kMaxStages = 4;
constexpr int kSmemBudget = 216 * 1024;

struct R8Args {
  const uint8_t *codes, *scales;
  const void *dy;
  int64_t m, ld;
  int k, n, pitch, groups, k_blocks, stages, chunk, test_stall;
  float *partial;     // [pair of column blocks][gridDim.x][128 columns of dy][128 columns of the input]
  float *partial_db;  // [gridDim.x][n] or NULL
  int32_t *status;
  long long wait_cycles;
};

struct R8Barriers {
  uint64_t full[kMaxStages];   // producers -> MMA
  uint64_t empty[kMaxStages];  // MMA -> producers
  uint64_t acc_full[2];        // MMA -> epilogue
  uint64_t acc_empty[2];       // epilogue -> MMA
};

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two neighbouring codes (bytes b = c + 128 of a word, 2 * H and 2 * H + 1) times the scale, as two bf16. 0x4300 | (b & 0x7f) is
// 128 + (b & 0x7f) in bf16, and 0x4300 | (~b & 0x80) is 256 where c is negative, else 128: their difference is c, exactly.
template <int H>
__device__ __forceinline__ uint32_t two_values(uint32_t word, __nv_bfloat162 scale) {
  const uint32_t w = __byte_perm(word, 0x43434343u, H == 0 ? 0x4140 : 0x4342);
  const uint32_t lo = w & 0xff7fff7fu, hi = (w & 0xff80ff80u) ^ 0x00800080u;
  __nv_bfloat162 a, b;
  __builtin_memcpy(&a, &lo, 4);
  __builtin_memcpy(&b, &hi, 4);
  a = __hmul2(__hsub2(a, b), scale);
  uint32_t out;
  __builtin_memcpy(&out, &a, 4);
  return out;
}

// hi, mid and lo of 8 fp32 values (four pairs), as 8 bf16 each. Cutting instead of rounding keeps the sum exact (8 bits each).
// Infinities and NaN go into hi alone (what is left of them would be NaN).
__device__ __forceinline__ void three_parts(const Pair (&v)[4], uint32_t (&hi)[4], uint32_t (&mid)[4], uint32_t (&lo)[4]) {
  const Pair minus = pair(-1.f, -1.f);
  auto upper = [](Pair p) { return static_cast<Pair>(p & 0xffff0000ffff0000ull); };
  Pair h[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = upper(v[i]);
    r[i] = fma2(h[i], minus, v[i]);
  }
  // a rest that is NaN: a value that is not finite (the rests themselves are far too small to add up to an infinity)
  const float any = sum2(add2(add2(r[0], r[1]), add2(r[2], r[3])));
  if (any != any) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = halves(v[i]), a = halves(h[i]), b = halves(r[i]);
      if ((__float_as_uint(f.x) & 0x7f800000u) == 0x7f800000u) a.x = f.x != f.x ? __uint_as_float(0x7fc00000u) : f.x, b.x = 0.f;
      if ((__float_as_uint(f.y) & 0x7f800000u) == 0x7f800000u) a.y = f.y != f.y ? __uint_as_float(0x7fc00000u) : f.y, b.y = 0.f;
      h[i] = pair(a.x, a.y), r[i] = pair(b.x, b.y);
    }
  }
  auto pack = [](Pair p) { return __byte_perm(static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32), 0x7632); };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair m = upper(r[i]);
    hi[i] = pack(h[i]);
    mid[i] = pack(m);
    lo[i] = pack(fma2(m, minus, r[i]));
  }
}

// SPANS: 64-column spans of a block of dy. VECTOR: bytes of the vectors that rows of dy are read in, all of them whole. 32-byte
// vectors of fp32 take half the passes through L1 that pairs of 16-byte ones do.
template <typename T, int VECTOR, int SPANS>
__global__ void __launch_bounds__(kThreads, 1) rows8_wgrad(const __grid_constant__ R8Args a) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  constexpr int kCols = 64 * SPANS;
  constexpr uint32_t kStageBytes = (2 + kParts * SPANS) * kSpan;
  constexpr int kAccCols = kParts == 3 ? 2 * kCols : kCols;  // of a buffer in tensor memory
  constexpr int kTmem = 2 * kAccCols;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(8) R8Barriers bars;
  __shared__ float db_side[kProdWarps][128];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_slot;
  volatile int *abort_flag = &abort_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int x_at = static_cast<int>(blockIdx.y % a.k_blocks) * 128, g_at = static_cast<int>(blockIdx.y / a.k_blocks) * 128;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  float *const sums = reinterpret_cast<float *>(smem_raw + (base - smem_addr(smem_raw)) + static_cast<size_t>(a.stages) * kStageBytes);  // [kCols][128]
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_slot)), "r"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    abort_slot = 0;
    for (int s = 0; s < kMaxStages; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&bars.full[s])), "r"(32 * kProdWarps) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&bars.empty[s])) : "memory");
    }
    for (int b = 0; b < 2; ++b) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&bars.acc_full[b])) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&bars.acc_empty[b])), "r"(32 * kEpiWarps) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  dependency_wait();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_d = tmem_base_slot;
  const int64_t n_tiles = (a.m + kPos - 1) / kPos;
  const int64_t tile_lo = n_tiles * blockIdx.x / gridDim.x, tile_hi = n_tiles * (blockIdx.x + 1) / gridDim.x;

  if (warp >= kFirstProd) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    // ================= producers =================
    // Every thread has a unit of 16 codes and one or two of 8 values of dy per stage. What it loads of the stage after the next
    // replaces a unit as soon as this one is written, so that a load has two stages' time to arrive.
    constexpr int kThr = 32 * kProdWarps;
    constexpr int kUnitsPerRow = 8 * SPANS;                 // of dy
    constexpr int kGUnits = kPos * kUnitsPerRow / kThr;
    constexpr int kGRows = kThr / kUnitsPerRow;             // rows from a thread's unit to its next
    static_assert(kPos * 8 == kThr, "a unit of codes per thread");
    const int pt = tid - 32 * kFirstProd;
    const int xu = pt & 7, gu = pt % kUnitsPerRow, xrow = pt >> 3, grow = pt / kUnitsPerRow;
    const int xcol = x_at + xu * 16, gcol = g_at + gu * 8;
    const bool x_in = xcol < a.pitch;
    const int64_t row_end = tile_hi * kPos < a.m ? tile_hi * kPos : a.m;  // of this block
    int64_t row = tile_lo * kPos;                                         // first of the stage that is loaded
    const uint8_t *codes = a.codes + (row + xrow) * a.pitch + xcol, *scales = a.scales + (row + xrow) * a.groups + xcol / kGroup;
    const T *dy = static_cast<const T *>(a.dy) + (row + grow) * a.ld + gcol;
    constexpr int W = sizeof(T) == 4 ? 8 : 4;
    struct Raw {  // of a stage, as it was loaded
      uint4 codes;
      uint32_t scale;
      uint32_t dy[kGUnits][W];
    };
    auto load_codes = [&](Raw &raw) {
      raw.codes = make_uint4(0, 0, 0, 0);
      raw.scale = 0;
      if (x_in && row + xrow < row_end) {
        raw.codes = __ldg(reinterpret_cast<const uint4 *>(codes));
        raw.scale = __ldg(scales);
      }
    };
    auto load_dy = [&](Raw &raw, int j) {
      uint32_t(&v)[W] = raw.dy[j];
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = 0;
      if (row + grow + j * kGRows >= row_end) return;
      const T *p = dy + static_cast<int64_t>(j * kGRows) * a.ld;
      if constexpr (VECTOR == 32) {
        if (gcol < a.n)
          asm("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
              : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4 % W]), "=r"(v[5 % W]), "=r"(v[6 % W]), "=r"(v[7 % W])
              : "l"(p));
      } else if constexpr (VECTOR > static_cast<int>(sizeof(T))) {
        constexpr int kWords = VECTOR / 4, kStep = VECTOR / static_cast<int>(sizeof(T));  // words and values of a vector
#pragma unroll
        for (int i = 0; i < W / kWords; ++i)
          if (gcol + i * kStep < a.n) {
            if constexpr (VECTOR == 16) {
              const uint4 t = __ldg(reinterpret_cast<const uint4 *>(p) + i);
              v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
            } else if constexpr (VECTOR == 8) {
              const uint2 t = __ldg(reinterpret_cast<const uint2 *>(p) + i);
              v[2 * i] = t.x, v[2 * i + 1] = t.y;
            } else {
              v[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
            }
          }
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (gcol + i < a.n) v[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (gcol + i < a.n) v[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t *>(p) + i)) << (16 * (i & 1));
      }
    };
    auto onward = [&]() {
      row += kPos;
      codes += static_cast<int64_t>(kPos) * a.pitch;
      scales += static_cast<int64_t>(kPos) * a.groups;
      dy += static_cast<int64_t>(kPos) * a.ld;
    };
    // where a unit goes, from the start of a stage
    const int odd = xu >> 2;  // the second span's lanes start with their odd chunk: other banks
    const uint32_t x_first = (xu >> 2) * kSpan + swizzled_offset<false>(xrow, (xu & 3) * 2 + odd);
    const uint32_t x_second = (xu >> 2) * kSpan + swizzled_offset<false>(xrow, (xu & 3) * 2 + 1 - odd);
    const uint32_t g_first = (2 + (gu >> 3)) * kSpan + swizzled_offset<false>(grow, gu & 7);
    static_assert(kGRows % 8 == 0, "the swizzle repeats every eight rows");
    Pair db[4] = {};
    const bool want_db = a.partial_db != nullptr && x_at == 0;
    auto put_codes = [&](const Raw &raw, uint32_t stage) {
      const __nv_bfloat162 s = __float2bfloat162_rn(rows8::scale_of(raw.scale));
      const uint32_t w[4] = {raw.codes.x, raw.codes.y, raw.codes.z, raw.codes.w};
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = two_values<0>(w[i], s), v[2 * i + 1] = two_values<1>(w[i], s);
      st_shared16(stage + (odd ? x_second : x_first), v[0], v[1], v[2], v[3]);
      st_shared16(stage + (odd ? x_first : x_second), v[4], v[5], v[6], v[7]);
    };
    auto put_dy = [&](const Raw &raw, int j, uint32_t stage) {
      const uint32_t(&r)[W] = raw.dy[j];
      const uint32_t at = stage + g_first + j * kGRows * 128;
      if constexpr (sizeof(T) == 4) {
        Pair v[4];
        uint32_t hi[4], mid[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = pair(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        }
        if (want_db) {
#pragma unroll
          for (int i = 0; i < 4; ++i) db[i] = add2(db[i], v[i]);
        }
        three_parts(v, hi, mid, lo);
        st_shared16(at, hi[0], hi[1], hi[2], hi[3]);
        st_shared16(at + SPANS * kSpan, mid[0], mid[1], mid[2], mid[3]);
        st_shared16(at + 2 * SPANS * kSpan, lo[0], lo[1], lo[2], lo[3]);
      } else {
        if (want_db) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            db[i] = add2(db[i], pair(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u)));
        }
        st_shared16(at, r[0], r[1], r[2], r[3]);
      }
    };
    Ring ring(a.stages);
    auto load = [&](Raw &raw) {
      load_codes(raw);
#pragma unroll
      for (int j = 0; j < kGUnits; ++j) load_dy(raw, j);
      onward();
    };
    auto hand_over = [&](Raw &raw) {
      const int s = ring.stage;
      if (ring.reused() && !wait_bar(&bars.empty[s], ring.emptied(), abort_flag, a.status, a.wait_cycles)) return false;
      const uint32_t stage = base + static_cast<uint32_t>(s) * kStageBytes;
      put_codes(raw, stage);
      load_codes(raw);
#pragma unroll
      for (int j = 0; j < kGUnits; ++j) {
        put_dy(raw, j, stage);
        load_dy(raw, j);
      }
      onward();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (!(a.test_stall && ring.round == 0 && s == 0)) mbar_arrive(&bars.full[s]);
      ring.next();
      return true;
    };
    Raw even, odd_raw;
    load(even);
    load(odd_raw);
    for (int64_t tile = tile_lo; tile < tile_hi; tile += 2) {
      if (!hand_over(even)) break;
      if (tile + 1 < tile_hi && !hand_over(odd_raw)) break;
    }
    if (want_db) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 t = halves(db[i]);
#pragma unroll
        for (int o = kUnitsPerRow; o < 32; o <<= 1) {
          t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
          t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        }
        if (lane < kUnitsPerRow) db_side[warp - kFirstProd][gu * 8 + 2 * i] = t.x, db_side[warp - kFirstProd][gu * 8 + 2 * i + 1] = t.y;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kProdWarps) : "memory");
      if (pt < kCols && g_at + pt < a.n) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kProdWarps; ++w) t += db_side[w][pt];
        a.partial_db[static_cast<int64_t>(blockIdx.x) * a.n + g_at + pt] = t;
      }
    }
  } else if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssuerRegs));
    if (warp == kMmaWarp) {
    // ================= MMA issuer: the whole warp walks the tiles, one lane issues =================
    auto wait_all = [&](uint64_t *bar, uint32_t parity) {
      return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, a.status, a.wait_cycles)) != 0;
    };
    const uint32_t idesc = make_idesc_mn(1, 128, kCols), idesc_wide = make_idesc_mn(1, 128, kParts == 3 ? 2 * kCols : kCols);
    Ring ring(a.stages);
    int64_t chunk = 0;
    int in_chunk = 0;
    bool alive = true;
    for (int64_t tile = tile_lo; tile < tile_hi && alive; ++tile) {
      const int buf = static_cast<int>(chunk & 1);
      if (in_chunk == 0 && chunk >= 2) {  // the epilogue has read the chunk that used this buffer before
        alive = wait_all(&bars.acc_empty[buf], static_cast<uint32_t>(((chunk >> 1) - 1) & 1));
        if (!alive) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const int s = ring.stage;
      alive = wait_all(&bars.full[s], ring.filled());
      if (!alive) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem_d + buf * kAccCols;
      const uint32_t x0 = base + static_cast<uint32_t>(s) * kStageBytes, g0 = x0 + 2 * kSpan;
#pragma unroll
      for (int j = 0; j < kPos / 16; ++j) {
        const uint32_t go_on = (in_chunk > 0 || j > 0) ? 1u : 0u;
        const uint64_t xa = make_desc_mn_sw128<false>(x0 + j * 2048, kSpan);
        mma_ss<false>(d, xa, make_desc_mn_sw128<false>(g0 + j * 2048, kSpan), idesc_wide, go_on);
        if constexpr (kParts == 3)
          mma_ss<false>(d + kCols, xa, make_desc_mn_sw128<false>(g0 + 2 * SPANS * kSpan + j * 2048, kSpan), idesc, 1u);
      }
      commit_to(&bars.empty[s]);
      if (++in_chunk == a.chunk || tile + 1 == tile_hi) {
        commit_to(&bars.acc_full[buf]);
        in_chunk = 0;
        ++chunk;
      }
      ring.next();
    }
    if (!alive) {  // what was issued ends before tensor memory is given back
      const long long t0 = clock64();
      while (clock64() - t0 < 200000) {
      }
    }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
    // ================= epilogue: lane = column of the input, half of the columns of dy per four warps =================
    constexpr int kHalf = kCols / 2;
    const int first = (warp >> 2) * kHalf, row = (warp & 3) * 32 + lane;
    const int64_t n_chunks = (tile_hi - tile_lo + a.chunk - 1) / a.chunk;
    bool alive = true;
    for (int64_t chunk = 0; chunk < n_chunks; ++chunk) {
      const int buf = static_cast<int>(chunk & 1);
      alive = __all_sync(0xffffffffu, wait_bar(&bars.acc_full[buf], static_cast<uint32_t>((chunk >> 1) & 1), abort_flag, a.status,
                                               a.wait_cycles)) != 0;
      if (!alive) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t taddr = tmem_d + (static_cast<uint32_t>((warp & 3) * 32) << 16) + buf * kAccCols + first;
      float *sum = sums + first * 128 + row;
#pragma unroll 1
      for (int c = 0; c < kHalf; c += 8, sum += 8 * 128) {
        uint32_t v[8], w[8];
        tmem_ld8(v, taddr + c);
        if constexpr (kParts == 3) tmem_ld8(w, taddr + kCols + c);
        float old[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) old[i] = chunk > 0 ? sum[i * 128] : 0.f;
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i)
          sum[i * 128] = old[i] + (kParts == 3 ? __uint_as_float(v[i]) + __uint_as_float(w[i]) : __uint_as_float(v[i]));
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(&bars.acc_empty[buf]);
    }
    if (alive && x_at + row < a.k) {
      float *out = a.partial + ((static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 128 + first) * 128 + row;
      for (int c = 0; c < kHalf && g_at + first + c < a.n; ++c) out[c * 128] = sums[(first + c) * 128 + row];
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_d), "r"(kTmem) : "memory");
  }
}

// dw[o][i] and db[o] from [pair of column blocks][parts][per columns of dy][128 columns of the input]: warp q of a block adds the
// partials q, q + 8, ... of 32 outputs, the eight sums are added in order. (A thread per output and all its
// partials took 11 us for 148 partials of 128 x 100, a chain of loads.)
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) rows8_wgrad_join(const float *partial, const float *partial_db, T *dw, T *db, int k,
                                                                    int n, int k_blocks, int parts, int per) {
  dependency_wait();
  __shared__ float side[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = blockIdx.x * 32ll + lane, kn = static_cast<int64_t>(k) * n;
  const float *p = nullptr;
  int64_t step = 0;
  if (i < kn) {
    const int o = static_cast<int>(i / k), c = static_cast<int>(i % k);
    const int64_t pair = c / 128 + static_cast<int64_t>(k_blocks) * (o / 128);
    p = partial + (pair * parts * per + o % 128) * 128 + c % 128;
    step = per * 128;
  } else if (db != nullptr && i < kn + n) {
    p = partial_db + (i - kn);
    step = n;
  }
  float s = 0.f;
  if (p != nullptr) {
    for (int q = warp; q < parts; q += 8 * kJoinWarps) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = q + u * kJoinWarps < parts ? p[(q + u * kJoinWarps) * step] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  }
  side[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && p != nullptr) {
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) s += side[w][lane];
    if (i < kn)
      dw[i] = from_f32<T>(s);
    else
      db[i - kn] = from_f32<T>(s);
  }
}

__device__ int32_t r8_status;  // set when a bounded wait ran out, cleared by cxg_rows8_wgrad_status

int parts_of(int k, int n, int64_t m) {
  const int64_t pairs = static_cast<int64_t>((k + 127) / 128) * ((n + 127) / 128);
  const int64_t tiles = (m + kPos - 1) / kPos, parts = pairs < kNumSM ? kNumSM / pairs : 1;
  return static_cast<int>(parts < tiles ? parts : tiles);
}

template <typename... P>
void launch_join(int out_dtype, cudaStream_t st, const float *partial, const float *partial_db, void *dw, void *db, int k, int n, P... p) {
  const int64_t outs = static_cast<int64_t>(k) * n + (db != nullptr ? n : 0);
  const unsigned blocks = static_cast<unsigned>((outs + 31) / 32);
  if (out_dtype == CXG_F32)
    launch_dependent(rows8_wgrad_join<float>, blocks, 32 * kJoinWarps, 0, st, partial, partial_db, static_cast<float *>(dw),
                     static_cast<float *>(db), k, n, p...);
  else
    launch_dependent(rows8_wgrad_join<__nv_bfloat16>, blocks, 32 * kJoinWarps, 0, st, partial, partial_db,
                     static_cast<__nv_bfloat16 *>(dw), static_cast<__nv_bfloat16 *>(db), k, n, p...);
}

}  // namespace
}  // namespace cxg

using namespace cxg;

extern "C" int cxg_rows8_wgrad_workspace_size(int64_t m, int k, int n, size_t *bytes) {
  CXG_REQUIRE(bytes != nullptr, CXG_ENULL, "cxg_rows8_wgrad_workspace_size: bytes is NULL");
  CXG_REQUIRE(m >= 0 && k > 0 && n > 0, CXG_EINVAL, "cxg_rows8_wgrad_workspace_size: bad sizes");
  const Rows8NarrowPlan narrow = rows8_narrow_plan(m, k, n);
  const size_t pairs = static_cast<size_t>((k + 127) / 128) * ((n + 127) / 128), parts = static_cast<size_t>(parts_of(k, n, m));
  const size_t need = parts * (pairs * 128 * 128 + n), few = static_cast<size_t>(narrow.parts) * (narrow.columns * 128 + n);
  *bytes = (need > few ? need : few) * sizeof(float);
  return CXG_OK;
}

extern "C" int cxg_rows8_wgrad(const void *codes, const void *scales, int64_t m, int k, const void *dy, int dtype, int64_t ld, int n,
                               uint32_t flags, void *dw, void *db, int out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  CXG_REQUIRE(m >= 0 && k > 0 && n > 0 && ld >= n && (dtype == CXG_F32 || dtype == CXG_BF16) &&
                  (out_dtype == CXG_F32 || out_dtype == CXG_BF16),
              CXG_EINVAL, "cxg_rows8_wgrad: bad sizes or type");
  CXG_REQUIRE(dw != nullptr, CXG_ENULL, "cxg_rows8_wgrad: dw is NULL");
  const int k_blocks = (k + 127) / 128, n_blocks = (n + 127) / 128;
  CXG_REQUIRE(static_cast<int64_t>(k_blocks) * n_blocks <= 65535 && static_cast<int64_t>(k) * n < (1ll << 31), CXG_EUNSUPPORTED,
              "cxg_rows8_wgrad: a weight of %d x %d", n, k);
  cudaStream_t st = as_stream(stream);
  if (m == 0) {
    const size_t size = out_dtype == CXG_F32 ? 4 : 2;
    cudaError_t e = cudaMemsetAsync(dw, 0, size * static_cast<size_t>(k) * n, st);
    if (e == cudaSuccess && db != nullptr) e = cudaMemsetAsync(db, 0, size * n, st);
    return e == cudaSuccess ? CXG_OK : set_error(CXG_ECUDA, "cxg_rows8_wgrad: %s", cudaGetErrorString(e));
  }
  CXG_REQUIRE(codes && scales && dy, CXG_ENULL, "cxg_rows8_wgrad: NULL argument");
  CXG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, CXG_EINVAL, "cxg_rows8_wgrad: codes must be 16-byte aligned");
  size_t need = 0;
  cxg_rows8_wgrad_workspace_size(m, k, n, &need);
  CXG_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, CXG_EWORKSPACE,
              "cxg_rows8_wgrad: workspace %zu bytes, need %zu", workspace_bytes, need);
  const Rows8NarrowPlan narrow = rows8_narrow_plan(m, k, n);
  if (narrow.columns > 0 && ld == n && (reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(scales)) % 16 == 0) {
    Rows8Narrow a = {};
    a.codes = static_cast<const uint8_t *>(codes), a.scales = static_cast<const uint8_t *>(scales), a.dy = dy;
    a.m = m, a.k = k, a.n = n, a.groups = rows8::groups_of(k), a.pitch = a.groups * kGroup;
    a.partial = static_cast<float *>(workspace);
    a.partial_db = db != nullptr ? a.partial + static_cast<size_t>(narrow.parts) * narrow.columns * 128 : nullptr;
    const cudaError_t e = rows8_narrow_run(a, narrow, dtype, st);
    if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_wgrad: %s", cudaGetErrorString(e));
    launch_join(out_dtype, st, a.partial, a.partial_db, dw, db, k, n, 1, narrow.parts, narrow.columns);
    count_launches(2);
    return check_launch("cxg_rows8_wgrad (narrow)");
  }
  const int parts = parts_of(k, n, m), elem = dtype == CXG_F32 ? 4 : 2;
  R8Args a = {};
  a.codes = static_cast<const uint8_t *>(codes), a.scales = static_cast<const uint8_t *>(scales), a.dy = dy;
  a.m = m, a.ld = ld, a.k = k, a.n = n, a.groups = rows8::groups_of(k), a.pitch = a.groups * kGroup, a.k_blocks = k_blocks;
  a.test_stall = (flags & CXG_WGRAD_TEST_STALL) ? 1 : 0;
  a.partial = static_cast<float *>(workspace);
  a.partial_db = db != nullptr ? a.partial + static_cast<size_t>(k_blocks) * n_blocks * parts * (128 * 128) : nullptr;
  a.wait_cycles = wait_limit_cycles();
  const int spans = n > 64 ? 2 : 1;
  const int stage = (2 + (dtype == CXG_F32 ? 3 : 1) * spans) * kSpan;
  const int sums = 64 * spans * 128 * static_cast<int>(sizeof(float)), fit = (kSmemBudget - 1024 - sums) / stage;
  a.stages = fit < kMaxStages ? fit : kMaxStages;
  a.chunk = (dtype == CXG_F32 ? 512 : 1024) / kPos;
  const int smem = 1024 + a.stages * stage + sums;
  void *word = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&word, r8_status);
  a.status = static_cast<int32_t *>(word);
  const uint64_t bits = static_cast<uint64_t>(ld) * elem | static_cast<uint64_t>(n) * elem | reinterpret_cast<uintptr_t>(dy);
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(k_blocks * n_blocks));
  auto go = [&](auto kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_dependent(kernel, grid, kThreads, smem, st, a);
  };
  auto by_spans = [&](auto one, auto two) { spans == 1 ? go(one) : go(two); };
  using bf16 = __nv_bfloat16;
  if (dtype == CXG_F32)
    bits % 32 == 0   ? by_spans(rows8_wgrad<float, 32, 1>, rows8_wgrad<float, 32, 2>)
    : bits % 16 == 0 ? by_spans(rows8_wgrad<float, 16, 1>, rows8_wgrad<float, 16, 2>)
    : bits % 8 == 0  ? by_spans(rows8_wgrad<float, 8, 1>, rows8_wgrad<float, 8, 2>)
                     : by_spans(rows8_wgrad<float, 4, 1>, rows8_wgrad<float, 4, 2>);
  else
    bits % 16 == 0  ? by_spans(rows8_wgrad<bf16, 16, 1>, rows8_wgrad<bf16, 16, 2>)
    : bits % 8 == 0 ? by_spans(rows8_wgrad<bf16, 8, 1>, rows8_wgrad<bf16, 8, 2>)
    : bits % 4 == 0 ? by_spans(rows8_wgrad<bf16, 4, 1>, rows8_wgrad<bf16, 4, 2>)
                    : by_spans(rows8_wgrad<bf16, 2, 1>, rows8_wgrad<bf16, 2, 2>);
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_wgrad: %s", cudaGetErrorString(e));
  launch_join(out_dtype, st, a.partial, a.partial_db, dw, db, k, n, k_blocks, parts, 128);
  count_launches(2);
  return check_launch("cxg_rows8_wgrad");
}

extern "C" int cxg_rows8_wgrad_status(void *stream) {
  void *word = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&word, r8_status);
  if (e != cudaSuccess) return set_error(CXG_ECUDA, "cxg_rows8_wgrad_status: %s", cudaGetErrorString(e));
  return take_status_word(word, stream, "cxg_rows8_wgrad");
}
