// fp4_gemm.cu -- products of 4-bit matrices on the tensor cores.
//
// out[m][n] = ga gb sum_k a[m][k] b[n][k], a and b the codes times their block scales. The
// sm_100a tensor core takes the codes from shared memory and the block scales from tensor
// memory (tcgen05.mma block_scale), multiplies them into every product and sums in fp32, so
// nothing is decoded and no partial sum leaves tensor memory before the last K step.
//
// A CTA (one per SM, persistent) computes tiles of 128 rows of a by BN rows of b. K steps of 256
// values: 128 bytes of codes a row (one 128-byte swizzle row) and the scale tiles of those 256
// columns, which lie back to back in memory (fp4.cuh). Warp 0 issues b's copies and warp 10 those
// of a (a copy costs its thread about 90 cycles, a step has 6), warp 1 the scale copies into tensor
// memory and the MMAs (4 of K = 64 a step), warps 2..9 store tiles.
// Scale columns in tensor memory have two slots: the copies for step k + 2 are issued when the
// MMAs of step k have retired. A scale operand starts at a whole scale tile (4 columns), so BN
// is a multiple of 128.
//
// With swiglu, b holds gate and up rows: a tile takes 128 rows of each, and the epilogue turns the
// two halves of its columns into the 4-bit blocks of gate * silu(up), so the fp32 product never
// reaches memory.
//
// Tensor memory has 512 columns. At BN = 128 two accumulators lie side by side. At BN = 256
// two of them and the scales do not fit: the accumulators overlap by 96 columns, which the
// epilogue reads first, and the next tile starts as soon as those are in registers.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "fmoe.h"
#include "fmoe_common.cuh"
#include "fmoe_kernels.cuh"
#include "fp4.cuh"
#include "fp4_kernels.cuh"
#include "sm100.cuh"

namespace fmoe {
namespace {

using namespace fp4;
using namespace sm100;

constexpr int kThreads = 352;
constexpr int kEpiWarps = 8;
constexpr int kStepCols = 256;      // K values per step
constexpr int kABytes = 128 * 128;
constexpr int kMaxExperts = 1024;   // of a grouped product; their row tiles and rows lie in
constexpr int kStatic = (2 * kMaxExperts + 4) * 4;  // static shared memory
constexpr int kSmemLimit = 232448 - kStatic;
constexpr int kOverlap = 96;        // columns two 256-column accumulators share

enum Epilogue { kStore, kSwiglu };

// S > 1: a cluster of S CTAs takes a tile of at most 32 rows together, each a part of K (see
// the kernel). The parts meet in `kExchange` bytes of shared memory: a slice of BN / S columns
// from each other CTA.
template <int kFormat, int BN, int S>
struct Cfg {
  static constexpr int kSlice = BN / S;                               // columns a CTA finishes
  static constexpr int kExchange = (S - 1) * kSlice * 32 * 4;
  static constexpr int kScaleTiles = kStepCols / tile_cols(kFormat);  // per 128 rows and step
  static constexpr int kRunBytes = kScaleTiles * kTileBytes;
  static constexpr int kRuns = BN / 128;                              // 128-row runs of b
  static constexpr int kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes + (1 + kRuns) * kRunBytes;
  static constexpr int kFixed = 1024 + 512;
  static constexpr int kStagesRaw = (kSmemLimit - kFixed - kExchange) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kSmemBytes = kFixed + kExchange + kStages * kStageBytes;
  // tensor memory
  static constexpr bool kOverlapped = BN > 128;
  static constexpr int kAcc1 = kOverlapped ? BN - kOverlap : BN;      // second accumulator
  static constexpr int kScales = kAcc1 + BN;                          // first scale column
  static constexpr int kSfaCols = kScaleTiles * 4;
  static constexpr int kSlotCols = kSfaCols * (1 + kRuns);
  static_assert(kScales + 2 * kSlotCols <= 512, "tensor memory budget");
  static_assert(BN % 128 == 0, "scale operands start at whole scale tiles");
  static_assert(kStages >= 3, "pipeline depth");
  static_assert(kStageBytes % 1024 == 0, "stage alignment");
};

// True for one lane of a fully active warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// scale tile (128 rows x 4 blocks) -> 4 tensor memory columns: lane l, column j holds the four
// scale bytes of row 32 j + l
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF)            // start address
         | ((uint64_t)8 << 16) | ((uint64_t)8 << 32)  // 8-row groups 128 B apart
         | ((uint64_t)1 << 46);                       // descriptor version; no swizzle
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

template <int kFormat>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (kFormat == FMOE_MXFP4) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X "
        "[%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X "
        "[%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  }
}

// Instruction descriptor: e2m1 x e2m1 -> fp32, K-major, 128 x N x 64. mxfp4: the MMA's two
// scales are bytes `half` and `half + 1` of the four in the column.
template <int kFormat>
__device__ __forceinline__ uint32_t idesc_fp4(int n, int half) {
  return (1u << 7) | (1u << 10)                              // A, B = e2m1
         | ((uint32_t)half << 4) | ((uint32_t)half << 29)    // scale bytes of B, of A
         | ((uint32_t)(n >> 3) << 17)                        // N / 8
         | (kFormat == FMOE_MXFP4 ? 1u << 23 : 0u)           // scales are e8m0 (else e4m3)
         | (1u << 27);                                       // M / 128
}

// The scale copies and MMAs of a K step (kMmas of K = 64) on one stage. Scale tiles are 512
// bytes: 32 in descriptor units.
template <int kFormat, int BN, int S, int kMmas>
__device__ __forceinline__ void issue_step(uint32_t d, uint64_t ad, uint64_t bd, uint64_t sd,
                                           uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  using C = Cfg<kFormat, BN, S>;
  constexpr int kPer = kFormat == FMOE_MXFP4 ? 2 : 1;  // MMAs per scale tile
#pragma unroll
  for (int j = 0; j < (kMmas + kPer - 1) / kPer; ++j) {
    copy_scales(sfa + 4 * j, sd + 32 * j);
#pragma unroll
    for (int r = 0; r < C::kRuns; ++r)
      copy_scales(sfb + 4 * (j * C::kRuns + r), sd + (1 + r) * (C::kRunBytes / 16) + 32 * j);
  }
#pragma unroll
  for (int q = 0; q < kMmas; ++q) {
    const int j = q / kPer;
    mma_fp4<kFormat>(d, ad + 2 * q, bd + 2 * q, idesc_fp4<kFormat>(BN, q % kPer * 2), sfa + 4 * j,
                     sfb + 4 * j * C::kRuns, q > 0 ? 1u : accumulate);
  }
}

struct Tile {
  int m;        // row tile of a
  int rows;     // rows present
  int n;        // column tile
  int e;        // matrix of b
};

struct GemmFp4Args {
  const uint8_t* sa;
  const uint8_t* sb;
  const float* ga;
  const float* gb;
  void* out;
  int64_t M;
  int N, K;
  int m_tiles, n_tiles, panel;  // dense: tiles in panels of `panel` row tiles, rows first
  int dtype;
  int experts;                  // grouped: > 0
  const int* tile_first;
  const int* count;
  const float* row_w;
  // swiglu: the 4-bit blocks of the N / 2 values a row
  uint8_t* codes;
  uint8_t* scales;
  const float* gc;
  bool early;
  unsigned* sink;
};

// Tile i of the launch. Grouped (first / count: the experts' row tiles and rows in shared
// memory): an expert's tiles follow one another, its row tiles first, so that CTAs that run
// together read the same rows of b.
__device__ __forceinline__ bool tile_of(const GemmFp4Args& p, const int* first, const int* count,
                                        int64_t i, Tile& t) {
  if (p.experts == 0) {
    if (i >= (int64_t)p.m_tiles * p.n_tiles) return false;
    const int64_t per = (int64_t)p.panel * p.n_tiles;
    const int m = (int)(i / per) * p.panel;
    const int high = min(p.panel, p.m_tiles - m);
    const int r = (int)(i % per);
    t.m = m + r % high;
    t.n = r / high;
    t.rows = (int)min((int64_t)128, p.M - (int64_t)t.m * 128);
    t.e = 0;
    return true;
  }
  if (i >= (int64_t)first[p.experts] * p.n_tiles) return false;
  const int r = (int)(i / p.n_tiles);
  int low = 0, high = p.experts;  // first[low] <= r < first[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (first[mid] <= r) low = mid;
    else high = mid;
  }
  const int tiles = first[low + 1] - first[low];
  const int j = (int)(i - (int64_t)first[low] * p.n_tiles);
  t.e = low;
  t.m = first[low] + j % tiles;
  t.n = j / tiles;
  t.rows = min(128, count[low] - j % tiles * 128);
  return true;
}

__device__ __forceinline__ uint32_t pack2(int dtype, float x, float y) {
  if (dtype == FMOE_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The factor of a row's sums: two global scales and the row's weight. Their product may leave fp32
// where the results do not (two scales of 3e-23 multiply to nothing). Then `digits` is the product
// with an exponent that keeps a sum times it a normal number (sums of nvfp4 products lie in 2^-20 ..
// 2^39, or are 0), and the result what is to be multiplied by after it, a power of two (beyond fp32
// the results are 0 or infinite). Otherwise the result is the product, and `split` is false.
__device__ __forceinline__ float factor_of(float ga, float gb, float w, bool& split,
                                           float& digits) {
  const float ab = ga * gb, all = ab * w;
  split = false;
  if (fminf(fabsf(ab), fabsf(all)) >= 0x1p-126f && fmaxf(fabsf(ab), fabsf(all)) < 0x1p127f)
    return all;
  const double d = (double)ga * (double)gb * (double)w;  // three floats' exponents fit
  const int e = (int)(__double_as_longlong(d) >> 52 & 0x7ff) - 1023;
  if (d == 0.0 || e > 1000) return (float)d;  // an infinity, NaN
  const int low = max(-80, min(80, e));
  split = true;
  digits = (float)(d * __longlong_as_double((long long)(1023 + low - e) << 52));
  return ldexpf(1.0f, min(e - low, 127));
}

// Stores columns n .. n + 31 of the warp's 32 rows; lane l holds row m0 + l of `rows` and its 32
// values. Where rows are not whole 32-byte sectors the lanes exchange values (a 32 x 32
// transposition in registers), so that a store writes neighbouring columns of one row: 24 tiles
// with a row pitch of 2000 bytes took 23 us with a row per lane, 9 us so.
__device__ __forceinline__ void store32(const GemmFp4Args& p, int64_t m0, int rows, int n,
                                        uint32_t (&v)[32], float alpha, bool wide) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
  if (wide && n + 32 <= p.N) {
    if (lane >= rows) return;
    const int64_t at = (m0 + lane) * p.N + n;
    if (p.dtype == FMOE_F32) {
      float* o = static_cast<float*>(p.out) + at;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = v[i + j];
        st_global_v8(o + i, w);
      }
    } else {
      uint16_t* o = static_cast<uint16_t*>(p.out) + at;
#pragma unroll
      for (int i = 0; i < 32; i += 16) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j] = pack2(p.dtype, __uint_as_float(v[i + 2 * j]), __uint_as_float(v[i + 2 * j + 1]));
        st_global_v8(o + i, w);
      }
    }
    return;
  }
#pragma unroll
  for (int s = 16; s; s >>= 1) {
    const bool upper = lane & s;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i & s) continue;
      const uint32_t give = upper ? v[i] : v[i + s];
      const uint32_t take = __shfl_xor_sync(0xffffffffu, give, s);
      if (upper) v[i] = take;
      else v[i + s] = take;
    }
  }
  // now lane l holds column n + l, v[i] of row m0 + i
  if (n + lane >= p.N) return;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (i >= rows) break;
    const int64_t at = (m0 + i) * p.N + n + lane;
    const float x = __uint_as_float(v[i]);
    if (p.dtype == FMOE_F32) static_cast<float*>(p.out)[at] = x;
    else if (p.dtype == FMOE_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
    else static_cast<__half*>(p.out)[at] = __float2half_rn(x);
  }
}

// Columns [col, col + 32) of a row's halves: gate * silu(up), as 4-bit blocks. Returns the scale
// bytes, one (mxfp4) or two.
template <int kFormat>
__device__ __forceinline__ uint32_t swiglu32(const uint32_t (&gate)[32], const uint32_t (&up)[32],
                                             float alpha, const NvDivisor& divisor, uint4& codes) {
  float v[32];
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = swiglu(__uint_as_float(gate[i]) * alpha, __uint_as_float(up[i]) * alpha);
    top[i / 16] = max(top[i / 16], __float_as_uint(v[i]) & 0x7fffffffu);
  }
  if (kFormat == FMOE_MXFP4) top[0] = top[1] = max(top[0], top[1]);
  uint32_t bytes = 0;
  uint32_t w[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v[16 * h + i];
    const uint32_t b = encode16<kFormat>(x, top[h], divisor, w[2 * h], w[2 * h + 1]);
    bytes |= kFormat == FMOE_MXFP4 ? b : b << (8 * h);
  }
  codes = make_uint4(w[0], w[1], w[2], w[3]);
  return bytes;
}

// ---- the cluster's exchange -----------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of the same shared memory location in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                           uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void peer_arrive(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}
// mbar_wait for a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity,
                                                  const volatile int* abort) {
  const uint32_t a = smem_addr(bar);
  const uint64_t t0 = globaltimer();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*abort || globaltimer() - t0 > kWaitTimeoutNs) return false;
  }
}
// All threads of all CTAs of the cluster.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\t"
               "barrier.cluster.wait.acquire;" ::
                   : "memory");
}

// kSplit > 1 (at most 32 rows, so fewer tiles than would keep every SM reading): the CTAs of a
// cluster share one tile, each a part of the K steps. CTA r finishes the tile's slice r of the
// columns: the others store their sums of that slice into its shared memory, it adds them in the
// order of the ranks. 16 x 4096 x 7168: 8.3 us, 15 with whole tiles.
template <int kFormat, int BN, Epilogue kEpi, int kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_a32,
                    const __grid_constant__ CUtensorMap map_b, const GemmFp4Args p) {
  using C = Cfg<kFormat, BN, kSplit>;
  __shared__ int s_first[kMaxExperts + 1], s_count[kMaxExperts];
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* exchange = stages + S * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(exchange + C::kExchange);
  uint64_t* full = bars;         // [S] copies -> MMA
  uint64_t* empty = bars + 8;    // [S] MMA -> copies
  uint64_t* tfull = bars + 16;   // [2] MMA -> epilogue
  uint64_t* tempty = bars + 18;  // [2] epilogue -> MMA
  uint64_t* mma_done = bars + 20;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 22);
  int* err = reinterpret_cast<int*>(bars + 23);
  uint64_t* xfull = bars + 24;   // the other CTAs' sums of this one's slice have come

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 2);  // the issuers of a and of b
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], kEpiWarps);
    }
    mbar_init(mma_done, 1);
    if (kSplit > 1) mbar_init(xfull, 32 * (kSplit - 1));
    *abort_flag = 0;
    *err = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_a32);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  if constexpr (kSplit > 1) cluster_sync();  // the peers' barriers are there
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Within the expert layer (p.early) the plan and the weights were complete before the kernel in
  // front of this one passed its own wait, which this grid starts behind: the weights' copies
  // need not wait for it.
  if (!p.early) {
    pdl_wait();
    pdl_trigger();
  }
  if (p.experts > 0) {
    for (int e = threadIdx.x; e <= p.experts; e += kThreads) {
      s_first[e] = p.tile_first[e];
      if (e < p.experts) s_count[e] = p.count[e];
    }
    __syncthreads();
  }
  if (p.early && warp != 0) {
    pdl_wait();
    pdl_trigger();
  }

  const int steps = (p.K + kStepCols - 1) / kStepCols;
  const int across = tiles_across(p.K, kFormat);  // scale tiles per 128 rows
  const uint32_t rank = kSplit > 1 ? cluster_rank() : 0;
  // the tile's K steps [k0, k1) of this CTA
  const int k0 = steps * (int)rank / kSplit, k1 = steps * ((int)rank + 1) / kSplit;
  // Tile j of this CTA (round-robin; a cluster has one); false: no more.
  auto next = [&](int64_t j, Tile& t) {
    if (kSplit > 1) return j == 0 && tile_of(p, s_first, s_count, blockIdx.x / kSplit, t);
    return tile_of(p, s_first, s_count, blockIdx.x + j * gridDim.x, t);
  };
  // how many tiles back the accumulator of a tile must have been read
  constexpr int kBack = C::kOverlapped ? 1 : 2;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------------ copies of b
      const uint64_t keep = policy_evict_last(), once = policy_evict_first();
      int it = 0;
      bool ok = true;
      Tile t;
      for (int64_t j = 0; ok && next(j, t); ++j) {
        // the 128-row runs of b: next to each other, or gate and up rows
        int row[C::kRuns], runs = 0;
        const uint8_t* sb[C::kRuns];
#pragma unroll
        for (int r = 0; r < C::kRuns; ++r) {
          row[r] = kEpi == kSwiglu ? t.n * 128 + r * (p.N / 2) : t.n * BN + r * 128;
          if (row[r] < p.N) ++runs;  // a run past b's last row is not there
          sb[r] = p.sb + ((int64_t)t.e * tiles_down(p.N) + row[r] / 128) * across * kTileBytes;
        }
        // an expert with one row tile reads its weights once
        const bool reread = p.experts == 0 || s_first[t.e + 1] - s_first[t.e] > 1;
        const uint64_t policy = reread ? keep : once;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (!mbar_wait(&empty[s], ((it / S) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* st = stages + s * C::kStageBytes;
          uint8_t* sc = st + kABytes + C::kBBytes;
          const int have = min(C::kScaleTiles, across - k * C::kScaleTiles) * kTileBytes;
          const int64_t at = (int64_t)k * C::kScaleTiles * kTileBytes;
          mbar_arrive_expect_tx(&full[s], runs * (128 * 128 + have));
#pragma unroll
          for (int r = 0; r < C::kRuns; ++r) {
            if (r >= runs) break;
            tma_load_3d(st + kABytes + r * 128 * 128, &map_b, &full[s], k * 128, row[r], t.e,
                        policy);
            bulk_load_1d(sc + (1 + r) * C::kRunBytes, sb[r] + at, have, &full[s]);
          }
        }
      }
      if (!ok) {
        atomicOr(err, kErrTimeoutProducer);
        *abort_flag = 1;
      }
      // every copy must land before the CTA's shared memory is released (where the other issuer
      // gave up, the wait runs out: the copies have landed by then)
      static const int zero = 0;
      for (int j = it > S ? it - S : 0; j < it; ++j) mbar_wait(&full[j % S], (j / S) & 1, &zero);
    }
    __syncwarp();
  } else if (warp == 10) {
    if (lane == 0) {
      // ------------------------------------------------------------------ copies of a
      const uint64_t keep = policy_evict_last();
      int it = 0;
      bool ok = true;
      Tile t;
      for (int64_t j = 0; ok && next(j, t); ++j) {
        const uint8_t* sa = p.sa + (int64_t)t.m * across * kTileBytes;
        // few rows: boxes of 32 (the other rows of the stage keep what they held; a row of a
        // only reaches its own row of the product)
        const int boxes = t.rows > 64 ? 0 : (t.rows + 31) / 32;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (!mbar_wait(&empty[s], ((it / S) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* st = stages + s * C::kStageBytes;
          const int have = min(C::kScaleTiles, across - k * C::kScaleTiles) * kTileBytes;
          mbar_arrive_expect_tx(&full[s], (boxes ? boxes * 4096 : kABytes) + have);
          if (boxes == 0) tma_load_2d(st, &map_a, &full[s], k * 128, t.m * 128, keep);
          for (int x = 0; x < boxes; ++x)
            tma_load_2d(st + x * 4096, &map_a32, &full[s], k * 128, t.m * 128 + 32 * x, keep);
          bulk_load_1d(st + kABytes + C::kBBytes, sa + (int64_t)k * C::kScaleTiles * kTileBytes,
                       have, &full[s]);
        }
      }
      if (!ok) {
        atomicOr(err, kErrTimeoutProducer);
        *abort_flag = 1;
      }
      static const int zero = 0;
      for (int j = it > S ? it - S : 0; j < it; ++j) mbar_wait(&full[j % S], (j / S) & 1, &zero);
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------------------- MMAs
    // The whole warp runs this loop and one elected lane issues: the operands stay in uniform
    // registers.
    int it = 0, n = 0;
    bool ok = true;
    Tile t;
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t st0 = __shfl_sync(0xffffffffu, smem_addr(stages), 0);
    for (int64_t j = 0; ok && next(j, t); ++j) {
      if (n >= kBack &&
          !mbar_wait(&tempty[(n - kBack) & 1], ((n - kBack) >> 1) & 1, abort_flag))
        ok = false;
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = base + (n & 1) * C::kAcc1;
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % S;
        // the scale slot's last reader, two steps back
        if ((it >= 2 && !mbar_wait(&empty[(it - 2) % S], ((it - 2) / S) & 1, abort_flag)) ||
            !mbar_wait(&full[s], (it / S) & 1, abort_flag))
          ok = false;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = st0 + s * C::kStageBytes;
        const uint32_t sfa = base + C::kScales + (it & 1) * C::kSlotCols;
        const uint32_t sfb = sfa + C::kSfaCols;
        const uint64_t ad = smem_desc_kmajor(st, 128);
        const uint64_t bd = smem_desc_kmajor(st + kABytes, 128);
        const uint64_t sd = scale_desc(st + kABytes + C::kBBytes);
        const int mmas = min(4, (p.K - k * kStepCols + 63) / 64);
        if (elect_one()) {
          if (mmas == 4) issue_step<kFormat, BN, kSplit, 4>(d, ad, bd, sd, sfa, sfb, k != k0);
          else if (mmas == 3) issue_step<kFormat, BN, kSplit, 3>(d, ad, bd, sd, sfa, sfb, k != k0);
          else if (mmas == 2) issue_step<kFormat, BN, kSplit, 2>(d, ad, bd, sd, sfa, sfb, k != k0);
          else issue_step<kFormat, BN, kSplit, 1>(d, ad, bd, sd, sfa, sfb, k != k0);
          tc_commit(&empty[s]);
          if (k == k1 - 1) tc_commit(&tfull[n & 1]);
        }
        __syncwarp();
      }
      ++n;
    }
    if (!ok && lane == 0) {
      atomicOr(err, kErrTimeoutMma);
      *abort_flag = 1;
    }
    // all issued MMAs must retire before tensor memory is released
    static const int zero = 0;
    if (elect_one()) {
      tc_commit(mma_done);
      mbar_wait(mma_done, 0, &zero);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------------- epilogue
    const int q = warp & 3;                   // tensor memory lanes 32 q .. 32 q + 31
    const int half = (warp - 2) >> 2;         // columns half * BN / 2 ..
    const float ga = p.ga ? *p.ga : 1.0f;
    const NvDivisor divisor = nv_divisor(kEpi == kSwiglu && p.gc ? *p.gc : 1.0f);
    const bool wide = (int64_t)p.N * (p.dtype == FMOE_F32 ? 4 : 2) % 32 == 0 &&
                      reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
    constexpr int kChunks = BN / 64;          // 32-column chunks of this warp
    int n = 0;
    bool ok = true;
    Tile t;
    for (int64_t j = 0; ok && next(j, t); ++j) {
      const int row = q * 32 + lane;
      const int64_t m = (int64_t)t.m * 128 + row, m0 = m - lane;
      const int rows = t.rows - q * 32;  // of this warp's 32
      bool split;  // (loaded while the tile is multiplied)
      float digits = 1.0f;
      const float alpha = factor_of(ga, p.gb ? p.gb[t.e] : 1.0f,
                                    p.row_w && row < t.rows ? p.row_w[m] : 1.0f, split, digits);
      split = __any_sync(0xffffffffu, split);
      if (!mbar_wait(&tfull[n & 1], (n >> 1) & 1, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + (n & 1) * C::kAcc1 + ((uint32_t)(q * 32) << 16);
      const int n0 = t.n * BN;
      if (__builtin_expect(split, false)) {
        // the digits' part in place, before anyone reads: this warp's columns, or its gate and up
        // columns. (A second multiplication wherever the sums are used, which no ordinary tile needs,
        // took the expert layer of 16 tokens from 94 to 102 us by its code alone.)
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 8) {
          const uint32_t at = acc + (kEpi == kSwiglu ? half * 64 + (c & 63) + (c & 64) * 2
                                                     : half * (BN / 2) + c);
          uint32_t v[8];
          tmem_ld_32x32b<8>(at, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * digits);
          tmem_st_32x32b_x8(at, v);
        }
        tmem_st_wait();
      }
      if constexpr (kSplit > 1) {
        // ---- a tile that the cluster shares: rows 0..31, so only the warps of lanes 0..31
        static_assert(kEpi == kStore && !C::kOverlapped, "a cluster's tile");
        constexpr int V = C::kSlice;
        const bool mine = q == 0 && (int)rank / (kSplit / 2) == half;
        if (q == 0 && (kSplit > 2 || !mine)) {
#pragma unroll
          for (int j = 0; j < kSplit / 2; ++j) {
            const int s = half * (kSplit / 2) + j;
            if (s == (int)rank) continue;
            const uint32_t src = rank < (uint32_t)s ? rank : rank - 1;
            const uint32_t to =
                peer_addr(smem_addr(exchange), s) + src * (V * 128) + (uint32_t)lane * 16;
#pragma unroll
            for (int c = 0; c < V / 32; ++c) {
              uint32_t v[32];
              tmem_ld_32x32b<32>(acc + s * V + 32 * c, v);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 8; ++x)
                peer_store(to + (c * 8 + x) * 512, v[4 * x], v[4 * x + 1], v[4 * x + 2],
                           v[4 * x + 3]);
            }
            peer_arrive(peer_addr(smem_addr(xfull), s));
          }
        }
        if (mine) {
          if (!mbar_wait_cluster(xfull, 0, abort_flag)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          // the slice: the ranks' parts added in their order
#pragma unroll
          for (int c = 0; c < V / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b<32>(acc + (int)rank * V + 32 * c, v);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              float sum[4] = {};
#pragma unroll
              for (int r = 0; r < kSplit; ++r) {
                float4 f;
                if (r == (int)rank) {
                  f = make_float4(__uint_as_float(v[4 * x]), __uint_as_float(v[4 * x + 1]),
                                  __uint_as_float(v[4 * x + 2]), __uint_as_float(v[4 * x + 3]));
                } else {
                  const int src = r < (int)rank ? r : r - 1;
                  f = *reinterpret_cast<const float4*>(exchange + src * (V * 128) +
                                                       (c * 8 + x) * 512 + lane * 16);
                }
                sum[0] += f.x;
                sum[1] += f.y;
                sum[2] += f.z;
                sum[3] += f.w;
              }
#pragma unroll
              for (int y = 0; y < 4; ++y) v[4 * x + y] = __float_as_uint(sum[y]);
            }
            store32(p, m0, rows, n0 + (int)rank * V + 32 * c, v, alpha, wide);
          }
        }
      } else if constexpr (kEpi == kSwiglu) {
        // this warp's 64 gate columns (col) and 64 up columns (128 + col). The side that lies in
        // the columns shared with the next tile comes first: up in the first accumulator
        // (160..255), gate in the second (0..95).
        const bool first = (n & 1) == 0;
        const uint32_t col = half * 64;
        uint32_t s0[32], s1[32], o[32];
        const uint32_t side = acc + col + (first ? 128 : 0), other = acc + col + (first ? 0 : 128);
        tmem_ld_32x32b<32>(side, s0);
        tmem_ld_32x32b<32>(side + 32, s1);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[n & 1]);
        const int I = p.N / 2, c0 = t.n * 128 + (int)col;
        uint8_t* dst = p.codes + m * (I / 2) + c0 / 2;
        uint32_t bytes = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_ld_32x32b<32>(other + 32 * h, o);
          tmem_ld_wait();
          uint4 codes;
          uint32_t b;
          if (first) b = swiglu32<kFormat>(o, h ? s1 : s0, alpha, divisor, codes);
          else b = swiglu32<kFormat>(h ? s1 : s0, o, alpha, divisor, codes);
          bytes |= b << (kFormat == FMOE_MXFP4 ? 8 * h : 16 * h);
          if (row < t.rows) *reinterpret_cast<uint4*>(dst + 16 * h) = codes;
        }
        if (row < t.rows) {
          const int block = c0 / block_of(kFormat);
          uint8_t* sc = p.scales +
                        ((int64_t)t.m * tiles_across(I, kFormat) + block / 4) * kTileBytes +
                        scale_offset(row, block);
          if (kFormat == FMOE_MXFP4) *reinterpret_cast<uint16_t*>(sc) = (uint16_t)bytes;
          else *reinterpret_cast<uint32_t*>(sc) = bytes;
        }
      } else if constexpr (!C::kOverlapped) {
        const uint32_t col = half * (BN / 2);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b<32>(acc + col + 32 * c, v);
          tmem_ld_wait();
          if (c == kChunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[n & 1]);
          }
          store32(p, m0, rows, n0 + col + 32 * c, v, alpha, wide);
        }
      } else {
        // the columns that the next tile's accumulator shares with this one come first:
        // 160..255 of the first accumulator (upper half's 32..127), 0..95 of the second (lower
        // half's 0..95)
        const bool first = (n & 1) == 0;
        const uint32_t col = half * 128;
        const bool shares = first == (half == 1);
        const uint32_t c0 = col + (shares && first ? 32 : 0);
        uint32_t v0[32], v1[32], v2[32];
        if (shares) {
          tmem_ld_32x32b<32>(acc + c0, v0);
          tmem_ld_32x32b<32>(acc + c0 + 32, v1);
          tmem_ld_32x32b<32>(acc + c0 + 64, v2);
          tmem_ld_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[n & 1]);
        if (shares) {
          store32(p, m0, rows, n0 + c0, v0, alpha, wide);
          store32(p, m0, rows, n0 + c0 + 32, v1, alpha, wide);
          store32(p, m0, rows, n0 + c0 + 64, v2, alpha, wide);
          const uint32_t c1 = first ? col : col + 96;
          tmem_ld_32x32b<32>(acc + c1, v0);
          tmem_ld_wait();
          store32(p, m0, rows, n0 + c1, v0, alpha, wide);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_32x32b<32>(acc + col + 32 * c, v0);
            tmem_ld_wait();
            store32(p, m0, rows, n0 + col + 32 * c, v0, alpha, wide);
          }
        }
      }
      ++n;
    }
    if (!ok && lane == 0) {
      atomicOr(err, kErrTimeoutEpilogue);
      *abort_flag = 1;
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *err != 0 && p.sink) report_device_error(p.sink, *err);
  if constexpr (kSplit > 1) cluster_sync();  // no peer writes to this CTA's memory any more
}

struct Maps {
  CUtensorMap a, a32, b;
};

template <int kFormat, int BN, Epilogue kEpi, int kSplit>
cudaError_t launch(const Maps& maps, const GemmFp4Args& p, int clusters, cudaStream_t stream) {
  using C = Cfg<kFormat, BN, kSplit>;
  auto* fn = fp4_gemm_kernel<kFormat, BN, kEpi, kSplit>;
  static thread_local int configured = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (configured != dev) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    configured = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * kSplit));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kSplit;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kSplit > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, maps.a, maps.a32, maps.b, p);
}

template <int kFormat>
cudaError_t launch(int bn, int split, bool swiglu, const Maps& maps, const GemmFp4Args& p,
                   int clusters, cudaStream_t stream) {
  if (swiglu) return launch<kFormat, 256, kSwiglu, 1>(maps, p, clusters, stream);
  if (bn == 256) return launch<kFormat, 256, kStore, 1>(maps, p, clusters, stream);
  if (split == 4) return launch<kFormat, 128, kStore, 4>(maps, p, clusters, stream);
  if (split == 2) return launch<kFormat, 128, kStore, 2>(maps, p, clusters, stream);
  return launch<kFormat, 128, kStore, 1>(maps, p, clusters, stream);
}

int bad(const std::string& msg) {
  set_last_error(msg);
  return FMOE_ERR_VALUE;
}

}  // namespace

int launch_fp4_gemm(const Fp4Gemm& g, cudaStream_t stream) {
  const int sms = num_sms();
  GemmFp4Args p = {};
  p.sa = static_cast<const uint8_t*>(g.sa);
  p.sb = static_cast<const uint8_t*>(g.sb);
  p.ga = g.ga;
  p.gb = g.gb;
  p.out = g.out;
  p.M = g.M;
  p.N = g.N;
  p.K = g.K;
  p.dtype = g.dtype;
  p.experts = g.experts;
  p.tile_first = g.tile_first;
  p.count = g.count;
  p.row_w = g.row_w;
  p.codes = static_cast<uint8_t*>(g.codes);
  p.scales = static_cast<uint8_t*>(g.scales);
  p.gc = g.gc;
  p.early = g.early;
  p.m_tiles = (int)tiles_down(g.M);
  const bool swiglu = g.codes != nullptr;
  const int steps = (g.K + kStepCols - 1) / kStepCols;
  int bn = 256, split = 1;
  if (g.experts == 0) {
    // A K step's time goes by the bytes it brings to the SM (about 60 a cycle): 54 KB at BN 256,
    // 36 KB at 128. The cheaper of the two in rounds of tiles over the SMs: 1024 x 4096 x 7168
    // runs 128 tiles of 256 in 19.7 us, 256 tiles of 128 in 28 us; 128 x 4096 x 7168 takes 15 us
    // with tiles of 128, 18 us with tiles of 256.
    auto rounds = [&](int n) {
      return ((int64_t)p.m_tiles * ((g.N + n - 1) / n) + sms - 1) / sms;
    };
    if (rounds(128) * 36 <= rounds(256) * 54) bn = 128;
    // few rows and too few tiles: tiles shared by 2 or 4 CTAs, as long as each has two K steps;
    // at most one tile a cluster
    if (g.M <= 32 && bn == 128) {
      const int tiles = (g.N + bn - 1) / bn;
      while (split < 4 && tiles * split * 2 <= sms && steps >= 4 * split) split *= 2;
    }
  }
  p.n_tiles = (g.N + bn - 1) / bn;
  p.panel = 8;
  p.sink = device_error_sink(stream);
  Maps maps;
  int v = make_byte_map(&maps.a, g.a, g.K / 2, g.M, 0, 128, 128, "a");
  if (v == FMOE_OK) v = make_byte_map(&maps.a32, g.a, g.K / 2, g.M, 0, 128, 32, "a");
  if (v == FMOE_OK)
    v = make_byte_map(&maps.b, g.b, g.K / 2, g.N, g.experts > 0 ? g.experts : 1, 128, 128, "b");
  if (v != FMOE_OK) return v;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  const int clusters = (int)(tiles < sms / split ? tiles : sms / split);
  const cudaError_t e = g.format == FMOE_MXFP4
                            ? launch<FMOE_MXFP4>(bn, split, swiglu, maps, p, clusters, stream)
                            : launch<FMOE_NVFP4>(bn, split, swiglu, maps, p, clusters, stream);
  if (e == cudaSuccess) return FMOE_OK;
  set_last_error(std::string("4-bit product: ") + cudaGetErrorString(e));
  return FMOE_ERR_RUNTIME;
}

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_fp4_matmul(const fmoe_fp4_matrix* a, const fmoe_fp4_matrix* b, void* out,
                               int32_t dtype, void* stream) {
  int v = fp4_check(a, "a");
  if (v != FMOE_OK) return v;
  if ((v = fp4_check(b, "b")) != FMOE_OK) return v;
  if (a->format != b->format) return bad("a and b must have the same format");
  if (a->cols != b->cols) return bad("a and b must have the same number of columns");
  if (a->batch != 1 || b->batch != 1) return bad("a and b must be single matrices");
  if (a->rows > (int64_t)1 << 22 || b->rows > (int64_t)1 << 22)
    return bad("a and b must have at most 2^22 rows");
  if (dtype < FMOE_F32 || dtype > FMOE_F16) {
    set_last_error("dtype must be FMOE_F32, FMOE_BF16 or FMOE_F16");
    return FMOE_ERR_TYPE;
  }
  if (a->rows == 0 || b->rows == 0) return FMOE_OK;
  if ((v = fp4_check_pointers(a, "a")) != FMOE_OK) return v;
  if ((v = fp4_check_pointers(b, "b")) != FMOE_OK) return v;
  if (!out || reinterpret_cast<uintptr_t>(out) % 16) return bad("out must be 16-byte aligned");
  Fp4Gemm g = {};
  g.format = a->format;
  g.a = a->codes;
  g.sa = a->scales;
  g.M = a->rows;
  g.b = b->codes;
  g.sb = b->scales;
  g.N = (int)b->rows;
  g.K = (int)a->cols;
  g.ga = a->global_scale;
  g.gb = b->global_scale;
  g.out = out;
  g.dtype = dtype;
  return launch_fp4_gemm(g, static_cast<cudaStream_t>(stream));
}
