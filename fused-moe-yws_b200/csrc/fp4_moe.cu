// fp4_moe.cu -- the expert layer on 4-bit weights (fmoe_fp4_forward).
//
//   plan      (token, k) pairs of the local experts in expert order, stable; every expert's rows
//             start at a multiple of 128, the row tile of the products
//   quantise  the pairs' hidden rows, gathered, to 4-bit blocks
//   product 1 with W13, SwiGLU and quantisation to 4-bit blocks in its epilogue
//   product 2 with W2, times the routing weight, to fp32 rows
//   combine   a token's rows summed in the order of its picks
//
// Nothing returns to the host: the number of row tiles stays on the device, buffers are sized
// for every pair being local.
#include <cuda_runtime.h>

#include <string>

#include "fmoe.h"
#include "fmoe_common.cuh"
#include "fmoe_kernels.cuh"
#include "fp4.cuh"
#include "fp4_kernels.cuh"

namespace fmoe {
namespace {

constexpr int kPlanThreads = 1024;   // pairs per CTA of the plan
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanExperts = 256;    // local experts (kMaxLocalExperts)

struct PlanArgs {
  const int* idx;      // [T, K]
  const float* w;      // [T, K]
  int64_t pairs;       // T * K
  int K, experts, offset;
  int* cta_count;      // [CTAs, experts]
  int* count;          // [experts]
  int* tile_first;     // [experts + 1]
  int* row_token;      // [capacity]: token of a row, -1 behind an expert's last
  float* row_w;        // [capacity]
  int* token_row;      // [T, K]: row of a pair, -1 for one that is not local
};

__device__ __forceinline__ int local_expert(const PlanArgs& a, int64_t i) {
  if (i >= a.pairs) return -1;
  const int g = a.idx[i];
  if (g < a.offset) return -1;
  return g - a.offset < a.experts ? g - a.offset : -1;
}

// The CTA's pairs per expert.
__global__ void __launch_bounds__(kPlanThreads) fp4_plan_count_kernel(PlanArgs a) {
  __shared__ int s_count[kPlanExperts];
  for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) s_count[e] = 0;
  pdl_wait();
  pdl_trigger();
  __syncthreads();
  const int e = local_expert(a, (int64_t)blockIdx.x * kPlanThreads + threadIdx.x);
  const unsigned same = __match_any_sync(0xffffffffu, e);
  if (e >= 0 && (int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&s_count[e], __popc(same));
  __syncthreads();
  for (int i = threadIdx.x; i < a.experts; i += kPlanThreads)
    a.cta_count[(int64_t)blockIdx.x * a.experts + i] = s_count[i];
}

// Every pair's row. Each CTA sums the counts of all CTAs itself: the experts' totals give the
// row tiles, the CTAs before it its first rows. With one CTA its own counts are all there are.
__global__ void __launch_bounds__(kPlanThreads) fp4_plan_rows_kernel(PlanArgs a) {
  __shared__ int s_warp[kPlanWarps][kPlanExperts];  // pairs of a warp, then of those before it
  __shared__ int s_total[kPlanExperts], s_before[kPlanExperts];
  __shared__ int s_tile[kPlanExperts + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int warps = blockDim.x / 32;  // a single CTA has as many as its pairs need
  for (int w = warp; w < warps; w += warps)
    for (int x = lane; x < a.experts; x += 32) s_warp[w][x] = 0;
  __syncthreads();
  const int64_t i = (int64_t)blockIdx.x * kPlanThreads + tid;
  const int e = local_expert(a, i);
  const float weight = i < a.pairs ? a.w[i] : 0.0f;
  const unsigned same = __match_any_sync(0xffffffffu, e);
  const int rank = __popc(same & ((1u << lane) - 1u));
  if (e >= 0 && rank == 0) s_warp[warp][e] = __popc(same);
  __syncthreads();
  for (int x = tid; x < a.experts; x += blockDim.x) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int n = s_warp[w][x];
      s_warp[w][x] = run;
      run += n;
    }
    int total = run, before = 0;
    if (gridDim.x > 1) {
      total = 0;
      constexpr int kBatch = 8;  // loads in flight
      for (int c = 0; c < (int)gridDim.x; c += kBatch) {
        int n[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
          n[q] = c + q < (int)gridDim.x ? a.cta_count[(int64_t)(c + q) * a.experts + x] : 0;
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          if (c + q < (int)blockIdx.x) before += n[q];
          total += n[q];
        }
      }
    }
    s_total[x] = total;
    s_before[x] = before;
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int b = 0; b < a.experts; b += 32) {
      const int x = b + lane;
      const int tiles = x < a.experts ? (s_total[x] + 127) / 128 : 0;
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      if (x < a.experts) s_tile[x] = run + sum - tiles;
      run += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s_tile[a.experts] = run;
  }
  __syncthreads();
  if (i < a.pairs) {
    int row = -1;
    if (e >= 0) {
      row = s_tile[e] * 128 + s_before[e] + s_warp[warp][e] + rank;
      a.row_token[row] = (int)(i / a.K);
      a.row_w[row] = weight;
    }
    a.token_row[i] = row;
  }
  // the rows behind each expert's last
  for (int x = blockIdx.x * warps + warp; x < a.experts; x += gridDim.x * warps)
    for (int r = s_tile[x] * 128 + s_total[x] + lane; r < s_tile[x + 1] * 128; r += 32)
      a.row_token[r] = -1;
  if (blockIdx.x == 0) {
    for (int x = tid; x <= a.experts; x += blockDim.x) {
      a.tile_first[x] = s_tile[x];
      if (x < a.experts) a.count[x] = s_total[x];
    }
  }
}

// out[t] = the sum of a token's rows in the order of its picks, rounded once. The rows are fp32 at
// every batch size: a token's result is the same whatever batch it is in. (Rows in bf16 would
// halve them but add as much error again as the result's own rounding.) A thread takes 8 columns
// (one sector of a row).
__global__ void __launch_bounds__(128) fp4_combine_kernel(const int* token_row, const float* rows,
                                                          __nv_bfloat16* out, int H, int K) {
  __shared__ int s_row[32];
  const int64_t t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < K) s_row[threadIdx.x] = token_row[t * K + threadIdx.x];
  __syncthreads();
  const int c = ((int)blockIdx.y * 128 + (int)threadIdx.x) * 8;
  if (c >= H) return;
  float sum[8] = {};
  for (int k = 0; k < K; ++k) {
    if (s_row[k] < 0) continue;
    const float4* p = reinterpret_cast<const float4*>(rows + (int64_t)s_row[k] * H + c);
    const float4 a = p[0], b = p[1];
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  }
  uint4 packed;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(sum[2 * i], sum[2 * i + 1]);
  *reinterpret_cast<uint4*>(out + t * H + c) = packed;
}

struct Layout {
  int64_t rows;  // capacity: every pair local, an expert's rows padded to 128
  int64_t ctas;
  size_t cta_count, count, tile_first, row_token, row_w, token_row, xq, xs, hidden, cq, cs, ow,
      total;
};

// Gate and up rows start at whole scale tiles of W13: SwiGLU and quantisation run in the first
// product's epilogue. Otherwise they are a pass of their own over an fp32 product.
bool fused(const fmoe_fp4_problem* p) { return p->intermediate_size % 128 == 0; }

Layout layout_of(const fmoe_fp4_problem* p) {
  Layout L = {};
  const int64_t pairs = p->num_tokens * p->top_k;
  const int64_t used = pairs < p->num_local_experts ? pairs : p->num_local_experts;
  L.rows = (pairs + 127 * used + 127) / 128 * 128;
  L.ctas = (pairs + kPlanThreads - 1) / kPlanThreads;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  };
  const size_t rows = (size_t)L.rows, tiles = rows / 128;
  L.cta_count = take((size_t)L.ctas * p->num_local_experts * 4);
  L.count = take((size_t)p->num_local_experts * 4);
  L.tile_first = take((size_t)(p->num_local_experts + 1) * 4);
  L.row_token = take(rows * 4);
  L.row_w = take(rows * 4);
  L.token_row = take((size_t)pairs * 4);
  L.xq = take(rows * (p->hidden_size / 2));
  L.xs = take(tiles * fp4::tiles_across(p->hidden_size, p->format) * fp4::kTileBytes);
  L.hidden = take(fused(p) ? 0 : rows * 2 * p->intermediate_size * 4);
  L.cq = take(rows * (p->intermediate_size / 2));
  L.cs = take(tiles * fp4::tiles_across(p->intermediate_size, p->format) * fp4::kTileBytes);
  L.ow = take(rows * p->hidden_size * 4);
  L.total = off;
  return L;
}

int bad(const std::string& msg) {
  set_last_error(msg);
  return FMOE_ERR_VALUE;
}

int check(const fmoe_fp4_problem* p) {
  if (!p) return bad("problem must not be NULL");
  if (p->num_tokens < 0 || p->num_tokens > (int64_t)1 << 20)
    return bad("num_tokens must be in [0, 2^20]");
  if (p->top_k < 1 || p->top_k > 32) return bad("top_k must be in [1, 32]");
  if (p->local_expert_offset < 0) return bad("local_expert_offset must not be negative");
  if (p->num_local_experts < 1 || p->num_local_experts > kPlanExperts)
    return bad("num_local_experts must be in [1, 256]");
  if (p->hidden_size < 32 || p->hidden_size % 32 != 0 || p->hidden_size > 16384)
    return bad("hidden_size must be a positive multiple of 32 (<= 16384)");
  if (p->intermediate_size < 32 || p->intermediate_size % 32 != 0 || p->intermediate_size > 16384)
    return bad("intermediate_size must be a positive multiple of 32 (<= 16384)");
  if (p->format != FMOE_MXFP4 && p->format != FMOE_NVFP4)
    return bad("format must be FMOE_MXFP4 or FMOE_NVFP4");
  if (p->dtype < FMOE_F32 || p->dtype > FMOE_F16) {
    set_last_error("dtype must be FMOE_F32, FMOE_BF16 or FMOE_F16");
    return FMOE_ERR_TYPE;
  }
  return FMOE_OK;
}

int cuda_failed(cudaError_t e) {
  set_last_error(std::string("4-bit expert layer: ") + cudaGetErrorString(e));
  return FMOE_ERR_RUNTIME;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_fp4_workspace_size(const fmoe_fp4_problem* p, size_t* bytes) {
  const int v = check(p);
  if (v != FMOE_OK) return v;
  if (!bytes) return bad("bytes must not be NULL");
  *bytes = layout_of(p).total;
  return FMOE_OK;
}

extern "C" int fmoe_fp4_forward(const fmoe_fp4_problem* p, const fmoe_fp4_tensors* t,
                                void* workspace, size_t workspace_bytes, void* stream_ptr) {
  int v = check(p);
  if (v != FMOE_OK) return v;
  if (!t) return bad("tensors must not be NULL");
  if (p->num_tokens == 0) return FMOE_OK;
  const void* ptrs[] = {t->hidden_states, t->topk_idx, t->topk_w, t->w13, t->w13_scales,
                        t->w2, t->w2_scales, t->output};
  const char* names[] = {"hidden_states", "topk_idx", "topk_w", "w13", "w13_scales",
                         "w2", "w2_scales", "output"};
  for (int i = 0; i < 8; ++i)
    if (!ptrs[i] || reinterpret_cast<uintptr_t>(ptrs[i]) % 16)
      return bad(std::string(names[i]) + " must be non-NULL and 16-byte aligned");
  for (const float* scale : {t->input_scale, t->intermediate_scale, t->w13_global, t->w2_global})
    if (reinterpret_cast<uintptr_t>(scale) % 4)
      return bad("global scales must be aligned to their type");
  if (p->format == FMOE_MXFP4 && (t->input_scale || t->intermediate_scale || t->w13_global ||
                                  t->w2_global))
    return bad("mxfp4 has no global scale");
  const Layout L = layout_of(p);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < L.total) {
    set_last_error("workspace must be 256-byte aligned and hold " + std::to_string(L.total) +
                   " bytes");
    return FMOE_ERR_WORKSPACE;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int H = p->hidden_size, I = p->intermediate_size, E = p->num_local_experts;

  PlanArgs plan = {};
  plan.idx = t->topk_idx;
  plan.w = t->topk_w;
  plan.pairs = p->num_tokens * p->top_k;
  plan.K = p->top_k;
  plan.experts = E;
  plan.offset = p->local_expert_offset;
  plan.cta_count = reinterpret_cast<int*>(ws + L.cta_count);
  plan.count = reinterpret_cast<int*>(ws + L.count);
  plan.tile_first = reinterpret_cast<int*>(ws + L.tile_first);
  plan.row_token = reinterpret_cast<int*>(ws + L.row_token);
  plan.row_w = reinterpret_cast<float*>(ws + L.row_w);
  plan.token_row = reinterpret_cast<int*>(ws + L.token_row);
  cudaError_t e = cudaSuccess;
  if (L.ctas > 1)
    e = launch_pdl(fp4_plan_count_kernel, dim3((unsigned)L.ctas), dim3(kPlanThreads), 0, stream,
                   plan);
  if (e == cudaSuccess)
    e = launch_pdl(fp4_plan_rows_kernel, dim3((unsigned)L.ctas),
                   dim3(L.ctas > 1 ? kPlanThreads : (unsigned)((plan.pairs + 127) / 128 * 128)), 0,
                   stream, plan);
  if (e != cudaSuccess) return cuda_failed(e);

  Fp4QuantArgs q = {};
  q.x = t->hidden_states;
  q.row_stride = H;
  q.rows = L.rows;
  q.cols = H;
  q.global = t->input_scale;
  q.codes = ws + L.xq;
  q.scales = ws + L.xs;
  q.row_index = plan.row_token;
  q.tiles_dev = plan.tile_first + E;
  if ((e = launch_fp4_quantize(q, p->format, p->dtype, 1, stream)) != cudaSuccess)
    return cuda_failed(e);

  Fp4Gemm g = {};
  g.format = p->format;
  g.a = q.codes;
  g.sa = q.scales;
  g.M = L.rows;
  g.b = t->w13;
  g.sb = t->w13_scales;
  g.N = 2 * I;
  g.K = H;
  g.ga = t->input_scale;
  g.gb = t->w13_global;
  g.experts = E;
  g.early = true;
  g.tile_first = plan.tile_first;
  g.count = plan.count;
  if (fused(p)) {
    g.codes = ws + L.cq;
    g.scales = ws + L.cs;
    g.gc = t->intermediate_scale;
  } else {
    g.out = ws + L.hidden;
    g.dtype = FMOE_F32;
  }
  if ((v = launch_fp4_gemm(g, stream)) != FMOE_OK) return v;

  if (!fused(p)) {
    q.x = ws + L.hidden;
    q.row_stride = 2 * I;
    q.cols = I;
    q.global = t->intermediate_scale;
    q.codes = ws + L.cq;
    q.scales = ws + L.cs;
    q.swiglu = true;
    if ((e = launch_fp4_quantize(q, p->format, FMOE_F32, 1, stream)) != cudaSuccess)
      return cuda_failed(e);
  }

  g.codes = g.scales = nullptr;
  g.a = ws + L.cq;
  g.sa = ws + L.cs;
  g.b = t->w2;
  g.sb = t->w2_scales;
  g.N = H;
  g.K = I;
  g.ga = t->intermediate_scale;
  g.gb = t->w2_global;
  g.out = ws + L.ow;
  g.dtype = FMOE_F32;
  g.row_w = plan.row_w;
  if ((v = launch_fp4_gemm(g, stream)) != FMOE_OK) return v;

  const unsigned T = (unsigned)p->num_tokens;
  e = launch_pdl(fp4_combine_kernel, dim3(T, (unsigned)((H / 8 + 127) / 128)), dim3(128), 0, stream,
                 (const int*)plan.token_row, reinterpret_cast<const float*>(ws + L.ow),
                 static_cast<__nv_bfloat16*>(t->output), H, p->top_k);
  return e == cudaSuccess ? FMOE_OK : cuda_failed(e);
}
