// fp4_quant.cu -- quantisation of a matrix to 4-bit blocks, and back.
//
// Bound by memory: 2 to 4 bytes a value in, 4.5 bits out (and back). A CTA takes 128 rows x 128
// columns: the 1 KB (nvfp4) or 512 bytes (mxfp4) of scales of that square lie back to back
// (fp4.cuh), so they are gathered in shared memory and leave in whole lines. A thread takes 16
// consecutive values of a row: one nvfp4 block, or half an mxfp4 block, whose other half its
// neighbour holds; four rows' loads are in flight together.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "fmoe.h"
#include "fmoe_common.cuh"
#include "fmoe_kernels.cuh"
#include "fp4.cuh"
#include "fp4_kernels.cuh"
#include "sm100.cuh"

namespace fmoe {
namespace {

using namespace fp4;

constexpr int kCols = 128;             // columns per CTA
constexpr int kThreads = 256;
constexpr int kAcross = kCols / 16;    // threads a row
constexpr int kDown = kThreads / kAcross;
static_assert(kDown == 32, "rows 32 apart share their place in a scale tile");

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T as_type(float v);
template <>
__device__ __forceinline__ float as_type<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half as_type<__half>(float v) { return __float2half_rn(v); }

// 16 consecutive elements as they lie in memory, by loads of kAlign bytes (the type's size where
// nothing better is aligned). Neighbouring lanes take neighbouring 32- or 64-byte pieces, so
// 16-byte accesses touch every sector in two instructions: with 32-byte stores the
// dequantisation of 4096 x 7168 to bf16 went from 17.9 to 10.8 us.
template <typename T>
struct Raw {
  uint32_t w[4 * sizeof(T)];
};
template <typename T, int kAlign>
__device__ __forceinline__ Raw<T> load16(const T* p) {
  Raw<T> r;
  if constexpr (kAlign == 32) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 4; i += 8)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]),
                     "=r"(r.w[i + 4]), "=r"(r.w[i + 5]), "=r"(r.w[i + 6]), "=r"(r.w[i + 7])
                   : "l"(reinterpret_cast<const uint32_t*>(p) + i));
  } else if constexpr (kAlign == 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i)
      reinterpret_cast<uint4*>(r.w)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      r.w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
    }
  }
  return r;
}
template <typename T, bool kSectors>
__device__ __forceinline__ void store16(T* p, const uint32_t (&w)[4 * sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) * 4; i += kSectors ? 8 : 4) {
    uint32_t* q = reinterpret_cast<uint32_t*>(p) + i;
    if constexpr (kSectors) {
      const uint32_t v[8] = {w[i],     w[i + 1], w[i + 2], w[i + 3],
                             w[i + 4], w[i + 5], w[i + 6], w[i + 7]};
      sm100::st_global_v8(q, v);
    } else {
      *reinterpret_cast<uint4*>(q) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
}

template <typename T2>
__device__ __forceinline__ T2 as_pair(uint32_t w) {
  return *reinterpret_cast<const T2*>(&w);
}

// The values, and the bits of the largest magnitude as fp32 (NaN above the infinity above the
// numbers). 16-bit types are compared two at a time.
template <typename T>
__device__ __forceinline__ uint32_t unpack16(const Raw<T>& r, float (&v)[16]) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = __uint_as_float(r.w[i]);
      top = max(top, r.w[i] & 0x7fffffffu);
    }
    return top;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 top = as_pair<T2>(0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = __hmax2_nan(top, as_pair<T2>(r.w[i] & 0x7fff7fffu));
      const T* e = reinterpret_cast<const T*>(&r.w[i]);
      v[2 * i] = as_float<T>(e[0]);
      v[2 * i + 1] = as_float<T>(e[1]);
    }
    const T* t = reinterpret_cast<const T*>(&top);
    return __float_as_uint(as_float<T>(__hmax_nan(t[0], t[1])));
  }
}

template <int kFormat, typename T, int kAlign, bool kSwiglu = false>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 4)
    fp4_quantize_kernel(Fp4QuantArgs a) {
  __shared__ __align__(16) uint8_t s_scale[kCols / tile_cols(kFormat) * kTileBytes];
  const int tid = threadIdx.x;
  const int c0 = blockIdx.y * kCols, e = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  const int across = tiles_across(a.cols, kFormat);
  const int first = c0 / tile_cols(kFormat);
  const int here = min(kCols / tile_cols(kFormat), across - first);
  const NvDivisor divisor = nv_divisor(a.global ? a.global[a.global_step * e] : 1.0f);
  const T* x = static_cast<const T*>(a.x) + e * a.batch_stride;
  uint8_t* codes = a.codes + (int64_t)e * a.rows * (a.cols / 2);
  const int c = c0 + tid % kAcross * 16;
  // (a row tile each, but for gathered rows: there are fewer tiles than the buffers have room for)
  const int tiles = a.tiles_dev ? *a.tiles_dev : (int)tiles_down(a.rows);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t m0 = (int64_t)tile * kTileRows;
    // A thread's rows are 32 apart (r = 32 u + tid / 8): kRows of them at a time, their loads in
    // flight together. Whole warps stay together: an mxfp4 block belongs to two lanes.
    constexpr int kRows = kSwiglu ? 2 : 4;
    const int r = tid / kAcross;
    const int64_t m = m0 + r;
    const T* from = x + m * a.row_stride + c;
    uint8_t* to = codes + m * (a.cols / 2) + c / 2;
    const int left = c < a.cols ? (int)min((int64_t)kTileRows, a.rows - m) : 0;  // rows from m on
#pragma unroll
    for (int g = 0; g < kTileRows / kDown; g += kRows) {
      Raw<T> raw[kRows], second[kSwiglu ? kRows : 1];
      bool mine[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int d = (g + u) * kDown;
        mine[u] = d < left;
        const T* p = from + d * a.row_stride;
        if (a.row_index) {
          const int src = mine[u] ? a.row_index[m + d] : -1;
          mine[u] = src >= 0;
          if (!kSwiglu) p = x + src * a.row_stride + c;
        }
        raw[u] = {};
        if (kSwiglu) second[kSwiglu ? u : 0] = {};
        if (mine[u]) {
          raw[u] = load16<T, kAlign>(p);
          if constexpr (kSwiglu) second[u] = load16<T, kAlign>(p + a.cols);
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        uint8_t* scale = s_scale + tid % kAcross * 16 / block_of(kFormat) / 4 * kTileBytes + r * 16 +
                         (g + u) * 4 + tid % kAcross * 16 / block_of(kFormat) % 4;
        if (!__any_sync(0xffffffffu, mine[u])) {  // few rows a tile: most warps have none
          *scale = 0;
          continue;
        }
        float v[16];
        uint32_t top = unpack16<T>(raw[u], v);
        if constexpr (kSwiglu) {
          float up[16];
          unpack16<T>(second[u], up);
          top = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = swiglu(v[i], up[i]);
            top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
          }
        }
        if constexpr (kFormat == FMOE_MXFP4) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        uint32_t lo, hi;
        const uint32_t byte = encode16<kFormat>(v, top, divisor, lo, hi);
        if (mine[u])
          *reinterpret_cast<uint2*>(to + (int64_t)(g + u) * kDown * (a.cols / 2)) =
              make_uint2(lo, hi);
        *scale = mine[u] ? (uint8_t)byte : 0;
      }
    }
    __syncthreads();
    uint8_t* out = a.scales +
                   (((int64_t)e * tiles_down(a.rows) + tile) * across + first) * kTileBytes;
    for (int i = tid; i < here * kTileBytes / 16; i += kThreads)
      reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(s_scale)[i];
    __syncthreads();
  }
}

template <int kFormat, typename T, bool kSectors>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(Fp4QuantArgs a) {
  __shared__ __align__(16) uint8_t s_scale[kCols / tile_cols(kFormat) * kTileBytes];
  const int tid = threadIdx.x;
  const int64_t m0 = (int64_t)blockIdx.x * kTileRows;
  const int c0 = blockIdx.y * kCols, e = blockIdx.z;
  const int across = tiles_across(a.cols, kFormat);
  const int first = c0 / tile_cols(kFormat);
  const int here = min(kCols / tile_cols(kFormat), across - first);
  const uint8_t* in = a.scales +
                      (((int64_t)e * tiles_down(a.rows) + blockIdx.x) * across + first) * kTileBytes;
  for (int i = tid; i < here * kTileBytes / 16; i += kThreads)
    reinterpret_cast<uint4*>(s_scale)[i] = reinterpret_cast<const uint4*>(in)[i];
  __syncthreads();
  const float global = a.global ? a.global[a.global_step * e] : 1.0f;
  const uint8_t* codes = a.codes + (int64_t)e * a.rows * (a.cols / 2);
  T* out = static_cast<T*>(a.out) + (int64_t)e * a.rows * a.cols;
  const int c = c0 + tid % kAcross * 16;
  if (c >= a.cols) return;
  constexpr int kRows = kTileRows / kDown;
  uint2 raw[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int64_t m = m0 + tid / kAcross + u * kDown;
    raw[u] = m < a.rows ? *reinterpret_cast<const uint2*>(codes + m * (a.cols / 2) + c / 2)
                        : make_uint2(0, 0);
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = tid / kAcross + u * kDown;
    const int64_t m = m0 + r;
    if (m >= a.rows) break;
    const int block = (c - c0) / block_of(kFormat);
    const float s = __fmul_rn(
        scale_value<kFormat>(s_scale[block / 4 * kTileBytes + scale_offset(r, block)]), global);
    float lo[8], hi[8];
    decode8(raw[u].x, lo);
    decode8(raw[u].y, hi);
    alignas(16) uint32_t packed[4 * sizeof(T)];
    T* t = reinterpret_cast<T*>(packed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = as_type<T>(__fmul_rn(lo[i], s));
      t[8 + i] = as_type<T>(__fmul_rn(hi[i], s));
    }
    store16<T, kSectors>(out + m * a.cols + c, packed);
  }
}

dim3 grid_of(const Fp4QuantArgs& a, int batch) {
  const int across = (a.cols + kCols - 1) / kCols;
  int64_t down = tiles_down(a.rows);
  if (a.tiles_dev) {
    // a few CTAs for every one that fits an SM: a grid over the whole capacity spent 18 of 40 us
    // on CTAs without rows (4096 tokens, 32 of 256 experts)
    const int64_t most = (24 * num_sms() + across - 1) / across;
    down = down < most ? down : most;
  }
  return dim3((unsigned)down, (unsigned)across, (unsigned)batch);
}

template <int kFormat, typename T>
cudaError_t quantize(const Fp4QuantArgs& a, int batch, cudaStream_t stream) {
  auto aligned = [&](int bytes) {
    const int64_t step = bytes / (int64_t)sizeof(T);
    return reinterpret_cast<uintptr_t>(a.x) % bytes == 0 && a.row_stride % step == 0 &&
           a.batch_stride % step == 0;
  };
  auto* fn = aligned(32)   ? fp4_quantize_kernel<kFormat, T, 32>
             : aligned(16) ? fp4_quantize_kernel<kFormat, T, 16>
                           : fp4_quantize_kernel<kFormat, T, 0>;
  return launch_pdl(fn, grid_of(a, batch), dim3(kThreads), 0, stream, a);
}

template <int kFormat>
cudaError_t quantize(const Fp4QuantArgs& a, int dtype, int batch, cudaStream_t stream) {
  if (a.swiglu)  // the expert layer's own fp32 buffer: aligned
    return launch_pdl(fp4_quantize_kernel<kFormat, float, 32, true>, grid_of(a, batch),
                      dim3(kThreads), 0, stream, a);
  if (dtype == FMOE_F32) return quantize<kFormat, float>(a, batch, stream);
  if (dtype == FMOE_BF16) return quantize<kFormat, __nv_bfloat16>(a, batch, stream);
  return quantize<kFormat, __half>(a, batch, stream);
}

template <int kFormat, typename T>
cudaError_t dequantize(const Fp4QuantArgs& a, int batch, cudaStream_t stream) {
  const dim3 grid = grid_of(a, batch);
  if (reinterpret_cast<uintptr_t>(a.out) % 32 == 0)
    fp4_dequantize_kernel<kFormat, T, true><<<grid, kThreads, 0, stream>>>(a);
  else
    fp4_dequantize_kernel<kFormat, T, false><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <int kFormat>
cudaError_t dequantize(const Fp4QuantArgs& a, int dtype, int batch, cudaStream_t stream) {
  if (dtype == FMOE_F32) return dequantize<kFormat, float>(a, batch, stream);
  if (dtype == FMOE_BF16) return dequantize<kFormat, __nv_bfloat16>(a, batch, stream);
  return dequantize<kFormat, __half>(a, batch, stream);
}

int bad(const std::string& msg) {
  set_last_error(msg);
  return FMOE_ERR_VALUE;
}

int bad_dtype(const char* what) {
  set_last_error(std::string(what) + " must be FMOE_F32, FMOE_BF16 or FMOE_F16");
  return FMOE_ERR_TYPE;
}

int done(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return FMOE_OK;
  set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
  return FMOE_ERR_RUNTIME;
}

Fp4QuantArgs args_of(const fmoe_fp4_matrix* q) {
  Fp4QuantArgs a = {};
  a.rows = q->rows;
  a.cols = (int)q->cols;
  a.global = q->global_scale;
  a.global_step = q->batch > 1 ? 1 : 0;
  a.codes = static_cast<uint8_t*>(q->codes);
  a.scales = static_cast<uint8_t*>(q->scales);
  return a;
}

}  // namespace

int fp4_check(const fmoe_fp4_matrix* q, const char* name) {
  const std::string n = name;
  if (!q) return bad(n + " must not be NULL");
  if (q->format != FMOE_MXFP4 && q->format != FMOE_NVFP4)
    return bad(n + ": format must be FMOE_MXFP4 or FMOE_NVFP4");
  if (q->rows < 0 || q->rows > (int64_t)1 << 30) return bad(n + ": rows must be in [0, 2^30]");
  if (q->cols < 32 || q->cols % 32 != 0 || q->cols > 65536)
    return bad(n + ": cols must be a multiple of 32 in [32, 65536]");
  if (q->batch < 1 || q->batch > 1024) return bad(n + ": batch must be in [1, 1024]");
  if (q->format == FMOE_MXFP4 && q->global_scale)
    return bad(n + ": mxfp4 has no global scale");
  return FMOE_OK;
}

int fp4_check_pointers(const fmoe_fp4_matrix* q, const char* name) {
  const std::string n = name;
  if (!q->codes || !q->scales) return bad(n + ": codes and scales must not be NULL");
  if (reinterpret_cast<uintptr_t>(q->codes) % 16 || reinterpret_cast<uintptr_t>(q->scales) % 16)
    return bad(n + ": codes and scales must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(q->global_scale) % 4)
    return bad(n + ": global_scale must be aligned to its type");
  return FMOE_OK;
}

cudaError_t launch_fp4_quantize(const Fp4QuantArgs& a, int format, int dtype, int batch,
                                cudaStream_t stream) {
  return format == FMOE_MXFP4 ? quantize<FMOE_MXFP4>(a, dtype, batch, stream)
                              : quantize<FMOE_NVFP4>(a, dtype, batch, stream);
}

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_fp4_scale_bytes(const fmoe_fp4_matrix* q, size_t* bytes) {
  const int v = fp4_check(q, "matrix");
  if (v != FMOE_OK) return v;
  if (!bytes) return bad("bytes must not be NULL");
  *bytes = (size_t)q->batch * fp4::tiles_down(q->rows) *
           fp4::tiles_across((int)q->cols, q->format) * fp4::kTileBytes;
  return FMOE_OK;
}

extern "C" int fmoe_fp4_quantize(const fmoe_fp4_matrix* q, const void* x, int32_t dtype,
                                 int64_t row_stride, int64_t batch_stride, void* stream) {
  int v = fp4_check(q, "matrix");
  if (v != FMOE_OK) return v;
  if (dtype < FMOE_F32 || dtype > FMOE_F16) return bad_dtype("dtype");
  if (q->rows == 0) return FMOE_OK;
  if ((v = fp4_check_pointers(q, "matrix")) != FMOE_OK) return v;
  if (!x || reinterpret_cast<uintptr_t>(x) % (dtype == FMOE_F32 ? 4 : 2))
    return bad("x must not be NULL and be aligned to its type");
  if (row_stride < 0 || batch_stride < 0) return bad("strides must not be negative");
  Fp4QuantArgs a = args_of(q);
  a.x = x;
  a.row_stride = row_stride;
  a.batch_stride = batch_stride;
  return done(launch_fp4_quantize(a, q->format, dtype, q->batch,
                                  static_cast<cudaStream_t>(stream)), "quantisation");
}

extern "C" int fmoe_fp4_dequantize(const fmoe_fp4_matrix* q, void* out, int32_t dtype,
                                   void* stream) {
  int v = fp4_check(q, "matrix");
  if (v != FMOE_OK) return v;
  if (dtype < FMOE_F32 || dtype > FMOE_F16) return bad_dtype("dtype");
  if (q->rows == 0) return FMOE_OK;
  if ((v = fp4_check_pointers(q, "matrix")) != FMOE_OK) return v;
  if (!out || reinterpret_cast<uintptr_t>(out) % 16) return bad("out must be 16-byte aligned");
  Fp4QuantArgs a = args_of(q);
  a.out = out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return done(q->format == FMOE_MXFP4 ? dequantize<FMOE_MXFP4>(a, dtype, q->batch, s)
                                      : dequantize<FMOE_NVFP4>(a, dtype, q->batch, s),
              "dequantisation");
}
