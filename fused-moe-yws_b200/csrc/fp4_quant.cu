// fp4_quant.cu -- quantisation of a matrix to 4-bit blocks, and back.
//
// A CTA takes 128 rows x 256 columns: the 2 KB (nvfp4) or 1 KB (mxfp4) of scales of that
// square lie back to back (fp4.cuh), so they are gathered in shared memory and leave in whole
// lines. A thread takes 16 consecutive values of a row: one nvfp4 block, or half an mxfp4
// block, whose other half its neighbour holds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "fmoe.h"
#include "fmoe_common.cuh"
#include "fmoe_kernels.cuh"
#include "fp4.cuh"
#include "fp4_kernels.cuh"

namespace fmoe {
namespace {

using namespace fp4;

constexpr int kCols = 256;      // columns per CTA
constexpr int kThreads = 256;   // 16 rows at a time, 16 threads a row

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

// 16 consecutive elements, by 16-byte loads where the address allows them.
template <typename T, bool kWide>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  if constexpr (kWide) {
    constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
      uint4 raw = *reinterpret_cast<const uint4*>(p + i * kPer);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i * kPer + j] = as_float<T>(e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = as_float<T>(p[i]);
  }
}

// gate * silu(up) with the fast exponential and division: a few units in the last place
__device__ __forceinline__ float swiglu(float gate, float up) {
  return gate * __fdividef(up, 1.0f + __expf(-up));
}

template <int kFormat, typename T, bool kWide, bool kSwiglu = false>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(Fp4QuantArgs a) {
  __shared__ __align__(16) uint8_t s_scale[kCols / tile_cols(kFormat) * kTileBytes];
  const int tid = threadIdx.x;
  const int64_t m0 = (int64_t)blockIdx.x * kTileRows;
  const int c0 = blockIdx.y * kCols, e = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  if (a.tiles_dev && (int)blockIdx.x >= *a.tiles_dev) return;  // row tiles nobody uses
  const int across = tiles_across(a.cols, kFormat);
  const int first = c0 / tile_cols(kFormat);
  const int here = min(kCols / tile_cols(kFormat), across - first);
  for (int i = tid; i < here * kTileBytes / 4; i += kThreads)
    reinterpret_cast<uint32_t*>(s_scale)[i] = 0;
  __syncthreads();
  const float global = a.global ? a.global[a.global_step * e] : 1.0f;
  const T* x = static_cast<const T*>(a.x) + e * a.batch_stride;
  uint8_t* codes = a.codes + (int64_t)e * a.rows * (a.cols / 2);
  const int c = c0 + (tid & 15) * 16;
  for (int r = tid >> 4; r < kTileRows; r += kThreads / 16) {
    const int64_t m = m0 + r;
    int64_t src = m;
    if (m < a.rows && a.row_index) src = a.row_index[m];
    // whole warps stay together: an mxfp4 block belongs to two lanes
    const bool mine = m < a.rows && src >= 0 && c < a.cols;
    float v[16] = {};
    uint32_t top = 0;
    if (mine) {
      if constexpr (kSwiglu) {
        float up[16];
        load16<T, kWide>(x + m * a.row_stride + c, v);
        load16<T, kWide>(x + m * a.row_stride + a.cols + c, up);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = swiglu(v[i], up[i]);
      } else {
        load16<T, kWide>(x + src * a.row_stride + c, v);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    uint32_t byte;
    if constexpr (kFormat == FMOE_MXFP4) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      float by;
      byte = mx_scale(top, by);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __fmul_rn(v[i], by);
    } else {
      float by;
      byte = nv_scale(top, global, by);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = by > 0.0f ? __fdiv_rn(v[i], by) : __fmul_rn(v[i], 0.0f);
    }
    if (mine) {
      const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
      const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
      *reinterpret_cast<uint2*>(codes + m * (a.cols / 2) + c / 2) =
          make_uint2(encode8(lo), encode8(hi));
      const int block = (c - c0) / block_of(kFormat);
      s_scale[block / 4 * kTileBytes + scale_offset(r, block)] = (uint8_t)byte;
    }
  }
  __syncthreads();
  uint8_t* out = a.scales +
                 (((int64_t)e * tiles_down(a.rows) + blockIdx.x) * across + first) * kTileBytes;
  for (int i = tid; i < here * kTileBytes / 16; i += kThreads)
    reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(s_scale)[i];
}

template <int kFormat, typename T>
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
  const int c = c0 + (tid & 15) * 16;
  if (c >= a.cols) return;
  for (int r = tid >> 4; r < kTileRows && m0 + r < a.rows; r += kThreads / 16) {
    const int64_t m = m0 + r;
    const uint2 raw = *reinterpret_cast<const uint2*>(codes + m * (a.cols / 2) + c / 2);
    const int block = (c - c0) / block_of(kFormat);
    const float s = __fmul_rn(
        scale_value<kFormat>(s_scale[block / 4 * kTileBytes + scale_offset(r, block)]), global);
    float lo[8], hi[8];
    decode8(raw.x, lo);
    decode8(raw.y, hi);
    constexpr int kPer = 16 / (int)sizeof(T);
    uint4 packed[16 / kPer];
    T* t = reinterpret_cast<T*>(packed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = as_type<T>(__fmul_rn(lo[i], s));
      t[8 + i] = as_type<T>(__fmul_rn(hi[i], s));
    }
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i)
      *reinterpret_cast<uint4*>(out + m * a.cols + c + i * kPer) = packed[i];
  }
}

dim3 grid_of(const Fp4QuantArgs& a, int batch) {
  return dim3((unsigned)tiles_down(a.rows), (unsigned)((a.cols + kCols - 1) / kCols),
              (unsigned)batch);
}

template <int kFormat, typename T>
cudaError_t quantize(const Fp4QuantArgs& a, int batch, cudaStream_t stream) {
  const int64_t step = 16 / (int64_t)sizeof(T);
  const bool wide = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.row_stride % step == 0 &&
                    a.batch_stride % step == 0;
  auto* fn = wide ? fp4_quantize_kernel<kFormat, T, true> : fp4_quantize_kernel<kFormat, T, false>;
  return launch_pdl(fn, grid_of(a, batch), dim3(kThreads), 0, stream, a);
}

template <int kFormat>
cudaError_t quantize(const Fp4QuantArgs& a, int dtype, int batch, cudaStream_t stream) {
  if (a.swiglu)  // the expert layer's own fp32 buffer: aligned
    return launch_pdl(fp4_quantize_kernel<kFormat, float, true, true>, grid_of(a, batch),
                      dim3(kThreads), 0, stream, a);
  if (dtype == FMOE_F32) return quantize<kFormat, float>(a, batch, stream);
  if (dtype == FMOE_BF16) return quantize<kFormat, __nv_bfloat16>(a, batch, stream);
  return quantize<kFormat, __half>(a, batch, stream);
}

template <int kFormat>
cudaError_t dequantize(const Fp4QuantArgs& a, int dtype, int batch, cudaStream_t stream) {
  const dim3 grid = grid_of(a, batch);
  if (dtype == FMOE_F32)
    fp4_dequantize_kernel<kFormat, float><<<grid, kThreads, 0, stream>>>(a);
  else if (dtype == FMOE_BF16)
    fp4_dequantize_kernel<kFormat, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(a);
  else
    fp4_dequantize_kernel<kFormat, __half><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
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
  if (!x) return bad("x must not be NULL");
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
