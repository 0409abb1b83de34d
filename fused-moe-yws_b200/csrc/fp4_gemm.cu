// fp4_gemm.cu -- products of 4-bit matrices.
//
// out[m][n] = ga gb sum_k a[m][k] b[n][k], with a and b the codes times their block scales,
// summed in fp32. One CTA per 64 x 64 tile, both operands decoded to fp32 in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "fmoe.h"
#include "fmoe_kernels.cuh"
#include "fp4.cuh"
#include "fp4_kernels.cuh"

namespace fmoe {
namespace {

using namespace fp4;

struct ProductArgs {
  const uint8_t *a, *b, *sa, *sb;
  const float *ga, *gb;
  int64_t M, N;
  int K;
  void* out;
};

constexpr int kT = 64, kK = 32;

template <int kFormat>
__device__ __forceinline__ void stage(float (*s)[kT + 1], const uint8_t* codes,
                                      const uint8_t* scales, int64_t r0, int64_t rows, int k0,
                                      int K) {
  // 64 rows x 32 columns: 256 threads, 8 values each
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
  float v[8] = {};
  if (r0 + r < rows) {
    const int64_t m = r0 + r;
    decode8(*reinterpret_cast<const uint32_t*>(codes + m * (K / 2) + (k0 + c) / 2), v);
    const int block = (k0 + c) / block_of(kFormat);
    const int64_t tile = m / kTileRows * tiles_across(K, kFormat) + block / 4;
    const float f = scale_value<kFormat>(
        scales[tile * kTileBytes + scale_offset((int)(m % kTileRows), block)]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[c + i][r] = v[i];
}

template <int kFormat, typename T>
__global__ void __launch_bounds__(256) fp4_product_kernel(ProductArgs p) {
  __shared__ float s_a[kK][kT + 1], s_b[kK][kT + 1];
  const int64_t m0 = (int64_t)blockIdx.x * kT, n0 = (int64_t)blockIdx.y * kT;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kK) {
    stage<kFormat>(s_a, p.a, p.sa, m0, p.M, k0, p.K);
    stage<kFormat>(s_b, p.b, p.sb, n0, p.N, k0, p.K);
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(s_a[k][tm + 16 * i], s_b[k][tn + 16 * j], acc[i][j]);
    __syncthreads();
  }
  const float g = (p.ga ? *p.ga : 1.0f) * (p.gb ? *p.gb : 1.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m < p.M && n < p.N) static_cast<T*>(p.out)[m * p.N + n] = (T)(acc[i][j] * g);
    }
}

template <int kFormat>
cudaError_t product(const ProductArgs& p, int dtype, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.M + kT - 1) / kT), (unsigned)((p.N + kT - 1) / kT));
  if (dtype == FMOE_F32)
    fp4_product_kernel<kFormat, float><<<grid, 256, 0, stream>>>(p);
  else if (dtype == FMOE_BF16)
    fp4_product_kernel<kFormat, __nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  else
    fp4_product_kernel<kFormat, __half><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

int bad(const std::string& msg) {
  set_last_error(msg);
  return FMOE_ERR_VALUE;
}

}  // namespace
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
  ProductArgs p = {static_cast<const uint8_t*>(a->codes), static_cast<const uint8_t*>(b->codes),
                   static_cast<const uint8_t*>(a->scales), static_cast<const uint8_t*>(b->scales),
                   a->global_scale, b->global_scale, a->rows, b->rows, (int)a->cols, out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->format == FMOE_MXFP4 ? product<FMOE_MXFP4>(p, dtype, s)
                                                : product<FMOE_NVFP4>(p, dtype, s);
  if (e == cudaSuccess) return FMOE_OK;
  set_last_error(std::string("4-bit product: ") + cudaGetErrorString(e));
  return FMOE_ERR_RUNTIME;
}
