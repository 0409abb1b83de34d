// fp4_kernels.cuh -- argument blocks and launch entry points of the 4-bit kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "fmoe.h"
#include "fp4.cuh"

namespace fmoe {

struct Fp4QuantArgs {
  const void* x;           // quantise: [batch][rows] of `cols` values
  int64_t row_stride, batch_stride;
  void* out;               // dequantise: [batch, rows, cols]
  int64_t rows;
  int cols;
  const float* global;     // nvfp4 global scale(s), or null: 1
  int global_step;         // distance between the matrices' global scales
  uint8_t* codes;          // [batch, rows, cols / 2]
  uint8_t* scales;         // tiles, fp4.cuh
  const int* row_index;    // or null: row m is taken from x's row row_index[m]; below 0: none
  const int* tiles_dev;    // or null: row tiles from *tiles_dev on are not touched
  bool swiglu;             // x is fp32 [rows, 2 cols], the value x[c] * silu(x[cols + c]) of the
                           // same row; row_index only tells which rows there are
};

// Argument checks of one matrix: sizes and format; pointers.
int fp4_check(const fmoe_fp4_matrix* q, const char* name);
int fp4_check_pointers(const fmoe_fp4_matrix* q, const char* name);

// A product out[m][n] = sum_k a[m][k] b[n][k]. Dense (experts == 0): M rows of a, one b.
// Grouped: row tile r of a (128 rows) belongs to the expert e with tile_first[e] <= r <
// tile_first[e + 1] and is multiplied by b's matrix e; an expert's count[e] rows fill its tiles
// from the front, the rows behind them are not written.
struct Fp4Gemm {
  int format;
  const void* a;          // codes [rows of a, K / 2]
  const void* sa;
  int64_t M;              // rows of a; grouped: its capacity, a multiple of 128
  const void* b;          // codes [experts, N, K / 2]
  const void* sb;
  int N, K;
  const float* ga;        // global scales or null; one per expert for b
  const float* gb;
  void* out;              // [M, N]
  int dtype;
  int experts;
  const int* tile_first;  // [experts + 1] on the device
  const int* count;       // [experts] on the device
  const float* row_w;     // or null: factor of each row of out
  bool early;             // b, tile_first and count were complete before the kernel in front of
                          // this one on the stream passed its dependency wait
  // Or, instead of out: b's rows are N / 2 gate and N / 2 up rows (N / 2 a multiple of 128), and
  // gate * silu(up) goes to a 4-bit matrix [M, N / 2] with the global scale gc (null: 1).
  void* codes;
  void* scales;
  const float* gc;
};
int launch_fp4_gemm(const Fp4Gemm& g, cudaStream_t stream);

cudaError_t launch_fp4_quantize(const Fp4QuantArgs& a, int format, int dtype, int batch,
                                cudaStream_t stream);

}  // namespace fmoe
