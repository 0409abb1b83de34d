// fp4_kernels.cuh -- argument blocks and launch entry points of the 4-bit kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "fmoe.h"

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
  const int* rows_dev;     // or null: row tiles from *rows_dev on are not touched
};

// Argument checks of one matrix: sizes and format; pointers.
int fp4_check(const fmoe_fp4_matrix* q, const char* name);
int fp4_check_pointers(const fmoe_fp4_matrix* q, const char* name);

cudaError_t launch_fp4_quantize(const Fp4QuantArgs& a, int format, int dtype, int batch,
                                cudaStream_t stream);

}  // namespace fmoe
