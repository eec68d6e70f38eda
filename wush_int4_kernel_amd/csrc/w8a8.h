// w8a8.h -- what the W8A8 sources share: w8a8.hip (quantization, streaming
// product, the choice between the kernels) and gemm_w8a8.hip (tiles).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wush {

// Output tiles of tile_rows x tile_cols (256x256, 256x128, 128x128, 64x128,
// 64x64, 32x128, 32x64),
// K % 64 == 0, in `splits` slices of K; with more than one, `part` holds
// splits * M * N int32.
int launch_gemm_w8a8(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, uint16_t* y, int dtype, int M,
                     int N, int K, int tile_rows, int tile_cols, int splits, int* part, hipStream_t stream);

}  // namespace wush
