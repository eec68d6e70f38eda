// fp8.h -- what the e4m3 sources share: fp8.hip (quantization, the choice between
// the kernels), gemm_fp8.hip (tiles) and moe.hip (experts).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wush {

constexpr int kFp8Block = 128;                   // channels (and weight rows) that share a scale

constexpr int kOutF32 = 2;                       // beside WUSH_DTYPE_BF16 and WUSH_DTYPE_F16

// y = x w^T of one matrix, or of one for each expert.
struct Fp8Gemm {
    const uint8_t* x;                            // codes (rows, K)
    const float* xs;                             // their scales (K / 128, ldx): block by block
    int64_t ldx;
    const uint8_t* w;                            // codes (N, K), of each expert
    const float* ws;                             // their scales (N / 128, K / 128), of each expert
    void* y;                                     // (M, N); experts: one row for each sorted row
    int out;                                     // type of y
    float* part;                                 // with splits > 1: splits * M * N partial sums
    int M, N, K, splits;
    // experts: tiles of rows {expert, first row, end of the expert's rows}, their number, and
    // the row of x that each sorted row stands for (null: itself)
    const int4* tiles;
    const int* ntiles;
    const int* row_of;
    int most_tiles;
};

struct Fp8Tile {
    int rows, cols, depth;
    double stage;                                // us that a K block takes a workgroup on a full chip
};
constexpr Fp8Tile kFp8Tiles[] = {{256, 256, 2, 1.6}, {128, 128, 4, 0.6}, {64, 128, 3, 0.43}, {32, 128, 3, 0.39}, {32, 64, 4, 0.2}};

// Tiles of tile_rows x tile_cols, one of kFp8Tiles; K % 16 == 0.
int launch_gemm_fp8(const Fp8Gemm& g, int tile_rows, int tile_cols, hipStream_t stream);

}  // namespace wush
