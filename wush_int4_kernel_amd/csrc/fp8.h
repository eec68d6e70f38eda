// fp8.h -- what the e4m3 sources share: fp8.hip (quantization, the choice between the kernels),
// gemm_fp8.hip and gemm_fp8_runs.hip (tiles), fp8_gemv.hip (few rows) and moe.hip (experts).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wush {

constexpr int kFp8Block = 128;                   // channels (and weight rows) that share a scale

// Type of y beside WUSH_DTYPE_BF16 and WUSH_DTYPE_F16
constexpr int kOutF32 = 2;

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
    // experts' outputs: fp32; act: codes of silu(gate) * up, N / 2 a row, with their scales in hs (N / 256, ldh);
    // shared: fp16, with powers of two in hs (rows, N / 64)
    int act, shared;
    float* hs;
    int64_t ldh;
    int wide;                                    // products in fp16 matrix instructions, which cut none (with act: always)
    int once;                                    // weights are mostly read for one tile of rows only
};

struct Fp8Tile {
    int rows, cols;
    bool runs;                                   // gemm_fp8_runs.hip: N % 8 == 0 only
    double stage;                                // us that a K block takes a workgroup on a full chip
};
constexpr Fp8Tile kFp8Tiles[] = {{256, 256, false, 1.63}, {128, 256, true, 1.02}, {64, 256, true, 0.8}, {128, 128, false, 0.72},
                                 {64, 128, false, 0.57},  {32, 128, false, 0.41}, {32, 64, false, 0.28}};

// Tiles of tile_rows x tile_cols, one of kFp8Tiles; K % 16 == 0.
int launch_gemm_fp8(const Fp8Gemm& g, int tile_rows, int tile_cols, hipStream_t stream);

// The same over experts, fp32 out, tiles of kFp8RowsTile x kFp8RowsTile * 2.
constexpr int kFp8RowsTile = 32;
int launch_gemm_fp8_rows(const Fp8Gemm& g, hipStream_t stream);

// Tiles of tile_rows (64 or 128) x 256 by workgroups that take one after another: one matrix with N % 8 == 0 and
// 16-byte aligned y, or experts with act or shared.
constexpr int kFp8Workgroups = 256;              // one for each of the chip's CUs
int launch_gemm_fp8_runs(const Fp8Gemm& g, int tile_rows, hipStream_t stream);

// Up to four rows (one with K up to 32768, two up to 16384, three and four up to 8192: fp8_gemv_shape) on dot products:
// x as bf16 or fp16 rows of y's type (xs null), or as codes with scales xs (K / 128, M).
bool fp8_gemv_shape(int64_t M, int64_t K);
int launch_fp8_gemv(const void* x, int64_t row_stride, const float* xs, const uint8_t* w, const float* ws, uint16_t* y,
                    int dtype, int64_t M, int64_t N, int64_t K, hipStream_t stream);

// A layer of experts for few tokens; h: T * k * I fp32 of workspace.
struct Fp8Experts {
    const void* x;
    int64_t row_stride;
    const float* weights;
    const int32_t* ids;
    const uint8_t *w_up, *w_down;
    const float *s_up, *s_down;
    float* h;
    void* y;
    int dtype, T, k, E, H, I;
};
constexpr int kFp8GemvPairs = 512;                // of tokens and choices, at most
bool fp8_experts_gemv_shape(int64_t T, int64_t k, int64_t H, int64_t I);
int launch_fp8_experts_gemv(const Fp8Experts& a, hipStream_t stream);

}  // namespace wush
