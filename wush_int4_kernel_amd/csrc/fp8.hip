// fp8.hip -- linear layers in 8-bit floating point (e4m3: four exponent and three
// fraction bits, largest 448): activations scaled for each token and block of 128 channels,
// weights for each block of 128 x 128.
//
//   A_bm = max(amax_{k in b} |x_mk|, 448 * 2^-126),  xs_bm = A_bm / 448,  q_mk = e4m3(448 x_mk / A_bm)
//   y_mn = sum_b (sum_{k in b} q_mk w_nk) xs_bm ws_{n / 128, b}        (fp32 sums, rounded once)
//
// Scales lie block by block, (K / 128, rows): a tile's rows of one block are then one load.
#include "fp8.h"
#include "fp8_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

template <int DT, int ROWS>
__global__ __launch_bounds__(256) void quant_fp8_block_kernel(const uint16_t* __restrict__ x, uint8_t* __restrict__ q,
                                                              float* __restrict__ s, int64_t rows, int K, int64_t stride) {
    fp8_quant<DT, ROWS>(x, q, s, rows, K, stride, (int)blockIdx.x, (int)blockIdx.y, (int)threadIdx.x);
}

template <int DT>
int launch_quant(const void* x, uint8_t* q, float* s, int64_t rows, int64_t K, int64_t stride, hipStream_t stream) {
    const uint16_t* p = static_cast<const uint16_t*>(x);
    const Fp8QuantGrid g = fp8_quant_grid(rows, K);
    const dim3 grid((unsigned)g.x, (unsigned)g.y);
    if (g.rows == 1) quant_fp8_block_kernel<DT, 1><<<grid, 256, 0, stream>>>(p, q, s, rows, (int)K, stride);
    else quant_fp8_block_kernel<DT, 16><<<grid, 256, 0, stream>>>(p, q, s, rows, (int)K, stride);
    return (int)hipGetLastError();
}

// ---------------------------------------------------------------- the choice
struct Plan {
    int kernel, rows, cols, splits;
};

// Up to four rows take dot products where they fit (fp8_gemv_shape), all else the tile and the split of K with the least
// estimated time, in microseconds: rounds of workgroups with the time of their stages (3/4 of it on an empty chip), or the
// weights' way from HBM (slower where several row tiles read them), whichever is longer, a part of the shorter, and for a
// split its launch and partial sums.  The constants are fitted to 94 shapes from 5 x 8192 x 28672 to 4000 x 4096 x 4096,
// weights from HBM: 0.8% slower than the fastest of all tiles and splits on average, 12% at worst.
Plan plan_of(int64_t M, int64_t N, int64_t K, size_t room) {
    if (fp8_gemv_shape(M, K)) return {WUSH_FP8_DOT, (int)M, 1, 1};
    Plan best = {WUSH_FP8_TILES, 32, 64, 1};
    const int64_t stages = (K + 127) / 128;
    double least = 1e30;
    for (const auto& t : kFp8Tiles) {
        if ((t.rows > 64 && t.rows >= 2 * M) || (t.runs && N % 8 != 0)) continue;
        const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols);
        for (int s = 1; s <= 8 && (s == 1 || (stages / s >= 4 && t.cols < 256)); ++s) {
            if (s > 1 && (size_t)M * N * 4 * s > room) break;
            const double groups = (double)tiles * s, full = groups / 256 < 1 ? groups / 256 : 1;
            const double rounds = groups <= 1024 ? (double)(int64_t)((groups + 255) / 256) : groups / 256;
            const double work = rounds * (double)((stages + s - 1) / s) * t.stage * (0.75 + 0.25 * full);
            const double hbm = (double)N * K / (M <= t.rows ? 6.3e6 : 4.4e6);
            double us = 4.6 + rounds + (work > hbm ? work + 0.08 * hbm : hbm + 0.08 * work);
            if (s > 1) us += 2.1 + (double)M * N * (8.0 * s + 2) / 4.4e6;
            if (us < least) {
                least = us;
                best = {WUSH_FP8_TILES, t.rows, t.cols, s};
            }
        }
    }
    return best;
}

}  // namespace
}  // namespace wush

extern "C" {

static constexpr int64_t kMostRows = 1 << 26;

static bool fp8_sizes(int64_t M, int64_t N, int64_t K) {
    return M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_FP8_MAX_K && M <= kMostRows && N <= kMostRows;
}

int wush_quant_fp8_block(const void* x, int dtype, uint8_t* q, float* s, int64_t rows, int64_t K, int64_t row_stride,
                         hipStream_t stream) {
    WUSH_REQUIRE(fp8_sizes(rows, 0, K));
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (rows == 0) return (int)hipSuccess;
    WUSH_REQUIRE(x && q && s);
    WUSH_REQUIRE(((uintptr_t)x & 15u) == 0 && ((uintptr_t)q & 15u) == 0 && ((uintptr_t)s & 3u) == 0);
    WUSH_REQUIRE(rows == 1 || (row_stride >= 0 && row_stride % 8 == 0));
    if (rows == 1) row_stride = 0;                // the stride of a single row does not enter any address
    return dtype == WUSH_DTYPE_BF16 ? wush::launch_quant<WUSH_DTYPE_BF16>(x, q, s, rows, K, row_stride, stream)
                                    : wush::launch_quant<WUSH_DTYPE_F16>(x, q, s, rows, K, row_stride, stream);
}

size_t wush_gemm_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (!fp8_sizes(M, N, K) || M == 0 || N == 0) return 0;
    const wush::Plan p = wush::plan_of(M, N, K, SIZE_MAX);
    return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
}

int wush_gemm_fp8_plan(int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int32_t plan[4]) {
    WUSH_REQUIRE(plan && M > 0 && N > 0 && fp8_sizes(M, N, K));
    const wush::Plan p = wush::plan_of(M, N, K, workspace_bytes);
    plan[0] = p.kernel;
    plan[1] = p.rows;
    plan[2] = p.cols;
    plan[3] = p.splits;
    return (int)hipSuccess;
}

int wush_gemm_fp8(const uint8_t* xq, const float* xs, const uint8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                  int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(fp8_sizes(M, N, K));
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    WUSH_REQUIRE(xq && xs && wq && ws && y);
    WUSH_REQUIRE((((uintptr_t)xq | (uintptr_t)wq) & 15u) == 0 && (((uintptr_t)xs | (uintptr_t)ws) & 3u) == 0 && ((uintptr_t)y & (N % 8 == 0 ? 15u : 1u)) == 0);
    const bool usable = workspace && ((uintptr_t)workspace & 15u) == 0;
    const wush::Plan p = wush::plan_of(M, N, K, usable ? workspace_bytes : 0);
    if (p.kernel == WUSH_FP8_DOT)
        return wush::launch_fp8_gemv(xq, 0, xs, wq, ws, static_cast<uint16_t*>(y), dtype, M, N, K, stream);
    wush::Fp8Gemm g = {};
    g.x = xq;
    g.xs = xs;
    g.ldx = M;
    g.w = wq;
    g.ws = ws;
    g.y = y;
    g.out = dtype;
    g.part = static_cast<float*>(workspace);
    g.M = (int)M;
    g.N = (int)N;
    g.K = (int)K;
    g.splits = p.splits;
    g.once = M <= p.rows;
    if (p.rows < 256 && p.cols == 256) return wush::launch_gemm_fp8_runs(g, p.rows, stream);
    return wush::launch_gemm_fp8(g, p.rows, p.cols, stream);
}

static size_t fp8_scale_bytes(int64_t M, int64_t K) { return ((size_t)M * ((K + 127) / 128) * 4 + 15) & ~(size_t)15; }

size_t wush_linear_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (!fp8_sizes(M, N, K) || M == 0 || N == 0 || wush::fp8_gemv_shape(M, K)) return 0;
    return (size_t)M * K + fp8_scale_bytes(M, K) + wush_gemm_fp8_workspace_bytes(M, N, K);
}

int wush_linear_fp8(const void* x, int64_t row_stride, const uint8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                    int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(fp8_sizes(M, N, K));
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    const size_t need = wush_linear_fp8_workspace_bytes(M, N, K);
    WUSH_REQUIRE(x && wq && ws && y && workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0)));
    WUSH_REQUIRE((((uintptr_t)x | (uintptr_t)wq) & 15u) == 0 && ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)y & (N % 8 == 0 ? 15u : 1u)) == 0);
    WUSH_REQUIRE(M == 1 || (row_stride >= 0 && row_stride % 8 == 0));
    if (M == 1) row_stride = 0;
    if (wush::fp8_gemv_shape(M, K))
        return wush::launch_fp8_gemv(x, row_stride, nullptr, wq, ws, static_cast<uint16_t*>(y), dtype, M, N, K, stream);
    uint8_t* q = static_cast<uint8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + (size_t)M * K);
    const int st = wush_quant_fp8_block(x, dtype, q, s, M, K, row_stride, stream);
    if (st) return st;
    const size_t held = (size_t)M * K + fp8_scale_bytes(M, K);
    return wush_gemm_fp8(q, s, wq, ws, y, dtype, M, N, K, q + held, workspace_bytes - held, stream);
}

}  // extern "C"
