// w8a8.hip -- linear layers in 8-bit integers: activations scaled per token,
// weights per output channel.
//
//   s_m  = max(amax_k |x_mk| / 127, 2^-126)
//   q_mk = clamp(rint(x_mk * (1 / s_m)), -127, 127)
//   y_mn = ((sum_k q_mk w_nk) * s_m) * ws_n       (exact int32 sum, fp32 scaling)
//
// A row of x with a non-finite value gets s = NaN and zero codes, so its
// outputs are NaN.  Every step is one IEEE operation, so codes and scales are
// the same bits in any implementation of these formulas; the integer sum does
// not depend on its order, so the product is the same bits for every split of K.
#include "w8a8.h"
#include "wush_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr float kScaleFloor = 0x1p-126f;
constexpr int kQuantThreads = 1024;

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == WUSH_DTYPE_BF16) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            v[2 * i] = f16_to_f32(u[i] & 0xffffu);
            v[2 * i + 1] = f16_to_f32(u[i] >> 16);
        }
    }
}

// Codes of eight values, and their largest magnitude.  Magnitudes are compared as
// bits (sign cleared): a NaN's are above those of infinity, so that one
// maximum finds both the scale and a non-finite value.
template <int DT>
__device__ __forceinline__ uint2 codes_of(const uint4& w, float inv) {
    float v[8];
    unpack8<DT>(w, v);
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        o[i >> 2] |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(v[i] * inv), -127.0f, 127.0f) & 0xffu) << (8 * (i & 3));
    return make_uint2(o[0], o[1]);
}
__device__ __forceinline__ uint32_t largest8(const uint4& w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = max(mx, max(u[j] & 0x7fffu, (u[j] >> 16) & 0x7fffu));
    return mx;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}
template <int DT>
__device__ __forceinline__ float token_scale(uint32_t largest) {
    if (largest >= (DT == WUSH_DTYPE_BF16 ? 0x7f80u : 0x7c00u)) return __builtin_nanf("");
    return fmaxf((DT == WUSH_DTYPE_BF16 ? bf16_to_f32(largest) : f16_to_f32(largest)) / 127.0f, kScaleFloor);
}

// One workgroup per row, of as many threads as it has groups of 8 values, up to
// kQuantThreads; a thread keeps its NU groups in registers between the two passes (NU 0: rows
// too long for that, read twice).  Latency-bound for few rows: 203 x 8192 WUSH_Q1 us, with 256
// threads that read the row twice 5.0; 4096 x 8192 WUSH_Q2 us.
template <int DT, int NU>
__global__ __launch_bounds__(kQuantThreads) void quant_int8_token_kernel(const uint16_t* __restrict__ x,
                                                                         int8_t* __restrict__ q,
                                                                         float* __restrict__ s, int K,
                                                                         int64_t stride) {
    const int64_t row = blockIdx.x;
    const int threads = blockDim.x, units = K / 8;
    const uint4* px = reinterpret_cast<const uint4*>(x + row * stride);
    uint2* pq = reinterpret_cast<uint2*>(q + row * K);
    uint4 v[NU ? NU : 1];
    uint32_t mx = 0;
    if constexpr (NU > 0) {
#pragma unroll
        for (int u = 0; u < NU; ++u) v[u] = px[min((int)threadIdx.x + u * threads, units - 1)];
#pragma unroll
        for (int u = 0; u < NU; ++u) mx = max(mx, largest8(v[u]));
    } else {
        for (int i = threadIdx.x; i < units; i += threads) mx = max(mx, largest8(px[i]));
    }
    __shared__ uint32_t part[kQuantThreads / 64];
    mx = wave_max(mx);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < threads / 64; ++i) mx = max(mx, part[i]);
    const float sc = token_scale<DT>(mx);
    if (threadIdx.x == 0) s[row] = sc;
    const bool bad = sc != sc;
    const float inv = 1.0f / sc;
    if constexpr (NU > 0) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int i = threadIdx.x + u * threads;
            if (i < units) pq[i] = bad ? make_uint2(0, 0) : codes_of<DT>(v[u], inv);
        }
    } else {
        for (int i = threadIdx.x; i < units; i += threads) pq[i] = bad ? make_uint2(0, 0) : codes_of<DT>(px[i], inv);
    }
}

// y rows as fp16 or bf16, each rounded once from fp32
__device__ __forceinline__ uint16_t out_bits(float f, int dt) {
    return dt == WUSH_DTYPE_F16 ? f32_to_f16_bits(f) : (uint16_t)(f != f ? 0x7fc0u : f32_to_bf16_rne(f));
}

// One or two rows of activations: the weight stream.  A wavefront takes whole
// weight rows, 1 KiB of contiguous codes an instruction, four instructions ahead, and
// multiplies on v_dot4_i32_i8 with the activation codes, which every workgroup holds in
// LDS.  SRC: codes and scales given, or (a whole linear layer) made by every
// workgroup for itself, while its first weights are on their way: that is
// cheaper than a launch.
enum { kCodes = -1 };                             // else the activations' dtype
constexpr int kGemvWaves = 4, kGemvAhead = 4;

template <int MM, int SRC>
__global__ __launch_bounds__(64 * kGemvWaves) void w8a8_gemv_kernel(const void* __restrict__ xp, int64_t stride,
                                                                    const float* __restrict__ xs,
                                                                    const int8_t* __restrict__ wq,
                                                                    const float* __restrict__ ws,
                                                                    uint16_t* __restrict__ y, int dt, int N, int K) {
    extern __shared__ __align__(16) uint8_t codes[];          // MM rows of Kp bytes, zero past K
    __shared__ uint32_t part[MM][kGemvWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = (K + 1023) >> 10, Kp = chunks << 10;
    const int total = (int)gridDim.x * kGemvWaves;
    const int groups = (chunks + kGemvAhead - 1) / kGemvAhead;
    int row = (int)blockIdx.x * kGemvWaves + wave;

    // group g of row n; a lane past the row's end reads its last 16 bytes,
    // which meet zero activations
    v4i w[kGemvAhead];
    auto fetch = [&](int n, int g) {
        const int8_t* p = wq + (size_t)min(n, N - 1) * K;
#pragma unroll
        for (int u = 0; u < kGemvAhead; ++u)
            w[u] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p + min((g * kGemvAhead + u) * 1024 + 16 * lane, K - 16)));
    };
    fetch(row, 0);

    float sx[MM];
#pragma unroll
    for (int m = 0; m < MM; ++m) {
        uint2* q = reinterpret_cast<uint2*>(codes + m * Kp);
        if constexpr (SRC == kCodes) {
            const uint2* x = reinterpret_cast<const uint2*>(static_cast<const int8_t*>(xp) + m * stride);
            for (int i = tid; i < Kp / 8; i += 64 * kGemvWaves) q[i] = i < K / 8 ? x[i] : make_uint2(0, 0);
            sx[m] = xs[m];
        } else {
            const uint4* x = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(xp) + m * stride);
            uint32_t mx = 0;
            for (int i = tid; i < K / 8; i += 64 * kGemvWaves) mx = max(mx, largest8(x[i]));
            mx = wave_max(mx);
            if (lane == 0) part[m][wave] = mx;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kGemvWaves; ++i) mx = max(mx, part[m][i]);
            sx[m] = token_scale<SRC>(mx);
            const bool bad = sx[m] != sx[m];
            const float inv = 1.0f / sx[m];
            for (int i = tid; i < Kp / 8; i += 64 * kGemvWaves) q[i] = i < K / 8 && !bad ? codes_of<SRC>(x[i], inv) : make_uint2(0, 0);
        }
    }
    __syncthreads();

    for (; row < N; row += total) {
        int acc[MM] = {};
        for (int g = 0; g < groups; ++g) {
            v4i now[kGemvAhead];
#pragma unroll
            for (int u = 0; u < kGemvAhead; ++u) now[u] = w[u];
            if (g + 1 < groups) fetch(row, g + 1);
            else if (row + total < N) fetch(row + total, 0);
#pragma unroll
            for (int u = 0; u < kGemvAhead; ++u) {
                const int c = g * kGemvAhead + u;
                if (c >= chunks) break;
#pragma unroll
                for (int m = 0; m < MM; ++m) {
                    const v4i x = *reinterpret_cast<const v4i*>(codes + m * Kp + c * 1024 + 16 * lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m] = __builtin_amdgcn_sdot4(now[u][e], x[e], acc[m], false);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            int v = acc[m];
#pragma unroll
            for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
            if (lane == 0) y[(size_t)m * N + row] = out_bits((float)v * sx[m] * ws[row], dt);
        }
    }
}

// Streaming product: 16 rows of activations (grid.y) against 16 CB weight rows
// (grid.x), K split over the workgroup's KW wavefronts, whose int32 partial
// sums meet in LDS.  v_mfma_i32_16x16x64_i8 with the weights as row operand: a
// lane loads 16 bytes of its row, straight from HBM into the operand register.
// Any K % 16 == 0: past the end of a row the weights count as zero.
template <int CB, int KW>
__global__ __launch_bounds__(64 * KW) void w8a8_stream_kernel(const int8_t* __restrict__ xq,
                                                              const float* __restrict__ xs,
                                                              const int8_t* __restrict__ wq,
                                                              const float* __restrict__ ws,
                                                              uint16_t* __restrict__ y, int dt, int M, int N, int K) {
    constexpr int U = 8;                          // steps of 64 codes in flight
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16 * CB, m0 = blockIdx.y * 16;
    const int steps = (K + 63) >> 6;
    const int s0 = (int)((long long)steps * wave / KW), s1 = (int)((long long)steps * (wave + 1) / KW);
    const int8_t* wrow[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) wrow[c] = wq + (size_t)min(n0 + 16 * c + l16, N - 1) * K + 16 * kq;
    const int8_t* xrow = xq + (size_t)min(m0 + l16, M - 1) * K + 16 * kq;
    const v4i zero = {0, 0, 0, 0};
    v4i acc[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[c] = zero;
    int s = s0;
    for (; s + U <= s1 && (s + U) * 64 <= K; s += U) {
        v4i w[U][CB], x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int c = 0; c < CB; ++c) w[u][c] = *reinterpret_cast<const v4i*>(wrow[c] + (s + u) * 64);
            x[u] = *reinterpret_cast<const v4i*>(xrow + (s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CB; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][c], x[u], acc[c], 0, 0, 0);
    }
    for (; s < s1; ++s) {
        const bool in = s * 64 + 16 * kq < K;
        const v4i x = in ? *reinterpret_cast<const v4i*>(xrow + s * 64) : zero;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            const v4i w = in ? *reinterpret_cast<const v4i*>(wrow[c] + s * 64) : zero;
            acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc[c], 0, 0, 0);
        }
    }
    // lane (l16, kq) holds weight rows 4 kq + r of activation row l16
    __shared__ int part[KW][CB][16][17];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][c][l16][4 * kq + r] = acc[c][r];
    __syncthreads();
    for (int o = threadIdx.x; o < 256 * CB; o += 64 * KW) {
        const int m = o / (16 * CB), c = o / 16 % CB, n = o % 16;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += part[w][c][m][n];
        const int col = n0 + 16 * c + n;
        if (m0 + m < M && col < N) y[(size_t)(m0 + m) * N + col] = out_bits((float)sum * xs[m0 + m] * ws[col], dt);
    }
}

// ---------------------------------------------------------------- the choice
// One or two rows whose codes fit 64 KiB of LDS take the GEMV.
constexpr int kGemvRows = 2, kGemvLds = 64 * 1024;
bool gemv_shape(int64_t M, int64_t K) { return M <= kGemvRows && M * ((K + 1023) / 1024 * 1024) <= kGemvLds; }

struct Plan {
    int rows, cols, splits;                       // rows 0: the streaming kernel
};

// K % 64 == 0 takes tiles: those, and the split of K, with the least estimated
// time, in microseconds.  A workgroup's stage of 128 codes takes `stage` on a full
// chip (fitted to 4096 x 57344 x 8192 and, for the small tiles, 16 and 64 x 57344 x
// 8192), 0.7 of it on an empty one; the whole no less than the weights' way from HBM.  A
// split costs a launch and its partial sums both ways.
Plan plan_of(int64_t M, int64_t N, int64_t K, size_t room) {
    Plan best = {0, 0, 1};
    if (K % 64 != 0) return best;
    static const struct { int rows, cols; double stage; } kTiles[] = {
        {256, 256, 1.60}, {256, 128, 0.92}, {128, 128, 0.58}, {64, 128, 0.37}, {64, 64, 0.26}, {32, 128, 0.32}, {32, 64, 0.20}};
    const int64_t stages = (K + 127) / 128;
    double least = 1e30;
    for (const auto& t : kTiles) {
        if (t.rows > 32 && t.rows >= 2 * M) continue;
        const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols);
        for (int s = 1; s <= 8 && (s == 1 || stages / s >= 4); ++s) {
            if (s > 1 && (size_t)M * N * 4 * s > room) break;
            const double groups = (double)tiles * s, full = groups / 256 < 1 ? groups / 256 : 1;
            const double rounds = groups <= 1024 ? (double)(int64_t)((groups + 255) / 256) : groups / 256;
            const double work = rounds * (double)((stages + s - 1) / s) * t.stage * (0.7 + 0.3 * full);
            const double hbm = (double)N * K / 6.3e6;
            double us = 4.0 + 1.0 * rounds + (work > hbm ? work : hbm);
            if (s > 1) us += 2.5 + (double)M * N * (8.0 * s + 2) / 4.5e6;
            if (us < least) {
                least = us;
                best = {t.rows, t.cols, s};
            }
        }
    }
    return best;
}

template <int DT>
int launch_quant(const void* x, int8_t* q, float* s, int64_t rows, int64_t K, int64_t stride, hipStream_t stream) {
    const uint16_t* p = static_cast<const uint16_t*>(x);
    const int64_t units = K / 8;
    const unsigned threads = units < kQuantThreads ? (unsigned)((units + 63) / 64 * 64) : kQuantThreads;
    const dim3 grid((unsigned)rows);
    if (units <= threads) quant_int8_token_kernel<DT, 1><<<grid, threads, 0, stream>>>(p, q, s, (int)K, stride);
    else if (units <= 2 * threads) quant_int8_token_kernel<DT, 2><<<grid, threads, 0, stream>>>(p, q, s, (int)K, stride);
    else if (units <= 4 * threads) quant_int8_token_kernel<DT, 4><<<grid, threads, 0, stream>>>(p, q, s, (int)K, stride);
    else quant_int8_token_kernel<DT, 0><<<grid, threads, 0, stream>>>(p, q, s, (int)K, stride);
    return (int)hipGetLastError();
}

template <int SRC>
int launch_gemv(const void* x, int64_t stride, const float* xs, const int8_t* wq, const float* ws, void* y, int dtype,
                int64_t M, int64_t N, int64_t K, hipStream_t stream) {
    const int64_t want = (N + kGemvWaves - 1) / kGemvWaves;
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);   // 8 workgroups a CU
    const size_t lds = (size_t)M * ((K + 1023) / 1024 * 1024);
    uint16_t* o = static_cast<uint16_t*>(y);
    if (M == 1) w8a8_gemv_kernel<1, SRC><<<grid, 64 * kGemvWaves, lds, stream>>>(x, stride, xs, wq, ws, o, dtype, (int)N, (int)K);
    else w8a8_gemv_kernel<2, SRC><<<grid, 64 * kGemvWaves, lds, stream>>>(x, stride, xs, wq, ws, o, dtype, (int)N, (int)K);
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace wush

extern "C" {

int wush_quant_int8_token(const void* x, int dtype, int8_t* q, float* s, int64_t rows, int64_t K, int64_t row_stride,
                          hipStream_t stream) {
    WUSH_REQUIRE(rows >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (rows == 0) return (int)hipSuccess;
    WUSH_REQUIRE(x && q && s && rows <= 0x7fffffffLL);
    WUSH_REQUIRE(((uintptr_t)x & 15u) == 0 && ((uintptr_t)q & 15u) == 0 && ((uintptr_t)s & 3u) == 0);
    WUSH_REQUIRE(rows == 1 || (row_stride >= 0 && row_stride % 8 == 0));
    return dtype == WUSH_DTYPE_BF16 ? wush::launch_quant<WUSH_DTYPE_BF16>(x, q, s, rows, K, row_stride, stream)
                                    : wush::launch_quant<WUSH_DTYPE_F16>(x, q, s, rows, K, row_stride, stream);
}

size_t wush_gemm_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0 || wush::gemv_shape(M, K)) return 0;
    const wush::Plan p = wush::plan_of(M, N, K, SIZE_MAX);
    return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
}

int wush_gemm_w8a8(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                   int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(M <= 0x7fffffffLL && N <= 0x7fffffffLL);
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    WUSH_REQUIRE(xq && xs && wq && ws && y);
    WUSH_REQUIRE(((uintptr_t)xq & 15u) == 0 && ((uintptr_t)wq & 15u) == 0 && ((uintptr_t)xs & 3u) == 0 &&
                 ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)y & 1u) == 0);
    if (wush::gemv_shape(M, K)) return wush::launch_gemv<wush::kCodes>(xq, K, xs, wq, ws, y, dtype, M, N, K, stream);
    uint16_t* o = static_cast<uint16_t*>(y);
    const bool usable = workspace && ((uintptr_t)workspace & 15u) == 0;
    const wush::Plan p = wush::plan_of(M, N, K, usable ? workspace_bytes : 0);
    if (p.rows)
        return wush::launch_gemm_w8a8(xq, xs, wq, ws, o, dtype, (int)M, (int)N, (int)K, p.rows, p.cols, p.splits,
                                      static_cast<int*>(workspace), stream);
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)((M + 15) / 16));
    WUSH_REQUIRE(grid.y <= 65535u);
    wush::w8a8_stream_kernel<2, 4><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, o, dtype, (int)M, (int)N, (int)K);
    return (int)hipGetLastError();
}

size_t wush_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || wush::gemv_shape(M, K)) return 0;
    return (size_t)M * K + (((size_t)M * 4 + 15) & ~(size_t)15) + wush_gemm_w8a8_workspace_bytes(M, N, K);
}

int wush_linear_w8a8(const void* x, int64_t row_stride, const int8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                     int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(M <= 0x7fffffffLL && N <= 0x7fffffffLL);
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    const size_t need = wush_linear_w8a8_workspace_bytes(M, N, K), scales = ((size_t)M * 4 + 15) & ~(size_t)15;
    WUSH_REQUIRE(x && wq && ws && y && workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0)));
    WUSH_REQUIRE((((uintptr_t)x | (uintptr_t)wq) & 15u) == 0 && ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)y & 1u) == 0);
    WUSH_REQUIRE(M == 1 || row_stride % 8 == 0);
    if (wush::gemv_shape(M, K))
        return dtype == WUSH_DTYPE_BF16
                   ? wush::launch_gemv<WUSH_DTYPE_BF16>(x, row_stride, nullptr, wq, ws, y, dtype, M, N, K, stream)
                   : wush::launch_gemv<WUSH_DTYPE_F16>(x, row_stride, nullptr, wq, ws, y, dtype, M, N, K, stream);
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + (size_t)M * K);
    const int st = wush_quant_int8_token(x, dtype, q, s, M, K, row_stride, stream);
    if (st) return st;
    return wush_gemm_w8a8(q, s, wq, ws, y, dtype, M, N, K, reinterpret_cast<uint8_t*>(s) + scales,
                          workspace_bytes - (size_t)M * K - scales, stream);
}

}  // extern "C"
