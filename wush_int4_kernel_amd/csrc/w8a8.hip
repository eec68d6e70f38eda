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
constexpr int kQuantThreads = 256;

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

__device__ __forceinline__ uint32_t pack4(const float (&v)[8], int o, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float r = __builtin_amdgcn_fmed3f(__builtin_rintf(v[o + i] * inv), -127.0f, 127.0f);
        w |= ((uint32_t)(int)r & 0xffu) << (8 * i);
    }
    return w;
}

// One workgroup per row.  Largest magnitudes are compared as bits (sign
// cleared): above those of infinity for a NaN, so one maximum finds both the
// scale and a non-finite value.
template <int DT>
__global__ __launch_bounds__(kQuantThreads) void quant_int8_token_kernel(const uint16_t* __restrict__ x,
                                                                         int8_t* __restrict__ q,
                                                                         float* __restrict__ s, int K,
                                                                         int64_t stride) {
    const int64_t row = blockIdx.x;
    const uint4* px = reinterpret_cast<const uint4*>(x + row * stride);
    uint2* pq = reinterpret_cast<uint2*>(q + row * K);
    uint32_t mx = 0;
    for (int i = threadIdx.x; i < K / 8; i += kQuantThreads) {
        const uint4 w = px[i];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = max(mx, max(u[j] & 0x7fffu, (u[j] >> 16) & 0x7fffu));
    }
    __shared__ uint32_t part[kQuantThreads / 64];
#pragma unroll
    for (int d = 32; d; d >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 64; ++i) mx = max(mx, part[i]);
    const bool bad = mx >= (DT == WUSH_DTYPE_BF16 ? 0x7f80u : 0x7c00u);
    const float amax = DT == WUSH_DTYPE_BF16 ? bf16_to_f32(mx) : f16_to_f32(mx);
    const float sc = bad ? __builtin_nanf("") : fmaxf(amax / 127.0f, kScaleFloor);
    if (threadIdx.x == 0) s[row] = sc;
    const float inv = 1.0f / sc;
    for (int i = threadIdx.x; i < K / 8; i += kQuantThreads) {
        float v[8];
        unpack8<DT>(px[i], v);
        pq[i] = bad ? make_uint2(0, 0) : make_uint2(pack4(v, 0, inv), pack4(v, 4, inv));
    }
}

// y rows as fp16 or bf16, each rounded once from fp32
__device__ __forceinline__ uint16_t out_bits(float f, int dt) {
    return dt == WUSH_DTYPE_F16 ? f32_to_f16_bits(f) : (uint16_t)(f != f ? 0x7fc0u : f32_to_bf16_rne(f));
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
    WUSH_REQUIRE(rows == 1 || (row_stride >= K && row_stride % 8 == 0));
    const uint16_t* px = static_cast<const uint16_t*>(x);
    if (dtype == WUSH_DTYPE_BF16)
        wush::quant_int8_token_kernel<WUSH_DTYPE_BF16><<<(unsigned)rows, wush::kQuantThreads, 0, stream>>>(px, q, s, (int)K, row_stride);
    else
        wush::quant_int8_token_kernel<WUSH_DTYPE_F16><<<(unsigned)rows, wush::kQuantThreads, 0, stream>>>(px, q, s, (int)K, row_stride);
    return (int)hipGetLastError();
}

size_t wush_gemm_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) { return 0; }

size_t wush_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return (size_t)M * K + (((size_t)M * 4 + 15) & ~(size_t)15) + wush_gemm_w8a8_workspace_bytes(M, N, K);
}

int wush_linear_w8a8(const void* x, int64_t row_stride, const int8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                     int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K && M <= 0x7fffffffLL);
    if (M == 0 || N == 0) return (int)hipSuccess;
    const size_t need = wush_linear_w8a8_workspace_bytes(M, N, K), scales = ((size_t)M * 4 + 15) & ~(size_t)15;
    WUSH_REQUIRE(x && wq && ws && y && workspace && ((uintptr_t)workspace & 15u) == 0 && workspace_bytes >= need);
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + (size_t)M * K);
    const int st = wush_quant_int8_token(x, dtype, q, s, M, K, row_stride, stream);
    if (st) return st;
    return wush_gemm_w8a8(q, s, wq, ws, y, dtype, M, N, K, reinterpret_cast<uint8_t*>(s) + scales,
                          workspace_bytes - (size_t)M * K - scales, stream);
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
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)((M + 15) / 16));
    WUSH_REQUIRE(grid.y <= 65535u);
    wush::w8a8_stream_kernel<2, 8><<<grid, 512, 0, stream>>>(xq, xs, wq, ws, static_cast<uint16_t*>(y), dtype, (int)M, (int)N, (int)K);
    return (int)hipGetLastError();
}

}  // extern "C"
