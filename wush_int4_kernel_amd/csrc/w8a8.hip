// w8a8.hip -- linear layers in 8-bit integers: activations scaled per token,
// weights per output channel.
//
//   s_m  = max(amax_k |x_mk| / 127, 2^-126)
//   q_mk = clamp(rint(x_mk * (1 / s_m)), -127, 127)
//   y_mn = ((sum_k q_mk w_nk) * s_m) * ws_n       (exact int32 sum, fp32 scaling)
//
// A row of x with a non-finite value gets s = NaN and zero codes, so its
// outputs are NaN.  Every step is one IEEE operation, so codes and scales are
// the same bits wherever these are (a product with 1 / 127 in place of the division, which
// tensor libraries make of one by a constant on the GPU, is an ulp off now and then, and codes
// at ties with it); the integer sum does
// not depend on its order, so the product is the same bits for every split of K.
#include "w8a8.h"
#include "wush_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr float kScaleFloor = 0x1p-126f;
constexpr int kQuantThreads = 1024;
constexpr int64_t kQuantRows = 1 << 21;           // of a launch, at most

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
// too long for that, read twice).  Latency-bound for few rows: 203 x 8192 4.2 us, with 256
// threads that read the row twice 5.0; 4096 x 8192 (100 MB) 25 us.
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

// A whole layer for one or two short rows, M K <= kGemvCodes: a wavefront takes whole
// weight rows, 1 KiB of contiguous codes an instruction, the next row's loads ahead of this
// one's v_dot4_i32_i8.  Every workgroup makes the activations' codes for itself, in LDS, while
// its first weights are on their way: cheaper than a launch (1 x 1024 x 2048 4.2 us, not 5.9, 2 x 1024 x
// 2048 5.1, not 6.2; 1 x 24576 x 4096 18.4, not 19.4; 1 x 4096 x 4096, 7.6 with weights from HBM, the same).  For
// longer rows it is not: 1 x 8192 x 8192 17.4 us against 15.3, 2 x 8192 x 28672 92 against 44.
constexpr int kGemvWaves = 4, kGemvRows = 2, kGemvCodes = 4096;

template <int MM, int DT>
__global__ __launch_bounds__(64 * kGemvWaves) void w8a8_gemv_kernel(const uint16_t* __restrict__ xp, int64_t stride,
                                                                    const int8_t* __restrict__ wq,
                                                                    const float* __restrict__ ws,
                                                                    uint16_t* __restrict__ y, int N, int K) {
    constexpr int kChunks = kGemvCodes / 1024 / MM;           // of a row, at most
    __shared__ __align__(16) uint8_t codes[MM][1024 * kChunks];   // zero past K
    __shared__ uint32_t part[MM][kGemvWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = (K + 1023) >> 10, Kp = chunks << 10;
    const int total = (int)gridDim.x * kGemvWaves;
    int row = (int)blockIdx.x * kGemvWaves + wave;

    // a lane past the row's end reads its last 16 bytes, which meet zero activations
    v4i w[kChunks];
    auto fetch = [&](int n) {
        const int8_t* p = wq + (size_t)min(n, N - 1) * K;
#pragma unroll
        for (int u = 0; u < kChunks; ++u)
            if (u < chunks) w[u] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p + min(u * 1024 + 16 * lane, K - 16)));
    };
    fetch(row);

    float sx[MM];
#pragma unroll
    for (int m = 0; m < MM; ++m) {
        uint2* q = reinterpret_cast<uint2*>(codes[m]);
        const uint4* x = reinterpret_cast<const uint4*>(xp + m * stride);
        uint32_t mx = 0;
        for (int i = tid; i < K / 8; i += 64 * kGemvWaves) mx = max(mx, largest8(x[i]));
        mx = wave_max(mx);
        if (lane == 0) part[m][wave] = mx;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kGemvWaves; ++i) mx = max(mx, part[m][i]);
        sx[m] = token_scale<DT>(mx);
        const bool bad = sx[m] != sx[m];
        const float inv = 1.0f / sx[m];
        for (int i = tid; i < Kp / 8; i += 64 * kGemvWaves) q[i] = i < K / 8 && !bad ? codes_of<DT>(x[i], inv) : make_uint2(0, 0);
    }
    __syncthreads();

    for (; row < N; row += total) {
        v4i now[kChunks];
#pragma unroll
        for (int u = 0; u < kChunks; ++u) now[u] = w[u];
        if (row + total < N) fetch(row + total);
        int acc[MM] = {};
#pragma unroll
        for (int u = 0; u < kChunks; ++u) {
            if (u >= chunks) break;
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                const v4i x = *reinterpret_cast<const v4i*>(codes[m] + u * 1024 + 16 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m] = __builtin_amdgcn_sdot4(now[u][e], x[e], acc[m], false);
            }
        }
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            int v = acc[m];
#pragma unroll
            for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
            if (lane == 0) y[(size_t)m * N + row] = out_bits((float)v * sx[m] * ws[row], DT);
        }
    }
}

// Up to kDotRows rows of codes: a wavefront takes R weight rows, 1 KiB of contiguous
// codes of each at a time, against activation codes that stay in the caches.  Bound by the weights'
// stream: 1 x 57344 x 8192 65 us, 7.2 TB/s.  The tiles of gemm_w8a8.hip, whose
// loads take 128 bytes of a row at a time, need 98 us there, and MFMAs on operands loaded
// straight from HBM, 64 bytes of a row at a time, 79.  For four rows the two come close (24576 x 4096
// 23.9 us against 25.4, 8192 x 28672 48 against 44, 57344 x 8192 83 against 92); for
// eight the tiles are faster (92 against 105).
constexpr int kDotRows = 4;
template <int MM, int R>
__global__ __launch_bounds__(256) void w8a8_dot_kernel(const int8_t* __restrict__ xq, const float* __restrict__ xs,
                                                       const int8_t* __restrict__ wq, const float* __restrict__ ws,
                                                       uint16_t* __restrict__ y, int dt, int N, int K) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = ((int)blockIdx.x * 4 + wave) * R;
    if (n0 >= N) return;
    const int8_t *pw[R], *px[MM];
#pragma unroll
    for (int r = 0; r < R; ++r) pw[r] = wq + (size_t)min(n0 + r, N - 1) * K;
#pragma unroll
    for (int m = 0; m < MM; ++m) px[m] = xq + (size_t)m * K;
    int acc[R][MM] = {};
    auto chunk = [&](int at, bool in) {
        v4i w[R], x[MM];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(pw[r] + at));
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            x[m] = *reinterpret_cast<const v4i*>(px[m] + at);
            if (!in) x[m] = (v4i){0, 0, 0, 0};
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < MM; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][m] = __builtin_amdgcn_sdot4(w[r][e], x[m][e], acc[r][m], false);
    };
    const int whole = K >> 10;
#pragma unroll R > 2 ? 2 : 4
    for (int c = 0; c < whole; ++c) chunk((c << 10) + 16 * lane, true);
    const int at = (whole << 10) + 16 * lane;
    if (whole << 10 < K) chunk(min(at, K - 16), at < K);      // a lane past the row's end: zero activations
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            int v = acc[r][m];
#pragma unroll
            for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
            if (lane == 0 && n0 + r < N) y[(size_t)m * N + n0 + r] = out_bits((float)v * xs[m] * ws[n0 + r], dt);
        }
}

// Streaming product: 16 rows of activations (grid.y) against 16 CB weight rows
// (grid.x), K split over the workgroup's KW wavefronts, whose int32 partial
// sums meet in LDS.  v_mfma_i32_16x16x64_i8 with the weights as row operand: a
// lane loads 16 bytes of its row, straight from HBM into the operand register.
// Any K % 16 == 0: past the end of a row the weights count as zero.  Every 16 rows
// load all weights again: right for few rows only (5 x 8192 x 4112 10.4 us, tiles at K = 4096 12.6; 32
// rows 17.0 and 12.6, 300 rows 102 and 21, 2000 rows 623 and 69).
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
// R: more weight rows a wavefront load the activations less often, but leave fewer
// wavefronts.  us at R = 1, 2, 4: 1 x 24576 x 4096 17.0, 17.9, 21.4, 1 x 57344 x 8192 65, 68, 73; 2 x 4096 x 4096
// 5.9, 6.3, 8.2, 2 x 57344 x 8192 86, 74, 74; 3 x 1024 x 2048 4.2, 5.1, 6.7, 4 x 8192 x 8192 22.0, 18.4, 19.8, 4 x 57344 x 8192
// 125, 98, 83.
int dot_rows(int64_t M, int64_t N, int64_t K) {
    if (M == 1) return 1;
    if (M == 2) return N * K < 1 << 26 ? 1 : 2;
    return N * K < 1 << 24 ? 1 : N * K < 1 << 27 ? 2 : 4;
}

struct Plan {
    int kernel, rows, cols, splits;
};

// M <= kDotRows takes the dot products.
// Else K % 64 == 0 takes tiles: those, and the split of K, with the least estimated
// time, in microseconds.  A workgroup's stage of 128 codes takes `stage` on a full
// chip, 0.6 of it on an empty one, and no less than HBM's latency over the stages in flight;
// the whole takes no less than the weights' way from HBM.  A split costs a launch and its
// partial sums both ways.  The estimates are there to be compared with each other.  The constants are fitted to 60 shapes from 5 x 8192 x 28672 to 300 rows, weights
// from HBM: 1.6% slower than the fastest of all tiles and splits on average, 15% at worst; without the
// latency 5.4% and 50%.  Other K take the streaming kernel, which any K % 16 == 0 suits (tiles need
// whole steps of 64 codes).
Plan plan_of(int64_t M, int64_t N, int64_t K, size_t room) {
    if (M <= kDotRows) return {WUSH_W8A8_DOT, (int)M, 4 * dot_rows(M, N, K), 1};
    Plan best = {WUSH_W8A8_STREAM, 16, 32, 1};
    if (K % 64 != 0) return best;
    static const struct { int rows, cols, depth; double stage; } kTiles[] = {
        {256, 256, 2, 1.60}, {256, 128, 3, 0.92}, {128, 128, 4, 0.58}, {64, 128, 3, 0.43},
                {64, 64, 4, 0.26}, {32, 128, 3, 0.39}, {32, 64, 4, 0.20}};
    const int64_t stages = (K + 127) / 128;
    double least = 1e30;
    for (const auto& t : kTiles) {
        if (t.rows > 32 && t.rows >= 2 * M) continue;
        const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols);
        for (int s = 1; s <= 8 && (s == 1 || stages / s >= 4); ++s) {
            if (s > 1 && (size_t)M * N * 4 * s > room) break;
            const double groups = (double)tiles * s, full = groups / 256 < 1 ? groups / 256 : 1;
            const double rounds = groups <= 1024 ? (double)(int64_t)((groups + 255) / 256) : groups / 256;
            const double busy = t.stage * (0.6 + 0.4 * full), idle = 0.72 / (t.depth - 1);
            const double work = rounds * (double)((stages + s - 1) / s) * (busy > idle ? busy : idle);
            const double hbm = (double)N * K / 7e6;
            double us = 4.0 + 1.0 * rounds + (work > hbm ? work : hbm);
            if (s > 1) us += 3.3 + (double)M * N * (8.0 * s + 2) / 4.5e6;
            if (us < least) {
                least = us;
                best = {WUSH_W8A8_TILES, t.rows, t.cols, s};
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
    // a launch has fewer than 2^32 threads
    for (int64_t r = 0; r < rows; r += kQuantRows) {
        const uint16_t* xr = r ? p + r * stride : p;              // one row's stride may be anything
        int8_t* qr = q + r * K;
        float* sr = s + r;
        const dim3 grid((unsigned)(rows - r < kQuantRows ? rows - r : kQuantRows));
        if (units <= threads) quant_int8_token_kernel<DT, 1><<<grid, threads, 0, stream>>>(xr, qr, sr, (int)K, stride);
        else if (units <= 2 * threads) quant_int8_token_kernel<DT, 2><<<grid, threads, 0, stream>>>(xr, qr, sr, (int)K, stride);
        else if (units <= 4 * threads) quant_int8_token_kernel<DT, 4><<<grid, threads, 0, stream>>>(xr, qr, sr, (int)K, stride);
        else quant_int8_token_kernel<DT, 0><<<grid, threads, 0, stream>>>(xr, qr, sr, (int)K, stride);
        const int st = (int)hipGetLastError();
        if (st) return st;
    }
    return (int)hipSuccess;
}

template <int DT>
int launch_gemv(const void* x, int64_t stride, const int8_t* wq, const float* ws, void* y, int64_t M, int64_t N, int64_t K,
                hipStream_t stream) {
    const int64_t want = (N + kGemvWaves - 1) / kGemvWaves;
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);   // 8 workgroups a CU
    const uint16_t* p = static_cast<const uint16_t*>(x);
    uint16_t* o = static_cast<uint16_t*>(y);
    if (M == 1) w8a8_gemv_kernel<1, DT><<<grid, 64 * kGemvWaves, 0, stream>>>(p, stride, wq, ws, o, (int)N, (int)K);
    else w8a8_gemv_kernel<2, DT><<<grid, 64 * kGemvWaves, 0, stream>>>(p, stride, wq, ws, o, (int)N, (int)K);
    return (int)hipGetLastError();
}

template <int MM>
int launch_dot(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, uint16_t* y, int dtype, int64_t N,
               int64_t K, hipStream_t stream) {
    const int r = dot_rows(MM, N, K);
    const unsigned grid = (unsigned)((N + 4 * r - 1) / (4 * r));
    if (r == 1) w8a8_dot_kernel<MM, 1><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, y, dtype, (int)N, (int)K);
    if constexpr (MM > 1)
        if (r == 2) w8a8_dot_kernel<MM, 2><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, y, dtype, (int)N, (int)K);
    if constexpr (MM > 2)
        if (r == 4) w8a8_dot_kernel<MM, 4><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, y, dtype, (int)N, (int)K);
    return (int)hipGetLastError();
}

bool gemv_shape(int64_t M, int64_t K) { return M <= kGemvRows && M * K <= kGemvCodes; }

}  // namespace
}  // namespace wush

extern "C" {

static constexpr int64_t kMostRows = 0x7fff0000LL;    // rounded up to tiles, still an int

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
    if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0) return 0;
    const wush::Plan p = wush::plan_of(M, N, K, SIZE_MAX);
    return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
}

int wush_gemm_w8a8_plan(int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int32_t plan[4]) {
    WUSH_REQUIRE(plan && M > 0 && N > 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(M <= kMostRows && N <= kMostRows);
    const wush::Plan p = wush::plan_of(M, N, K, workspace_bytes);
    plan[0] = p.kernel;
    plan[1] = p.rows;
    plan[2] = p.cols;
    plan[3] = p.splits;
    return (int)hipSuccess;
}

int wush_gemm_w8a8(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                   int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(M <= kMostRows && N <= kMostRows);
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    WUSH_REQUIRE(xq && xs && wq && ws && y);
    WUSH_REQUIRE(((uintptr_t)xq & 15u) == 0 && ((uintptr_t)wq & 15u) == 0 && ((uintptr_t)xs & 3u) == 0 &&
                 ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)y & 1u) == 0);
    uint16_t* o = static_cast<uint16_t*>(y);
    switch (M) {
        case 1: return wush::launch_dot<1>(xq, xs, wq, ws, o, dtype, N, K, stream);
        case 2: return wush::launch_dot<2>(xq, xs, wq, ws, o, dtype, N, K, stream);
        case 3: return wush::launch_dot<3>(xq, xs, wq, ws, o, dtype, N, K, stream);
        case 4: return wush::launch_dot<4>(xq, xs, wq, ws, o, dtype, N, K, stream);
    }
    const bool usable = workspace && ((uintptr_t)workspace & 15u) == 0;
    const wush::Plan p = wush::plan_of(M, N, K, usable ? workspace_bytes : 0);
    if (p.kernel == WUSH_W8A8_TILES)
        return wush::launch_gemm_w8a8(xq, xs, wq, ws, o, dtype, (int)M, (int)N, (int)K, p.rows, p.cols, p.splits,
                                      static_cast<int*>(workspace), stream);
    // a grid has 65535 rows of workgroups at most
    constexpr int64_t kRows = 16 * 65535;
    for (int64_t m = 0; m < M; m += kRows) {
        const int64_t rows = M - m < kRows ? M - m : kRows;
        const dim3 grid((unsigned)((N + 31) / 32), (unsigned)((rows + 15) / 16));
        wush::w8a8_stream_kernel<2, 4><<<grid, 256, 0, stream>>>(xq + m * K, xs + m, wq, ws, o + m * N, dtype, (int)rows, (int)N, (int)K);
        const int st = (int)hipGetLastError();
        if (st) return st;
    }
    return (int)hipSuccess;
}

size_t wush_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || wush::gemv_shape(M, K)) return 0;
    return (size_t)M * K + (((size_t)M * 4 + 15) & ~(size_t)15) + wush_gemm_w8a8_workspace_bytes(M, N, K);
}

int wush_linear_w8a8(const void* x, int64_t row_stride, const int8_t* wq, const float* ws, void* y, int dtype, int64_t M,
                     int64_t N, int64_t K, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    WUSH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(M <= kMostRows && N <= kMostRows);
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (M == 0 || N == 0) return (int)hipSuccess;
    const size_t need = wush_linear_w8a8_workspace_bytes(M, N, K), scales = ((size_t)M * 4 + 15) & ~(size_t)15;
    WUSH_REQUIRE(x && wq && ws && y && workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0)));
    WUSH_REQUIRE((((uintptr_t)x | (uintptr_t)wq) & 15u) == 0 && ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)y & 1u) == 0);
    WUSH_REQUIRE(M == 1 || (row_stride >= 0 && row_stride % 8 == 0));
    if (wush::gemv_shape(M, K))
        return dtype == WUSH_DTYPE_BF16
                   ? wush::launch_gemv<WUSH_DTYPE_BF16>(x, row_stride, wq, ws, y, M, N, K, stream)
                   : wush::launch_gemv<WUSH_DTYPE_F16>(x, row_stride, wq, ws, y, M, N, K, stream);
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + (size_t)M * K);
    const int st = wush_quant_int8_token(x, dtype, q, s, M, K, row_stride, stream);
    if (st) return st;
    return wush_gemm_w8a8(q, s, wq, ws, y, dtype, M, N, K, reinterpret_cast<uint8_t*>(s) + scales,
                          workspace_bytes - (size_t)M * K - scales, stream);
}

}  // extern "C"
