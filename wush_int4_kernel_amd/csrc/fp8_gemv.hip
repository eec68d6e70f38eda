// fp8_gemv.hip -- e4m3 products for one to four rows, and a layer of experts for few tokens: every
// weight is read once, straight from memory into dot products, so that the weights' stream is all there is.
//
// A wavefront takes whole weight rows, 1 KiB of contiguous codes an instruction, 16 a lane.  The
// activations' codes that meet a lane's weights stay, as fp32, in its registers from the first row to the
// last: a workgroup quantizes x itself (a block of 128 is eight lanes), while its first
// weights are on their way.  Weights become fp32 two at a time (v_cvt_pk_f32_fp8) and are multiplied in fp32: no product is
// rounded, and 41 bytes of weights a clock and CU for one row are three times what memory delivers.
// 1 x 4096 x 4096: 5.2 us, 3.2 TB/s, more than half of it launch and latency.  One token's layer, 6 of 64 experts of 2048 x 1408
// (52 MB): 15.3 us in two launches, 3.4 TB/s.
#include "fp8.h"
#include "fp8_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef unsigned int u32v4 __attribute__((ext_vector_type(4)));

// 16 channels of x from channel k on, zeros past K
struct Sixteen {
    uint4 a, b;
};
__device__ __forceinline__ Sixteen load16(const uint16_t* __restrict__ x, int k, int K) {
    if (k >= K) return {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    const uint4* p = reinterpret_cast<const uint4*>(x + k);
    return {p[0], p[1]};
}
// their codes, and the scale of their block, which eight lanes have
template <int DT>
__device__ __forceinline__ uint4 quantized16(const Sixteen& x, float& scale) {
    float t[2][8];
    fp8_unpack8<DT>(x.a, t[0]);
    fp8_unpack8<DT>(x.b, t[1]);
    const float amax = fp8_amax(row8_max(max(fp8_largest8(t[0]), fp8_largest8(t[1]))));
    const Fp8Divisor by = fp8_divisor(amax);
    scale = fp8_scale(amax);
    uint32_t c[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float* s = t[q >> 1] + 4 * (q & 1);
        c[q] = fp8_codes4(s[0], s[1], s[2], s[3], by, amax != amax);
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
}

// The values of 16 codes
__device__ __forceinline__ void values16(const u32v4& codes, float (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float t[4];
        fp8_values4(codes[q], t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
    }
}

// 16 weights against a lane's 16 values
__device__ __forceinline__ float dot16(const u32v4& w, const float (&x)[16]) {
    float p = 0.0f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float v[4];
        fp8_values4(w[q], v);
#pragma unroll
        for (int i = 0; i < 4; ++i) p = __builtin_fmaf(v[i], x[4 * q + i], p);
    }
    return p;
}

__device__ __forceinline__ uint16_t out_bits(float f, int dt) {
    return dt == WUSH_DTYPE_F16 ? f32_to_f16_bits(f) : (uint16_t)(f != f ? 0x7fc0u : f32_to_bf16_rne(f));
}

// M rows of x; K in KS slices of at most 1024 C, one a wavefront, whose sums meet in LDS; R weight rows at a time.
// CODES: x as codes with scales xs (K / 128, M), else as bf16 or fp16 rows.
template <int M, int C, int KS, int R, bool CODES, int DT>
__global__ __launch_bounds__(256) void fp8_gemv_kernel(const void* __restrict__ xp, int64_t stride,
                                                       const float* __restrict__ xs, const uint8_t* __restrict__ w,
                                                       const float* __restrict__ ws, uint16_t* __restrict__ y, int dt, int N,
                                                       int K) {
    constexpr int G = 4 / KS, V = (M == 3 ? 4 : M) * R;          // row groups of a workgroup, sums of a group
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave % KS, group = wave / KS;
    const int KB = (K + 127) >> 7, groups = (N + R - 1) / R;
    int k[C], kb[C];                                             // this lane's channels; past K the row's last, which meet zeros
    bool in[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (slice * C + c) * 1024 + 16 * lane;
        in[c] = at < K;
        k[c] = min(at, K - 16);
        kb[c] = k[c] >> 7;
    }
    u32v4 wn[R][C];
    auto fetch = [&](int g) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c)
                wn[r][c] = __builtin_nontemporal_load(reinterpret_cast<const u32v4*>(w + (size_t)min(g * R + r, N - 1) * K + k[c]));
    };
    int g = (int)blockIdx.x * G + group;
    fetch(min(g, groups - 1));
    float x[M][C][16], xscale[M][C];
    if constexpr (CODES) {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const u32v4 zero = {0, 0, 0, 0};
                const u32v4 q = *reinterpret_cast<const u32v4*>(static_cast<const uint8_t*>(xp) + (size_t)m * K + k[c]);
                values16(in[c] ? q : zero, x[m][c]);
                xscale[m][c] = in[c] ? xs[(size_t)kb[c] * M + m] : 0.0f;
            }
    } else {
        constexpr int kUnits = C * KS * 64;                      // of 16 channels
        __shared__ uint4 codes[M][kUnits];
        __shared__ float scales[M][kUnits / 8];
        for (int u = threadIdx.x; u < M * kUnits; u += 256) {
            const int m = u / kUnits, at = u % kUnits;
            float s;
            codes[m][at] = quantized16<DT>(load16(static_cast<const uint16_t*>(xp) + m * stride, 16 * at, K), s);
            if ((at & 7) == 0) scales[m][at >> 3] = s;
        }
        WUSH_LDS_BARRIER();
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (slice * C + c) * 64 + lane;
                const uint4 q = codes[m][at];
                values16((u32v4){q.x, q.y, q.z, q.w}, x[m][c]);
                xscale[m][c] = scales[m][at >> 3];
            }
    }
    __shared__ float part[2][4][V];
    int turn = 0;
    for (int g0 = (int)blockIdx.x * G; g0 < groups; g0 += (int)gridDim.x * G, turn ^= 1) {
        g = g0 + group;
        const int gc = min(g, groups - 1);
        u32v4 now[R][C];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) now[r][c] = wn[r][c];
        float s[R][C];                                           // scales of the rows' blocks
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) s[r][c] = ws[(size_t)(min(gc * R + r, N - 1) >> 7) * KB + kb[c]];
        if (g0 + (int)gridDim.x * G < groups) fetch(min(g + (int)gridDim.x * G, groups - 1));
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int m = 0; m < M; ++m) acc[m * R + r] = __builtin_fmaf(dot16(now[r][c], x[m][c]), s[r][c] * xscale[m][c], acc[m * R + r]);
        const float sum = wave_reduce_scatter<V>(acc, lane);
        const int v = wave_rs_index<V>(lane);
        const bool mine = (lane & (64 / V - 1)) == 0;
        if constexpr (KS == 1) {
            const int n = g * R + v % R;
            if (mine && v / R < M && n < N) y[(size_t)(v / R) * N + n] = out_bits(sum, dt);
        } else {
            if (mine) part[turn][wave][v] = sum;
            WUSH_LDS_BARRIER();
            if (threadIdx.x < G * V) {
                const int q = threadIdx.x / V, u = threadIdx.x % V, n = (g0 + q) * R + u % R;
                float t = part[turn][q * KS][u];
#pragma unroll
                for (int i = 1; i < KS; ++i) t += part[turn][q * KS + i][u];
                if (u / R < M && n < N) y[(size_t)(u / R) * N + n] = out_bits(t, dt);
            }
        }
    }
}

// ------------------------------------------------------------------- experts
// h = silu(gate) * up of pair blockIdx.y's token and expert, R columns a wavefront
template <int C, int R, int DT>
__global__ __launch_bounds__(256) void fp8_experts_up_kernel(const uint16_t* __restrict__ x, int64_t stride,
                                                             const int32_t* __restrict__ ids, const uint8_t* __restrict__ w,
                                                             const float* __restrict__ ws, float* __restrict__ h, int k, int E,
                                                             int H, int I) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p = blockIdx.y;
    constexpr int U = (C * 64 + 255) / 256;                      // units of 16 channels that a thread quantizes
    Sixteen raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load16(x + (p / k) * stride, 16 * ((int)threadIdx.x + 256 * u), H);
    const int e = ids[p];
    if ((unsigned)e >= (unsigned)E) return;
    const int n0 = ((int)blockIdx.x * 4 + wave) * R;             // I is a multiple of 4 R
    const int KB = (H + 127) >> 7;
    const uint8_t* we = w + ((size_t)e * 2 * I + n0) * H;
    const float* se = ws + ((size_t)e * (2 * I >> 7) + (n0 >> 7)) * KB;
    u32v4 wn[2 * R][C];
    float s[2][C], v[C][16];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int kk = min(c * 1024 + 16 * lane, H - 16);
#pragma unroll
        for (int r = 0; r < 2 * R; ++r)
            wn[r][c] = __builtin_nontemporal_load(reinterpret_cast<const u32v4*>(we + (size_t)(r < R ? r : r - R + I) * H + kk));
        s[0][c] = se[kk >> 7];
        s[1][c] = se[(size_t)(I >> 7) * KB + (kk >> 7)];
    }
    __shared__ uint4 codes[C * 64];
    __shared__ float scales[C * 8];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = threadIdx.x + 256 * i;
        float t;
        const uint4 q = quantized16<DT>(raw[i], t);
        if (u < C * 64) {
            codes[u] = q;
            if ((u & 7) == 0) scales[u >> 3] = t;
        }
    }
    WUSH_LDS_BARRIER();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint4 q = codes[c * 64 + lane];
        values16((u32v4){q.x, q.y, q.z, q.w}, v[c]);
        const float t = scales[c * 8 + (lane >> 3)];
        s[0][c] *= t;
        s[1][c] *= t;
    }
    float acc[2 * R];
#pragma unroll
    for (int r = 0; r < 2 * R; ++r) {
        acc[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[r] = __builtin_fmaf(dot16(wn[r][c], v[c]), s[r >= R][c], acc[r]);
    }
#pragma unroll
    for (int r = 0; r < 2 * R; ++r) acc[r] = wave_sum_dpp(acc[r]);
    if (lane < R) {
        float g = acc[0], u = acc[R];
#pragma unroll
        for (int r = 1; r < R; ++r)
            if (lane == r) {
                g = acc[r];
                u = acc[R + r];
            }
        h[(size_t)p * I + n0 + lane] = fp8_silu(g) * u;
    }
}

// R columns of token blockIdx.y's output: wavefront w takes choices w, w + waves, ...; their sums meet in LDS
template <int C, int R>
__global__ __launch_bounds__(512) void fp8_experts_down_kernel(const float* __restrict__ h, const int32_t* __restrict__ ids,
                                                               const float* __restrict__ weights,
                                                               const uint8_t* __restrict__ w, const float* __restrict__ ws,
                                                               uint16_t* __restrict__ y, int dt, int k, int E, int H, int I) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t t = blockIdx.y;
    const int n0 = (int)blockIdx.x * R, KB = I >> 7;             // H is a multiple of R, and 128 of R
    float sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = 0.0f;
    for (int j = wave; j < k; j += waves) {
        const int64_t p = t * k + j;
        const int e = ids[p];
        if ((unsigned)e >= (unsigned)E) continue;
        const uint8_t* we = w + ((size_t)e * H + n0) * I;
        const float* se = ws + ((size_t)e * ((H + 127) >> 7) + (n0 >> 7)) * KB;
        u32v4 wn[R][C];
        float v[C][16];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int kk = min(c * 1024 + 16 * lane, I - 16);
#pragma unroll
            for (int r = 0; r < R; ++r) wn[r][c] = __builtin_nontemporal_load(reinterpret_cast<const u32v4*>(we + (size_t)r * I + kk));
        }
        const float weight = weights[p];
        float s[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = c * 1024 + 16 * lane, kk = min(at, I - 16);
            const float4* q = reinterpret_cast<const float4*>(h + p * I + kk);
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 f = q[i];
                v[c][4 * i] = f.x, v[c][4 * i + 1] = f.y, v[c][4 * i + 2] = f.z, v[c][4 * i + 3] = f.w;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = max(mx, __float_as_uint(v[c][i]) & 0x7fffffffu);
            const float amax = fp8_amax(row8_max(mx)), factor = fp8_factor(amax);
            // the block's scales; nothing past I
            s[c] = at < I ? fp8_scale(amax) * se[kk >> 7] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float q4[4];
                fp8_values4(fp8_codes4_by(v[c][4 * i], v[c][4 * i + 1], v[c][4 * i + 2], v[c][4 * i + 3], factor), q4);
#pragma unroll
                for (int d = 0; d < 4; ++d) v[c][4 * i + d] = at < I ? q4[d] : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float d = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) d = __builtin_fmaf(dot16(wn[r][c], v[c]), s[c], d);
            sum[r] = __builtin_fmaf(d, weight, sum[r]);
        }
    }
    __shared__ float part[8][R];
    const float mine = wave_reduce_scatter<R>(sum, lane);
    if ((lane & (64 / R - 1)) == 0) part[wave][wave_rs_index<R>(lane)] = mine;
    __syncthreads();
    if (threadIdx.x < R) {
        float o = part[0][threadIdx.x];
        for (int i = 1; i < waves; ++i) o += part[i][threadIdx.x];
        y[t * H + n0 + threadIdx.x] = out_bits(o, dt);
    }
}

// -------------------------------------------------------------- the choice
constexpr int kGemvRows = 4, kGemvValues = 8;                    // M; 1024 channels of a row in registers, M C of them

// slices and chunks of K for M rows, or none
bool gemv_split(int64_t M, int64_t K, int& C, int& KS) {
    const int64_t chunks = (K + 1023) / 1024, most = kGemvValues / (M == 3 ? 4 : M);
    for (KS = 1; KS <= 4; KS *= 2)
        for (C = 1; C <= most; C *= 2)
            if (chunks <= (int64_t)C * KS) return true;
    return false;
}

struct GemvArgs {
    const void* x;
    int64_t stride;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    uint16_t* y;
    int dt, N, K;
    hipStream_t stream;
};

template <int M, int C, int KS, bool CODES, int DT>
int launch_gemv3(const GemvArgs& a) {
    constexpr int R = M * C >= 8 ? 1 : M * C >= 4 ? 2 : M >= 2 ? 2 : 4, G = 4 / KS;
    const long long groups = ((long long)a.N + R - 1) / R, want = (groups + G - 1) / G;
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);
    fp8_gemv_kernel<M, C, KS, R, CODES, DT><<<grid, 256, 0, a.stream>>>(a.x, a.stride, a.xs, a.w, a.ws, a.y, a.dt, a.N, a.K);
    return (int)hipGetLastError();
}
template <int M, int C, int KS>
int launch_gemv2(const GemvArgs& a) {
    if (a.xs) return launch_gemv3<M, C, KS, true, 0>(a);
    return a.dt == WUSH_DTYPE_BF16 ? launch_gemv3<M, C, KS, false, WUSH_DTYPE_BF16>(a) : launch_gemv3<M, C, KS, false, WUSH_DTYPE_F16>(a);
}
template <int M, int C>
int launch_gemv1(const GemvArgs& a, int KS) {
    if (KS == 1) return launch_gemv2<M, C, 1>(a);
    if constexpr (C * (M == 3 ? 4 : M) == kGemvValues) return KS == 2 ? launch_gemv2<M, C, 2>(a) : launch_gemv2<M, C, 4>(a);
    return (int)hipErrorInvalidValue;
}
template <int M>
int launch_gemv(const GemvArgs& a, int C, int KS) {
    if (C == 1) return launch_gemv1<M, 1>(a, KS);
    if (C == 2) return launch_gemv1<M, 2>(a, KS);
    if constexpr (M <= 2)
        if (C == 4) return launch_gemv1<M, 4>(a, KS);
    if constexpr (M == 1)
        if (C == 8) return launch_gemv1<M, 8>(a, KS);
    return (int)hipErrorInvalidValue;
}

template <int C>
int launch_experts(const Fp8Experts& a, hipStream_t stream) {
    constexpr int R = C >= 8 ? 1 : C >= 4 ? 2 : 4;
    const dim3 grid((unsigned)(a.I / (4 * R)), (unsigned)(a.T * a.k));
    const uint16_t* x = static_cast<const uint16_t*>(a.x);
    if (a.dtype == WUSH_DTYPE_BF16)
        fp8_experts_up_kernel<C, R, WUSH_DTYPE_BF16><<<grid, 256, 0, stream>>>(x, a.row_stride, a.ids, a.w_up, a.s_up, a.h, a.k, a.E, a.H, a.I);
    else
        fp8_experts_up_kernel<C, R, WUSH_DTYPE_F16><<<grid, 256, 0, stream>>>(x, a.row_stride, a.ids, a.w_up, a.s_up, a.h, a.k, a.E, a.H, a.I);
    return (int)hipGetLastError();
}
template <int C>
int launch_experts_down(const Fp8Experts& a, hipStream_t stream) {
    constexpr int R = C >= 4 ? 4 : 8;
    const dim3 grid((unsigned)(a.H / R), (unsigned)a.T);
    fp8_experts_down_kernel<C, R><<<grid, 64 * (a.k < 8 ? a.k : 8), 0, stream>>>(
        a.h, a.ids, a.weights, a.w_down, a.s_down, static_cast<uint16_t*>(a.y), a.dtype, a.k, a.E, a.H, a.I);
    return (int)hipGetLastError();
}

}  // namespace

bool fp8_gemv_shape(int64_t M, int64_t K) {
    int C, KS;
    return M <= kGemvRows && gemv_split(M, K, C, KS);
}

int launch_fp8_gemv(const void* x, int64_t row_stride, const float* xs, const uint8_t* w, const float* ws, uint16_t* y,
                    int dtype, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
    int C, KS;
    WUSH_REQUIRE(M >= 1 && M <= kGemvRows && N >= 1 && gemv_split(M, K, C, KS));
    const GemvArgs a = {x, row_stride, xs, w, ws, y, dtype, (int)N, (int)K, stream};
    switch (M) {
        case 1: return launch_gemv<1>(a, C, KS);
        case 2: return launch_gemv<2>(a, C, KS);
        case 3: return launch_gemv<3>(a, C, KS);
        default: return launch_gemv<4>(a, C, KS);
    }
}

bool fp8_experts_gemv_shape(int64_t T, int64_t k, int64_t H, int64_t I) {
    return T * k <= kFp8GemvPairs && H <= 8192 && I <= 4096;
}

int launch_fp8_experts_gemv(const Fp8Experts& a, hipStream_t stream) {
    WUSH_REQUIRE(fp8_experts_gemv_shape(a.T, a.k, a.H, a.I) && a.H % 16 == 0 && a.I % 128 == 0);
    const int st = a.H <= 1024 ? launch_experts<1>(a, stream) : a.H <= 2048 ? launch_experts<2>(a, stream)
                 : a.H <= 4096 ? launch_experts<4>(a, stream) : launch_experts<8>(a, stream);
    if (st) return st;
    return a.I <= 1024 ? launch_experts_down<1>(a, stream) : a.I <= 2048 ? launch_experts_down<2>(a, stream)
                                                           : launch_experts_down<4>(a, stream);
}

}  // namespace wush
