// gemm_w8a8.hip -- W8A8 products on int8 MFMA tiles: y = (xq @ wq^T) * xs * ws,
// an exact int32 sum over all of K.
//
// Workgroup: 4 wavefronts in 2 x 2, one per SIMD, each owning 16 RB x 16 CB
// outputs.  K advances a row's 128-byte line per stage: whole lines are DMA'd
// into LDS, 8 rows per instruction, NB stages deep, and read as operands, 16
// bytes a lane, for two v_mfma_i32_16x16x64_i8 steps.  Every LDS read and DMA
// is placed behind an MFMA; a step's operands are read during the step before.
//
// 4096 x 57344 x 8192: 1.48-1.52 ms, 2.5-2.6 POP/s (a library int8 product on the
// same card 2.1-2.3); 203 x 8192 x 8192 25.5 us, 13 x 24576 x 4096 17 to 22 us (weights from the last
// cache, or from HBM).  The large tiles are bound by what feeds them: without the DMAs the largest
// shape takes 1.19 ms, without the MFMAs 1.28 (64 KB a stage and CU, 11.7 TB/s over the
// chip).  Issuing the DMAs earlier or in bursts changes nothing; stages of 64 codes, five deep, are slower (1.63 ms): a DMA of half
// lines costs what whole lines do.
#include "gemm_h16_device.h"
#include "w8a8.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// c += a * b (int32, exact), accumulator in place.  The compiler does not know
// this is an MFMA: callers wait before reading c.
__device__ __forceinline__ void mfma_i8_inplace(v4i& c, const v4i& a, const v4i& b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

__device__ __forceinline__ uint32_t bf16_bits(float f) { return f != f ? 0x7fc0u : f32_to_bf16_rne(f); }

template <bool BF16>
__device__ __forceinline__ uint2 pack_out(const v4f& v) {
    if constexpr (BF16)
        return make_uint2(bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16);
    else
        return __builtin_bit_cast(uint2, __builtin_convertvector(v, h4));
}

// n of the outstanding DMAs may stay in flight, n = (stages - 1) * per, known
// at compile time for each number of stages
template <int PER, int MOST>
__device__ __forceinline__ void wait_all_but(int stages) {
    if constexpr (MOST > 0) {
        if (stages >= MOST) {
            WUSH_WAIT_VMCNT(MOST * PER);
            return;
        }
        wait_all_but<PER, MOST - 1>(stages);
    } else {
        WUSH_WAIT_VMCNT(0);
    }
}

template <int RB, int CB, int NB, bool BF16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
void gemm_w8a8_kernel(const int8_t* __restrict__ xq, const float* __restrict__ xs, const int8_t* __restrict__ wq,
                      const float* __restrict__ ws, uint16_t* __restrict__ y, int* __restrict__ part, int M, int N, int K,
                      int splits) {
    constexpr int TR = 32 * RB, TC = 32 * CB;
    constexpr int DA = TR / 32, DB = TC / 32, ND = DA + DB;      // DMAs per wavefront and stage (8 rows each)
    constexpr int kA = TR * 128, kBuf = kA + TC * 128;
    constexpr int kStage = 4 * (16 * RB) * (32 * CB);            // outputs staged, 32 CB bytes a row
    constexpr int kSmem = NB * kBuf > kStage ? NB * kBuf : kStage;
    static_assert(DA * 32 == TR && DB * 32 == TC && kSmem <= 160 * 1024 && (NB - 2) * ND < 64);
    __shared__ __align__(16) uint8_t smem[kSmem];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, l16 = lane & 15, kq = lane >> 4;
    const int wr = wave >> 1, wc = wave & 1;
    const int NR = (M + TR - 1) / TR, NC = (N + TC - 1) / TC;
    const int split = (int)blockIdx.x / (NR * NC);
    int tm, tn;
    h16_tile((int)blockIdx.x - split * (NR * NC), NR, NC, tm, tn);
    const int m0 = tm * TR, n0 = tn * TC;
    const int NS = (K + 127) >> 7;                               // stages, the last half one if K % 128 == 64
    const int first = (int)((long long)NS * split / splits), last = (int)((long long)NS * (split + 1) / splits);
    const bool half = (K & 127) != 0;
    // The sum does not depend on its order: column c of the tiles begins at stage c (of the
    // whole ones; a half one stays last), so that workgroups in step do not ask for
    // addresses a multiple of K apart, which fall on few of HBM's channels.  64 x 57344 x 8192 95 us, from the
    // same stage on 107; 64 x 24576 x 4096 26, not 30; 256 x 57344 x 8192 128, not 143; none slower.
    const int whole = last - first - (half && last == NS ? 1 : 0);
    const int turn = whole > 0 ? tn % whole : 0;
    const uint32_t lds0 = lds_addr(smem);

    // DMA k of a stage: 8 rows; lane l fetches piece (l % 8) ^ f(r) of row r = 8
    // k' + l / 8, f(r) = (r / 2) % 8, so that 16 consecutive rows' reads of one
    // piece hit distinct banks.  Rows past M or N read the last one; pieces
    // past a half stage's end the ones before (never multiplied).
    uint32_t voff[ND], back[2][2];
#pragma unroll
    for (int k = 0; k < ND; ++k) {
        const int r = 8 * (k < DA ? wave * DA + k : wave * DB + k - DA) + (lane >> 3);
        const int lim = (k < DA ? M - m0 : N - n0) - 1;
        const int piece = (lane & 7) ^ ((r >> 1) & 7);
        voff[k] = (uint32_t)min(r, lim) * (uint32_t)K + 16u * piece;
        const int e = k < DA ? k : k - DA;
        if (e < 2) back[k >= DA][e] = piece >= 4 ? 64u : 0u;     // the same for every k of one parity
    }
    const int8_t* abase = xq + (size_t)m0 * K;
    const int8_t* bbase = wq + (size_t)n0 * K;
    auto issue = [&](int st, int buf, int k) {
        const int at = st - first >= whole ? st : st + turn - (st + turn >= first + whole ? whole : 0);
        const size_t o = (size_t)at * 128;
        const uint32_t dst = lds0 + buf * kBuf;
        const uint32_t v = voff[k] - (half && st == NS - 1 ? back[k >= DA][(k < DA ? k : k - DA) & 1] : 0u);
        if (k < DA) dma16_uniform(abase + o, v, dst + (wave * DA + k) * 1024);
        else dma16_uniform(bbase + o, v, dst + kA + (wave * DB + k - DA) * 1024);
    };

    v4i acc[RB][CB], a[2][RB], b[2][CB];
    const int fsw = (l16 >> 1) & 7;
    const uint8_t* arow = smem + (wr * RB * 16 + l16) * 128;
    const uint8_t* brow = smem + kA + (wc * CB * 16 + l16) * 128;
    // read q (columns first) of step s of the stage in buffer buf
    auto read = [&](int s, int buf, int q) {
        const int o = buf * kBuf + 16 * ((4 * s + kq) ^ fsw);
        if (q < CB) b[s][q] = *reinterpret_cast<const v4i*>(brow + o + q * 2048);
        else a[s][q - CB] = *reinterpret_cast<const v4i*>(arow + o + (q - CB) * 2048);
    };

#pragma unroll
    for (int s = 0; s < NB; ++s)
        if (first + s < last)
#pragma unroll
            for (int k = 0; k < ND; ++k) issue(first + s, s, k);
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
    wait_all_but<ND, NB - 1>(last - first - 1);
    WUSH_LDS_BARRIER();
#pragma unroll
    for (int q = 0; q < RB + CB; ++q) read(0, 0, q);
    asm volatile("s_nop 7");                     // the zeroed accumulators before the first MFMA
    __builtin_amdgcn_sched_barrier(0);

    constexpr int kReads = RB + CB, kMf = RB * CB;
    int buf = 0;                                 // LDS buffer of stage st
    int st = first;
    // one stage; REFILL: its buffer takes stage st + NB.  Operands read past the
    // last stage are what the buffer happens to hold, and are not used.
    auto stage = [&](auto refill) {
        const int nbuf = buf + 1 == NB ? 0 : buf + 1;
        static_for<kMf>([&](auto mc) {           // the second step's operands are read behind the first
            constexpr int m = mc.value, i = m / CB, j = m % CB;
            mfma_i8_inplace(acc[i][j], b[0][j], a[0][i]);
            constexpr int q0 = m * kReads / kMf, q1 = (m + 1) * kReads / kMf;
            static_for<q1 - q0>([&](auto qc) { read(1, buf, q0 + qc.value); });
            __builtin_amdgcn_sched_barrier(0);
        });
        // stage st + 1 has landed in all wavefronts' view, and all have read this one
        if constexpr (refill.value) WUSH_WAIT_VMCNT((NB - 2) * ND);
        else wait_all_but<ND, NB - 2>(last - st - 2);
        WUSH_LDS_BARRIER();
        __builtin_amdgcn_sched_barrier(0);
        if (!refill.value && half && st == NS - 1) return;       // a half stage, always the last one
        static_for<kMf>([&](auto mc) {
            constexpr int m = mc.value, i = m / CB, j = m % CB;
            mfma_i8_inplace(acc[i][j], b[1][j], a[1][i]);
            constexpr int q0 = m * kReads / kMf, q1 = (m + 1) * kReads / kMf;
            static_for<q1 - q0>([&](auto qc) { read(0, nbuf, q0 + qc.value); });
            constexpr int d0 = m * ND / kMf, d1 = (m + 1) * ND / kMf;
            if constexpr (refill.value) static_for<d1 - d0>([&](auto dc) { issue(st + NB, buf, d0 + dc.value); });
            __builtin_amdgcn_sched_barrier(0);
        });
        buf = nbuf;
    };
    for (; st + NB < last; ++st) stage(std::true_type{});
    for (; st < last; ++st) stage(std::false_type{});
    WUSH_WAIT_VMCNT(0);
    asm volatile("s_nop 15\n\ts_nop 15");        // the last MFMAs' results
    __syncthreads();

    const int mw = m0 + wr * RB * 16, nw = n0 + wc * CB * 16;
    if (splits > 1) {                            // partial sums, four columns a lane
        int* p = part + (size_t)split * M * N;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int m = mw + 16 * i + l16;
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                const int n = nw + 16 * j + 4 * kq;
                const v4i v = acc[i][j];
                int* o = p + (size_t)m * N + n;
                if (m >= M || n >= N) continue;
                if ((N & 3) == 0) *reinterpret_cast<v4i*>(o) = v;
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < N) o[r] = v[r];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        return;
    }
    // outputs through LDS: rows of 32 CB bytes, chunk c of row r at c ^ (r % chunks)
    constexpr int kRow = 32 * CB, kChunks = kRow / 16;
    uint8_t* stg = smem + wave * (16 * RB * kRow);
    uint8_t* wst = stg + l16 * kRow + (kq & 1) * 8;
    float sx[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) sx[i] = xs[min(mw + 16 * i + l16, M - 1)];
#pragma unroll
    for (int j = 0; j < CB; ++j) {
        float sw[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sw[r] = ws[min(nw + 16 * j + 4 * kq + r, N - 1)];
        uint8_t* w = wst + ((2 * j + (kq >> 1)) ^ (l16 & (kChunks - 1))) * 16;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            v4f v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][j][r] * sx[i] * sw[r];
            *reinterpret_cast<uint2*>(w + i * 16 * kRow) = pack_out<BF16>(v);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if ((N & 7) != 0 || (reinterpret_cast<uintptr_t>(y) & 15u) != 0) {
        if ((N & 1) == 0 && (reinterpret_cast<uintptr_t>(y) & 3u) == 0)
            store_staged<kRow, uint32_t>(stg, 16 * RB, y, mw, M, nw, N, lane);
        else
            store_staged<kRow, uint16_t>(stg, 16 * RB, y, mw, M, nw, N, lane);
        return;
    }
    constexpr int kRows = 64 / kChunks;          // rows per store instruction
    const int r0 = lane / kChunks, c = lane % kChunks;
#pragma unroll 8
    for (int k = 0; k < 16 * RB / kRows; ++k) {
        const int r = k * kRows + r0;
        const uint4 v = *reinterpret_cast<const uint4*>(stg + r * kRow + ((c ^ (r & (kChunks - 1))) * 16));
        if (mw + r < M && nw + c * 8 < N) *reinterpret_cast<uint4*>(y + (size_t)(mw + r) * N + nw + c * 8) = v;
    }
}

// Sums of the slices' partial sums, scaled; E outputs of one row a thread
template <int E>
__global__ __launch_bounds__(256) void w8a8_sum_kernel(const int* __restrict__ part, const float* __restrict__ xs,
                                                       const float* __restrict__ ws, uint16_t* __restrict__ y, int dtype,
                                                       int M, int N, int splits) {
    const size_t o = ((size_t)blockIdx.x * 256 + threadIdx.x) * E, total = (size_t)M * N;
    if (o >= total) return;
    const int m = (int)(o / N), n = (int)(o % N);
    v4i s = {0, 0, 0, 0};
    for (int k = 0; k < splits; ++k) {
        const int* p = part + (size_t)k * total + o;
        if constexpr (E == 4) s += *reinterpret_cast<const v4i*>(p);
        else s[0] += *p;
    }
    const float sx = xs[m];
    v4f v = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < E; ++r) v[r] = (float)s[r] * sx * ws[n + r];
    const uint2 w = dtype == WUSH_DTYPE_BF16 ? pack_out<true>(v) : pack_out<false>(v);
    if constexpr (E == 4) {
        if ((reinterpret_cast<uintptr_t>(y) & 7u) == 0) *reinterpret_cast<uint2*>(y + o) = w;
        else
#pragma unroll
            for (int r = 0; r < 4; ++r) y[o + r] = (uint16_t)((r < 2 ? w.x : w.y) >> (16 * (r & 1)));
    } else {
        y[o] = (uint16_t)w.x;
    }
}

template <int RB, int CB, int NB>
void launch_tile(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, uint16_t* y, int dtype, int M, int N,
                 int K, int splits, int* part, unsigned grid, hipStream_t stream) {
    if (dtype == WUSH_DTYPE_BF16)
        gemm_w8a8_kernel<RB, CB, NB, true><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, y, part, M, N, K, splits);
    else
        gemm_w8a8_kernel<RB, CB, NB, false><<<grid, 256, 0, stream>>>(xq, xs, wq, ws, y, part, M, N, K, splits);
}

}  // namespace

int launch_gemm_w8a8(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, uint16_t* y, int dtype, int M,
                     int N, int K, int tile_rows, int tile_cols, int splits, int* part, hipStream_t stream) {
    WUSH_REQUIRE(M > 0 && N > 0 && K > 0 && K % 64 == 0 && splits >= 1 && splits <= (K + 127) / 128);
    const long long tiles = (long long)((M + tile_rows - 1) / tile_rows) * ((N + tile_cols - 1) / tile_cols) * splits;
    WUSH_REQUIRE(tiles <= 0x7fffffffLL);
    const unsigned grid = (unsigned)tiles;
    const int key = tile_rows << 16 | tile_cols;
    switch (key) {
        case 256 << 16 | 256: launch_tile<8, 8, 2>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 256 << 16 | 128: launch_tile<8, 4, 3>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 128 << 16 | 128: launch_tile<4, 4, 4>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 64 << 16 | 128: launch_tile<2, 4, 3>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 64 << 16 | 64: launch_tile<2, 2, 4>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 32 << 16 | 128: launch_tile<1, 4, 3>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        case 32 << 16 | 64: launch_tile<1, 2, 4>(xq, xs, wq, ws, y, dtype, M, N, K, splits, part, grid, stream); break;
        default: return (int)hipErrorInvalidValue;
    }
    int st = (int)hipGetLastError();
    if (st || splits == 1) return st;
    const long long total = (long long)M * N;
    const int e = N % 4 == 0 ? 4 : 1;
    const long long blocks = (total / e + 255) / 256;
    WUSH_REQUIRE(blocks <= 0x7fffffffLL);
    if (e == 4) w8a8_sum_kernel<4><<<(unsigned)blocks, 256, 0, stream>>>(part, xs, ws, y, dtype, M, N, splits);
    else w8a8_sum_kernel<1><<<(unsigned)blocks, 256, 0, stream>>>(part, xs, ws, y, dtype, M, N, splits);
    return (int)hipGetLastError();
}

}  // namespace wush
