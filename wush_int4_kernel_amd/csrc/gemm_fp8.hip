// gemm_fp8.hip -- products of e4m3 codes with a scale for each row of x and block of 128
// channels, and for each block of 128 x 128 weights, on MFMA tiles:
//   y_mn = sum_b (sum_{k in block b} x_mk w_nk) xs_bm ws_{n / 128, b}
// Inner sums are one v_mfma_f32_16x16x128_f8f6f4 each; the outer one is an fp32
// multiply-add of its four results a lane with the product of the two scales.
//
// Workgroup: WR x WC wavefronts, each owning 16 RB x 16 CB outputs.  A stage is one block
// of K: rows' 128-byte lines are DMA'd into LDS, 8 rows per instruction, NB stages deep,
// and the stage's scales with them.  A wavefront walks its columns' operands in a ring of BR
// register slots, read BR - 1 columns ahead; its rows' operands are replaced, during the last
// column, by the next stage's.  The multiply-adds run kLag products behind the MFMAs, so that
// none waits for its result.
//
// 4096 x 57344 x 8192 with 256 x 256 tiles: 1.59 ms, 2.42 PFLOP/s, where the clock falls to 1.84 GHz (the library's
// product with one scale for all: 1.31 ms).  The smaller tiles are bound by the bytes that LDS can have on their way:
// about 96 KiB a CU and some 2 us of loaded latency are 12 TB/s for x and w together (203 x 8192 x 8192: 33 us).
#include "fp8.h"
#include "fp8_device.h"
#include "gemm_h16_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

__device__ __forceinline__ uint32_t bf16_bits(float f) { return f != f ? 0x7fc0u : f32_to_bf16_rne(f); }

template <bool BF16>
__device__ __forceinline__ uint2 pack_out(const v4f& v) {
    if constexpr (BF16)
        return make_uint2(bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16);
    else
        return __builtin_bit_cast(uint2, __builtin_convertvector(v, h4));
}

// n of the outstanding DMAs may stay in flight, n = stages * PER, known
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

// kPlain: one matrix.  kRows: each expert's, over its rows.
enum { kPlain, kRows };

// NT: one row tile, whose weights are read once.
template <int RB, int CB, int WR, int WC, int NB, int BR, int OCC, int MODE, int OUT, bool F16, bool NT>
__global__ __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(OCC, OCC)))
void gemm_fp8_kernel(const Fp8Gemm g) {
    constexpr int NW = WR * WC, TR = 16 * RB * WR, TC = 16 * CB * WC;
    constexpr int DA = TR / 8 / NW, DB = TC / 8 / NW, ND = DA + DB + 1;    // DMAs per wavefront and stage, one of scales
    constexpr int kChunksA = (TR + 63) / 64;                     // wavefronts that fetch x's scales, the others w's
    constexpr int kA = TR * 128, kSx = kA + TC * 128, kSw = kSx + kChunksA * 256, kBuf = kSw + 256;
    constexpr int kStage = NW * (16 * RB) * (32 * CB);           // outputs staged, 32 CB bytes a row
    constexpr bool GROUPED = MODE != kPlain;
    constexpr int kSmem = NB * kBuf > kStage ? NB * kBuf : kStage;
    constexpr int kMf = RB * CB, kLag = 3, kTmp = 4;
    static_assert(DA * 8 * NW == TR && DB * 8 * NW == TC && kChunksA < NW && CB % BR == 0 && BR >= 2 && CB >= 2);
    static_assert(kMf % kTmp == 0 && kSmem <= 160 * 1024 && (NB - 1) * ND < 64 && (CB * 16) <= 128);
    __shared__ __align__(16) uint8_t smem[kSmem];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, l16 = lane & 15, kq = lane >> 4;
    const int wr = wave / WC, wc = wave % WC;
    const int N = g.N, K = g.K;
    const int NC = (N + TC - 1) / TC, KB = (K + 127) >> 7;
    int tm, tn, m0, M, split = 0, first = 0, last = KB;
    const uint8_t* wbase = g.w;
    const float* wsbase = g.ws;
    if constexpr (GROUPED) {
        const int NR = *g.ntiles;
        if ((int)blockIdx.x >= NR * NC) return;
        // An XCD (workgroups i, i + 8, ...) takes a run of row tiles, all columns of one
        // before the next: an expert's row tiles share its weights in the XCD's L2.
        const int q = (NR * NC) >> 3, r = (NR * NC) & 7, xcd = (int)blockIdx.x & 7;
        const int s = xcd * q + min(xcd, r) + ((int)blockIdx.x >> 3);
        tm = s / NC;
        tn = s - tm * NC;
        const int4 t = g.tiles[tm];
        m0 = __builtin_amdgcn_readfirstlane(t.y);
        M = __builtin_amdgcn_readfirstlane(t.z);
        const int e = __builtin_amdgcn_readfirstlane(t.x);
        wbase += (size_t)e * N * K;
        wsbase += (size_t)e * ((N + 127) >> 7) * KB;
    } else {
        M = g.M;
        const int NR = (M + TR - 1) / TR;
        split = (int)blockIdx.x / (NR * NC);
        h16_tile((int)blockIdx.x - split * (NR * NC), NR, NC, tm, tn);
        m0 = tm * TR;
        first = (int)((long long)KB * split / g.splits);
        last = (int)((long long)KB * (split + 1) / g.splits);
    }
    const int n0 = tn * TC;
    const int tail = (K & 127) >> 4;                             // 16-byte pieces of a last, shorter block; 0: none
    // Column c of the tiles begins at stage c (of the whole blocks), so that workgroups in step do
    // not ask for addresses a multiple of K apart, which fall on few of HBM's channels.
    const int whole = last - first - (tail && last == KB ? 1 : 0);
    const int turn = whole > 0 ? tn % whole : 0;
    const uint32_t lds0 = lds_addr(smem);

    // DMA k of a stage: 8 rows; lane l fetches piece (l % 8) ^ f(r) of row r = 8
    // k' + l / 8, f(r) = (r / 2) % 8, so that 16 consecutive rows' reads of one
    // piece hit distinct banks.  Rows past M or N read the last one; pieces
    // past a short block's end its first one, whose activations are zeroed before use.
    uint32_t voff[ND - 1], past[2][2];
#pragma unroll
    for (int k = 0; k < ND - 1; ++k) {
        const int r = 8 * (k < DA ? wave * DA + k : wave * DB + k - DA) + (lane >> 3);
        const int piece = (lane & 7) ^ ((r >> 1) & 7);
        int row;
        if (k < DA) {
            row = min(r, M - m0 - 1);
            if constexpr (GROUPED) {
                row += m0;
                if (g.row_of) row = g.row_of[row];
            }
        } else {
            row = min(r, N - n0 - 1);
        }
        voff[k] = (uint32_t)row * (uint32_t)K + 16u * piece;
        const int e = k < DA ? k : k - DA;
        if (e < 2) past[k >= DA][e] = piece >= tail ? 16u * piece : 0u;    // the same for every k of one parity
    }
    const uint8_t* abase = GROUPED ? g.x : g.x + (size_t)m0 * K;
    const uint8_t* bbase = wbase + (size_t)n0 * K;
    // the scales' DMA: 64 of x's, or those of w's TC / 128 blocks
    const uint8_t* sbase;
    size_t sstep;
    uint32_t soff, sdst;
    if (wave < kChunksA) {
        int row = min(64 * wave + lane, M - m0 - 1);
        if constexpr (GROUPED) {
            row += m0;
            if (g.row_of) row = g.row_of[row];
        }
        sbase = reinterpret_cast<const uint8_t*>(GROUPED ? g.xs : g.xs + m0);
        sstep = (size_t)g.ldx * 4;
        soff = (uint32_t)row * 4u;
        sdst = kSx + wave * 256;
    } else {
        const int nb = min(lane & (TC / 128 > 1 ? TC / 128 - 1 : 0), ((N - 1) >> 7) - (n0 >> 7));
        sbase = reinterpret_cast<const uint8_t*>(wsbase + (size_t)(n0 >> 7) * KB);
        sstep = 4;
        soff = (uint32_t)(nb * KB) * 4u;
        sdst = kSw;
    }
    auto issue = [&](int st, int buf, int k) {
        const int at = st - first >= whole ? st : st + turn - (st + turn >= first + whole ? whole : 0);
        const uint32_t dst = lds0 + buf * kBuf;
        if (k == ND - 1) {
            const uint8_t* b = sbase + at * sstep;
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(soff), "s"(b), "s"(dst + sdst) : "m0");
            return;
        }
        const size_t o = (size_t)at * 128;
        const uint32_t v = voff[k] - (tail && at == KB - 1 ? past[k >= DA][(k < DA ? k : k - DA) & 1] : 0u);
        if (k < DA) dma16_uniform(abase + o, v, dst + (wave * DA + k) * 1024);
        else if constexpr (NT) dma16_uniform_nt(bbase + o, v, dst + kA + (wave * DB + k - DA) * 1024);
        else dma16_uniform(bbase + o, v, dst + kA + (wave * DB + k - DA) * 1024);
    };

    v4f acc[RB][CB];
    v8i a[RB], b[BR];
    float sc[RB], old[RB];                       // products of the scales: this stage's, the last one's
    const int fsw = (l16 >> 1) & 7;
    const uint8_t* arow = smem + (wr * RB * 16 + l16) * 128;
    const uint8_t* brow = smem + kA + (wc * CB * 16 + l16) * 128;
    const int p0 = 16 * (kq ^ fsw), p1 = 16 * ((4 + kq) ^ fsw);
    auto pieces = [&](const uint8_t* p) {
        const v4i lo = *reinterpret_cast<const v4i*>(p + p0), hi = *reinterpret_cast<const v4i*>(p + p1);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto read_a = [&](int buf, int i) { a[i] = pieces(arow + buf * kBuf + i * 2048); };
    auto read_b = [&](int buf, int j) { b[j % BR] = pieces(brow + buf * kBuf + j * 2048); };
    float sx[RB], sw;
    auto read_s = [&](int buf) {
        const uint8_t* p = smem + buf * kBuf;
#pragma unroll
        for (int i = 0; i < RB; ++i) sx[i] = *reinterpret_cast<const float*>(p + kSx + 4 * ((wr * RB + i) * 16 + l16));
        sw = *reinterpret_cast<const float*>(p + kSw + 4 * ((wc * CB * 16) >> 7));
    };

#pragma unroll
    for (int s = 0; s < NB; ++s)
        if (first + s < last)
#pragma unroll
            for (int k = 0; k < ND; ++k) issue(first + s, s, k);
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        sc[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < CB; ++j) acc[i][j] = (v4f){0, 0, 0, 0};
    }
    wait_all_but<ND, NB - 1>(last - first - 1);
    WUSH_LDS_BARRIER();
    __builtin_amdgcn_sched_barrier(0);
    read_s(0);
#pragma unroll
    for (int i = 0; i < RB; ++i) read_a(0, i);
#pragma unroll
    for (int j = 0; j < BR - 1; ++j) read_b(0, j);
    __builtin_amdgcn_sched_barrier(0);

    int buf = 0;                                 // LDS buffer of stage st
    int st = first;
    // what both forms of a stage begin with
    auto begin = [&] {
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            old[i] = sc[i];
            sc[i] = sx[i] * sw;
        }
        if (tail && st == KB - 1) {              // a short block, always the last: no activations past its end
            const v4i zero = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const v4i lo = kq < tail ? __builtin_shufflevector(a[i], a[i], 0, 1, 2, 3) : zero;
                const v4i hi = 4 + kq < tail ? __builtin_shufflevector(a[i], a[i], 4, 5, 6, 7) : zero;
                a[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    };
    // stage st + 1 has landed in all wavefronts' view, and all have read this one's columns
    auto landed = [&](auto refill) {
        if constexpr (refill.value) WUSH_WAIT_VMCNT((NB - 2) * ND);
        else wait_all_but<ND, NB - 2>(last - st - 2);
        WUSH_LDS_BARRIER();
        __builtin_amdgcn_sched_barrier(0);
    };
    // share q of n of the refill's DMAs
    auto refill_part = [&](auto qc, auto nc) {
        constexpr int q = qc.value, n = nc.value;
        static_for<(q + 1) * ND / n - q * ND / n>([&](auto dc) { issue(st + NB, buf, q * ND / n + dc.value); });
    };
    constexpr int kTurn = CB - BR + 1;           // the column from which on the next stage is read
    if constexpr (!F16) {
        v4f tmp[kTmp];
#pragma unroll
        for (int t = 0; t < kTmp; ++t) tmp[t] = (v4f){0, 0, 0, 0};
        auto add = [&](int m, const float (&s)[RB]) {
            const int i = m % RB, j = m / RB;
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(tmp[m % kTmp][r], s[i], acc[i][j][r]);
        };
        // one stage; REFILL: its buffer takes stage st + NB.  Operands read past the
        // last stage are what the buffer happens to hold, and are not used.
        auto stage = [&](auto refill) {
            const int nbuf = buf + 1 == NB ? 0 : buf + 1;
            begin();
            static_for<kMf>([&](auto mc) {
                constexpr int m = mc.value, i = m % RB, j = m / RB;
                if constexpr (i == 0 && j == kTurn) landed(refill);
                tmp[m % kTmp] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j % BR], a[i], (v4f){0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                if constexpr (i == 0) {
                    constexpr int jn = j + BR - 1;
                    if constexpr (jn < CB) read_b(buf, jn);
                    else read_b(nbuf, jn - CB);
                }
                if constexpr (j == CB - 1) read_a(nbuf, i);
                if constexpr (m == kMf - 1) read_s(nbuf);
                if constexpr (m >= kLag) add(m - kLag, sc);
                else add(kMf + m - kLag, old);
                if constexpr (refill.value && j >= kTurn)
                    refill_part(std::integral_constant<int, m - kTurn * RB>{}, std::integral_constant<int, (BR - 1) * RB>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            buf = nbuf;
        };
        for (; st + NB < last; ++st) stage(std::true_type{});
        for (; st < last; ++st) stage(std::false_type{});
#pragma unroll
        for (int m = kMf - kLag; m < kMf; ++m) add(m, sc);
    } else {
        // Operands widened to fp16, which is exact, and four v_mfma_f32_16x16x32_f16 a block; a column's
        // multiply-adds run behind the next column's MFMAs.
        v4f tmp[2][RB];
        h8 wa[RB][4], wb[4];
#pragma unroll
        for (int i = 0; i < RB; ++i) tmp[(CB - 1) & 1][i] = (v4f){0, 0, 0, 0};
        auto add = [&](int j, int i, const float (&s)[RB]) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(tmp[j & 1][i][r], s[i], acc[i][j][r]);
        };
        auto stage = [&](auto refill) {
            const int nbuf = buf + 1 == NB ? 0 : buf + 1;
            begin();
#pragma unroll
            for (int i = 0; i < RB; ++i) fp8_widen(a[i], wa[i]);
            static_for<CB>([&](auto jc) {
                constexpr int j = jc.value, jn = j + BR - 1;
                if constexpr (j == kTurn) {
                    landed(refill);
#pragma unroll
                    for (int i = 0; i < RB; ++i) read_a(nbuf, i);
                    read_s(nbuf);
                }
                fp8_widen(b[j % BR], wb);
                if constexpr (jn < CB) read_b(buf, jn);
                else read_b(nbuf, jn - CB);
                __builtin_amdgcn_sched_barrier(0);
                static_for<4 * RB>([&](auto mc) {
                    constexpr int q = mc.value / RB, i = mc.value % RB;
                    tmp[j & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[q], wa[i][q], q ? tmp[j & 1][i] : (v4f){0, 0, 0, 0}, 0, 0, 0);
                    if constexpr (q == 1) {
                        if constexpr (j > 0) add(j - 1, i, sc);
                        else add(CB - 1, i, old);
                    }
                    if constexpr (refill.value && j >= kTurn)
                        refill_part(std::integral_constant<int, (j - kTurn) * 4 * RB + mc.value>{},
                                    std::integral_constant<int, (BR - 1) * 4 * RB>{});
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
            buf = nbuf;
        };
        for (; st + NB < last; ++st) stage(std::true_type{});
        for (; st < last; ++st) stage(std::false_type{});
#pragma unroll
        for (int i = 0; i < RB; ++i) add(CB - 1, i, sc);
    }
    WUSH_WAIT_VMCNT(0);
    __syncthreads();

    const int mw = m0 + wr * RB * 16, nw = n0 + wc * CB * 16;
    if (OUT == kOutF32 || g.splits > 1) {        // four columns a lane
        float* p = OUT == kOutF32 ? static_cast<float*>(g.y) : g.part + (size_t)split * M * N;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int m = mw + 16 * i + l16;
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                const int n = nw + 16 * j + 4 * kq;
                float* o = p + (size_t)m * N + n;
                if (m >= M || n >= N) continue;
                if ((N & 3) == 0) *reinterpret_cast<v4f*>(o) = acc[i][j];
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < N) o[r] = acc[i][j][r];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        return;
    }
    if constexpr (OUT != kOutF32) {
        // outputs through LDS: rows of 32 CB bytes, chunk c of row r at c ^ (r % chunks)
        uint16_t* y = static_cast<uint16_t*>(g.y);
        constexpr int kRow = 32 * CB, kChunks = kRow / 16;
        uint8_t* stg = smem + wave * (16 * RB * kRow);
        uint8_t* wst = stg + l16 * kRow + (kq & 1) * 8;
#pragma unroll
        for (int j = 0; j < CB; ++j) {
            uint8_t* w = wst + ((2 * j + (kq >> 1)) ^ (l16 & (kChunks - 1))) * 16;
#pragma unroll
            for (int i = 0; i < RB; ++i) *reinterpret_cast<uint2*>(w + i * 16 * kRow) = pack_out<OUT == WUSH_DTYPE_BF16>(acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if ((N & 7) != 0 || (reinterpret_cast<uintptr_t>(y) & 15u) != 0) {
            if ((N & 1) == 0 && (reinterpret_cast<uintptr_t>(y) & 3u) == 0)
                store_staged<kRow, uint32_t>(stg, 16 * RB, y, mw, M, nw, N, lane);
            else
                store_staged<kRow, uint16_t>(stg, 16 * RB, y, mw, M, nw, N, lane);
            return;
        }
        constexpr int kRows = 64 / kChunks;      // rows per store instruction
        const int r0 = lane / kChunks, c = lane % kChunks;
#pragma unroll 8
        for (int k = 0; k < 16 * RB / kRows; ++k) {
            const int r = k * kRows + r0;
            const uint4 v = *reinterpret_cast<const uint4*>(stg + r * kRow + ((c ^ (r & (kChunks - 1))) * 16));
            if (mw + r < M && nw + c * 8 < N) *reinterpret_cast<uint4*>(y + (size_t)(mw + r) * N + nw + c * 8) = v;
        }
    }
}

// Sums of the slices' partial sums; E outputs of one row a thread
template <int E>
__global__ __launch_bounds__(256) void fp8_sum_kernel(const float* __restrict__ part, uint16_t* __restrict__ y, int dtype,
                                                      size_t total, int splits) {
    const size_t o = ((size_t)blockIdx.x * 256 + threadIdx.x) * E;
    if (o >= total) return;
    v4f s = {0, 0, 0, 0};
    for (int k = 0; k < splits; ++k) {
        const float* p = part + (size_t)k * total + o;
        if constexpr (E == 4) s += *reinterpret_cast<const v4f*>(p);
        else s[0] += *p;
    }
    const uint2 w = dtype == WUSH_DTYPE_BF16 ? pack_out<true>(s) : pack_out<false>(s);
    if constexpr (E == 4) {
        if ((reinterpret_cast<uintptr_t>(y) & 7u) == 0) *reinterpret_cast<uint2*>(y + o) = w;
        else
#pragma unroll
            for (int r = 0; r < 4; ++r) y[o + r] = (uint16_t)((r < 2 ? w.x : w.y) >> (16 * (r & 1)));
    } else {
        y[o] = (uint16_t)w.x;
    }
}

template <int RB, int CB, int WR, int WC, int NB, int BR, int OCC>
int launch_plain(const Fp8Gemm& g, unsigned grid, hipStream_t stream) {
    constexpr int T = 64 * WR * WC;
    constexpr int BF = WUSH_DTYPE_BF16, HF = WUSH_DTYPE_F16;
    const bool bf = g.out == BF;
    if (g.M <= 16 * RB * WR) {
        if (bf) gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, OCC, kPlain, BF, false, true><<<grid, T, 0, stream>>>(g);
        else gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, OCC, kPlain, HF, false, true><<<grid, T, 0, stream>>>(g);
    } else {
        if (bf) gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, OCC, kPlain, BF, false, false><<<grid, T, 0, stream>>>(g);
        else gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, OCC, kPlain, HF, false, false><<<grid, T, 0, stream>>>(g);
    }
    return (int)hipGetLastError();
}

}  // namespace

// for few rows an expert: mostly one tile of each
int launch_gemm_fp8_rows(const Fp8Gemm& g, hipStream_t stream) {
    constexpr int RB = 2, CB = 2, WR = 1, WC = 2, NB = 4, BR = 2, T = 64 * WR * WC, TC = 16 * CB * WC;
    static_assert(16 * RB * WR == kFp8RowsTile && TC == 2 * kFp8RowsTile);
    const long long cols = (g.N + TC - 1) / TC;
    WUSH_REQUIRE(g.tiles && g.ntiles && g.N > 0 && g.K > 0 && g.K % 16 == 0 && g.splits == 1 && !g.act && !g.shared);
    WUSH_REQUIRE(g.most_tiles * cols < (1 << 23));               // a launch has fewer than 2^32 threads
    const unsigned grid = (unsigned)(g.most_tiles * cols);
    if (g.wide) gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, 1, kRows, kOutF32, true, true><<<grid, T, 0, stream>>>(g);
    else gemm_fp8_kernel<RB, CB, WR, WC, NB, BR, 1, kRows, kOutF32, false, true><<<grid, T, 0, stream>>>(g);
    return (int)hipGetLastError();
}

int launch_gemm_fp8(const Fp8Gemm& g, int tile_rows, int tile_cols, hipStream_t stream) {
    WUSH_REQUIRE(g.M > 0 && g.N > 0 && g.K > 0 && g.K % 16 == 0 && g.splits >= 1 && g.splits <= (g.K + 127) / 128);
    WUSH_REQUIRE(!g.tiles && (g.splits == 1 || g.part));
    const long long tiles = (long long)((g.M + tile_rows - 1) / tile_rows) * ((g.N + tile_cols - 1) / tile_cols) * g.splits;
    WUSH_REQUIRE(tiles < (1 << 23));                             // a launch has fewer than 2^32 threads
    const unsigned grid = (unsigned)tiles;
    int st;
    switch (tile_rows << 16 | tile_cols) {
        case 256 << 16 | 256: st = launch_plain<4, 8, 4, 2, 2, 4, 2>(g, grid, stream); break;
        case 128 << 16 | 128: st = launch_plain<4, 4, 2, 2, 4, 4, 1>(g, grid, stream); break;
        case 64 << 16 | 128: st = launch_plain<2, 4, 2, 2, 3, 4, 1>(g, grid, stream); break;
        case 32 << 16 | 128: st = launch_plain<1, 4, 2, 2, 3, 4, 1>(g, grid, stream); break;
        case 32 << 16 | 64: st = launch_plain<2, 2, 1, 2, 4, 2, 1>(g, grid, stream); break;
        default: return (int)hipErrorInvalidValue;
    }
    if (st || g.splits == 1) return st;
    const size_t total = (size_t)g.M * g.N;
    const int e = g.N % 4 == 0 ? 4 : 1;
    const size_t blocks = (total / e + 255) / 256;
    WUSH_REQUIRE(blocks <= 0x7fffffffu / 256);
    uint16_t* y = static_cast<uint16_t*>(g.y);
    if (e == 4) fp8_sum_kernel<4><<<(unsigned)blocks, 256, 0, stream>>>(g.part, y, g.out, total, g.splits);
    else fp8_sum_kernel<1><<<(unsigned)blocks, 256, 0, stream>>>(g.part, y, g.out, total, g.splits);
    return (int)hipGetLastError();
}

}  // namespace wush
