// gemm_fp8_runs.hip -- the products of gemm_fp8.hip for many rows: one workgroup a
// CU takes tile after tile, and the loads of a tile's first stages are issued during the last stages of
// the one before, so that neither its way from memory nor the outputs' way to it is waited for.
//
// Workgroup: eight wavefronts, WR x WC, each owning 16 RB x 256 / WC outputs.  Stages and their order as in gemm_fp8.hip.
// Outputs leave straight from registers, four columns of a lane made 16 by swaps between the
// lanes of a row: LDS belongs to the next tile by then.
//
// 27 x 57344 x 8192, tiles of 64 x 256: 71 us, 6.6 TB/s of weights (one tile a workgroup: 82).  The experts' layer of 4096 tokens,
// 8 of 128 experts of 4096 x 1024: 265 to 290 us for the down projections, where LDS reads take as long as the MFMAs, and 745 to
// 790 for the gate and up projections, in fp16 instructions (0.7 PFLOP/s), where the issue of vector instructions takes longest: 250
// and 64 MFMAs of 9 cycles each for a block of K in a wavefront, half of them to widen codes.
#include "fp8.h"
#include "fp8_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// One matrix (kPlain); each expert's, over its rows, outputs in fp32 (kWide) or in fp16 with shared powers of
// two (kShared); each expert's gate and up projection together, whose products leave as codes of
// silu(gate) * up (kAct): half of a wavefront's columns are the gate's, the other half the same ones of the up projection.
enum { kPlain, kWide, kShared, kAct };

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16)
        return (a != a ? 0x7fc0u : f32_to_bf16_rne(a)) | (b != b ? 0x7fc0u : f32_to_bf16_rne(b)) << 16;
    else
        return __builtin_bit_cast(uint32_t, (h2){(_Float16)a, (_Float16)b});
}

// v[j] of the four 16-lane rows r -> v[r] of rows j: a transposition
__device__ __forceinline__ void rows_transpose(uint32_t (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(v[i], v[i + 2], false, false);
        v[i] = r[0];
        v[i + 2] = r[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const auto r = __builtin_amdgcn_permlane16_swap(v[i], v[i + 1], false, false);
        v[i] = r[0];
        v[i + 1] = r[1];
    }
}

template <int RB, int WR, int WC, int NB, int MODE, bool BF16, bool F16, bool NT>
__global__ __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gemm_fp8_runs_kernel(const Fp8Gemm g) {
    constexpr int NW = WR * WC, TR = 16 * RB * WR, TC = 256;
    constexpr int CB = 16 / WC, BR = F16 ? 2 : 4, kMf = RB * CB, kLag = 3, kTmp = 4, kTurn = CB - BR + 1;
    constexpr int DA = TR / 8 / NW, DB = TC / 8 / NW, ND = DA + DB + 1;    // DMAs per wavefront and stage, one of scales
    constexpr int kChunksA = TR / 64;                            // wavefronts that fetch x's scales, the others w's
    constexpr int kA = TR * 128, kSx = kA + TC * 128, kSw = kSx + kChunksA * 256, kBuf = kSw + 256;
    constexpr int kSmem = NB * kBuf + (MODE == kAct ? TR * WC * 4 : 0);
    constexpr bool GROUPED = MODE != kPlain;
    constexpr int NSW = MODE == kAct ? 2 : 1;                    // scales of w that a wavefront's columns have
    constexpr int kStores = MODE == kAct ? RB : MODE == kWide ? RB * CB : RB * CB / 2;    // stores of a whole tile, at least
    constexpr int kHalf = 8 * CB;                                // kAct: columns of the gate that a wavefront has
    static_assert(kSmem <= 160 * 1024 && (NB - 2) * ND + kStores < 64 && 8 * DB <= kHalf && kChunksA < NW);
    __shared__ __align__(16) uint8_t smem[kSmem];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, l16 = lane & 15, kq = lane >> 4;
    const int wr = wave / WC, wc = wave % WC;
    const int N = g.N, K = g.K, I = N >> 1;
    const int NC = MODE == kAct ? I >> 7 : (N + TC - 1) / TC, KB = (K + 127) >> 7;
    const int tail = (K & 127) >> 4;                             // 16-byte pieces of a last, shorter block; 0: none
    const int whole = KB - (tail != 0);                          // blocks that are whole
    const int NR = GROUPED ? *g.ntiles : (g.M + TR - 1) / TR;
    // Tiles in order: experts', all columns of a row tile before the next (an expert's row tiles
    // share its weights); one matrix's, groups of 8 row tiles walked together.  An XCD
    // (workgroups i, i + 8, ...) takes a run of them, its workgroups in turn.
    const int total = NR * NC, xcd = (int)blockIdx.x & 7;
    const int q8 = total >> 3, r8 = total & 7;
    const int run_end = xcd * q8 + min(xcd, r8) + q8 + (xcd < r8 ? 1 : 0);
    const int step = ((int)gridDim.x + 7 - xcd) >> 3;            // workgroups of the XCD
    int next = xcd * q8 + min(xcd, r8) + ((int)blockIdx.x >> 3);
    if (next >= run_end) return;
    const uint32_t lds0 = lds_addr(smem);

    // ------------------------------------------------ the tile whose loads are being issued
    int ist = 0, iturn = 0;
    const uint8_t *abase = nullptr, *bbase = nullptr, *sbase = nullptr;
    size_t sstep = 0;
    uint32_t voff[DA + DB], soff = 0;
    const int r0 = 8 * DB * wave;                                // this wavefront's first LDS row of w
    const uint32_t piece = ((uint32_t)lane & 7u) ^ (((uint32_t)lane >> 4) & 3u);     // of even groups of 8 rows; of odd ones ^ 4
    const uint32_t flip = DA & 1 ? 4u * (wave & 1) : 0u;         // this wavefront's first group of x
    auto place = [&](int s, int& tm, int& tn) {
        if constexpr (GROUPED) {
            tm = s / NC;
            tn = s - tm * NC;
        } else {
            const int G = s / (8 * NC), h = min(8, NR - G * 8), w = s - G * (8 * NC);
            tm = G * 8 + w % h;
            tn = w / h;
        }
    };
    auto row_range = [&](int tm, int& m0, int& M) {
        if constexpr (GROUPED) {
            const int4 t = g.tiles[tm];
            m0 = __builtin_amdgcn_readfirstlane(t.y);
            M = __builtin_amdgcn_readfirstlane(t.z);
        } else {
            m0 = tm * TR;
            M = g.M;
        }
    };
    auto open = [&](int s) {
        int tm, tn, im0, iM;
        place(s, tm, tn);
        row_range(tm, im0, iM);
        const uint8_t* wb = g.w;
        const float* wsb = g.ws;
        if constexpr (GROUPED) {
            const int e = __builtin_amdgcn_readfirstlane(g.tiles[tm].x);
            wb += (size_t)e * N * K;
            wsb += (size_t)e * ((N + 127) >> 7) * KB;
        }
        ist = 0;
        // Column c of the tiles begins at block c (of the whole ones), so that workgroups in step do
        // not ask for addresses a multiple of K apart, which fall on few of HBM's channels.
        iturn = whole > 0 ? tn % whole : 0;
        abase = GROUPED ? g.x : g.x + (size_t)im0 * K;
        // kAct: LDS rows are, for each wavefront column, kHalf of the gate's and the same of the up projection's
        const int n0 = MODE == kAct ? (r0 & kHalf ? I : 0) + tn * 128 + r0 / (2 * kHalf) * kHalf + r0 % kHalf : tn * TC + r0;
        bbase = wb + (size_t)(MODE == kAct ? n0 : min(n0, N - 1)) * K;
#pragma unroll
        for (int k = 0; k < DA + DB; ++k) {
            int row = 8 * (k < DA ? wave * DA + k : k - DA) + (lane >> 3);
            if (k < DA) {
                row = min(row, iM - im0 - 1);
                if constexpr (GROUPED) {
                    row += im0;
                    if (MODE == kAct) row = g.row_of[row];
                }
            } else if (MODE != kAct) {
                row = max(min(row, N - n0 - 1), 0);
            }
            voff[k] = (uint32_t)row * (uint32_t)K + 16u * (piece ^ (k < DA ? flip ^ (k & 1 ? 4u : 0u) : (k - DA) & 1 ? 4u : 0u));
        }
        if (wave < kChunksA) {
            int row = min(64 * wave + lane, iM - im0 - 1);
            if constexpr (GROUPED) {
                row += im0;
                if (MODE == kAct) row = g.row_of[row];
            }
            sbase = reinterpret_cast<const uint8_t*>(GROUPED ? g.xs : g.xs + im0);
            sstep = (size_t)g.ldx * 4;
            soff = (uint32_t)row * 4u;
        } else {
            const int nb = MODE == kAct ? tn : 2 * tn;
            sbase = reinterpret_cast<const uint8_t*>(wsb + (size_t)nb * KB);
            sstep = 4;
            soff = (uint32_t)((MODE == kAct ? (lane & 1) * (I >> 7) : min(lane & 1, ((N - 1) >> 7) - nb)) * KB) * 4u;
        }
    };
    // DMA k of stage ist into buffer buf: lane l fetches piece (l % 8) ^ f(r) of row r = 8 k' + l / 8,
    // f(r) = (r / 2) % 8, so that 16 consecutive rows' reads of one piece hit distinct banks.  Rows past the
    // end read the last one; pieces past a short block's end its first one, whose activations are zeroed before use.
    const uint8_t *ia, *ib, *is;                                 // this stage's addresses
    uint32_t idst, past[2], pastx;
    auto aim = [&](int buf) {
        const int at = ist >= whole ? ist : ist + iturn - (ist + iturn >= whole ? whole : 0);
        const bool cut = tail && at == KB - 1;
        ia = abase + (size_t)at * 128;
        ib = bbase + (size_t)at * 128;
        is = sbase + at * sstep;
        idst = lds0 + buf * kBuf;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t p = piece ^ (e ? 4u : 0u);
            past[e] = cut && p >= (uint32_t)tail ? 16u * p : 0u;
        }
        pastx = flip ? past[1] : past[0];
    };
    auto issue = [&](auto kc) {
        constexpr int k = kc.value;
        if constexpr (k == DA + DB) {
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                         : : "v"(soff), "s"(is), "s"(idst + (wave < kChunksA ? kSx + wave * 256 : kSw)) : "m0");
        } else if constexpr (k < DA) {
            dma16_uniform(ia, voff[k] - (DA & 1 ? pastx : past[k & 1]), idst + (wave * DA + k) * 1024);
        } else {
            if constexpr (NT) dma16_uniform_nt(ib, voff[k] - past[(k - DA) & 1], idst + kA + (wave * DB + k - DA) * 1024);
            else dma16_uniform(ib, voff[k] - past[(k - DA) & 1], idst + kA + (wave * DB + k - DA) * 1024);
        }
    };
    static_assert((DA == 1 || DA % 2 == 0) && DB % 2 == 0);
    // The stage after this one; behind the last of all, that one again, so that every stage issues as many loads.
    auto advance = [&] {
        if (++ist < KB) return;
        if (next + step < run_end) open(next += step);
        else ist = KB - 1;
    };

    // --------------------------------------------------------------- the pipeline's state
    v4f acc[RB][CB], tmp[F16 ? 2 * RB : kTmp];                   // F16: column j's products at (j & 1) * RB
    v8i a[RB], b[BR];
    float sc[NSW][RB], old[RB], sx[RB], sw[NSW];
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
    auto read_s = [&](int buf) {
        const uint8_t* p = smem + buf * kBuf;
#pragma unroll
        for (int i = 0; i < RB; ++i) sx[i] = *reinterpret_cast<const float*>(p + kSx + 4 * ((wr * RB + i) * 16 + l16));
        if constexpr (MODE == kAct) {
            sw[0] = *reinterpret_cast<const float*>(p + kSw);
            sw[1] = *reinterpret_cast<const float*>(p + kSw + 4);
        } else {
            sw[0] = *reinterpret_cast<const float*>(p + kSw + 4 * ((wc * CB * 16) >> 7));
        }
    };

    int cur = next, tm, tn, m0, M;                               // the tile being computed
    place(cur, tm, tn);
    row_range(tm, m0, M);
    open(next);
    for (int s = 0; s < NB; ++s) {
        aim(s);
        static_for<ND>(issue);
        advance();
    }
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int j = 0; j < CB; ++j) acc[i][j] = (v4f){0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < (F16 ? 2 * RB : kTmp); ++t) tmp[t] = (v4f){0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < RB; ++i) sc[NSW - 1][i] = 0.0f;      // the last tile's may be NaN, which no zero product undoes
    };
    clear();
    WUSH_WAIT_VMCNT(0);
    WUSH_LDS_BARRIER();
    __builtin_amdgcn_sched_barrier(0);
    read_s(0);
#pragma unroll
    for (int i = 0; i < RB; ++i) read_a(0, i);
#pragma unroll
    for (int j = 0; j < BR - 1; ++j) read_b(0, j);
    __builtin_amdgcn_sched_barrier(0);

    int buf = 0, st = 0;                         // LDS buffer of stage st
    auto add = [&](int m, const float (&s)[RB]) {
        const int i = m % RB, j = m / RB;
        const v4f& t = tmp[F16 ? (j & 1) * RB + i : m % kTmp];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(t[r], s[i], acc[i][j][r]);
        asm volatile("" : "+v"(acc[i][j]));      // here, and not where the compiler finds its next use
    };
    // the next stage has landed in all wavefronts' view, and all have read this one's columns
    auto next_landed = [&](auto first) {
        WUSH_WAIT_VMCNT((NB - 2) * ND + (first.value ? kStores : 0));
        WUSH_LDS_BARRIER();
        aim(buf);
        __builtin_amdgcn_sched_barrier(0);
    };
    // One stage, whose buffer takes the next one to be issued.  Operands read past the last stage are not used.
    // FIRST: one of a tile's first NB - 1, the loads of whose successors were issued before the last tile's
    // kStores stores (loads and stores complete, for the counter, in the order of their issue).
    auto stage = [&](auto first) {
        const int nbuf = buf + 1 == NB ? 0 : buf + 1;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            old[i] = sc[NSW - 1][i];
#pragma unroll
            for (int h = 0; h < NSW; ++h) sc[h][i] = sx[i] * sw[h];
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
        auto landed = [&] { next_landed(first); };
        auto refill_part = [&](auto qc, auto nc) {               // share q of n
            constexpr int q = qc.value, n = nc.value;
            static_for<(q + 1) * ND / n - q * ND / n>([&](auto dc) { issue(std::integral_constant<int, q * ND / n + dc.value>{}); });
        };
        if constexpr (!F16) {
            static_for<kMf>([&](auto mc) {
                constexpr int m = mc.value, i = m % RB, j = m / RB;
                if constexpr (i == 0 && j == kTurn) landed();
                tmp[m % kTmp] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j % BR], a[i], (v4f){0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                if constexpr (i == 0) {
                    constexpr int jn = j + BR - 1;
                    if constexpr (jn < CB) read_b(buf, jn);
                    else read_b(nbuf, jn - CB);
                }
                if constexpr (j == CB - 1) read_a(nbuf, i);
                if constexpr (m == kMf - 1) read_s(nbuf);
                if constexpr (m >= kLag) add(m - kLag, sc[(m - kLag) / RB * NSW / CB]);
                else add(kMf + m - kLag, old);
                if constexpr (j >= kTurn)
                    refill_part(std::integral_constant<int, m - kTurn * RB>{}, std::integral_constant<int, (BR - 1) * RB>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        } else {
            h8 wa[RB][4], wb[4];
#pragma unroll
            for (int i = 0; i < RB; ++i) fp8_widen(a[i], wa[i]);
            static_for<CB>([&](auto jc) {
                constexpr int j = jc.value, jn = j + BR - 1;
                if constexpr (j == kTurn) {
                    landed();
#pragma unroll
                    for (int i = 0; i < RB; ++i) read_a(nbuf, i);
                    read_s(nbuf);
                }
                fp8_widen(b[j % BR], wb);
                if constexpr (jn < CB) read_b(buf, jn);
                else read_b(nbuf, jn - CB);
                __builtin_amdgcn_sched_barrier(0);
                static_for<4 * RB>([&](auto mc) {
                    constexpr int q = mc.value / RB, i = mc.value % RB, t = (j & 1) * RB + i;
                    tmp[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[q], wa[i][q], q ? tmp[t] : (v4f){0, 0, 0, 0}, 0, 0, 0);
                    if constexpr (q == 1) {
                        if constexpr (j > 0) add((j - 1) * RB + i, sc[(j - 1) * NSW / CB]);
                        else add((CB - 1) * RB + i, old);
                    }
                    if constexpr (j >= kTurn)
                        refill_part(std::integral_constant<int, (j - kTurn) * 4 * RB + mc.value>{},
                                    std::integral_constant<int, (BR - 1) * 4 * RB>{});
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
        }
        asm volatile("" ::: "memory");           // the reads above stay above
        buf = nbuf;
        advance();
    };
    // One stage of a wavefront whose rows are all past the tile's last: its part of the loads only
    auto idle_stage = [&](auto first) {
        next_landed(first);
        static_for<ND>(issue);
        buf = buf + 1 == NB ? 0 : buf + 1;
        advance();
    };
    auto idle_tile = [&] {
        for (st = 0; st < min(NB - 1, KB); ++st) idle_stage(std::true_type{});
        for (; st < KB; ++st) idle_stage(std::false_type{});
        read_s(buf);
#pragma unroll
        for (int i = 0; i < RB; ++i) read_a(buf, i);
#pragma unroll
        for (int j = 0; j < BR - 1; ++j) read_b(buf, j);
        if constexpr (MODE == kAct) {
            WUSH_LDS_BARRIER();
            WUSH_LDS_BARRIER();
        }
        WUSH_WAIT_VMCNT(0);                      // no stores: as below
        __builtin_amdgcn_sched_barrier(0);
    };
    // The tile's outputs.  Rows past M hold what row M - 1 does, and are stored there.
    auto finish = [&] {
#pragma unroll
        for (int m = kMf - (F16 ? RB : kLag); m < kMf; ++m) add(m, sc[NSW - 1]);
        __builtin_amdgcn_sched_barrier(0);
        const int nw = tn * TC + wc * CB * 16;
        const bool full = MODE == kAct || tn * TC + TC <= N;
        if constexpr (MODE == kAct) {
            // h = silu(gate) * up; a row's 128 columns are in WC wavefronts
            uint32_t* part = reinterpret_cast<uint32_t*>(smem + NB * kBuf);
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                uint32_t mx = 0;
#pragma unroll
                for (int j = 0; j < CB / 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float h = fp8_silu(acc[i][j][r]) * acc[i][j + CB / 2][r];
                        acc[i][j][r] = h;
                        mx = max(mx, __float_as_uint(h) & 0x7fffffffu);
                    }
                mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
                mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
                if (kq == 0) part[WC * ((wr * RB + i) * 16 + l16) + wc] = mx;
            }
            WUSH_LDS_BARRIER();
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int row = (wr * RB + i) * 16 + l16, m = min(m0 + row, M - 1);
                uint32_t mx = part[WC * row];
#pragma unroll
                for (int w = 1; w < WC; ++w) mx = max(mx, part[WC * row + w]);
                const float amax = fp8_amax(mx);
                const float factor = fp8_factor(amax);
                if (kq == 0 && wc == 0) g.hs[(size_t)tn * g.ldh + m] = fp8_scale(amax);
                uint32_t c[CB / 2];
#pragma unroll
                for (int j = 0; j < CB / 2; ++j) c[j] = fp8_codes4_by(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], factor);
                uint8_t* out = static_cast<uint8_t*>(g.y) + (size_t)m * I + tn * 128 + wc * kHalf;
                if constexpr (CB == 8) {
                    rows_transpose(c);
                    *reinterpret_cast<uint4*>(out + 16 * kq) = make_uint4(c[0], c[1], c[2], c[3]);
                } else {
                    const auto r = __builtin_amdgcn_permlane16_swap(c[0], c[1], false, false);
                    *reinterpret_cast<uint2*>(out + 16 * (kq & 1) + 8 * (kq >> 1)) = make_uint2(r[0], r[1]);
                }
            }
            WUSH_LDS_BARRIER();                  // part is read before the next tile's is written
        } else if constexpr (MODE == kWide) {
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int m = min(m0 + (wr * RB + i) * 16 + l16, M - 1);
                float* out = static_cast<float*>(g.y) + (size_t)m * N + nw + 4 * kq;
#pragma unroll
                for (int j = 0; j < CB; ++j)
                    if (full || nw + 16 * j < N) *reinterpret_cast<v4f*>(out + 16 * j) = acc[i][j];
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            uint16_t* y = static_cast<uint16_t*>(g.y);
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int m = min(m0 + (wr * RB + i) * 16 + l16, M - 1);
#pragma unroll
                for (int h = 0; h < CB / 4; ++h) {
                    const int n0 = nw + 64 * h;
                    float by = 1.0f;
                    if constexpr (MODE == kShared) {
                        // the power of two that brings the largest finite value of the row's 64 columns to [2^14, 2^15): fp16 keeps
                        // 11 bits of each value down to 2^-28 of that one
                        uint32_t mx = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint32_t u = __float_as_uint(acc[i][4 * h + j][r]) & 0x7fffffffu;
                                mx = max(mx, u < 0x7f800000u && n0 + 16 * j < N ? u : 0u);
                            }
                        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
                        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
                        const int e = max((int)(mx >> 23), 16) - 127 - 14;   // the inverse is a normal number too
                        by = __uint_as_float((uint32_t)(127 - e) << 23);
                        if (kq == 0 && n0 < N) g.hs[(size_t)m * ((N + 63) >> 6) + (n0 >> 6)] = __uint_as_float((uint32_t)(127 + e) << 23);
                    }
                    uint32_t c[2][4];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) c[d][j] = pack2<BF16>(acc[i][4 * h + j][2 * d] * by, acc[i][4 * h + j][2 * d + 1] * by);
                        rows_transpose(c[d]);
                    }
                    const int n = n0 + 16 * kq;
                    uint16_t* out = y + (size_t)m * N + n;
                    if (full || n < N) *reinterpret_cast<uint4*>(out) = make_uint4(c[0][0], c[1][0], c[0][1], c[1][1]);
                    if (full || n + 8 < N) *reinterpret_cast<uint4*>(out + 8) = make_uint4(c[0][2], c[1][2], c[0][3], c[1][3]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!full) WUSH_WAIT_VMCNT(0);           // fewer stores than kStores: the next stages' loads have all landed
        __builtin_amdgcn_sched_barrier(0);
    };

    for (;;) {
        if (m0 + wr * RB * 16 < M) {
            for (st = 0; st < min(NB - 1, KB); ++st) stage(std::true_type{});
            for (; st < KB; ++st) stage(std::false_type{});
            finish();
        } else {
            idle_tile();
        }
        cur += step;
        if (cur >= run_end) break;
        place(cur, tm, tn);
        row_range(tm, m0, M);
        clear();
    }
    WUSH_WAIT_VMCNT(0);                          // no load may reach LDS that is another workgroup's by then
}

template <int RB, bool NT>
int launch(const Fp8Gemm& g, unsigned grid, hipStream_t stream) {
    constexpr int WR = 2, WC = 4, NB = 3, T = 64 * WR * WC;
    if (g.act) gemm_fp8_runs_kernel<RB, WR, WC, NB, kAct, false, true, NT><<<grid, T, 0, stream>>>(g);
    else if (g.tiles && g.shared) gemm_fp8_runs_kernel<RB, WR, WC, NB, kShared, false, false, NT><<<grid, T, 0, stream>>>(g);
    else if (g.tiles) gemm_fp8_runs_kernel<RB, WR, WC, NB, kWide, false, false, NT><<<grid, T, 0, stream>>>(g);
    else if (g.out == WUSH_DTYPE_BF16) gemm_fp8_runs_kernel<RB, WR, WC, NB, kPlain, true, false, NT><<<grid, T, 0, stream>>>(g);
    else gemm_fp8_runs_kernel<RB, WR, WC, NB, kPlain, false, false, NT><<<grid, T, 0, stream>>>(g);
    return (int)hipGetLastError();
}

}  // namespace

int launch_gemm_fp8_runs(const Fp8Gemm& g, int tile_rows, hipStream_t stream) {
    WUSH_REQUIRE((tile_rows == 64 || tile_rows == 128) && g.M > 0 && g.N > 0 && g.N % 8 == 0 && g.K > 0 && g.K % 16 == 0 && ((uintptr_t)g.y & 15u) == 0);
    WUSH_REQUIRE(!g.tiles || (g.ntiles && g.N % 16 == 0 && (g.act || !g.wide)));
    WUSH_REQUIRE(!g.act || (g.tiles && g.N % 256 == 0 && g.row_of && g.hs));
    const long long rows = g.tiles ? g.most_tiles : (g.M + tile_rows - 1) / tile_rows;
    const long long tiles = rows * (g.act ? g.N / 256 : (g.N + 255) / 256);
    WUSH_REQUIRE(tiles <= 0x7fffffffLL);
    const unsigned grid = (unsigned)(tiles < kFp8Workgroups ? tiles : kFp8Workgroups);
    if (tile_rows == 64) return g.once ? launch<2, true>(g, grid, stream) : launch<2, false>(g, grid, stream);
    return g.once ? launch<4, true>(g, grid, stream) : launch<4, false>(g, grid, stream);
}

}  // namespace wush
