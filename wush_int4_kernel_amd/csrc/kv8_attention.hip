// kv8_attention.hip -- attention over the 8-bit paged cache, for few query rows
// a sequence (one new token each, or a handful).
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(cap(scale q . k_t) - max),
//   cap(x) = x, or c tanh(x / c); t from max(pos - window + 1, 0) to pos.
//
// A sequence's rows for one key/value head, (new token, query head of the group)
// in that order, are taken 16 at a time.  A workgroup of four wavefronts walks a
// stretch of the cache in tiles of 64 tokens, each wavefront its own tiles with
// its own running maximum, sum and output, which meet in LDS at the end; stretches of
// one row meet in a second kernel.
//
// The cache is the row operand of both products.  Scores are exact integers: keys enter
// v_mfma_i32_16x16x64_i8 as the codes that they are, against q in 24-bit fixed
// point, three bytes (a power of two puts the row's largest value between 2^22 and 8355711;
// values above 2^-15 of it in bf16 and 2^-12 in fp16 are exact, smaller ones are off by
// at most 2^-23 of the largest: what fp32 sums round to).  Two bytes were off by 2^-15 of
// the largest, and a channel 300 times the others cost these 0.3%.  Converting the keys to fp16 took 160 of about 490 vector
// instructions a tile of 64 tokens, which bind a wavefront as much as the loads do.  The score tile comes out
// with a lane holding 16 consecutive tokens of one row (keys are loaded in the order that
// makes it so), which is the operand that the second product, v_mfma_f32_16x16x32_f16
// on values converted exactly, needs: the probabilities never leave their lanes.
//
// A token's value scale is folded into its exponent: with t = log2(e) s +
// log2(v_scale), weights are exp2(t - base), rounded once to fp16 (11 bits, normal
// down to 2^-26 of the largest), and the sum of the probabilities takes them, unrounded,
// times 1 / v_scale, in fp32.  The base follows the running maximum lazily, 2^12 below it: it
// moves, and the sums are rescaled, only when a weight would pass 2^15.
//
// Bound by HBM where the cache fills the chip (one token behind 131072, 8 heads of 128:
// 268 MB in 57 us with 6 to join, 4.7 TB/s; 64 ragged sequences up to 4096: 344 MB in 66 us,
// the CUs not quite evenly loaded), by a wavefront's instructions and latencies otherwise (3 x 300: 6.1 us).  Two
// tiles' loads in flight instead of one changed nothing; without the non-temporal hint
// 131072 tokens took 2 us more, but 8192-token stretches 20% less, so loads have none.
#include "kv8_attention.h"

namespace wush {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;

__device__ __forceinline__ float quarters_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarters_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The sequence that is taken at place w: by length, the longest first, every second
// round of the CUs the other way round, so that a CU's workgroups together hold about as
// much as another's.  A thread ranks one sequence; keys differ, so ranks do.
// 64 ragged sequences up to 4096 (8 heads of 128) 68 us, as they come 73; 48 of 4000 60, not 69; 100 of
// 2500 with heads of 64 38, not 45; 6% slower at worst of 34 shapes (128 of 1100 with heads of 64).  With
// caches below kLeastSorted tokens, or more sequences than kMostSorted, the ranking costs what it
// gives or more: 64 of 300 11.5 us, as they come 11.3; 256 of 1200 94 and 87.
constexpr int kMostSorted = 128, kLeastSorted = 1024;

__device__ __forceinline__ int by_length(const AttnArgs& a, int w) {
    const Kv8Batch& t = a.batch;
    __shared__ __align__(16) int key[kMostSorted];
    __shared__ int found;
    const int tid = threadIdx.x, mine = tid < t.seqs ? min(max(t.lens[tid], 0), 0x7fffff) << 8 | tid : -1;
    if (tid < kMostSorted) key[tid] = mine;
    __syncthreads();
    const int k = w / a.round, want = k & 1 ? min((k + 1) * a.round, t.seqs) - 1 - w % a.round : w;
    if (mine >= 0) {
        int rank = 0;
        for (int j = 0; j < t.seqs; j += 32)      // behind them: -1, below every key
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const int4 o = *reinterpret_cast<const int4*>(key + j + i);
                rank += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
            }
        if (rank == want) found = tid;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
}

template <int DT, int D, int CAP>
__global__ __launch_bounds__(64 * kWaves) void kv8_rows_kernel(const AttnArgs a) {
    constexpr int NJ = D / 64, NB = D / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, kq = lane >> 4;
    const Kv8Batch& t = a.batch;
    const int lg = a.cache.page_log2, ps = 1 << lg, G = a.group;
    // Stretches slowest: the first ones, which are full, start first, and full and
    // short ones spread over the XCDs (workgroup i runs on XCD i % 8).  With stretches fastest, two
    // a sequence, every other XCD had the full ones: 64 ragged sequences 87 us, not 73.
    const int h = (int)blockIdx.x % a.cache.heads, rest = (int)blockIdx.x / a.cache.heads;
    const int item = rest % a.items, split = rest / a.items;
    int row0;
    int b = item_rows(a, item, row0);
    if (a.round) b = by_length(a, b);
    const Kv8Seq s = kv8_seq(t, b);
    clear_rest(a);
    if (row0 < 0 || row0 >= s.count * G) return;
    const Span span = span_of(a, s, row0);
    const int begin = span.base + split * a.chunk;
    const int end = split == a.splits - 1 ? span.end : min(span.end, begin + a.chunk);
    if (begin >= end && split > 0) return;        // the joining kernel leaves it out too

    // this lane's row
    const int r = min(row0 + l16, s.count * G - 1);
    const int i = r / G, hq = h * G + r % G;
    const int64_t tok = s.first + i;
    const int pos = s.len - s.count + i;
    const int low = a.window > 0 ? pos - a.window + 1 : 0;
    const int last_low = s.len - s.count + min((row0 + 15) / G, s.count - 1) - a.window;   // tokens behind it are in every row's window

    v4i qh[NJ], qm[NJ], ql[NJ];                   // q = 65536 qh + 256 qm + ql, in units of its row
    float c;                                      // scores in powers of two, per unit of key scale
    {
        const uint16_t* p = a.q + tok * a.qt + hq * a.qh + 16 * kq;
        float x[2 * NJ][8], mx = 0.0f;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 2 * NJ; ++j) {
            load8<DT>(p + 64 * (j >> 1) + 8 * (j & 1), x[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                mx = fmaxf(mx, fabsf(x[j][e]));
                bad |= !(fabsf(x[j][e]) < __builtin_inff());
            }
        }
        mx = quarters_max(mx);
        int ex = mx > 0.0f ? 23 - __builtin_amdgcn_frexp_expf(mx) : 0;
        if (__builtin_amdgcn_ldexpf(mx, ex) > 8355711.0f) --ex;   // 127 in each byte
        c = row_factor(__builtin_amdgcn_ldexpf(a.scale * score_unit<CAP>(a), -ex));
        if (quarters_max(bad ? 1.0f : 0.0f) > 0.0f) c = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            uint32_t hi[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = bad ? 0 : (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x[2 * j + (e >> 3)][e & 7], ex));
                const int u = (n + 128) >> 8, w = (u + 128) >> 8;                // digits of -128 to 127
                hi[e >> 2] |= ((uint32_t)w & 0xffu) << (8 * (e & 3));
                mid[e >> 2] |= ((uint32_t)(u - 256 * w) & 0xffu) << (8 * (e & 3));
                lo[e >> 2] |= ((uint32_t)(n - 256 * u) & 0xffu) << (8 * (e & 3));
            }
            qh[j] = (v4i){(int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
            qm[j] = (v4i){(int)mid[0], (int)mid[1], (int)mid[2], (int)mid[3]};
            ql[j] = (v4i){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3]};
        }
    }

    const v4f zero = {0, 0, 0, 0};
    v4f acc[NB];
#pragma unroll
    for (int d = 0; d < NB; ++d) acc[d] = zero;
    float m = kLow, l = 0.0f;                     // the weights' base, their sum
    const int64_t tile_bytes = (int64_t)D << lg;
    const int32_t* table = t.table + (int64_t)b * t.table_stride;
    constexpr int kStep = kWaves * kTile;

    // The pages of the keys that this lane loads (four 16-token groups, one of
    // them by l16) and of the 16 tokens whose scores it holds (by kq); -1: none.
    auto page_of = [&](int tk) {
        const int id = table[min(tk, end - 1) >> lg];
        return tk < end && (uint32_t)id < (uint64_t)a.cache.pages ? id : -1;
    };
    const int ok = 16 * (l16 >> 2), ov = 16 * kq;
    v4i kk[4][NJ];
    uint4 vv[NB];
    float ks, vs;
    auto load_keys = [&](int t0, int idk, int idv) {
        const int8_t* pk = a.cache.k + ((int64_t)max(idk, 0) * a.cache.heads + h) * tile_bytes +
                           (((t0 + ok) & (ps - 1)) + (l16 & 3)) * D + 16 * kq;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < NJ; ++j) kk[n][j] = *reinterpret_cast<const v4i*>(pk + 4 * n * D + 64 * j);
        const int64_t vt = (int64_t)max(idv, 0) * a.cache.heads + h;
        ks = a.cache.ks[vt];
        vs = a.cache.vs[vt];
    };
    auto load_values = [&](int t0, int idv) {
        const int8_t* pv = a.cache.v + ((int64_t)max(idv, 0) * a.cache.heads + h) * tile_bytes + (l16 << lg) + ((t0 + ov) & (ps - 1));
#pragma unroll
        for (int d = 0; d < NB; ++d) vv[d] = *reinterpret_cast<const uint4*>(pv + ((int64_t)d << (lg + 4)));
    };

    // One tile.  A tile's keys go out while the last tile's weights are made, its
    // values behind the last tile's products: the registers that held those take
    // them.  Behind the end nothing goes out.
    auto tile = [&](int t0, int idv, bool masked, auto&& keys_ahead, auto&& values_ahead) {
        v4i sh[4], sm[4], sl[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) sh[n] = sm[n] = sl[n] = (v4i){0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                sh[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[n][j], qh[j], sh[n], 0, 0, 0);
                sm[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[n][j], qm[j], sm[n], 0, 0, 0);
                sl[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[n][j], ql[j], sl[n], 0, 0, 0);
            }
        // the lane's 16 tokens, of one page
        const float cs = kept_finite(c * ks);
        const float fv = vs < kValueFloor ? kValueFloor : vs;
        const float lv = __builtin_amdgcn_logf(fv);
        __builtin_amdgcn_sched_barrier(0);
        keys_ahead();
        __builtin_amdgcn_sched_barrier(0);
        v4f sc[4];
        const int tv = t0 + ov, last = idv >= 0 ? min(pos, end - 1) : -1;
        float top = kLow;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_fmaf((float)(256 * sh[n][e] + sm[n][e]), 256.0f, (float)sl[n][e]);
                sc[n][e] = capped<CAP>(a, x * cs) + lv;
            }
        if (masked) {
            asm volatile("" : "+v"(top));         // a branch: not computed for every tile
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = tv + 4 * n + e;
                    sc[n][e] = at <= last && at >= low ? sc[n][e] : -__builtin_inff();
                }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[n][e]);
        top = quarters_max(top);
        if (__any(top - m > kMostWeight)) {
            const float mn = fmaxf(m, base_of(top)), fade = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= fade;
#pragma unroll
            for (int d = 0; d < NB; ++d) acc[d] *= fade;
        }
        float sum = 0.0f;
        h8 p[2];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = __builtin_amdgcn_exp2f(sc[n][e] - m);
                sum += w;
                p[n >> 1][4 * (n & 1) + e] = (_Float16)w;
            }
        l += sum != 0.0f ? sum * __builtin_amdgcn_rcpf(fv) : 0.0f;    // a scale may be NaN where nothing is seen
#pragma unroll
        for (int d = 0; d < NB; ++d) {
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vv[d].x, vv[d].y), p[0], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vv[d].z, vv[d].w), p[1], acc[d], 0, 0, 0);
            if (d & 1) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        values_ahead();
    };

    int t0 = begin + wave * kTile;
    if (t0 < end) {
        int idk = page_of(t0 + ok), idv = page_of(t0 + ov);
        load_keys(t0, idk, idv);
        load_values(t0, idv);
        int nk = page_of(t0 + kStep + ok), nv = page_of(t0 + kStep + ov);
        const int least = s.len - s.count + row0 / G;             // the smallest position of these rows
        for (; t0 + kStep < end; t0 += kStep) {
            const int nnk = page_of(t0 + 2 * kStep + ok), nnv = page_of(t0 + 2 * kStep + ov);
            const auto keys = [&] { load_keys(t0 + kStep, nk, nv); };
            const auto values = [&] { load_values(t0 + kStep, nv); };
            const bool inside = t0 + kTile - 1 <= least && (a.window == 0 || t0 > last_low) && __all(idv >= 0);
            tile(t0, idv, !inside, keys, values);
            idv = nv;
            nk = nnk;
            nv = nnv;
        }
        tile(t0, idv, true, [] {}, [] {});
    }

    // join the wavefronts: a lane holds channels 16 d + 4 kq + e of row l16
    __shared__ float so[kWaves][16][D + 4];
    __shared__ float sm[kWaves][16], ssum[kWaves][16];
    l = quarters_sum(l);
    if (kq == 0) {
        sm[wave][l16] = m;
        ssum[wave][l16] = l;
    }
#pragma unroll
    for (int d = 0; d < NB; ++d) *reinterpret_cast<v4f*>(&so[wave][l16][16 * d + 4 * kq]) = acc[d];
    __syncthreads();
    constexpr int PD = D / 16;                    // channels a thread
    const int jr = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PD;
    if (row0 + jr >= s.count * G) return;
    float mm = kLow, ll = 0.0f, o[PD];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, sm[w][jr]);
#pragma unroll
    for (int e = 0; e < PD; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][jr] - mm);
        ll += ssum[w][jr] * f;
#pragma unroll
        for (int e = 0; e < PD; ++e) o[e] += so[w][jr][d0 + e] * f;
    }
    const int rr = row0 + jr;
    const int64_t row = (int64_t)(s.first + rr / G) * a.cache.heads * G + h * G + rr % G;
    if (a.splits == 1) {
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;      // no token seen: zeros
#pragma unroll
        for (int e = 0; e < PD; e += 2)
            *reinterpret_cast<uint32_t*>(a.out + row * D + d0 + e) = out16<DT>(o[e] * inv) | out16<DT>(o[e + 1] * inv) << 16;
        return;
    }
    float* part = a.part + (row * a.splits + split) * (D + kPartExtra);
#pragma unroll
    for (int e = 0; e < PD; ++e) part[d0 + e] = o[e];
    if (d0 == 0) {
        part[D] = mm;
        part[D + 1] = ll;
    }
}

// The stretches that hold tokens of a (token, query head), joined: by one
// wavefront, or, where there are more than kFewSplits, by a workgroup's four, which
// take every fourth stretch.  Four stretches at a time, so that their loads overlap.
// With 32 stretches a wavefront took 5 us more than a workgroup (decode of 1 x 131072), with 16
// up to 3, with 2 to 8 they are equal within 1; with many rows of few stretches a workgroup a row is
// slow (five chunks of 700 tokens 133 us, not 87).
constexpr int kFewSplits = 16;

template <int DT, int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Kv8Batch& t = a.batch;
    const int heads = a.cache.heads * a.group;
    const bool few = a.splits <= kFewSplits;
    const int64_t row = few ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    const int first = few ? 0 : wave, by = few ? 1 : 4;
    const int tok = (int)(row / heads);
    bool mine = tok < t.tokens;
    int n = 0;
    if (mine) {
        const int b = t.cu ? kv8_find(t, tok, 1, 0, 0) : tok;
        const Kv8Seq s = kv8_seq(t, b);
        const int i = tok - s.first;
        mine = i >= 0 && i < s.count;
        if (mine) {
            const Span span = span_of(a, s, (i * a.group + (int)(row % a.group)) & ~(a.tile_rows - 1));
            n = min(a.splits, max((span.end - span.base + a.chunk - 1) / a.chunk, 1));
        }
    }
    constexpr int PD = D / 64;
    typedef float vpd __attribute__((ext_vector_type(PD)));
    const float* part = a.part + row * a.splits * (D + kPartExtra);
    float mm = kLow;
    for (int k = lane; k < n; k += 64) mm = fmaxf(mm, part[(int64_t)k * (D + kPartExtra) + D]);
#pragma unroll
    for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    float ll = 0.0f;
    vpd o = 0.0f;
    for (int k0 = first; k0 < n; k0 += 4 * by) {
        vpd v[4];
        float f[4], w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* p = part + (int64_t)min(k0 + by * u, n - 1) * (D + kPartExtra);
            v[u] = *reinterpret_cast<const vpd*>(p + lane * PD);
            f[u] = p[D];
            w[u] = p[D + 1];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (k0 + by * u < n) {
                const float g = __builtin_amdgcn_exp2f(f[u] - mm);
                ll += w[u] * g;
                o += v[u] * g;
            }
    }
    if (!few) {
        __shared__ vpd so[4][64];
        __shared__ float sl[4];
        so[wave][lane] = o;
        if (lane == 0) sl[wave] = ll;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            o += so[w][lane];
            ll += sl[w];
        }
    }
    if (!mine) return;
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    uint16_t* out = a.out + row * D + lane * PD;
    if constexpr (PD == 2) *reinterpret_cast<uint32_t*>(out) = out16<DT>(o[0] * inv) | out16<DT>(o[1] * inv) << 16;
    else *out = (uint16_t)out16<DT>(o[0] * inv);
}

// A window of the longest sequence or more hides nothing; a shorter one, added to or taken
// from a position, stays in 32 bits.
int window_of(int64_t window) { return window >= WUSH_KV8_MAX_LENGTH ? 0 : (int)window; }

struct Plan {
    int tile_rows, splits, chunk;
    int64_t items;
    int round;                                    // AttnArgs::round
};

// For each tile height, 16 (kv8_rows_kernel), 128 and 256 (kv8_chunk.hip), the
// stretches of the cache per item with the least estimated time: a
// workgroup's pass over `step` tokens (`split` alone on its CU, `more` for each where several
// share it: the loads of one cover the latencies of another), `ends` passes' worth for its beginning
// and end, and where there is more than one stretch the joining.  `more` below `split`
// (16 rows only; for tall tiles `pass` below `alone` says the same, and their stretches have not been
// chosen by it) halves the stretches of long caches: 8 ragged sequences up to 32768 79 us, not 91 (8 heads of
// 128; of 64 48, not 61), 16 up to 8192 46, not 51, one of 131072 58 to 59 in both; over 104 shapes of decode and few new
// tokens 2.4% faster on average, 28% at best, 5% slower at worst (5 of 12000, page of 16); without `ends`
// 12 of 3000 took 18.0 us, not 15.1.  Of the three, the height with the least time: a
// start, and passes that take `alone` where a CU has one workgroup and `pass` for each where it has
// more.  Those constants are fitted to 72 shapes, 1 and 16 sequences of 1024 and 8192 with 41 to 1024 rows of
// new tokens, none with a cap: 1% slower than the fastest height on average, 19% at worst.  The estimates rank heights
// and are no times: neither what causality leaves out nor a cap's exponentials are in them (1 x 8192 new tokens 1092,
// measured 540; 5 x 700 with window and cap 21, measured 56).  16 rows below
// a fixed number of rows a sequence, tall ones above, was 15% slower on average and 98% at
// worst (16 sequences of 8192 with 32 heads of 64 and 170 new tokens: 467 us, now 267).
Plan plan_of(const Kv8Cache& c, int64_t seqs, int64_t tokens, bool ragged, int group, int64_t table_stride, int window,
             int64_t max_len) {
    static const struct { int rows, step; double split, more, ends, start, alone, pass; } kHeights[] = {
        {16, 256, 2.1, 1.65, 1.0, 0.5, 2.2, 1.65}, {128, kTile, 1.5, 1.5, 0.0, 3.0, 1.7, 1.2}, {256, kTile, 1.5, 1.5, 0.0, 8.0, 2.1, 2.1}};
    const int64_t rows = tokens * group;
    const double joined = 0.02 + (double)rows * c.heads * (c.dim + kPartExtra) * 8 / 4e6;   // a stretch's sums both ways
    Plan best = {16, 1, 1, 0, 0};
    double least = 1e30;
    for (const auto& t : kHeights) {
        const int64_t items = ragged ? rows / t.rows + seqs : seqs * ((group + t.rows - 1) / t.rows);
        int64_t range = table_stride << c.page_log2;
        if (max_len > 0 && max_len < range) range = max_len;
        if (window > 0 && window + 64 + t.rows / group < range) range = window + 64 + t.rows / group;
        if (range < 1) range = 1;
        if (range > WUSH_KV8_MAX_LENGTH) range = WUSH_KV8_MAX_LENGTH;
        const int64_t most = (range + t.step - 1) / t.step;
        double fewest = 1e30;
        int64_t splits = 1;
        for (int64_t n = 1; n <= most && n <= 256 && (n == 1 || items * c.heads * n <= 1024); n += n < 16 ? 1 : n / 16) {
            const int64_t deep = (items * c.heads * n + 255) / 256;          // workgroups of a CU
            const double us = (deep > 1 ? t.more * (double)deep : t.split) * c.dim / 128 * ((double)((most + n - 1) / n) + t.ends) +
                              (n > 1 ? 3.0 + joined * (double)n : 0.0);
            if (us < fewest) {
                fewest = us;
                splits = n;
            }
        }
        const double shared = t.pass * (double)(items * c.heads * splits) / 256;
        const double us = t.start + (0.15 + 0.85 * c.dim / 128) * (double)((most + splits - 1) / splits) * (shared > t.alone ? shared : t.alone) +
                          (splits > 1 ? 3.0 + joined * (double)splits : 0.0);
        if (us < least) {
            least = us;
            const int chunk = (int)((most + splits - 1) / splits * t.step);
            best = {t.rows, (int)((range + chunk - 1) / chunk), chunk, items, 0};
        }
    }
    // Sorted by length where a stretch has more workgroups than the chip CUs, and the cache is long enough.
    int64_t range = table_stride << c.page_log2;
    if (max_len > 0 && max_len < range) range = max_len;
    if (window > 0 && window < range) range = window;
    const int64_t wide = (int64_t)c.heads * ((group + 15) / 16);                // workgroups of a sequence
    if (best.tile_rows == 16 && !ragged && seqs <= kMostSorted && wide * seqs > 256 && range >= kLeastSorted)
        best.round = wide < 256 ? (int)(256 / wide) : 1;
    return best;
}

template <int DT, int D>
void launch_rows(const AttnArgs& a, unsigned grid, hipStream_t stream) {
    if (a.cap > kMostPlainCap) kv8_rows_kernel<DT, D, kWideCap><<<grid, 64 * kWaves, 0, stream>>>(a);
    else if (a.cap > 0.0f) kv8_rows_kernel<DT, D, kCap><<<grid, 64 * kWaves, 0, stream>>>(a);
    else kv8_rows_kernel<DT, D, kNoCap><<<grid, 64 * kWaves, 0, stream>>>(a);
}

template <int DT>
int launch(const AttnArgs& a, hipStream_t stream) {
    const int64_t blocks = (int64_t)a.items * a.cache.heads * a.splits;
    const int64_t rows = (int64_t)a.batch.tokens * a.cache.heads * a.group;
    WUSH_REQUIRE(blocks <= 0x7fffffffLL && rows <= 0x7fffffffLL);
    if (a.tile_rows > 16) {
        const int st = launch_kv8_chunk(a, DT, stream);
        if (st) return st;
    }
    const dim3 join((unsigned)(a.splits <= kFewSplits ? (rows + 3) / 4 : rows));
    if (a.cache.dim == 64) {
        if (a.tile_rows == 16) launch_rows<DT, 64>(a, (unsigned)blocks, stream);
        if (a.splits > 1) kv8_join_kernel<DT, 64><<<join, 256, 0, stream>>>(a);
    } else {
        if (a.tile_rows == 16) launch_rows<DT, 128>(a, (unsigned)blocks, stream);
        if (a.splits > 1) kv8_join_kernel<DT, 128><<<join, 256, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace wush

extern "C" {

static bool kv8_plan(const wush_kv8_cache* cache, int64_t seqs, int64_t tokens, int ragged, int64_t q_heads,
                     int64_t table_stride, int64_t window, int64_t max_len, wush::Kv8Cache* c, wush::Plan* p) {
    if (wush::kv8_cache_of(cache, c) || seqs <= 0 || tokens <= 0 || q_heads <= 0 || q_heads % c->heads) return false;
    *p = wush::plan_of(*c, seqs, tokens, ragged != 0, (int)(q_heads / c->heads), table_stride,
                       wush::window_of(window < 0 ? 0 : window), max_len);
    return true;
}

size_t wush_kv8_attention_workspace_bytes(const wush_kv8_cache* cache, int64_t seqs, int64_t tokens, int ragged,
                                          int64_t q_heads, int64_t table_stride, int64_t window, int64_t max_len) {
    wush::Kv8Cache c;
    wush::Plan p;
    if (!kv8_plan(cache, seqs, tokens, ragged, q_heads, table_stride, window, max_len, &c, &p)) return 0;
    return p.splits > 1 ? (size_t)tokens * q_heads * p.splits * (c.dim + wush::kPartExtra) * 4 : 0;
}

int wush_kv8_attention_plan(const wush_kv8_cache* cache, int64_t seqs, int64_t tokens, int ragged, int64_t q_heads,
                            int64_t table_stride, int64_t window, int64_t max_len, int32_t plan[4]) {
    wush::Kv8Cache c;
    wush::Plan p;
    WUSH_REQUIRE(plan && table_stride >= 0 && window >= 0 && max_len >= 0);
    WUSH_REQUIRE(kv8_plan(cache, seqs, tokens, ragged, q_heads, table_stride, window, max_len, &c, &p));
    plan[0] = p.tile_rows;
    plan[1] = p.splits;
    plan[2] = p.chunk;
    plan[3] = p.round;
    return (int)hipSuccess;
}

int wush_kv8_attention(const void* q, int dtype, int64_t q_token_stride, int64_t q_head_stride,
                       const wush_kv8_cache* cache, const int32_t* block_table, int64_t table_stride,
                       const int32_t* seq_lens, const int32_t* cu_q, int64_t seqs, int64_t tokens, int64_t q_heads,
                       float scale, int64_t window, float softcap, int64_t max_len, void* out, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    wush::AttnArgs a;
    const int st = wush::kv8_cache_of(cache, &a.cache);
    if (st) return st;
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    WUSH_REQUIRE(seqs >= 0 && tokens >= 0 && table_stride >= 0 && window >= 0 && max_len >= 0);
    WUSH_REQUIRE(q_heads > 0 && q_heads % a.cache.heads == 0 && q_heads <= 65535);
    WUSH_REQUIRE(scale - scale == 0.0f && softcap >= 0.0f && softcap < __builtin_inff());
    if (seqs == 0 || tokens == 0) return (int)hipSuccess;
    WUSH_REQUIRE(q && out && (block_table || table_stride == 0) && seq_lens && (cu_q || seqs == tokens));
    WUSH_REQUIRE(seqs <= 0x3fffffffLL && tokens <= 0x3fffffffLL);
    WUSH_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15u) == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0);
    const size_t need = wush_kv8_attention_workspace_bytes(cache, seqs, tokens, cu_q != nullptr, q_heads, table_stride,
                                                           window, max_len);
    WUSH_REQUIRE(need <= workspace_bytes && (need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0)));
    a.q = static_cast<const uint16_t*>(q);
    a.qt = q_token_stride;
    a.qh = q_head_stride;
    a.batch = {block_table, seq_lens, cu_q, table_stride, (int)seqs, (int)tokens};
    a.group = (int)(q_heads / a.cache.heads);
    a.window = wush::window_of(window);
    const wush::Plan p = wush::plan_of(a.cache, seqs, tokens, cu_q != nullptr, a.group, table_stride, a.window, max_len);
    WUSH_REQUIRE(p.items <= 0x7fffffffLL);
    a.tile_rows = p.tile_rows;
    a.tile_shift = __builtin_ctz(p.tile_rows);
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.items = (int)p.items;
    a.round = p.round;
    a.scale = scale;
    a.cap = softcap;
    a.out = static_cast<uint16_t*>(out);
    a.part = static_cast<float*>(workspace);
    return dtype == WUSH_DTYPE_BF16 ? wush::launch<WUSH_DTYPE_BF16>(a, stream) : wush::launch<WUSH_DTYPE_F16>(a, stream);
}

}  // extern "C"
