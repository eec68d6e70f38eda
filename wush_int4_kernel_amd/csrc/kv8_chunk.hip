// kv8_chunk.hip -- attention over the 8-bit paged cache for many query rows a
// sequence (prefill, chunks of it).  The formulas are kv8_attention.hip's.
//
// A workgroup of NW wavefronts takes 32 NW rows, (new token, query head of the
// group), of one sequence and key/value head, and walks the cache in tiles of 64
// tokens: codes are loaded, converted to fp16 (exact) once for all rows and put into
// LDS in operand order.  A wavefront keeps its 32 rows of q in registers and runs both products
// on v_mfma_f32_32x32x16_f16 with the cache as row operand: a lane holds one row's scores,
// which are, in the order that the values are put down in, its operand of the second product.
//
// Wavefronts alternate between a matrix phase, the second product of tile t - 1
// and the first of tile t with the staging of a share of the next tiles among them, and a vector
// phase, tile t's weights.  The workgroup's second half runs one phase behind the first, with a
// barrier between phases: of a SIMD's two wavefronts one feeds the matrix cores while the
// other computes.
//
// The base of the weights exp2(t - base), 2^12 below the running maximum, follows it lazily: it
// moves, and the sums are rescaled, only when a weight would pass 2^15; weights are
// rounded once to fp16 (11 bits, normal down to 2^-26 of the largest) for the product;
// their sum takes them unrounded (pages whose values are far smaller than others' have
// weights below fp16's range, and count in it all the same).
//
// 8192 new tokens, 32 query and 8 key/value heads of 128: 540-570 us, 1.0 PFLOP/s (a large
// fp16 matrix product reaches 1.43 on this card).  The matrix cores are busy for 47% of the
// time and the vector units for 60%, neither in full: a tile has 32 MFMAs and about 260 vector instructions a wavefront (32 of
// them exponentials, 80 between the MFMAs), and the halves wait for each other at the barriers.  All wavefronts in step took 613 us, no higher
// priority for the matrix phase 16% more, loads in the vector phase 5%.
#include "kv8_attention.h"

namespace wush {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kFar = 0x1p12f;                   // a base up to it is off by 2^-12 at most

template <int DT, int D, int NW, int CAP>
__global__ __launch_bounds__(64 * NW, 2) void kv8_chunk_kernel(const AttnArgs a) {
    constexpr int kThreads = 64 * NW;
    constexpr int NS = D / 16, NB = D / 32;       // steps of the first product, channel blocks of the second
    constexpr int kOp = kTile * D * 2;            // bytes of one operand's tile
    constexpr int kCodes = kTile * D / 16, kLoads = 2 * kCodes / kThreads;   // 16-byte chunks of one tensor's tile; a thread's of both
    __shared__ __align__(16) uint8_t smem[4 * kOp > NW * 32 * D * 2 ? 4 * kOp : NW * 32 * D * 2];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hf = lane >> 5;
    const Kv8Batch& t = a.batch;
    const int lg = a.cache.page_log2, ps = 1 << lg, G = a.group;
    // heads fastest (an XCD, every eighth workgroup, then keeps to few heads), the
    // last rows, which see the most, first
    const int h = (int)blockIdx.x % a.cache.heads, w = (int)blockIdx.x / a.cache.heads;
    const int split = w % a.splits, item = a.items - 1 - w / a.splits;
    int row0;
    const int b = item_rows(a, item, row0);
    const Kv8Seq s = kv8_seq(t, b);
    clear_rest(a);
    if (row0 < 0 || row0 >= s.count * G) return;
    const Span span = span_of(a, s, row0);
    const int begin = span.base + split * a.chunk;
    const int end = split == a.splits - 1 ? span.end : min(span.end, begin + a.chunk);
    if (begin >= end && split > 0) return;        // the joining kernel leaves it out too

    // this lane's row, and its wavefront's range of positions
    const int rows = s.count * G, wrow = row0 + 32 * wave;
    const int r = min(wrow + l32, rows - 1);
    const int before = s.len - s.count, pos = before + r / G;
    const int low = a.window > 0 ? pos - a.window + 1 : 0;
    const int pos0 = before + min(wrow, rows - 1) / G, pos1 = before + min(wrow + 31, rows - 1) / G;
    const int64_t tok = s.first + r / G;
    const int hq = h * G + r % G;

    h8 q[NS];
    float c;                                      // scores in powers of two, per unit of key scale; not negative
    bool bad = false;                             // a value is not finite: scores of 0, and NaN for what sees a token
    {
        const uint16_t* p = a.q + tok * a.qt + hq * a.qh + 8 * hf;
        float mx = 0.0f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            float x[8];
            load8<DT>(p + 16 * j, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                mx = fmaxf(mx, fabsf(x[e]));
                bad |= !(fabsf(x[e]) < __builtin_inff());
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        bad |= __shfl_xor((int)bad, 32) != 0;
        const int ex = mx > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
        c = row_factor(__builtin_amdgcn_ldexpf(fabsf(a.scale) * score_unit<CAP>(a), -ex));
        if (bad) c = 0.0f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            float x[8];
            load8<DT>(p + 16 * j, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) q[j][e] = bad ? (_Float16)0.0f : (_Float16)__builtin_amdgcn_ldexpf(a.scale < 0.0f ? -x[e] : x[e], ex);
        }
    }

    // The stretch's pages: a wavefront holds 128 of them, two a lane, from entry e0 of
    // the table on: tile numbers (page, this head), and the tiles' key scale and log2 and
    // reciprocal of the value scale.  The second 64 are loaded when the first are
    // used up, long before they are needed.  Where there is no page the log2 is
    // -inf (weights of zero); a NaN scale leaves the reciprocal 0 (the weights are NaN already).
    struct Pages {
        int tile;
        float ks, lv, rv;
    };
    const int32_t* table = t.table + (int64_t)b * t.table_stride;
    const int entries = end > 0 ? (end - 1 >> lg) + 1 : 0;
    auto entry = [&](int e) __attribute__((always_inline)) {
        const int id = table[min(e, max(entries - 1, 0))];
        const bool has = e < entries && id >= 0 && id < a.cache.pages;
        Pages r;
        r.tile = has ? id * a.cache.heads + h : 0;
        const float ks = a.cache.ks[r.tile];
        float vs = a.cache.vs[r.tile];
        r.ks = has ? ks : 0.0f;
        if (vs < kValueFloor) vs = kValueFloor;
        r.lv = has ? __builtin_amdgcn_logf(vs) : -__builtin_inff();
        r.rv = has && vs == vs ? 1.0f / vs : 0.0f;
        return r;
    };
    int e0 = begin >> lg;
    Pages page0 = {}, page1 = {};
    if (begin < end) {
        page0 = entry(e0 + lane);
        page1 = entry(e0 + 64 + lane);
    }
    auto pages_from = [&](int e) __attribute__((always_inline)) {                // the entries below e are done with
        if (e < e0 + 64) return;
        e0 += 64;
        page0 = page1;
        page1 = entry(e0 + 64 + lane);
    };
    // of token tk, the same in all lanes (a tile's entries lie in one of the halves)
    auto tile_at = [&](int tk) __attribute__((always_inline)) {
        const int e = (tk >> lg) - e0;
        return __builtin_amdgcn_readlane(e < 64 ? page0.tile : page1.tile, e & 63);
    };
    // Staging.  Chunks of 16 codes, kCodes of the keys' tile, by token (D / 16
    // each), and kCodes of the values', by channel inside a page's part of the tile (cpp
    // each), as they lie in memory: a wavefront's lie in one page.
    const int cpp = min(ps, kTile) >> 4, cpl = __builtin_ctz(cpp);
    uint4 raw[kLoads];
    uint32_t voff[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int n = (i * kThreads + tid) & (kCodes - 1);
        voff[i] = ((n >> cpl & (D - 1)) << lg) + 16 * (n & (cpp - 1));
    }
    auto of_keys = [&](int i) { return kThreads <= kCodes ? i * kThreads < kCodes : 64 * wave < kCodes; };
    const int tile_log2 = lg + __builtin_ctz(D);
    auto tile_of = [&](const int8_t* p, int n) { return p + ((uint64_t)(uint32_t)n << tile_log2); };
    // the thread's share of the keys of the tile at tk0 and of the values of the one at tv0
    auto load = [&](int tk0, int tv0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n0 = (i * kThreads + 64 * wave) & (kCodes - 1);            // the wavefront's first chunk
            if (of_keys(i)) {
                const int tk = tk0 + n0 / (D / 16);
                raw[i] = *reinterpret_cast<const uint4*>(tile_of(a.cache.k, tile_at(tk)) + (tk & (ps - 1)) * D + 16 * lane);
            } else {
                const int tv = tv0 + 16 * cpp * (n0 / D >> cpl);
                raw[i] = *reinterpret_cast<const uint4*>(tile_of(a.cache.v, tile_at(tv)) + (tv & (ps - 1)) + voff[i]);
            }
        }
    };
    // LDS: operand fragments of 1 KiB, lane l's 16 bytes in slot l, the slots' low
    // bits mixed with the fragment's number so that the stores spread over the banks
    // Piece k of a thread's staging, 8 codes converted and stored: 2 kLoads pieces.
    auto put = [&](int k, int kbuf, int vbuf) __attribute__((always_inline)) {
        const int i = k >> 1, n = (i * kThreads + tid) & (kCodes - 1);
        if (of_keys(i)) {
            const int tk = n / (D / 16), st = n % (D / 16);
            uint8_t* f = smem + kbuf * kOp + ((tk >> 5) * NS + st) * 1024 + 16 * ((tk & 31) ^ (st & 7));
            if (k & 1) *reinterpret_cast<h8*>(f + 512) = codes8(raw[i].z, raw[i].w);
            else *reinterpret_cast<h8*>(f) = codes8(raw[i].x, raw[i].y);
        } else {
            const int d = n >> cpl & (D - 1), ts = (n / D >> cpl) * cpp + (n & (cpp - 1));
            uint8_t* g = smem + (2 + vbuf) * kOp + ((d >> 5) * 4 + ts) * 1024 + 16 * ((d & 31) ^ ((ts & 1) << 2 | (ts & 2)));
            if (k & 1) *reinterpret_cast<h8*>(g + 512) = codes8(raw[i].y, raw[i].w);     // tokens 4-7, 12-15 of 16
            else *reinterpret_cast<h8*>(g) = codes8(raw[i].x, raw[i].z);                 // 0-3, 8-11
        }
    };
    v16f o[NB], sc[2];
    h8 p[4];
#pragma unroll
    for (int d = 0; d < NB; ++d) o[d] = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) p[g] = (_Float16)0.0f;
    float m = kLow, l = 0.0f;                     // the weights' base, their sum
    // The matrix phase: the second product of a tile and (QK) the first of the next,
    // their operands read kAhead fragments ahead of the MFMAs, and the staging: keys
    // into the buffer that kbuf is not, values into the one that kbuf is.
    constexpr int kAhead = 6, kFrags = 2 * NS;                    // 4 NB = 2 NS fragments each
    auto matrix = [&](auto qk, auto kbufc) __attribute__((always_inline)) {
        constexpr int kbuf = kbufc.value, vbuf = kbuf ^ 1;        // known, so that addresses are
        const uint8_t* vb = smem + (2 + vbuf) * kOp + 512 * hf;
        const uint8_t* kb = smem + kbuf * kOp + 512 * hf;
        constexpr int kTotal = qk.value ? 2 * kFrags : kFrags;
        h8 f[kAhead];
        auto read = [&](auto ic) __attribute__((always_inline)) {
            constexpr int i = ic.value;
            if constexpr (i < kFrags) {
                constexpr int g = i / NB, d = i % NB;
                f[ic.value % kAhead] = *reinterpret_cast<const h8*>(vb + (d * 4 + g) * 1024 + 16 * (l32 ^ ((g & 1) << 2 | (g & 2))));
            } else {
                constexpr int st = (i - kFrags) / 2, tb = i & 1;
                f[ic.value % kAhead] = *reinterpret_cast<const h8*>(kb + (tb * NS + st) * 1024 + 16 * (l32 ^ (st & 7)));
            }
        };
        static_for<kAhead>([&](auto ic) { read(ic); });
        if constexpr (qk.value) {
            sc[0] = 0.0f;
            sc[1] = 0.0f;
        }
        __builtin_amdgcn_sched_barrier(0);
        static_for<kTotal>([&](auto ic) {
            constexpr int i = ic.value;
            const h8 x = f[ic.value % kAhead];
            if constexpr (i < kFrags) o[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p[i / NB], o[i % NB], 0, 0, 0);
            else sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[(i - kFrags) / 2], sc[i & 1], 0, 0, 0);
            if constexpr (ic.value + kAhead < kTotal) read(std::integral_constant<int, ic.value + kAhead>{});
            // a piece of the staging behind every few MFMAs
            constexpr int kEvery = 2 * kFrags / (2 * kLoads + 1);
            if constexpr (qk.value && ic.value % kEvery == kEvery - 1 && ic.value / kEvery < 2 * kLoads)
                put(ic.value / kEvery, kbuf ^ 1, vbuf ^ 1);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // scores of the tile at t0 -> weights.  Register 8 g + e: token 16 g + 8 (e / 4) + 4 hf + e % 4.
    auto weights = [&](int t0) __attribute__((always_inline)) {
        float cg[4], lv[4], rv[4];
        {
            const int e = (t0 >> lg) - e0;
            const bool half = e < 64;
            const float ks = half ? page0.ks : page1.ks, ls = half ? page0.lv : page1.lv, rs = half ? page0.rv : page1.rv;
            auto of = [&](float v, int at) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), at)); };
            cg[0] = kept_finite(c * of(ks, e & 63));
            lv[0] = of(ls, e & 63);
            rv[0] = of(rs, e & 63);
#pragma unroll
            for (int g = 1; g < 4; ++g) {
                cg[g] = cg[0];
                lv[g] = lv[0];
                rv[g] = rv[0];
            }
            if (lg < 6) {                         // several pages a tile
#pragma unroll
                for (int g = 1; g < 4; ++g) {
                    const int at = (e & 63) + (16 * g >> lg);
                    cg[g] = kept_finite(c * of(ks, at));
                    lv[g] = of(ls, at);
                    rv[g] = of(rs, at);
                }
            }
        }
        const bool edge = t0 + kTile - 1 > pos0 || (a.window > 0 && t0 < pos1 - a.window + 1);
        if (CAP || edge) {                        // to final scores first, then the mask
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = capped<CAP>(a, sc[g >> 1][8 * (g & 1) + e] * cg[g]) + lv[g];
                    const int at = t0 + 16 * g + 8 * (e >> 2) + 4 * hf + (e & 3);
                    if (edge) x = at <= pos && at >= low ? x : -__builtin_inff();
                    sc[g >> 1][8 * (g & 1) + e] = x;
                }
                cg[g] = 1.0f;
                lv[g] = 0.0f;
            }
        }
        float top = kLow;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const v16f& x = sc[g >> 1];
            const int k = 8 * (g & 1);
            const float u = fmaxf(fmaxf(x[k], x[k + 1]), x[k + 2]), v = fmaxf(fmaxf(x[k + 3], x[k + 4]), x[k + 5]);
            const float w = fmaxf(fmaxf(u, v), fmaxf(x[k + 6], x[k + 7]));
            top = fmaxf(top, __builtin_fmaf(w, cg[g], lv[g]));
        }
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
        if (__any(top - m > kMostWeight)) {
            const float mn = fmaxf(m, base_of(top)), fade = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= fade;
#pragma unroll
            for (int d = 0; d < NB; ++d) o[d] *= fade;
        }
        // Far from zero the rounding of the base may exceed the weights' head-room: scores are
        // rounded as the maximum was, so that none passes it (with a cap they have been).
        if (!CAP && __any(fabsf(m) > kFar)) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sc[g >> 1][8 * (g & 1) + e] = __builtin_fmaf(sc[g >> 1][8 * (g & 1) + e], cg[g], lv[g]);
                cg[g] = 1.0f;
                lv[g] = 0.0f;
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float base = lv[g] - m;
            float sum;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                typedef float v2f __attribute__((ext_vector_type(2)));
                v2f x;
                x[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e], cg[g], base));
                x[1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e + 1], cg[g], base));
                const h2 pr = __builtin_convertvector(x, h2);
                p[g][e] = pr[0];
                p[g][e + 1] = pr[1];
                sum = e ? sum + x[0] : x[0];
                sum += x[1];
            }
            l = __builtin_fmaf(sum, rv[g], l);
        }
    };

    const int tiles = begin < end ? (end - begin + kTile - 1) / kTile : 0;
    if (tiles > 0) {
        // Phases: the first half of the workgroup runs M(0) V(0) M(1) V(1) ... M(tiles),
        // the second the same one phase later.  M(t) reads the values of t - 1 and the
        // keys of t (M(0)'s values are zeros), and stages keys of t + 1 and values of t
        // into the buffers whose last readers were the two M(t - 1), over by then.
        // (with one wavefront a SIMD all run in step, and one barrier a tile is enough:
        // what overlaps is another workgroup)
        constexpr bool kShift = NW == 8;
        const bool behind = kShift && wave >= NW / 2;
        load(begin, begin);
#pragma unroll
        for (int k = 0; k < 2 * kLoads; ++k)
            if (of_keys(k >> 1)) put(k, 0, 0);
        for (int i = tid; i < kOp / 16; i += kThreads) reinterpret_cast<uint4*>(smem + 3 * kOp)[i] = make_uint4(0, 0, 0, 0);
        // what M(u) stages; past the last tile, the last again, into buffers that nobody reads
        auto fetch = [&](int u) __attribute__((always_inline)) { load(begin + min(u + 1, tiles - 1) * kTile, begin + min(u, tiles - 1) * kTile); };
        fetch(0);
        WUSH_LDS_BARRIER();
        if (behind) WUSH_LDS_BARRIER();
        const std::integral_constant<int, 0> even;
        const std::integral_constant<int, 1> odd;
        auto step = [&](int i, auto parity) __attribute__((always_inline)) {
            __builtin_amdgcn_s_setprio(1);        // few instructions, all of them waited for
            matrix(std::true_type{}, parity);
            fetch(i + 1);
            __builtin_amdgcn_s_setprio(0);
            WUSH_LDS_BARRIER();
            pages_from(begin + i * kTile >> lg);
            weights(begin + i * kTile);
            if constexpr (kShift) WUSH_LDS_BARRIER();
        };
        int i = 0;
        for (; i + 1 < tiles; i += 2) {
            step(i, even);
            step(i + 1, odd);
        }
        if (i < tiles) {
            step(i, even);
            matrix(std::false_type{}, odd);
        } else {
            matrix(std::false_type{}, even);
        }
        WUSH_LDS_BARRIER();
        if (kShift && !behind) WUSH_LDS_BARRIER();
    }

    l += __shfl_xor(l, 32);
    if (bad && l != 0.0f) l = __builtin_nanf("");
    // register e of block d: channel 32 d + 8 (e / 4) + 4 hf + e % 4
    const bool mine = wrow + l32 < rows;
    if (a.splits > 1) {
        float* part = a.part + ((tok * a.cache.heads * G + hq) * a.splits + split) * (D + kPartExtra);
        if (mine) {
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<v4f*>(part + 32 * d + 8 * e + 4 * hf) =
                        (v4f){o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
            if (hf == 0) {
                part[D] = m;
                part[D + 1] = l;
            }
        }
        return;
    }
    // whole rows through LDS: 16-byte piece c of row r at c ^ (r % pieces)
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;                // no token seen: zeros
    constexpr int kPieces = D / 8;
    uint8_t* st = smem + wave * (32 * D * 2);
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int piece = (4 * d + e) ^ (l32 & (kPieces - 1));
            *reinterpret_cast<uint2*>(st + l32 * D * 2 + piece * 16 + 8 * hf) =
                make_uint2(out16<DT>(o[d][4 * e] * inv) | out16<DT>(o[d][4 * e + 1] * inv) << 16,
                           out16<DT>(o[d][4 * e + 2] * inv) | out16<DT>(o[d][4 * e + 3] * inv) << 16);
        }
    // (a wavefront reads what it wrote)
#pragma unroll
    for (int k = 0; k < 32 * kPieces / 64; ++k) {
        const int rr = (k * 64 + lane) / kPieces, pc = (k * 64 + lane) % kPieces;
        const uint4 v = *reinterpret_cast<const uint4*>(st + rr * D * 2 + (pc ^ (rr & (kPieces - 1))) * 16);
        const int row = wrow + rr;
        if (row < rows)
            *reinterpret_cast<uint4*>(a.out + ((int64_t)(s.first + row / G) * a.cache.heads * G + h * G + row % G) * D + 8 * pc) = v;
    }
}

template <int DT, int D, int NW>
void launch_one(const AttnArgs& a, unsigned grid, hipStream_t stream) {
    if (a.cap > kMostPlainCap) kv8_chunk_kernel<DT, D, NW, kWideCap><<<grid, 64 * NW, 0, stream>>>(a);
    else if (a.cap > 0.0f) kv8_chunk_kernel<DT, D, NW, kCap><<<grid, 64 * NW, 0, stream>>>(a);
    else kv8_chunk_kernel<DT, D, NW, kNoCap><<<grid, 64 * NW, 0, stream>>>(a);
}

template <int DT>
int launch(const AttnArgs& a, unsigned grid, hipStream_t stream) {
    if (a.cache.dim == 64) {
        if (a.tile_rows == 256) launch_one<DT, 64, 8>(a, grid, stream);
        else launch_one<DT, 64, 4>(a, grid, stream);
    } else {
        if (a.tile_rows == 256) launch_one<DT, 128, 8>(a, grid, stream);
        else launch_one<DT, 128, 4>(a, grid, stream);
    }
    return (int)hipGetLastError();
}

}  // namespace

int launch_kv8_chunk(const AttnArgs& a, int dtype, hipStream_t stream) {
    const long long blocks = (long long)a.items * a.cache.heads * a.splits;
    WUSH_REQUIRE(blocks <= 0x7fffffffLL && (a.tile_rows == 128 || a.tile_rows == 256));
    return dtype == WUSH_DTYPE_BF16 ? launch<WUSH_DTYPE_BF16>(a, (unsigned)blocks, stream)
                                    : launch<WUSH_DTYPE_F16>(a, (unsigned)blocks, stream);
}

}  // namespace wush
