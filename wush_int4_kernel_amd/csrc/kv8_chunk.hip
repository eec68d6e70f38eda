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
// and the first of tile t, and a vector phase, tile t's weights and the staging of its
// share of the next tiles.  The workgroup's second half runs one phase behind the first,
// with a barrier between phases: of a SIMD's two wavefronts one feeds the matrix cores while the other
// computes (both in step, neither unit was busy more than 60%: 2.7 us a tile).
//
// The running maximum follows lazily: it moves, and the sums are rescaled, only
// when a score passes it by 2^7; weights are exp2(t - maximum + 8), at most 2^15,
// rounded once to fp16 (11 bits, normal down to 2^-22 of the largest) for the product;
// their sum takes them unrounded (pages whose values are far smaller than others' have
// weights below fp16's range, and count in it all the same).
#include "kv8_attention.h"

namespace wush {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kHead = 8.0f, kSlack = 7.0f;
constexpr float kTinyScale = 0x1p-126f;

template <int DT, int D, int NW, bool CAP>
__global__ __launch_bounds__(64 * NW, 2) void kv8_chunk_kernel(const AttnArgs a) {
    constexpr int kThreads = 64 * NW;
    constexpr int NS = D / 16, NB = D / 32;       // steps of the first product, channel blocks of the second
    constexpr int kOp = kTile * D * 2;            // bytes of one operand's tile
    constexpr int kCodes = kTile * D / 16, kLoads = 2 * kCodes / kThreads;   // 16-byte chunks of one tensor's tile; a thread's of both
    __shared__ __align__(16) uint8_t smem[4 * kOp > NW * 32 * D * 2 ? 4 * kOp : NW * 32 * D * 2];
    __shared__ __align__(16) float meta[2][3][4]; // of 16 tokens each: key scale, log2 and reciprocal of the value scale

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
    if (row0 >= s.count * G) return;
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
    float c;                                      // scores in powers of two, per unit of key scale; positive
    {
        const uint16_t* p = a.q + tok * a.qt + hq * a.qh + 8 * hf;
        float mx = 0.0f;
        bool bad = false;
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
        const float up = __builtin_amdgcn_ldexpf(1.0f, ex > 100 ? 100 : ex);
        c = fabsf(a.scale) * (CAP ? 2.0f * kLog2e / a.cap : kLog2e) / up;
        if (bad) c = __builtin_nanf("");
        const float sup = a.scale < 0.0f ? -up : up;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            float x[8];
            load8<DT>(p + 16 * j, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) q[j][e] = bad ? (_Float16)0.0f : (_Float16)(x[e] * sup);
        }
    }

    typedef const __attribute__((address_space(4))) int32_t* sptr;
    const sptr table = (sptr)(uintptr_t)(t.table + (int64_t)b * t.table_stride);
    const int32_t most = (int32_t)a.cache.pages;
    // page of token tk, -1 for none; tk is the same in all lanes where it is called for staging
    auto page_at = [&](int tk) {
        const int id = table[min(tk, end - 1) >> lg];
        return tk < end && id >= 0 && id < most ? id : -1;
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
    auto tile_of = [&](const int8_t* p, int id) {
        return p + ((uint64_t)((uint32_t)max(id, 0) * (uint32_t)a.cache.heads + (uint32_t)h) << tile_log2);
    };
    // the thread's share of the keys of the tile at tk0 and of the values of the one at tv0
    auto load = [&](int tk0, int tv0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n0 = (i * kThreads + 64 * wave) & (kCodes - 1);            // the wavefront's first chunk
            if (of_keys(i)) {
                const int tk = tk0 + n0 / (D / 16);
                raw[i] = *reinterpret_cast<const uint4*>(tile_of(a.cache.k, page_at(tk)) + (tk & (ps - 1)) * D + 16 * lane);
            } else {
                const int tv = tv0 + 16 * cpp * (n0 / D >> cpl);
                raw[i] = *reinterpret_cast<const uint4*>(tile_of(a.cache.v, page_at(tv)) + (tv & (ps - 1)) + voff[i]);
            }
        }
    };
    float mks = 0.0f, mvs = 0.0f;
    bool mhas = false;
    auto load_meta = [&](int t0) {                // threads 0 to 3: scales of the tile's 16-token groups
        if (tid >= 4) return;
        const int tk = t0 + 16 * tid;
        const int id = t.table[(int64_t)b * t.table_stride + (min(tk, end - 1) >> lg)];
        mhas = tk < end && id >= 0 && id < most;
        const int64_t at = (int64_t)(mhas ? id : 0) * a.cache.heads + h;
        mks = a.cache.ks[at];
        mvs = a.cache.vs[at];
    };
    // LDS: operand fragments of 1 KiB, lane l's 16 bytes in slot l, the slots' low
    // bits mixed with the fragment's number so that the stores spread over the banks
    auto put = [&](int kbuf, int vbuf, bool with_keys, bool with_values) {
        uint8_t* kb = smem + kbuf * kOp;
        uint8_t* vb = smem + (2 + vbuf) * kOp;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n = (i * kThreads + tid) & (kCodes - 1);
            if (of_keys(i)) {
                if (!with_keys) continue;
                const int tk = n / (D / 16), st = n % (D / 16);
                uint8_t* f = kb + ((tk >> 5) * NS + st) * 1024 + 16 * ((tk & 31) ^ (st & 7));
                *reinterpret_cast<h8*>(f) = codes8(raw[i].x, raw[i].y);
                *reinterpret_cast<h8*>(f + 512) = codes8(raw[i].z, raw[i].w);
            } else {
                if (!with_values) continue;
                const int d = n >> cpl & (D - 1), ts = (n / D >> cpl) * cpp + (n & (cpp - 1));
                uint8_t* g = vb + ((d >> 5) * 4 + ts) * 1024 + 16 * ((d & 31) ^ ((ts & 1) << 2 | (ts & 2)));
                *reinterpret_cast<h8*>(g) = codes8(raw[i].x, raw[i].z);        // tokens 0-3, 8-11 of 16
                *reinterpret_cast<h8*>(g + 512) = codes8(raw[i].y, raw[i].w);  // 4-7, 12-15
            }
        }
    };
    auto put_meta = [&](int buf) {
        if (tid >= 4) return;
        const float vs = mvs < kValueFloor ? kValueFloor : mvs;
        meta[buf][0][tid] = !mhas ? 1.0f : mks < kTinyScale ? kTinyScale : mks;
        meta[buf][1][tid] = mhas ? __builtin_amdgcn_logf(vs) : -__builtin_inff();
        meta[buf][2][tid] = mhas ? 1.0f / vs : 0.0f;
    };

    v16f o[NB], sc[2];
    h8 p[4];
#pragma unroll
    for (int d = 0; d < NB; ++d) o[d] = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) p[g] = (_Float16)0.0f;
    float m = kLow, l = 0.0f;
    // The matrix phase: the second product of a tile (PV) and the first of the next
    // (QK), their operands read kAhead fragments ahead of the MFMAs.
    constexpr int kAhead = 4, kFrags = 2 * NS;                    // 4 NB = 2 NS fragments each
    auto matrix = [&](auto pv, auto qk, int vbuf, int kbuf) {
        const uint8_t* vb = smem + (2 + vbuf) * kOp + 512 * hf;
        const uint8_t* kb = smem + kbuf * kOp + 512 * hf;
        constexpr int kTotal = (pv.value ? kFrags : 0) + (qk.value ? kFrags : 0);
        h8 f[kAhead];
        auto read = [&](auto ic) {
            constexpr int i = pv.value ? ic.value : ic.value + kFrags;
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
            constexpr int i = pv.value ? ic.value : ic.value + kFrags;
            const h8 x = f[ic.value % kAhead];
            if constexpr (i < kFrags) o[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p[i / NB], o[i % NB], 0, 0, 0);
            else sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[(i - kFrags) / 2], sc[i & 1], 0, 0, 0);
            if constexpr (ic.value + kAhead < kTotal) read(std::integral_constant<int, ic.value + kAhead>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // scores of the tile at t0 -> weights.  Register 8 g + e: token 16 g + 8 (e / 4) + 4 hf + e % 4.
    auto weights = [&](int t0, int buf) {
        const v4f mk = *reinterpret_cast<const v4f*>(meta[buf][0]);
        v4f lv = *reinterpret_cast<const v4f*>(meta[buf][1]);
        const v4f rv = *reinterpret_cast<const v4f*>(meta[buf][2]);
        float cg[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            cg[g] = c * mk[g];
            if (cg[g] > kMostScale) cg[g] = kMostScale;
            if (cg[g] < kTinyScale) cg[g] = kTinyScale;
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
            float x = sc[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int e = 1; e < 8; ++e) x = fmaxf(x, sc[g >> 1][8 * (g & 1) + e]);
            top = fmaxf(top, __builtin_fmaf(x, cg[g], lv[g]));
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m + kSlack)) {
            const float mn = fmaxf(m, top), fade = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= fade;
#pragma unroll
            for (int d = 0; d < NB; ++d) o[d] *= fade;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float base = lv[g] - (m - kHead);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                typedef float v2f __attribute__((ext_vector_type(2)));
                v2f x;
                x[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e], cg[g], base));
                x[1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e + 1], cg[g], base));
                const h2 pr = __builtin_convertvector(x, h2);
                p[g][e] = pr[0];
                p[g][e + 1] = pr[1];
                sum += x[0];
                sum += x[1];
            }
            l += sum != 0.0f ? sum * rv[g] : 0.0f;                // a scale may be NaN where nothing is seen
        }
    };

    const int tiles = begin < end ? (end - begin + kTile - 1) / kTile : 0;
    if (tiles > 0) {
        // Phases: the first half of the workgroup runs M(0) V(0) M(1) V(1) ... M(tiles),
        // the second the same one phase later.  M(t) reads the values of t - 1 and the keys of t.  Keys of
        // t + 1 and values of t are staged during M(t) of either half: by the
        // second half ahead of its own V(t), by the first in its V(t), into
        // the buffers that M(t - 1), over for both, was the last to read.
        const int behind = wave >= NW / 2 ? 1 : 0;
        load(begin, begin);
        load_meta(begin);
        put(0, 0, true, false);
        put_meta(0);
        for (int i = tid; i < kOp / 16; i += kThreads) reinterpret_cast<uint4*>(smem + 3 * kOp)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        // staging step u: keys of tile u + 1, values of tile u, scales of tile u + 1
        auto fetch = [&](int u) {
            if (u >= tiles) return;
            load(begin + min(u + 1, tiles - 1) * kTile, begin + u * kTile);
            if (!behind && u + 1 < tiles) load_meta(begin + (u + 1) * kTile);
        };
        auto stage = [&](int u) {
            if (u >= tiles) return;
            put((u + 1) & 1, u & 1, u + 1 < tiles, true);
            if (!behind && u + 1 < tiles) put_meta((u + 1) & 1);
        };
        fetch(0);
        if (behind) {
            stage(0);
            fetch(1);
            WUSH_LDS_BARRIER();
        }
        const std::true_type yes;
        const std::false_type no;
        for (int i = 0; i < tiles; ++i) {         // (the first second product: zeros)
            matrix(yes, yes, (i + 1) & 1, i & 1);
            WUSH_LDS_BARRIER();
            weights(begin + i * kTile, i & 1);
            stage(i + behind);
            fetch(i + 1 + behind);
            WUSH_LDS_BARRIER();
        }
        matrix(yes, no, (tiles - 1) & 1, 0);
        WUSH_LDS_BARRIER();
        if (!behind) WUSH_LDS_BARRIER();
    }

    l += __shfl_xor(l, 32);
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
    if (a.cap > 0.0f) kv8_chunk_kernel<DT, D, NW, true><<<grid, 64 * NW, 0, stream>>>(a);
    else kv8_chunk_kernel<DT, D, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
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
