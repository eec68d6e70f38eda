// kv8_cache.hip -- writing and reading the 8-bit paged key/value cache.
//
// Append, for a token at position p of its sequence:
//   q', k' = q, k rotated by p: pairs (a, b) -> (a c - b s, b c + a s), with
//            (c, s) row p of the table, every product and sum rounded to fp32
//   a page's scale s' = max(s of the tokens already in it, amax(new) / 127, 2^-40)
//   new codes clamp(rint(x * (1 / s')), -127, 127), codes already there rint(code * (s / s'))
// over the tile's new tokens and channels.  A page that begins with a new token
// forgets its old scale.  A non-finite key or value makes its tile's scale NaN.
#include "kv8_device.h"

namespace wush {
namespace {

constexpr int kThreads = 256;
constexpr float kPageScaleFloor = 0x1p-40f;
// Values of at most so many new tokens in a page are stored byte by byte: 64 sequences,
// pages of 64, 1 token 5.8 us, through LDS 6.5; 8 tokens 11.5 and 11.8; 16 tokens in pages of 16
// 11.9 and 10.7.
constexpr int kFewTokens = 8;

// A thread's unit of a token's head: 16 channels, 8 from a and 8 from b on, so
// that it holds both of a pair: (i, i + rot / 2) or neighbours; behind the rotated
// channels 16 in a row.
struct Unit {
    int a, b, turn;                               // turn: first of its 8 pairs' table columns, -1: not rotated
};
__device__ __forceinline__ Unit unit_of(int u, int rot, bool interleaved) {
    if (16 * u >= rot) return {16 * u, 16 * u + 8, -1};
    if (interleaved) return {16 * u, 16 * u + 8, 8 * u};
    return {8 * u, 8 * u + (rot >> 1), 8 * u};
}

typedef float v8f __attribute__((ext_vector_type(8)));

struct Values {                                   // a unit's channels
    v8f a, b;
};
struct Turn {
    v8f c, s;
};

__device__ __forceinline__ v8f load_v8f(const float* p) {
    const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
    return (v8f){u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ Turn load_turn(const float* row, const Unit& u, int rot) {
    Turn t;
    t.c = 1.0f;
    t.s = 0.0f;
    if (u.turn >= 0) {
        t.c = load_v8f(row + u.turn);
        t.s = load_v8f(row + (rot >> 1) + u.turn);
    }
    return t;
}
// (a, b) -> (a c - b s, b c + a s) on the unit's eight pairs
__device__ __forceinline__ Values rotate(const Values& x, const Unit& u, const Turn& t, bool interleaved) {
    if (u.turn < 0) return x;
    if (!interleaved) return {x.a * t.c - x.b * t.s, x.b * t.c + x.a * t.s};
    const v8f p = __builtin_shufflevector(x.a, x.b, 0, 2, 4, 6, 8, 10, 12, 14);
    const v8f q = __builtin_shufflevector(x.a, x.b, 1, 3, 5, 7, 9, 11, 13, 15);
    const v8f r = p * t.c - q * t.s, v = q * t.c + p * t.s;
    return {__builtin_shufflevector(r, v, 0, 8, 1, 9, 2, 10, 3, 11), __builtin_shufflevector(r, v, 4, 12, 5, 13, 6, 14, 7, 15)};
}
template <int DT>
__device__ __forceinline__ v8f load8v(const uint16_t* p) {
    float y[8];
    load8<DT>(p, y);
    return (v8f){y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
}
template <int DT>
__device__ __forceinline__ void store8v(uint16_t* p, const v8f& v) {
    const float y[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    store8<DT>(p, y);
}
template <int DT>
__device__ __forceinline__ Values load_unit(const uint16_t* p, const Unit& u) {
    return {load8v<DT>(p + u.a), load8v<DT>(p + u.b)};
}
__device__ __forceinline__ uint32_t largest(const v8f& v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t qt, qh, kt, kh, vt, vh;               // token and head strides
    const float* cos_sin;
    int positions, rot, interleaved;
    Kv8Cache cache;
    Kv8Batch batch;
    int q_heads, items;
    int tile_blocks, q_each, q_parts;             // a thread's query heads; how many such groups of heads
    uint16_t* q_out;
};

__device__ __forceinline__ uint2 codes_of(const v8f& v, float inv) {
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        o[i >> 2] |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(v[i] * inv), -127.0f, 127.0f) & 0xffu) << (8 * (i & 3));
    return make_uint2(o[0], o[1]);
}

// four codes times a ratio <= 1
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r) {
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o |= ((uint32_t)(int)__builtin_rintf((float)(int8_t)(w >> (8 * i)) * r) & 0xffu) << (8 * i);
    return o;
}

// Workgroups of four wavefronts: W of them (page / 16, at most 4) take the new tokens of one
// (touched page, keys or values, head), a lane 16 channels of NP tokens; behind those
// workgroups that rotate the queries, a thread 16 channels of q_each heads of a token,
// whose table row it loads once.
//
// Measured (bf16, 8 key/value heads of 128): 4161 new tokens, 32 query heads, pages of 16,
// 96 MB, 20 us (4.8 TB/s); 64 single
// tokens, 64 query heads, pages of 64, 6.3 us, where the chain of loads (length, table,
// scale) and the launch are what it takes.
template <int DT, int D, int W, int NP>
__global__ __launch_bounds__(kThreads, NP > 2 ? 4 : 6) void kv8_append_kernel(const AppendArgs a) {
    constexpr int kUnits = D / 16, TP = 64 / kUnits, TW = 4 / W, kPage = W * TP * NP;
    constexpr int kRow = kPage + 4;               // bytes of a channel's tokens in LDS
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv8Batch& t = a.batch;
    const int lg = __builtin_ctz(kPage);
    const int un = lane % kUnits;

    if ((int)blockIdx.x >= a.tile_blocks) {
        const int64_t e = (int64_t)((int)blockIdx.x - a.tile_blocks) * kThreads + tid;
        const int64_t part = e / kUnits;
        const int tok = (int)(part / a.q_parts), h0 = (int)(part % a.q_parts) * a.q_each;
        if (tok >= t.tokens) return;
        const int b = t.cu ? kv8_find(t, tok, 1, 0, 0) : tok;
        const Kv8Seq s = kv8_seq(t, b);
        const int pos = min(max(s.len - s.count + tok - s.first, 0), a.positions - 1);
        const Unit u = unit_of(un, a.rot, a.interleaved);
        const Turn turn = load_turn(a.cos_sin + (int64_t)pos * a.rot, u, a.rot);
        const uint16_t* q = a.q + tok * a.qt + h0 * a.qh;
        uint16_t* o = a.q_out + ((int64_t)tok * a.q_heads + h0) * D;
        const int n = min(a.q_each, a.q_heads - h0);
        const bool given = tok >= s.first && tok - s.first < s.count;            // to a sequence; else zeros
#pragma unroll 2
        for (int h = 0; h < n; ++h) {
            Values x = {0.0f, 0.0f};
            if (given) x = rotate(load_unit<DT>(q + h * a.qh, u), u, turn, a.interleaved);
            store8v<DT>(o + h * D + u.a, x.a);
            store8v<DT>(o + h * D + u.b, x.b);
        }
        return;
    }

    __shared__ uint32_t part[4];
    __shared__ __align__(16) uint8_t stage[TW][D * kRow];
    const int slot = wave / W, within = wave % W;
    const int index = (int)blockIdx.x * TW + slot;                // ((item, keys or values), head)
    const int heads = a.cache.heads, h = index % heads;
    const bool values = index / heads & 1;
    const int w = index / heads >> 1;
    bool active = w < a.items;
    Kv8Seq s = {0, 0, 0};
    int page = 0, lo = 0, hi = 0, id = -1, b = 0;
    if (active) {
        b = t.cu ? kv8_find(t, w, 1, lg, 2) : w;
        s = kv8_seq(t, b);
        const int start = max(s.len - s.count, 0);
        page = (start >> lg) + (t.cu ? w - kv8_item_start(t, b, 1, lg, 2) : 0);
        lo = max(start - (page << lg), 0);                        // new tokens of the page: [lo, hi)
        hi = min(s.len - (page << lg), kPage);
        if (hi > lo && page < t.table_stride) id = t.table[(int64_t)b * t.table_stride + page];
        active = id >= 0 && id < a.cache.pages;
        if (!active) hi = lo;
    }
    const int64_t tile = active ? (int64_t)id * heads + h : 0;
    int8_t* codes = (values ? a.cache.v : a.cache.k) + tile * (D << lg);
    float* scale = (values ? a.cache.vs : a.cache.ks) + tile;
    const float old = lo > 0 && active ? *scale : 0.0f;

    // the new tokens, and their largest magnitude (as bits, so that a NaN is the largest)
    const Unit u = values ? Unit{16 * un, 16 * un + 8, -1} : unit_of(un, a.rot, a.interleaved);
    const uint16_t* src = values ? a.v + h * a.vh : a.k + h * a.kh;
    const int64_t step = values ? a.vt : a.kt;
    const int first = s.first + (page << lg) - (s.len - s.count);                // token at the page's start
    Values x[NP];
    uint32_t mx = 0;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = (p * W + within) * TP + lane / kUnits;
        x[p].a = 0.0f;
        x[p].b = 0.0f;
        if (i >= lo && i < hi) {
            const Turn turn = load_turn(a.cos_sin + (int64_t)min((page << lg) + i, a.positions - 1) * a.rot, u, a.rot);
            x[p] = rotate(load_unit<DT>(src + (first + i) * step, u), u, turn, a.interleaved);
            mx = max(mx, max(largest(x[p].a), largest(x[p].b)));
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
    if (lane == 0) part[wave] = mx;
    __syncthreads();                              // everyone has read the old scale, too
#pragma unroll
    for (int i = 0; i < W; ++i) mx = max(mx, part[slot * W + i]);
    const float fresh = mx >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(mx) / 127.0f, kPageScaleFloor);
    const float sc = __uint_as_float(max(__float_as_uint(fresh), __float_as_uint(old) & 0x7fffffffu));
    const bool bad = __float_as_uint(sc) >= 0x7f800000u;
    const float inv = bad ? 0.0f : 1.0f / sc;
    const bool grown = lo > 0 && sc != old && !bad;
    const float ratio = old / sc;
    const int me = within * 64 + lane;            // among the tile's threads
    if (active && me == 0) *scale = sc;

    if (active && !values && grown)
        for (int i = me; i < lo * D / 16; i += 64 * W) {
            uint4* p = reinterpret_cast<uint4*>(codes) + i;
            uint4 c = *p;
            c.x = rescale4(c.x, ratio); c.y = rescale4(c.y, ratio);
            c.z = rescale4(c.z, ratio); c.w = rescale4(c.w, ratio);
            *p = c;
        }
    uint8_t* st = stage[slot];
    const bool bytes = !grown && hi - lo <= kFewTokens;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = (p * W + within) * TP + lane / kUnits;
        if (i >= lo && i < hi) {
            const uint2 ca = bad ? make_uint2(0, 0) : codes_of(x[p].a, inv), cb = bad ? make_uint2(0, 0) : codes_of(x[p].b, inv);
            if (!values) {
                *reinterpret_cast<uint2*>(codes + i * D + u.a) = ca;
                *reinterpret_cast<uint2*>(codes + i * D + u.b) = cb;
            } else {
                const uint32_t c[4] = {ca.x, ca.y, cb.x, cb.y};
                // few tokens into a page whose scale stays: byte by byte, no reading
                // back of what lies around them
                if (bytes) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) codes[((16 * un + e) << lg) + i] = (int8_t)(c[e >> 2] >> (8 * (e & 3)));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) st[(16 * un + e) * kRow + i] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
                }
            }
        }
    }
    __syncthreads();
    if (!active || !values || bytes) return;
    // values: turned through LDS, whole 16-byte pieces of a channel, with what the
    // piece holds of other tokens kept
    const int c0 = grown ? 0 : lo >> 4, nc = ((hi + 15) >> 4) - c0;
    for (int i = me; i < nc * D; i += 64 * W) {
        const int d = i / nc, c = c0 + i % nc;
        uint4* p = reinterpret_cast<uint4*>(codes + (d << lg) + 16 * c);
        const bool whole = 16 * c >= lo && 16 * c + 16 <= hi;
        const uint4 had = whole ? make_uint4(0, 0, 0, 0) : *p;
        const uint32_t was[4] = {had.x, had.y, had.z, had.w};
        uint32_t now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t0 = 16 * c + 4 * j;
            const uint32_t fresh4 = *reinterpret_cast<const uint32_t*>(st + d * kRow + t0);
            uint32_t older = 0, mask = 0;         // bytes of older and of new tokens; what lies behind is none yet
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                older |= t0 + e < lo ? 0xffu << (8 * e) : 0u;
                mask |= t0 + e >= lo && t0 + e < hi ? 0xffu << (8 * e) : 0u;
            }
            const uint32_t kept = grown ? (rescale4(was[j], ratio) & older) | (was[j] & ~older) : was[j];
            now[j] = (fresh4 & mask) | (kept & ~mask);
        }
        *p = make_uint4(now[0], now[1], now[2], now[3]);
    }
}

// Pages as values: k, v (n, heads, page, D).  One workgroup per (page, head, keys or
// values).  Values are turned: through LDS, then eight channels by four tokens in
// registers.  64 pages of 64 tokens (25 MB): 7.4 us, of which the launch is about 3.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(const Kv8Cache c, const int32_t* __restrict__ ids,
                                                            uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    const int tid = threadIdx.x;
    const int lg = c.page_log2, row = (1 << lg) + 4;
    const bool values = blockIdx.x & 1;
    const int64_t out = blockIdx.x >> 1;          // (page, head) of the output
    const int id = ids[out / c.heads], h = (int)(out % c.heads);
    uint16_t* o = (values ? v : k) + out * (D << lg);
    const bool in = id >= 0 && id < c.pages;
    const int64_t tile = in ? (int64_t)id * c.heads + h : 0;
    const float s = in ? (values ? c.vs : c.ks)[tile] : __builtin_nanf("");
    const uint4* codes = reinterpret_cast<const uint4*>((values ? c.v : c.k) + tile * (D << lg));
    auto value = [&](uint32_t w, int e) { return (float)(int8_t)(w >> (8 * e)) * s; };
    if (!values) {
#pragma unroll 4
        for (int i = tid; i < (D << lg) / 16; i += kThreads) {
            const uint4 w = codes[i];
            store8v<DT>(o + (int64_t)i * 16, (v8f){value(w.x, 0), value(w.x, 1), value(w.x, 2), value(w.x, 3),
                                                   value(w.y, 0), value(w.y, 1), value(w.y, 2), value(w.y, 3)});
            store8v<DT>(o + (int64_t)i * 16 + 8, (v8f){value(w.z, 0), value(w.z, 1), value(w.z, 2), value(w.z, 3),
                                                       value(w.w, 0), value(w.w, 1), value(w.w, 2), value(w.w, 3)});
        }
        return;
    }
    __shared__ uint32_t stage[D * (128 + 4) / 4];
    uint8_t* st = reinterpret_cast<uint8_t*>(stage);
#pragma unroll 4
    for (int i = tid; i < (D << lg) / 16; i += kThreads) {
        const uint4 w = codes[i];
        uint32_t* p = reinterpret_cast<uint32_t*>(st + (i * 16 >> lg) * row + (i * 16 & ((1 << lg) - 1)));
        p[0] = w.x;
        p[1] = w.y;
        p[2] = w.z;
        p[3] = w.w;
    }
    __syncthreads();
    for (int i = tid; i < (D << lg) / 32; i += kThreads) {
        const int d0 = i % (D / 8) * 8, t0 = i / (D / 8) * 4;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const uint32_t*>(st + (d0 + e) * row + t0);
#pragma unroll
        for (int t = 0; t < 4; ++t)
            store8v<DT>(o + (t0 + t) * D + d0, (v8f){value(w[0], t), value(w[1], t), value(w[2], t), value(w[3], t),
                                                     value(w[4], t), value(w[5], t), value(w[6], t), value(w[7], t)});
    }
}

template <int DT>
int launch_append(const AppendArgs& a, dim3 grid, hipStream_t stream) {
    const int lg = a.cache.page_log2;
    if (a.cache.dim == 64) {
        if (lg == 4) kv8_append_kernel<DT, 64, 1, 1><<<grid, kThreads, 0, stream>>>(a);
        else if (lg == 5) kv8_append_kernel<DT, 64, 2, 1><<<grid, kThreads, 0, stream>>>(a);
        else if (lg == 6) kv8_append_kernel<DT, 64, 4, 1><<<grid, kThreads, 0, stream>>>(a);
        else kv8_append_kernel<DT, 64, 4, 2><<<grid, kThreads, 0, stream>>>(a);
    } else {
        if (lg == 4) kv8_append_kernel<DT, 128, 1, 2><<<grid, kThreads, 0, stream>>>(a);
        else if (lg == 5) kv8_append_kernel<DT, 128, 2, 2><<<grid, kThreads, 0, stream>>>(a);
        else if (lg == 6) kv8_append_kernel<DT, 128, 4, 2><<<grid, kThreads, 0, stream>>>(a);
        else kv8_append_kernel<DT, 128, 4, 4><<<grid, kThreads, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
}

// Pages of at most 2^22 (page, head)s a launch: a launch has fewer than 2^32 threads.
template <int DT>
int launch_read(const Kv8Cache& c, const int32_t* pages, int64_t n, uint16_t* k, uint16_t* v, hipStream_t stream) {
    const int64_t most = (1 << 22) / c.heads, page = (int64_t)c.heads * (c.dim << c.page_log2);
    for (int64_t at = 0; at < n; at += most, pages += most, k += most * page, v += most * page) {
        const dim3 grid((unsigned)((n - at < most ? n - at : most) * c.heads * 2));
        if (c.dim == 64) kv8_read_kernel<DT, 64><<<grid, kThreads, 0, stream>>>(c, pages, k, v);
        else kv8_read_kernel<DT, 128><<<grid, kThreads, 0, stream>>>(c, pages, k, v);
        const int st = (int)hipGetLastError();
        if (st) return st;
    }
    return (int)hipSuccess;
}

}  // namespace

int kv8_cache_of(const wush_kv8_cache* c, Kv8Cache* out) {
    WUSH_REQUIRE(c && c->k && c->v && c->k_scale && c->v_scale);
    WUSH_REQUIRE(c->pages > 0 && c->pages <= 0x7fffffffLL && c->heads > 0 && c->heads <= 65535);
    WUSH_REQUIRE(c->pages * c->heads <= 0x7fffffffLL);            // tiles: 2 TB and more beyond
    WUSH_REQUIRE(c->head_dim == 64 || c->head_dim == 128);
    WUSH_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128);
    WUSH_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15u) == 0 &&
                 (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3u) == 0);
    *out = {c->k, c->v, c->k_scale, c->v_scale, c->pages, c->heads, __builtin_ctz(c->page_size), c->head_dim};
    return 0;
}

}  // namespace wush

extern "C" {

int wush_kv8_append(const void* q, const void* k, const void* v, int dtype, const int64_t strides[6],
                    const float* cos_sin, int64_t positions, int64_t rot, int interleaved, const wush_kv8_cache* cache,
                    const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, const int32_t* cu_q,
                    int64_t seqs, int64_t tokens, int64_t q_heads, void* q_out, hipStream_t stream) {
    wush::AppendArgs a;
    const int st = wush::kv8_cache_of(cache, &a.cache);
    if (st) return st;
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    WUSH_REQUIRE(seqs >= 0 && tokens >= 0 && q_heads >= 0 && q_heads <= 65535 && table_stride >= 0);
    if (seqs == 0 || tokens == 0) return (int)hipSuccess;
    WUSH_REQUIRE(k && v && (cos_sin || rot == 0) && strides && (block_table || table_stride == 0) && seq_lens && (q_heads == 0 || (q && q_out)));
    WUSH_REQUIRE(seqs <= 0x3fffffffLL && tokens <= 0x3fffffffLL && (cu_q || seqs == tokens));
    WUSH_REQUIRE(positions > 0 && positions <= 0x7fffffffLL && rot >= 0 && rot <= a.cache.dim && rot % 16 == 0);
    uintptr_t bits = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out;
    WUSH_REQUIRE((bits & 15u) == 0);
    for (int i = 0; i < 6; ++i) WUSH_REQUIRE(strides[i] % 8 == 0);
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.qt = strides[0]; a.qh = strides[1]; a.kt = strides[2]; a.kh = strides[3]; a.vt = strides[4]; a.vh = strides[5];
    a.cos_sin = cos_sin;
    a.positions = (int)positions;
    a.rot = (int)rot;
    a.interleaved = interleaved != 0;
    a.batch = {block_table, seq_lens, cu_q, table_stride, (int)seqs, (int)tokens};
    a.q_heads = (int)q_heads;
    a.q_out = static_cast<uint16_t*>(q_out);
    WUSH_REQUIRE(((uintptr_t)cos_sin & 15u) == 0);
    // pages that new tokens can touch: one each, or tokens / page + 2 a sequence
    const int64_t items = cu_q ? (tokens >> a.cache.page_log2) + 2 * seqs : seqs;
    const int per = a.cache.page_log2 == 4 ? 4 : a.cache.page_log2 == 5 ? 2 : 1;  // (page, head)s a workgroup
    const int64_t tile_blocks = (items * a.cache.heads * 2 + per - 1) / per;
    // heads a query thread: more than one once the threads fill the chip several times
    int64_t each = tokens * q_heads * (a.cache.dim / 16) / (512 * 1024);
    each = each < 1 ? 1 : each > 8 ? 8 : each;
    a.q_each = (int)each;
    a.q_parts = (int)((q_heads + each - 1) / each);
    const int64_t q_blocks = (tokens * a.q_parts * (a.cache.dim / 16) + wush::kThreads - 1) / wush::kThreads;
    WUSH_REQUIRE(tile_blocks + q_blocks <= 0x7fffffffLL && items * a.cache.heads * 2 <= 0x7fffffffLL);
    a.items = (int)items;
    a.tile_blocks = (int)tile_blocks;
    const dim3 grid((unsigned)(tile_blocks + q_blocks));
    return dtype == WUSH_DTYPE_BF16 ? wush::launch_append<WUSH_DTYPE_BF16>(a, grid, stream)
                                    : wush::launch_append<WUSH_DTYPE_F16>(a, grid, stream);
}

int wush_kv8_read(const wush_kv8_cache* cache, const int32_t* pages, int64_t n, int dtype, void* k, void* v,
                  hipStream_t stream) {
    wush::Kv8Cache c;
    const int st = wush::kv8_cache_of(cache, &c);
    if (st) return st;
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    WUSH_REQUIRE(n >= 0);
    if (n == 0) return (int)hipSuccess;
    WUSH_REQUIRE(pages && k && v && (((uintptr_t)k | (uintptr_t)v) & 15u) == 0);
    WUSH_REQUIRE(n <= 0x3fffffffLL / c.heads);
    uint16_t *ko = static_cast<uint16_t*>(k), *vo = static_cast<uint16_t*>(v);
    return dtype == WUSH_DTYPE_BF16 ? wush::launch_read<WUSH_DTYPE_BF16>(c, pages, n, ko, vo, stream)
                                    : wush::launch_read<WUSH_DTYPE_F16>(c, pages, n, ko, vo, stream);
}

}  // extern "C"
