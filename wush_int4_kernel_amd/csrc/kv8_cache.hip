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

// Eight channels from d0 on of one token's head, rotated: out-of-rotation
// channels as they are.
template <int DT>
__device__ __forceinline__ void rotated8(const uint16_t* x, int d0, const float* cs, int rot, bool interleaved,
                                         float (&v)[8]) {
    load8<DT>(x + d0, v);
    if (d0 >= rot) return;
    const int half = rot >> 1;
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = cs[(d0 >> 1) + i], s = cs[half + (d0 >> 1) + i];
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * c - b * s;
            v[2 * i + 1] = b * c + a * s;
        }
        return;
    }
    const bool second = d0 >= half;
    const int i0 = second ? d0 - half : d0;
    float p[8];
    load8<DT>(x + (second ? i0 : d0 + half), p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = cs[i0 + i], s = cs[half + i0 + i];
        v[i] = second ? v[i] * c + p[i] * s : v[i] * c - p[i] * s;
    }
}

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t qt, qh, kt, kh, vt, vh;               // token and head strides
    const float* cos_sin;
    int positions, rot, interleaved;
    Kv8Cache cache;
    Kv8Batch batch;
    int q_heads, items;
    uint16_t* q_out;
};

__device__ __forceinline__ uint32_t code8(float x, float inv) {
    return (uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(x * inv), -127.0f, 127.0f) & 0xffu;
}

// four codes times a ratio <= 1
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r) {
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o |= ((uint32_t)(int)__builtin_rintf((float)(int8_t)(w >> (8 * i)) * r) & 0xffu) << (8 * i);
    return o;
}

// One workgroup per (touched page, head, keys or values), then workgroups that
// rotate the queries, eight channels a thread.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(const AppendArgs a) {
    const int tid = threadIdx.x;
    const Kv8Batch& t = a.batch;
    const int lg = a.cache.page_log2, ps = 1 << lg;
    const int tiles = a.items * a.cache.heads * 2;
    constexpr int TPT = D / 8;                    // threads per token

    if ((int)blockIdx.x >= tiles) {
        const int64_t e = (int64_t)(blockIdx.x - tiles) * kThreads + tid;
        const int64_t row = e / TPT;
        const int tok = (int)(row / a.q_heads), h = (int)(row % a.q_heads), d0 = (int)(e % TPT) * 8;
        if (tok >= t.tokens) return;
        const int b = t.cu ? kv8_find(t, tok, 1, 0, 0) : tok;
        const Kv8Seq s = kv8_seq(t, b);
        const int pos = min(max(s.len - s.count + tok - s.first, 0), a.positions - 1);
        float v[8];
        rotated8<DT>(a.q + tok * a.qt + h * a.qh, d0, a.cos_sin + (int64_t)pos * a.rot, a.rot, a.interleaved, v);
        store8<DT>(a.q_out + row * D + d0, v);
        return;
    }

    const bool values = blockIdx.x & 1;
    const int w = (int)(blockIdx.x >> 1) / a.cache.heads, h = (int)(blockIdx.x >> 1) % a.cache.heads;
    const int b = t.cu ? kv8_find(t, w, 1, lg, 2) : w;
    const Kv8Seq s = kv8_seq(t, b);
    const int start = max(s.len - s.count, 0);
    const int page = (start >> lg) + (t.cu ? w - kv8_item_start(t, b, 1, lg, 2) : 0);
    const int lo = max(start - (page << lg), 0);                  // new tokens of the page: [lo, hi)
    const int hi = min(s.len - (page << lg), ps);
    if (hi <= lo || page >= t.table_stride) return;
    const int id = t.table[(int64_t)b * t.table_stride + page];
    if (id < 0 || id >= a.cache.pages) return;
    const int64_t tile = (int64_t)id * a.cache.heads + h;
    int8_t* codes = (values ? a.cache.v : a.cache.k) + tile * (D << lg);
    float* scale = (values ? a.cache.vs : a.cache.ks) + tile;

    // the new tokens, eight channels a thread, and their largest magnitude (as
    // bits, so that a NaN is the largest)
    constexpr int TP = kThreads / TPT, NP = 128 / TP;
    const int tok0 = tid / TPT, d0 = tid % TPT * 8;
    const int first = s.first + (page << lg) - (s.len - s.count);  // token at the page's start
    float x[NP][8];
    uint32_t mx = 0;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = p * TP + tok0;
        if (i < lo || i >= hi) continue;
        const int tok = first + i;
        if (values) {
            load8<DT>(a.v + tok * a.vt + h * a.vh + d0, x[p]);
        } else {
            const int pos = min((page << lg) + i, a.positions - 1);
            rotated8<DT>(a.k + tok * a.kt + h * a.kh, d0, a.cos_sin + (int64_t)pos * a.rot, a.rot, a.interleaved, x[p]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(x[p][e]) & 0x7fffffffu);
    }
    __shared__ uint32_t part[kThreads / 64];
    __shared__ uint32_t stage[D * (128 + 4) / 4];
#pragma unroll
    for (int d = 32; d; d >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
    if ((tid & 63) == 0) part[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) mx = max(mx, part[i]);
    const float old = lo > 0 ? *scale : 0.0f;
    const float fresh = mx >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(mx) / 127.0f, kPageScaleFloor);
    const float sc = __uint_as_float(max(__float_as_uint(fresh), __float_as_uint(old) & 0x7fffffffu));
    const bool bad = __float_as_uint(sc) >= 0x7f800000u;
    const float inv = bad ? 0.0f : 1.0f / sc;
    const bool grown = lo > 0 && sc != old && !bad;
    const float ratio = old / sc;
    __syncthreads();                              // everyone has read the old scale
    if (tid == 0) *scale = sc;

    if (!values) {
        if (grown)
            for (int i = tid; i < lo * D / 16; i += kThreads) {
                uint4* p = reinterpret_cast<uint4*>(codes) + i;
                uint4 c = *p;
                c.x = rescale4(c.x, ratio); c.y = rescale4(c.y, ratio);
                c.z = rescale4(c.z, ratio); c.w = rescale4(c.w, ratio);
                *p = c;
            }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int i = p * TP + tok0;
            if (i < lo || i >= hi) continue;
            uint2 c = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c.x |= (bad ? 0u : code8(x[p][e], inv)) << (8 * e);
                c.y |= (bad ? 0u : code8(x[p][4 + e], inv)) << (8 * e);
            }
            *reinterpret_cast<uint2*>(codes + i * D + d0) = c;
        }
        return;
    }
    // values: codes turned through LDS, then whole 16-byte pieces of a channel,
    // with what the piece holds of other tokens kept
    uint8_t* st = reinterpret_cast<uint8_t*>(stage);
    const int row = ps + 4;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = p * TP + tok0;
        if (i < lo || i >= hi) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) st[(d0 + e) * row + i] = bad ? 0 : (uint8_t)code8(x[p][e], inv);
    }
    __syncthreads();
    const int c0 = grown ? 0 : lo >> 4, nc = ((hi + 15) >> 4) - c0;
    for (int i = tid; i < nc * D; i += kThreads) {
        const int d = i / nc, c = c0 + i % nc;
        uint4* p = reinterpret_cast<uint4*>(codes + ((int64_t)d << lg) + 16 * c);
        const bool whole = 16 * c >= lo && 16 * c + 16 <= hi;
        const uint4 had = whole ? make_uint4(0, 0, 0, 0) : *p;
        const uint32_t was[4] = {had.x, had.y, had.z, had.w};
        uint32_t now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t0 = 16 * c + 4 * j;
            const uint32_t fresh4 = *reinterpret_cast<const uint32_t*>(st + d * row + t0);
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

// Pages as values: k, v (n, heads, page, D).  One workgroup per (page, head, keys or values).
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(const Kv8Cache c, const int32_t* __restrict__ ids,
                                                            uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    const int tid = threadIdx.x;
    const int lg = c.page_log2, ps = 1 << lg;
    const bool values = blockIdx.x & 1;
    const int64_t out = blockIdx.x >> 1;          // (page, head) of the output
    const int id = ids[out / c.heads], h = (int)(out % c.heads);
    uint16_t* o = (values ? v : k) + out * (D << lg);
    const bool in = id >= 0 && id < c.pages;
    const int64_t tile = in ? (int64_t)id * c.heads + h : 0;
    const float s = in ? (values ? c.vs : c.ks)[tile] : __builtin_nanf("");
    const int8_t* codes = (values ? c.v : c.k) + tile * (D << lg);
    __shared__ uint32_t stage[D * (128 + 4) / 4];
    uint8_t* st = reinterpret_cast<uint8_t*>(stage);
    const int row = ps + 4;
    if (values) {
        for (int i = tid; i < (D << lg) / 4; i += kThreads) {
            const int d = i * 4 >> lg, t = i * 4 & (ps - 1);
            *reinterpret_cast<uint32_t*>(st + d * row + t) = reinterpret_cast<const uint32_t*>(codes)[i];
        }
        __syncthreads();
    }
    for (int i = tid; i < (D << lg) / 8; i += kThreads) {
        const int t = i / (D / 8), d0 = i % (D / 8) * 8;
        float x[8];
        if (values) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)st[(d0 + e) * row + t] * s;
        } else {
            const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = (float)(int8_t)(w.x >> (8 * e)) * s;
                x[4 + e] = (float)(int8_t)(w.y >> (8 * e)) * s;
            }
        }
        store8<DT>(o + (int64_t)i * 8, x);
    }
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
    WUSH_REQUIRE((bits & 15u) == 0 && ((uintptr_t)cos_sin & 3u) == 0);
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
    // pages that new tokens can touch: one each, or tokens / page + 2 a sequence
    const int64_t items = cu_q ? (tokens >> a.cache.page_log2) + 2 * seqs : seqs;
    const int64_t per_q = 256 * 8 / a.cache.dim;
    const int64_t blocks = items * a.cache.heads * 2 + (tokens * q_heads + per_q - 1) / per_q;
    WUSH_REQUIRE(blocks <= 0x7fffffffLL);
    a.items = (int)items;
    const dim3 grid((unsigned)blocks);
    if (dtype == WUSH_DTYPE_BF16) {
        if (a.cache.dim == 64) wush::kv8_append_kernel<WUSH_DTYPE_BF16, 64><<<grid, wush::kThreads, 0, stream>>>(a);
        else wush::kv8_append_kernel<WUSH_DTYPE_BF16, 128><<<grid, wush::kThreads, 0, stream>>>(a);
    } else {
        if (a.cache.dim == 64) wush::kv8_append_kernel<WUSH_DTYPE_F16, 64><<<grid, wush::kThreads, 0, stream>>>(a);
        else wush::kv8_append_kernel<WUSH_DTYPE_F16, 128><<<grid, wush::kThreads, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
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
    const dim3 grid((unsigned)(n * c.heads * 2));
    uint16_t *ko = static_cast<uint16_t*>(k), *vo = static_cast<uint16_t*>(v);
    if (dtype == WUSH_DTYPE_BF16) {
        if (c.dim == 64) wush::kv8_read_kernel<WUSH_DTYPE_BF16, 64><<<grid, wush::kThreads, 0, stream>>>(c, pages, ko, vo);
        else wush::kv8_read_kernel<WUSH_DTYPE_BF16, 128><<<grid, wush::kThreads, 0, stream>>>(c, pages, ko, vo);
    } else {
        if (c.dim == 64) wush::kv8_read_kernel<WUSH_DTYPE_F16, 64><<<grid, wush::kThreads, 0, stream>>>(c, pages, ko, vo);
        else wush::kv8_read_kernel<WUSH_DTYPE_F16, 128><<<grid, wush::kThreads, 0, stream>>>(c, pages, ko, vo);
    }
    return (int)hipGetLastError();
}

}  // extern "C"
