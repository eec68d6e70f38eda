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
// Both products run on v_mfma_f32_16x16x32_f16, with the cache as row operand.
// Codes are exact in fp16; a row of q is shifted by a power of two so that its
// largest value lies near 2^15 (exact for values down to 2^-29 of it).  The score tile
// comes out with a lane holding 16 consecutive tokens of one row (keys are loaded in
// the order that makes it so), which is the operand that the second product
// needs: the probabilities never leave their lanes.
//
// A token's value scale is folded into its exponent: with t = log2(e) s +
// log2(v_scale), weights are exp2(t - running max + 12), at most 2^12, rounded once
// to fp16 (11 bits, normal down to 2^-26 of the largest), and the sum of the
// probabilities takes them back times 1 / v_scale, in fp32.
#include "kv8_device.h"

namespace wush {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 64;                         // tokens a wavefront takes at a time
constexpr float kLow = -3e38f;                    // running maximum before any token: below every score
constexpr float kHead = 12.0f;                    // weights reach 2^12
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kValueFloor = 0x1p-40f;           // smallest scale of a page
constexpr float kMostScale = 0x1p97f;             // times 2^15 * 127 * 128: scores stay finite

struct AttnArgs {
    const uint16_t* q;
    int64_t qt, qh;
    Kv8Cache cache;
    Kv8Batch batch;
    int group, window, splits, chunk, items;
    float scale, cap;                             // cap 0: none
    uint16_t* out;
    float* part;                                  // (token, head, split): D sums, maximum, sum of weights
};

// 8 int8 codes -> fp16, exact: code ^ 0x80 = code + 128 in the low byte of 1024.0
__device__ __forceinline__ h8 codes8(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 r0 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - bias;
    const h2 r1 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - bias;
    const h2 r2 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
    const h2 r3 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
    return (h8){r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}

__device__ __forceinline__ float quarters_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarters_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Tokens that a tile of 16 rows beginning at row0 of its sequence may see:
// from base (a multiple of kTile) to end.
struct Span {
    int base, end;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Kv8Seq& s, int row0) {
    const int before = s.len - s.count;           // position of the first new token
    const int i0 = row0 / a.group, i1 = min((row0 + 15) / a.group, s.count - 1);
    Span r;
    r.base = a.window > 0 ? max(before + i0 - a.window + 1, 0) & ~(kTile - 1) : 0;
    const int64_t room = a.batch.table_stride << a.cache.page_log2;
    r.end = (int)min((int64_t)(before + i1 + 1), room);
    return r;
}

template <int DT, int D, bool CAP>
__global__ __launch_bounds__(64 * kWaves) void kv8_rows_kernel(const AttnArgs a) {
    constexpr int NJ = D / 64, NB = D / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, kq = lane >> 4;
    const Kv8Batch& t = a.batch;
    const int lg = a.cache.page_log2, ps = 1 << lg, G = a.group;
    const int split = blockIdx.x % a.splits;
    const int h = (int)(blockIdx.x / a.splits) % a.cache.heads, item = (int)(blockIdx.x / a.splits) / a.cache.heads;
    const int per = (G + 15) >> 4;
    const int b = t.cu ? kv8_find(t, item, G, 4, 1) : item / per;
    const int row0 = 16 * (t.cu ? item - kv8_item_start(t, b, G, 4, 1) : item % per);
    const Kv8Seq s = kv8_seq(t, b);
    if (row0 >= s.count * G) return;
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

    h8 q[2 * NJ];
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
        const int ex = mx > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
        const float up = __builtin_amdgcn_ldexpf(1.0f, ex > 100 ? 100 : ex);
        c = a.scale * (CAP ? 1.0f / a.cap : kLog2e) / up;
        if (quarters_max(bad ? 1.0f : 0.0f) > 0.0f) c = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < 2 * NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[j][e] = bad ? (_Float16)0.0f : (_Float16)(x[j][e] * up);
    }

    const v4f zero = {0, 0, 0, 0};
    v4f acc[NB];
#pragma unroll
    for (int d = 0; d < NB; ++d) acc[d] = zero;
    float m = kLow, l = 0.0f;
    const int64_t tile_bytes = (int64_t)D << lg;
    const int32_t* table = t.table + (int64_t)b * t.table_stride;

    for (int t0 = begin + wave * kTile; t0 < end; t0 += kWaves * kTile) {
        // pages of the keys this lane loads and of the tokens whose scores it holds
        auto page_of = [&](int tk) {
            const int id = tk < end ? table[tk >> lg] : -1;
            return id >= 0 && id < a.cache.pages ? id : -1;
        };
        const int tk = t0 + 16 * (l16 >> 2), tv = t0 + 16 * kq;
        const int idk = page_of(tk), idv = page_of(tv);
        const int8_t* pk = a.cache.k + ((int64_t)max(idk, 0) * a.cache.heads + h) * tile_bytes +
                           ((tk & (ps - 1)) + (l16 & 3)) * D + 16 * kq;
        const int64_t vt = (int64_t)max(idv, 0) * a.cache.heads + h;
        const int8_t* pv = a.cache.v + vt * tile_bytes + (l16 << lg) + (tv & (ps - 1));
        uint4 kk[4][NJ], vv[NB];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < NJ; ++j) kk[n][j] = *reinterpret_cast<const uint4*>(pk + 4 * n * D + 64 * j);
#pragma unroll
        for (int d = 0; d < NB; ++d) vv[d] = *reinterpret_cast<const uint4*>(pv + ((int64_t)d << (lg + 4)));
        const float ks = a.cache.ks[vt];
        float vs = a.cache.vs[vt];
        if (vs < kValueFloor) vs = kValueFloor;

        v4f sc[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            sc[n] = zero;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kk[n][j].x, kk[n][j].y), q[2 * j], sc[n], 0, 0, 0);
                sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kk[n][j].z, kk[n][j].w), q[2 * j + 1], sc[n], 0, 0, 0);
            }
        }
        // the lane's 16 tokens tv .. tv + 15, of one page
        float cs = c * ks;
        if (fabsf(cs) > kMostScale) cs = __builtin_copysignf(kMostScale, cs);
        const float lv = __builtin_amdgcn_logf(vs);
        const int last = idv >= 0 ? min(pos, end - 1) : -1;
        float top = kLow;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = sc[n][e] * cs;
                if constexpr (CAP) x = (a.cap * kLog2e) * (1.0f - 2.0f / (1.0f + __builtin_amdgcn_exp2f(x * (2.0f * kLog2e))));
                x += lv;
                const int at = tv + 4 * n + e;
                x = at <= last && at >= low ? x : -__builtin_inff();
                sc[n][e] = x;
                top = fmaxf(top, x);
            }
        const float mn = fmaxf(m, quarters_max(top));
        const float fade = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        float sum = 0.0f;
        h8 p[2];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = __builtin_amdgcn_exp2f(sc[n][e] - (mn - kHead));
                sum += w;
                p[n >> 1][4 * (n & 1) + e] = (_Float16)w;
            }
        l = l * fade + (sum != 0.0f ? sum * (1.0f / vs) : 0.0f);   // a scale may be NaN where nothing is seen
#pragma unroll
        for (int d = 0; d < NB; ++d) {
            acc[d] *= fade;
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vv[d].x, vv[d].y), p[0], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vv[d].z, vv[d].w), p[1], acc[d], 0, 0, 0);
        }
    }

    // join the wavefronts: a lane holds channels 16 d + 4 kq + e of row l16
    __shared__ float so[kWaves][16][D + 4];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    l = quarters_sum(l);
    if (kq == 0) {
        sm[wave][l16] = m;
        sl[wave][l16] = l;
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
        ll += sl[w][jr] * f;
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
    float* part = a.part + (row * a.splits + split) * (D + 2);
#pragma unroll
    for (int e = 0; e < PD; ++e) part[d0 + e] = o[e];
    if (d0 == 0) {
        part[D] = mm;
        part[D + 1] = ll;
    }
}

// One wavefront per (token, query head): the stretches that hold tokens, joined.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const Kv8Batch& t = a.batch;
    const int heads = a.cache.heads * a.group;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)t.tokens * heads) return;
    const int tok = (int)(row / heads);
    const int b = t.cu ? kv8_find(t, tok, 1, 0, 0) : tok;
    const Kv8Seq s = kv8_seq(t, b);
    const int i = tok - s.first;
    if (i < 0 || i >= s.count) return;
    const Span span = span_of(a, s, (i * a.group + (int)(row % a.group)) & ~15);
    const int n = min(a.splits, max((span.end - span.base + a.chunk - 1) / a.chunk, 1));
    const float* part = a.part + row * a.splits * (D + 2);
    float mm = kLow;
    for (int k = lane; k < n; k += 64) mm = fmaxf(mm, part[(int64_t)k * (D + 2) + D]);
#pragma unroll
    for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    constexpr int PD = D / 64;
    float ll = 0.0f, o[PD] = {};
    for (int k = 0; k < n; ++k) {
        const float* p = part + (int64_t)k * (D + 2);
        const float f = __builtin_amdgcn_exp2f(p[D] - mm);
        ll += p[D + 1] * f;
#pragma unroll
        for (int e = 0; e < PD; ++e) o[e] += p[lane * PD + e] * f;
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
    for (int e = 0; e < PD; ++e) a.out[row * D + lane * PD + e] = (uint16_t)out16<DT>(o[e] * inv);
}

struct Plan {
    int splits, chunk;
    int64_t items;
};

// Stretches of the cache per row tile: about 1024 workgroups, four to a CU.
Plan plan_of(const Kv8Cache& c, int64_t seqs, int64_t tokens, bool ragged, int group, int64_t table_stride, int window,
             int64_t max_len) {
    Plan p;
    p.items = ragged ? (tokens * group >> 4) + seqs : seqs * ((group + 15) / 16);
    int64_t range = table_stride << c.page_log2;
    if (max_len > 0 && max_len < range) range = max_len;
    if (window > 0 && window + 128 < range) range = window + 128;
    if (range < 1) range = 1;
    if (range > 1 << 30) range = 1 << 30;         // the last stretch takes what lies behind
    const int64_t step = kWaves * kTile, most = (range + step - 1) / step;
    int64_t splits = 1024 / (p.items * c.heads);
    splits = splits < 1 ? 1 : splits > most ? most : splits;
    p.chunk = (int)((most + splits - 1) / splits * step);
    p.splits = (int)((range + p.chunk - 1) / p.chunk);
    return p;
}

template <int DT>
int launch(const AttnArgs& a, hipStream_t stream) {
    const int64_t blocks = (int64_t)a.items * a.cache.heads * a.splits;
    const int64_t rows = (int64_t)a.batch.tokens * a.cache.heads * a.group;
    WUSH_REQUIRE(blocks <= 0x7fffffffLL && rows <= 0x7fffffffLL);
    const dim3 grid((unsigned)blocks), join((unsigned)((rows + 3) / 4));
    if (a.cache.dim == 64) {
        if (a.cap > 0.0f) kv8_rows_kernel<DT, 64, true><<<grid, 64 * kWaves, 0, stream>>>(a);
        else kv8_rows_kernel<DT, 64, false><<<grid, 64 * kWaves, 0, stream>>>(a);
        if (a.splits > 1) kv8_join_kernel<DT, 64><<<join, 256, 0, stream>>>(a);
    } else {
        if (a.cap > 0.0f) kv8_rows_kernel<DT, 128, true><<<grid, 64 * kWaves, 0, stream>>>(a);
        else kv8_rows_kernel<DT, 128, false><<<grid, 64 * kWaves, 0, stream>>>(a);
        if (a.splits > 1) kv8_join_kernel<DT, 128><<<join, 256, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace wush

extern "C" {

size_t wush_kv8_attention_workspace_bytes(const wush_kv8_cache* cache, int64_t seqs, int64_t tokens, int ragged,
                                          int64_t q_heads, int64_t table_stride, int64_t window, int64_t max_len) {
    wush::Kv8Cache c;
    if (wush::kv8_cache_of(cache, &c) || seqs <= 0 || tokens <= 0 || q_heads <= 0 || q_heads % c.heads) return 0;
    const int w = window <= 0 || window > 0x7fffffff ? 0 : (int)window;
    const wush::Plan p = wush::plan_of(c, seqs, tokens, ragged != 0, (int)(q_heads / c.heads), table_stride, w, max_len);
    return p.splits > 1 ? (size_t)tokens * q_heads * p.splits * (c.dim + 2) * 4 : 0;
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
    WUSH_REQUIRE(scale == scale && softcap >= 0.0f && softcap < __builtin_inff());
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
    a.window = window > 0x7fffffff ? 0 : (int)window;
    const wush::Plan p = wush::plan_of(a.cache, seqs, tokens, cu_q != nullptr, a.group, table_stride, a.window, max_len);
    WUSH_REQUIRE(p.items <= 0x7fffffffLL);
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.items = (int)p.items;
    a.scale = scale;
    a.cap = softcap;
    a.out = static_cast<uint16_t*>(out);
    a.part = static_cast<float*>(workspace);
    return dtype == WUSH_DTYPE_BF16 ? wush::launch<WUSH_DTYPE_BF16>(a, stream) : wush::launch<WUSH_DTYPE_F16>(a, stream);
}

}  // extern "C"
