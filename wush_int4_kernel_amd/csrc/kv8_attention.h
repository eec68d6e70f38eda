// kv8_attention.h -- what the attention kernels of the 8-bit cache share
// (kv8_attention.hip: few query rows a sequence, and the joining of stretches;
// kv8_chunk.hip: many).
#pragma once

#include "kv8_device.h"

namespace wush {

struct AttnArgs {
    const uint16_t* q;
    int64_t qt, qh;                               // token and head strides
    Kv8Cache cache;
    Kv8Batch batch;
    int group, window;
    int tile_rows;                                // query rows of a work item: 16, 128 or 256
    int tile_shift;                               // log2 of it
    int items;                                    // work items a key/value head
    int splits, chunk;                            // stretches of the cache, tokens of one
    int round;                                    // sequences whose workgroups make one round of the CUs; 0: taken as they come
    float scale, cap;                             // cap 0: none
    uint16_t* out;
    float* part;                                  // (token, head, split): D sums, the weights' base, their sum, 2 unused
};

constexpr int kPartExtra = 4;                     // floats of a partial result behind its D sums

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 64;                         // tokens taken at a time
constexpr float kLow = -3e38f;                    // the weights' base before any token: below every score
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMostWeight = 15.0f;              // weights reach 2^15: fp16 ends at 65504
constexpr float kValueFloor = 0x1p-40f;           // smallest scale of a page

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

// A row's factor, by which q was scaled: finite, so that a key scale of 0 gives scores of 0
__device__ __forceinline__ float row_factor(float c) {
    return __builtin_amdgcn_fmed3f(c, -3e38f, 3e38f);
}
// A row's factor times a key scale, below which scores stay finite: 2^89 * 2^23 * 127 * 128 = 2^126.  A NaN stays one.
__device__ __forceinline__ float kept_finite(float cs) {
    return fabsf(cs) > 0x1p89f ? __builtin_copysignf(0x1p89f, cs) : cs;
}

// Base of weights exp2(score - base) whose largest score is top: 2^12 below it, so that weights are
// normal in fp16 down to 2^-26 of the largest.  Far from zero (from 2^26 on) the difference is rounded, to 16 or to
// none: then the largest weight is 1.
__device__ __forceinline__ float base_of(float top) {
    const float base = top - 12.0f;
    return top - base > kMostWeight ? top : base;
}

// How scores are capped.  kCap's formula is off by up to 2^-22 of the cap, which up to kMostPlainCap is no more
// than a quarter of a weight's rounding; kWideCap's by 2^-20 of the score, for 11 more
// instructions a score (decode of 32 sequences of 4096 47.8 us, not 46.0, 2 x 4096 new tokens 653, not 403).
enum { kNoCap, kCap, kWideCap };
constexpr float kMostPlainCap = 256.0f;

// What a score in natural units is multiplied by before capped takes it
template <int CAP>
__device__ __forceinline__ float score_unit(const AttnArgs& a) {
    return CAP == kCap ? 2.0f * kLog2e / a.cap : kLog2e;
}

// A score in powers of two, cap tanh(score / cap) if there is a cap.
template <int CAP>
__device__ __forceinline__ float capped(const AttnArgs& a, float x) {
    if constexpr (CAP == kNoCap) return x;
    if constexpr (CAP == kCap) {                  // cap tanh(u) = cap (1 - 2 / (1 + exp(2 u)))
        const float top = a.cap * kLog2e;
        return __builtin_fmaf(-2.0f * top, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)), top);
    }
    // the same for |u| of 1/4 and more; below, tanh(u) = u (1 - u^2/3 + 2 u^4/15 - 17 u^6/315 + 62 u^8/2835 - ...)
    const float top = fminf(a.cap * kLog2e, 3e38f), v = x * (2.0f / a.cap);
    const float u = v * 0.34657359f, w = u * u;   // ln(2) / 2
    const float far = top * __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(fabsf(v))), 1.0f);
    const float p = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(62.0f / 2835, w, -17.0f / 315), w, 2.0f / 15), w, -1.0f / 3);
    return fabsf(u) < 0.25f ? __builtin_fmaf(x * w, p, x) : __builtin_copysignf(far, x);
}

// Tokens that a work item's rows, beginning at row0 of their sequence, may see:
// from base (a multiple of kTile) to end.
struct Span {
    int base, end;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Kv8Seq& s, int row0) {
    const int before = s.len - s.count;           // position of the first new token
    const int i0 = row0 / a.group, i1 = min((row0 + a.tile_rows - 1) / a.group, s.count - 1);
    Span r;
    r.base = a.window > 0 ? max(before + i0 - a.window + 1, 0) & ~(kTile - 1) : 0;
    const int64_t room = a.batch.table_stride << a.cache.page_log2;
    r.end = (int)min((int64_t)(before + i1 + 1), room);
    return r;
}

// Zeros for the tokens that cu gives to no sequence, before its first entry and from its last one on.
__device__ __forceinline__ void clear_rest(const AttnArgs& a) {
    const Kv8Batch& t = a.batch;
    if (!t.cu) return;
    const int first = min(max(t.cu[0], 0), t.tokens), last = min(max(t.cu[t.seqs], first), t.tokens);
    const int64_t row = (int64_t)a.cache.heads * a.group * a.cache.dim / 8, lo = first * row, hi = last * row;   // 16-byte pieces
    const int64_t n = lo + t.tokens * row - hi, by = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += by)
        reinterpret_cast<uint4*>(a.out)[i < lo ? i : i - lo + hi] = make_uint4(0, 0, 0, 0);
}

// Work item of a head -> sequence and first row of it, which is below 0 for items before the
// first sequence's
__device__ __forceinline__ int item_rows(const AttnArgs& a, int item, int& row0) {
    const Kv8Batch& t = a.batch;
    if (t.cu) {
        const int b = kv8_find(t, item, a.group, a.tile_shift, 1);
        row0 = (item - kv8_item_start(t, b, a.group, a.tile_shift, 1)) << a.tile_shift;
        return b;
    }
    const int per = (a.group + a.tile_rows - 1) >> a.tile_shift;
    row0 = (item % per) << a.tile_shift;
    return item / per;
}

}  // namespace

// kv8_chunk.hip: tiles of 128 or 256 rows
int launch_kv8_chunk(const AttnArgs& a, int dtype, hipStream_t stream);

}  // namespace wush
