// kv8_device.h -- what the kernels of the 8-bit paged key/value cache share:
// the cache's layout, the walk over ragged batches, conversions.
//
// Cache: pages of page_size tokens (16, 32, 64 or 128).  A (page, head) tile is
// contiguous: keys [token][D], values [D][token], int8, with one fp32 scale per
// tile and tensor.  Values lie channel by channel so that the product of the
// probabilities with them reads its operand (one channel, consecutive tokens)
// straight from memory; keys lie token by token for the same reason.
#pragma once

#include "wush_device.h"
#include "../../include/wush_int4.h"

namespace wush {

// a batch of sequences: new tokens [cu[b], cu[b + 1]) of b (without cu, one
// token each), behind which its length is lens[b]
struct Kv8Batch {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    int64_t table_stride;                         // entries per sequence
    int seqs, tokens;
};

struct Kv8Cache {
    int8_t *k, *v;
    float *ks, *vs;
    int64_t pages;
    int heads, page_log2, dim;
};

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

struct Kv8Seq {
    int first, count, len;                        // first new token, new tokens, length behind them
};

// Sequence b; device values out of range count as no tokens.  A length of at most
// WUSH_KV8_MAX_LENGTH keeps a position, with a window or some tiles added, in 32 bits.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch& t, int b) {
    Kv8Seq s;
    if (t.cu) {
        s.first = max(t.cu[b], 0);
        s.count = max(min(t.cu[b + 1], t.tokens) - s.first, 0);
    } else {
        s.first = b;
        s.count = 1;
    }
    s.len = t.lens[b];
    if (s.len < 0 || s.len > WUSH_KV8_MAX_LENGTH) s.len = 0;
    return s;
}

// The last b in [0, seqs) with cu[b] * mul / 2^shift + per * b <= w: work items are
// numbered so that sequence b's begin there (per = 1 or 2 spare ones each).
__device__ __forceinline__ int kv8_item_start(const Kv8Batch& t, int b, int mul, int shift, int per) {
    return (int)(((int64_t)max(t.cu[b], 0) * mul) >> shift) + per * b;
}
__device__ __forceinline__ int kv8_find(const Kv8Batch& t, int w, int mul, int shift, int per) {
    int lo = 0, hi = t.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (kv8_item_start(t, mid, mul, shift, per) <= w) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <int DT>
__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == WUSH_DTYPE_BF16) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            v[2 * i] = f16_to_f32(u[i] & 0xffffu);
            v[2 * i + 1] = f16_to_f32(u[i] >> 16);
        }
    }
}

// fp32 -> the output type, rounded to nearest even; a NaN stays one
template <int DT>
__device__ __forceinline__ uint32_t out16(float f) {
    if constexpr (DT == WUSH_DTYPE_F16) return f32_to_f16_bits(f);
    else return f != f ? 0x7fc0u : f32_to_bf16_rne(f);
}

template <int DT>
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
    uint4 w;
    w.x = out16<DT>(v[0]) | out16<DT>(v[1]) << 16;
    w.y = out16<DT>(v[2]) | out16<DT>(v[3]) << 16;
    w.z = out16<DT>(v[4]) | out16<DT>(v[5]) << 16;
    w.w = out16<DT>(v[6]) | out16<DT>(v[7]) << 16;
    *reinterpret_cast<uint4*>(p) = w;
}

}  // namespace

// the library's view of a caller's cache, or hipErrorInvalidValue (kv8_cache.hip)
int kv8_cache_of(const wush_kv8_cache* c, Kv8Cache* out);

}  // namespace wush
