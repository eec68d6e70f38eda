// fp8_device.h -- e4m3 codes of a block of 128 channels, shared by the kernels
// that quantize activations.
//
//   A = max(amax |x|, 448 * 2^-126),  scale = A / 448,  code = e4m3(448 x / A)
//
// The code is the nearest to the quotient itself, halves to even: 0.875 x is exact for bf16 and fp16
// values (7 x has 3 more bits), and no quotient of two such values is within 2^-22 of half a
// code's step without being it.  A
// product with the rounded reciprocal instead falls to one or the other side of those
// halves, which values of 8 bits meet often.  A block with a non-finite value gets the
// scale NaN and zero codes.
#pragma once

#include "wush_device.h"

namespace wush {
namespace {

constexpr float kFp8Largest = 448.0f;
constexpr float kFp8Floor = 448.0f * 0x1p-126f;

// largest: amax as fp32 bits, sign cleared (a NaN's are above infinity's)
__device__ __forceinline__ float fp8_amax(uint32_t largest) {
    return largest >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(largest), kFp8Floor);
}
__device__ __forceinline__ float fp8_scale(float amax) { return amax / kFp8Largest; }
// The division made once for a block: with a = A / 2^e in [1, 2), r = RN(1 / a) and v' = 0.875 v 2^(9 - e) (exact, or
// so small that its code is 0), q0 = RN(v' r) is within 1.5 ulps of v' / a, its remainder exact in an fma, and
// q1 = RN(q0 + remainder r) within an ulp, and the quotient itself where that is representable, as
// halves between codes are.
struct Fp8Divisor {
    float a, r;
    int shift;
};
__device__ __forceinline__ Fp8Divisor fp8_divisor(float amax) {
    Fp8Divisor d;
    const uint32_t u = __float_as_uint(amax);                    // a normal number, or NaN
    d.shift = 9 + 127 - (int)(u >> 23);
    d.a = __uint_as_float((u & 0x7fffffu) | 0x3f800000u);
    d.r = 1.0f / d.a;
    return d;
}
__device__ __forceinline__ float fp8_arg(float v, const Fp8Divisor& d) {
    const float w = __builtin_ldexpf(v * 0.875f, d.shift), q = w * d.r;
    return __builtin_fmaf(__builtin_fmaf(-q, d.a, w), d.r, q);
}

// four codes
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, const Fp8Divisor& by, bool bad) {
    if (bad) return 0;
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_arg(a, by), fp8_arg(b, by), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_arg(c, by), fp8_arg(d, by), p, true);
}

// values of four codes
__device__ __forceinline__ void fp8_values4(uint32_t codes, float (&v)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
}

// The same for values that are sums in fp32: a product with the rounded quotient 448 / A, off by less than
// 2^-22 of a code's value, since nothing puts such values onto the halves.
__device__ __forceinline__ float fp8_factor(float amax) { return kFp8Largest / amax; }
__device__ __forceinline__ uint32_t fp8_codes4_by(float a, float b, float c, float d, float factor) {
    if (factor != factor) return 0;
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a * factor, b * factor, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * factor, d * factor, p, true);
}

// x / (1 + exp(-x)): the hardware's exponential and reciprocal, each good to an ulp, with the exponent's
// rounding made up for, within 2^-21
__device__ __forceinline__ float fp8_silu(float x) {
    const float hi = x * -1.44269504f, lo = __builtin_fmaf(x, -1.44269504f, -hi) - x * 1.92596303e-8f;
    const float e = __builtin_amdgcn_exp2f(hi);
    // 0 and infinity as they are
    return x * __builtin_amdgcn_rcpf(1.0f + (__builtin_fabsf(hi) < 126.0f ? __builtin_fmaf(e, lo * 0.693147182f, e) : e));
}

// 32 codes as fp16, exactly (NaN stays NaN), in order
typedef int fp8_v8i __attribute__((ext_vector_type(8)));
typedef _Float16 fp8_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 fp8_h8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void fp8_widen(const fp8_v8i& v, fp8_h8 (&o)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        fp8_h2 p[4];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            p[2 * d] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * q + d], 1.0f, false);
            p[2 * d + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * q + d], 1.0f, true);
        }
        o[q] = (fp8_h8){p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
    }
}

// maximum over the 16 lanes of a row (of a block, where a lane holds 8 channels)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ uint32_t row8_max(uint32_t v) {       // over each half of a row: where a lane holds 16 channels
    v = dpp_max<0xB1>(v);        // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);        // quad_perm [2,3,0,1]
    return dpp_max<0x141>(v);    // row_half_mirror
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) { return dpp_max<0x140>(row8_max(v)); }    // row_mirror

// eight bf16 or fp16 values as fp32
template <int DT>
__device__ __forceinline__ void fp8_unpack8(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == 0) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            v[2 * i] = f16_to_f32(u[i] & 0xffffu);
            v[2 * i + 1] = f16_to_f32(u[i] >> 16);
        }
    }
}
__device__ __forceinline__ uint32_t fp8_largest8(const float (&v)[8]) {
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
    return mx;
}

// Codes and scales of x: 256 threads take ROWS rows and 16 / ROWS blocks of each, a row of 16 lanes a block, and
// kFp8QuantSteps times that along K.  Sixteen rows together write a block's scales as 64 bytes.
// 4096 x 4096 bf16: 15 us, 3.4 TB/s; 51 x 4096 4.2 us, which is a launch and one way to memory.
constexpr int kFp8QuantSteps = 4;

struct Fp8QuantGrid {
    int rows;                                    // ROWS
    int64_t x, y;                                // groups of rows, of blocks
};
inline Fp8QuantGrid fp8_quant_grid(int64_t rows, int64_t K) {
    const int64_t KB = (K + 127) / 128;
    if (rows < 16) return {1, rows, (KB + 16 * kFp8QuantSteps - 1) / (16 * kFp8QuantSteps)};
    return {16, (rows + 15) / 16, (KB + kFp8QuantSteps - 1) / kFp8QuantSteps};
}

template <int DT, int ROWS>
__device__ __forceinline__ void fp8_quant(const uint16_t* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ s,
                                          int64_t rows, int K, int64_t stride, int gx, int gy, int tid) {
    constexpr int BLOCKS = 16 / ROWS;
    const int group = tid >> 4, l16 = tid & 15;
    const int64_t row = (int64_t)gx * ROWS + group % ROWS;
    const int KB = (K + 127) >> 7;
    const int64_t at = row < rows ? row : rows - 1;
    const uint16_t* px = x + at * stride;
    uint4 w[kFp8QuantSteps];
    const int b0 = gy * BLOCKS * kFp8QuantSteps + group / ROWS;
#pragma unroll
    for (int u = 0; u < kFp8QuantSteps; ++u) {
        const int k = (b0 + u * BLOCKS) * 128 + 8 * l16;
        w[u] = k < K ? *reinterpret_cast<const uint4*>(px + k) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kFp8QuantSteps; ++u) {
        const int b = b0 + u * BLOCKS, k = b * 128 + 8 * l16;
        float v[8];
        fp8_unpack8<DT>(w[u], v);
        const float amax = fp8_amax(row16_max(fp8_largest8(v)));
        if (row >= rows || b >= KB) continue;
        if (l16 == 0) s[(size_t)b * rows + row] = fp8_scale(amax);
        const Fp8Divisor by = fp8_divisor(amax);
        if (k < K)
            *reinterpret_cast<uint2*>(q + row * K + k) = make_uint2(fp8_codes4(v[0], v[1], v[2], v[3], by, amax != amax),
                                                                    fp8_codes4(v[4], v[5], v[6], v[7], by, amax != amax));
    }
}

}  // namespace
}  // namespace wush
