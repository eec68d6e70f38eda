// moe.hip -- a feed-forward layer of experts: the router's choice, and the experts'
// gated layers in e4m3.
//
// Route: s = softmax(x) or sigmoid(x), c = s + bias; of each group of experts the sum of its best one or
// two c, the best groups stay; ids are the k largest c left, equal ones by the lowest
// index; weights s[ids], divided by their sum or not, times a factor.  Without a bias x itself orders the experts, and groups by
// their best one; with one, and for sums of two, the choice is that of 64-bit scores.  Weights and their sums are in 64 bits.
//
// Experts: rows of x by expert; a = q(x) up_e^T, h = silu(a_gate) a_up, o = q(h) down_e^T, y = sum of w o over a
// token's experts.  a and h are kept in fp32, o too but for bf16's fused way (see experts_plan), h and x quantized as in fp8_device.h.
#include <cmath>
#include <type_traits>

#include "fp8.h"
#include "fp8_device.h"
#include "../../include/wush_int4.h"

namespace wush {
namespace {

// ------------------------------------------------------------------- the router
typedef unsigned long long u64;

// Order of floats (doubles) as that of unsigned integers; NaN below all, 0 left for "not there".
__device__ __forceinline__ uint32_t order_key(float c) {
    if (c != c) return 1;
    const uint32_t b = __float_as_uint(c + 0.0f);                // -0 is 0
    return b >> 31 ? ~b : b | 1u << 31;
}
__device__ __forceinline__ u64 order_key(double c) {
    if (c != c) return 1;
    const u64 b = __builtin_bit_cast(u64, c + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ float order_value(uint32_t key) {
    return key <= 1 ? __builtin_nanf("") : __uint_as_float(key >> 31 ? key & ~(1u << 31) : ~key);
}
__device__ __forceinline__ double order_value(u64 key) {
    return key <= 1 ? __builtin_nan("") : __builtin_bit_cast(double, key >> 63 ? key & ~(1ull << 63) : ~key);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ u64 lane_value(u64 v, int lane) {
    return (u64)lane_value((uint32_t)(v >> 32), lane) << 32 | lane_value((uint32_t)v, lane);
}

// Maximum over the wavefront, in every lane: rows by DPP as in row16_max, row_bcast:15 and :31 fold them into the last
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t dpp_max_rows(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max_rows<0x143, 0xc>(dpp_max_rows<0x142, 0xa>(row16_max(v)));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ u64 wave_max(u64 v) {
    const uint32_t hi = wave_max((uint32_t)(v >> 32));
    return (u64)hi << 32 | wave_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

struct RouteArgs {
    const void* logits;
    int64_t stride;
    const float* bias;
    float* weights;
    int32_t* ids;
    int64_t rows;
    int dtype, E, k, groups, size, keep, best;   // size: experts of a group
    int lanes, shift;                            // of a group: a power of two, and its logarithm
    int sigmoid, renorm;
    float scale;
};

__device__ __forceinline__ float logit(const RouteArgs& p, int64_t row, int e) {
    const int64_t at = row * p.stride + e;
    if (p.dtype == WUSH_DTYPE_F32) return static_cast<const float*>(p.logits)[at];
    const uint32_t w = static_cast<const uint16_t*>(p.logits)[at];
    return p.dtype == WUSH_DTYPE_BF16 ? bf16_to_f32(w) : f16_to_f32(w);
}
__device__ __forceinline__ double sigmoid64(float x) { return 1.0 / (1.0 + exp(-(double)x)); }

// The k experts of the largest keys, equal ones by index, choice j and its key in lane j; `key` keeps what is not chosen.
// One lane holds a maximum but for equal keys: a ballot names it, and only for those the indexes are compared too.
// (Halving towards a border that k keys reach instead: 16384 x 256 23.5 us for 22.5, but 4096 x 128 in bf16, where
// equal keys are common and take every step, 8.6 for 5.5.)
template <int V, typename Key>
__device__ __forceinline__ void largest(Key (&key)[V], int first, int lanes, int lane, int k, int& id, Key& taken) {
    id = 0;
    taken = 0;
    for (int j = 0; j < k; ++j) {
        Key top = key[0];
        int e = first;
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (key[i] > top) {
                top = key[i];
                e = first + lanes * i;
            }
        const Key most = wave_max(top);
        const u64 at = __ballot(top == most);
        int chosen;
        if (at & (at - 1)) chosen = (int)~wave_max(top == most ? ~(uint32_t)e : 0u);
        else chosen = __builtin_amdgcn_readlane(e, __builtin_ctzll(at));
        if (lane == j) {
            id = chosen;
            taken = most;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (first + lanes * i == chosen && key[i] == most) key[i] = 0;
    }
}

// A group's two largest keys, in all of its lanes
template <int V, typename Key>
__device__ __forceinline__ void two_largest(const Key (&key)[V], int lanes, Key& a, Key& b) {
    a = b = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        b = max(b, min(a, key[i]));
        a = max(a, key[i]);
    }
    for (int d = 1; d < lanes; d <<= 1) {
        const Key oa = __shfl_xor(a, d), ob = __shfl_xor(b, d);
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
    }
}
// Groups whose score is above that of this lane's, equal ones by index
template <typename Key>
__device__ __forceinline__ int groups_above(Key score, const RouteArgs& p, int group) {
    int above = 0;
    for (int g = 0; g < p.groups; ++g) {
        const Key o = lane_value(score, g << p.shift);
        above += o > score || (o == score && g < group);
    }
    return above;
}

// A wavefront per row.  Lane group * lanes + sub holds experts group * size + sub + lanes * i.
// Without a bias (BIAS false) the logits order the experts as the scores do: 32-bit keys of logits, and scores of the
// chosen ones only, and of all for softmax's sum.  With one, scores in 32 bits decide wherever they are further apart than their
// errors: s is off by less than 2^-20 (a few units of the last bit; softmax, with a sum of up to 38 roundings, 2^-17), c = s + b by
// 2^-24 |c| more, and a sum of two by both of theirs and 2^-24 of itself: by magnitudes, since biases of opposite signs leave
// a small sum of large c.  A row in which two that matter are nearer, or that holds what is not finite, is chosen again in 64 bits.
// 4096 x 128 bf16, 8 of them: 5.5 us.  16384 x 256 fp32 with a bias, 8 groups: 23 us (64 bits throughout: 28), where
// the choices' chain of maxima and the chosen scores' exponentials bound it, not the 17 MB (3.4 us).  A row on 16 lanes instead
// of 64, which shares that chain among four rows, takes 30: one row that is chosen again holds up three.
template <int V, bool BIAS>
__global__ __launch_bounds__(256) void moe_route_kernel(const RouteArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const int group = lane >> p.shift, sub = lane & (p.lanes - 1), first = group * p.size + sub;
    const bool there = group < p.groups;
    float x[V], b[V];
    bool in[V];
    int at[V];                                   // every lane loads, at once: no branches between the loads
#pragma unroll
    for (int i = 0; i < V; ++i) {
        in[i] = there && sub + p.lanes * i < p.size;
        at[i] = in[i] ? first + p.lanes * i : 0;
    }
    if (p.dtype == WUSH_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = static_cast<const float*>(p.logits)[row * p.stride + at[i]];
    } else {
        uint32_t u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = static_cast<const uint16_t*>(p.logits)[row * p.stride + at[i]];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p.dtype == WUSH_DTYPE_BF16 ? bf16_to_f32(u[i]) : f16_to_f32(u[i]);
    }
    if constexpr (BIAS) {
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = p.bias[at[i]];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!in[i]) x[i] = -__builtin_inff();
        if (!BIAS || !in[i]) b[i] = 0.0f;
    }
    // softmax: the largest logit, whether the scores are NaN (inf - inf among them), and their sum where it is needed
    float mx = 0.0f;
    bool bad = false, nan = false;
    if (BIAS || !p.sigmoid) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            top = max(top, order_key(x[i]));
            nan |= x[i] != x[i];
        }
        nan = __any(nan);
        if (!p.sigmoid) {
            mx = order_value(wave_max(top));
            bad = nan || mx == __builtin_inff();
            if (!bad && mx == -__builtin_inff()) mx = 0.0f;      // nothing but -inf: every score 0
        }
    }
    double total = 1.0;
    auto sum64 = [&] {
        total = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) total += exp((double)x[i] - (double)mx);
        total = wave_sum(total);
        if (total == 0.0) total = 1.0;
    };
    if (!p.sigmoid && !p.renorm) sum64();

    int id;                                      // lane j: choice j
    if constexpr (!BIAS) {
        uint32_t key[V];
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = in[i] ? bad ? 1u : order_key(x[i]) : 0u;
        if (p.groups > 1) {
            uint32_t one, two;
            two_largest<V>(key, p.lanes, one, two);
            int above;
            if (p.best == 1) above = groups_above(one, p, group);
            else if (p.sigmoid) above = groups_above(order_key(sigmoid64(order_value(one)) + sigmoid64(order_value(two))), p, group);
            else above = groups_above(bad ? (u64)1 : order_key(exp((double)order_value(one) - (double)mx) + exp((double)order_value(two) - (double)mx)), p, group);
            if (above >= p.keep) {
#pragma unroll
                for (int i = 0; i < V; ++i) key[i] = 0;
            }
        }
        uint32_t taken;
        largest<V>(key, first, p.lanes, lane, p.k, id, taken);
    } else {
        const float kApart = p.sigmoid ? 0x1p-19f : 0x1p-16f;    // twice the errors
        constexpr float kPart = 0x1p-22f;
        uint32_t key[V];
        float sum = 0.0f, c[V];
        bool odd = bad || nan, wild = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // 1 / (1 + exp(-x)), or exp(x - max)
            const float e = __builtin_amdgcn_exp2f((p.sigmoid ? -x[i] : x[i] - mx) * 1.44269504f);
            c[i] = p.sigmoid ? __builtin_amdgcn_rcpf(1.0f + e) : e;
            sum += c[i];
        }
        const float by = p.sigmoid ? 1.0f : __builtin_amdgcn_rcpf(wave_sum_dpp(sum));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = c[i] * by + b[i];
            wild |= in[i] && !(__builtin_fabsf(c[i]) < 0x1p100f);
            key[i] = in[i] ? order_key(c[i]) : 0u;
        }
        odd |= __any(wild);
        if (p.groups > 1) {
            uint32_t one, two;
            two_largest<V>(key, p.lanes, one, two);
            const uint32_t score = p.best == 1 ? one : order_key(order_value(one) + order_value(two));
            const bool keep = groups_above(score, p, group) < p.keep;
            // the least of the groups that stay and the largest of the others
            const float last = order_value(~wave_max(keep && there ? ~score : 0u));
            const uint32_t out = wave_max(!keep && there ? score : 0u);
            // the errors' size, of any group: the two at the border may not have the largest
            const float size = p.best == 1 ? __builtin_fabsf(last) : __builtin_fabsf(order_value(one)) + __builtin_fabsf(order_value(two));
            odd |= out != 0 && __any(there && !(last - order_value(out) > 2.0f * (kApart + kPart * size)));
            if (!keep) {
#pragma unroll
                for (int i = 0; i < V; ++i) key[i] = 0;
            }
        }
        uint32_t taken;
        largest<V>(key, first, p.lanes, lane, p.k, id, taken);
        // each choice against the next, the last against the largest left
        uint32_t rest = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) rest = max(rest, key[i]);
        rest = wave_max(rest);
        uint32_t next = (uint32_t)__shfl((int)taken, lane + 1);
        if (lane == p.k - 1) next = rest;
        const float v = order_value(taken);
        odd |= __any(lane < p.k && next != 0 && !(v - order_value(next) > kApart + kPart * __builtin_fabsf(v)));
        if (odd) {
            if (!p.sigmoid && p.renorm) sum64();
            u64 key[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                double c = __builtin_nan("");
                if (in[i] && !bad) c = (p.sigmoid ? sigmoid64(x[i]) : exp((double)x[i] - (double)mx) / total) + (double)b[i];
                key[i] = in[i] ? order_key(c) : 0;
            }
            if (p.groups > 1) {
                u64 one, two;
                two_largest<V>(key, p.lanes, one, two);
                if (groups_above(p.best == 1 ? one : order_key(order_value(one) + order_value(two)), p, group) >= p.keep) {
#pragma unroll
                    for (int i = 0; i < V; ++i) key[i] = 0;
                }
            }
            u64 taken;
            largest<V>(key, first, p.lanes, lane, p.k, id, taken);
        }
    }
    // the chosen ones' scores
    const bool mine = lane < p.k;
    const float c = mine ? logit(p, row, id) : 0.0f;
    double w = !mine ? 0.0 : p.sigmoid ? sigmoid64(c) : bad ? __builtin_nan("") : exp((double)c - (double)mx);
    if (p.renorm) {
        const double sum = wave_sum(w);
        w = sum > 0.0 || sum != sum ? w / sum : 0.0;
    } else {
        w /= total;
    }
    if (mine) {
        p.weights[row * p.k + lane] = (float)(w * (double)p.scale);
        p.ids[row * p.k + lane] = id;
    }
}

template <int V>
void launch_route_v(const RouteArgs& a, hipStream_t stream) {
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    if (a.bias) moe_route_kernel<V, true><<<grid, 256, 0, stream>>>(a);
    else moe_route_kernel<V, false><<<grid, 256, 0, stream>>>(a);
}
// a launch has fewer than 2^32 threads: kRouteRows rows each
constexpr int64_t kRouteRows = 1 << 25;

int launch_route(RouteArgs a, hipStream_t stream) {
    const int v = (a.size + a.lanes - 1) / a.lanes;
    for (int64_t left = a.rows; left > 0; left -= kRouteRows) {
        a.rows = left < kRouteRows ? left : kRouteRows;
        if (v <= 1) launch_route_v<1>(a, stream);
        else if (v <= 2) launch_route_v<2>(a, stream);
        else if (v <= 4) launch_route_v<4>(a, stream);
        else if (v <= 8) launch_route_v<8>(a, stream);
        else if (v <= 16) launch_route_v<16>(a, stream);
        else launch_route_v<32>(a, stream);
        const int st = (int)hipGetLastError();
        if (st) return st;
        a.logits = static_cast<const uint8_t*>(a.logits) + kRouteRows * a.stride * (a.dtype == WUSH_DTYPE_F32 ? 4 : 2);
        a.weights += kRouteRows * a.k;
        a.ids += kRouteRows * a.k;
    }
    return (int)hipSuccess;
}

// ------------------------------------------------------------------- the experts
// Rows by expert.  One workgroup per kSortPairs (token, choice) pairs; each counts all
// pairs' experts for itself, those before its own apart, and so needs no other: row = the
// expert's first + its pairs in earlier workgroups + the rank among this one's.  The last two come
// from an LDS counter: which of an expert's rows a pair gets may differ from call to call, what
// is computed in that row does not depend on it.
// Alone, 408 pairs of 128 experts 3.8 us, 32768 10 us (their counts, 32 loads deep in each workgroup): latency.
constexpr int kSortThreads = 1024, kSortPairs = 1024, kMostExperts = 1024;

// The workgroups behind those `sorts` quantize x meanwhile, in four parts of 256 threads: 51 tokens 5 us, 4096 tokens 18
// (a launch for each: 4.8 and 4.8, 11 and 15).
struct BeginArgs {
    const int32_t* ids;
    int P, k, E, tile_rows;
    int *row_of, *pos, *ntiles;
    int4* tiles;
    const uint16_t* x;
    uint8_t* q;
    float* s;
    int64_t rows, stride;
    int K, sorts, gx, gy;
};
template <int DT, int ROWS>
__global__ __launch_bounds__(kSortThreads) void moe_begin_kernel(const BeginArgs a) {
    if ((int)blockIdx.x >= a.sorts) {
        const int part = ((int)blockIdx.x - a.sorts) * (kSortThreads / 256) + ((int)threadIdx.x >> 8);
        if (part < a.gx * a.gy) fp8_quant<DT, ROWS>(a.x, a.q, a.s, a.rows, a.K, a.stride, part % a.gx, part / a.gx, (int)threadIdx.x & 255);
        return;
    }
    const int32_t* __restrict__ ids = a.ids;
    const int P = a.P, k = a.k, E = a.E, tile_rows = a.tile_rows;
    int* __restrict__ row_of = a.row_of;
    int* __restrict__ pos = a.pos;
    int4* __restrict__ tiles = a.tiles;
    int* __restrict__ ntiles = a.ntiles;
    __shared__ int all[kMostExperts], before[kMostExperts], start[kMostExperts], tile0[kMostExperts];
    __shared__ int wave_rows[kSortThreads / 64], wave_tiles[kSortThreads / 64];
    const int tid = threadIdx.x, first = blockIdx.x * kSortPairs;
    all[tid] = before[tid] = 0;
    __syncthreads();
    const int own = first + tid < P ? ids[first + tid] : -1;
    const int mine = (unsigned)own < (unsigned)E ? own : -1;
    constexpr int kAhead = 8;                    // loads in flight
    for (int p0 = 0; p0 < P; p0 += kAhead * kSortThreads) {
        int e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int p = p0 + u * kSortThreads + tid;
            e[u] = p < P ? ids[p] : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int run = p0 + u * kSortThreads;               // one workgroup's
            if (run != first && (unsigned)e[u] < (unsigned)E) atomicAdd(run < first ? &before[e[u]] : &all[e[u]], 1);
        }
    }
    __syncthreads();
    int rank = 0;                                // among the expert's pairs up to this workgroup's
    if (mine >= 0) rank = atomicAdd(&before[mine], 1);
    __syncthreads();
    // exclusive sums over the experts, one a thread
    const int n = before[tid] + all[tid], t = (n + tile_rows - 1) / tile_rows;
    int sn = n, stl = t;
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int a = __shfl_up(sn, d), c = __shfl_up(stl, d);
        if (lane >= d) {
            sn += a;
            stl += c;
        }
    }
    if (lane == 63) {
        wave_rows[wave] = sn;
        wave_tiles[wave] = stl;
    }
    __syncthreads();
    int on = 0, ot = 0;
    for (int w = 0; w < wave; ++w) {
        on += wave_rows[w];
        ot += wave_tiles[w];
    }
    start[tid] = on + sn - n;
    tile0[tid] = ot + stl - t;
    __syncthreads();
    if (first + tid < P) {
        int r = -1;
        if (mine >= 0) {
            r = start[mine] + rank;
            row_of[r] = (first + tid) / k;
        }
        pos[first + tid] = r;
    }
    if (blockIdx.x == 0) {
        if (tid < E)
            for (int i = 0; i < t; ++i) tiles[tile0[tid] + i] = make_int4(tid, start[tid] + i * tile_rows, start[tid] + n, 0);
        if (tid == kSortThreads - 1) *ntiles = ot + stl;
    }
}

int launch_begin(const BeginArgs& a, int dtype, int rows, hipStream_t stream) {
    constexpr int parts = kSortThreads / 256;
    const unsigned grid = (unsigned)(a.sorts + (a.gx * a.gy + parts - 1) / parts);
    if (dtype == WUSH_DTYPE_BF16) {
        if (rows == 1) moe_begin_kernel<WUSH_DTYPE_BF16, 1><<<grid, kSortThreads, 0, stream>>>(a);
        else moe_begin_kernel<WUSH_DTYPE_BF16, 16><<<grid, kSortThreads, 0, stream>>>(a);
    } else {
        if (rows == 1) moe_begin_kernel<WUSH_DTYPE_F16, 1><<<grid, kSortThreads, 0, stream>>>(a);
        else moe_begin_kernel<WUSH_DTYPE_F16, 16><<<grid, kSortThreads, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
}

// h = silu(gate) * up of a row's 128 channels, quantized: 16 lanes a block
__global__ __launch_bounds__(256) void moe_act_kernel(const float* __restrict__ a, uint8_t* __restrict__ q,
                                                      float* __restrict__ s, int I, int64_t ld,
                                                      const int4* __restrict__ tiles, const int* __restrict__ ntiles) {
    const int nt = *ntiles, rows = nt ? tiles[nt - 1].z : 0;
    const int l16 = threadIdx.x & 15, blocks = I >> 7;
    const int64_t total = (int64_t)rows * blocks;
    for (int64_t u = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); u < total; u += (int64_t)gridDim.x * 16) {
        const int64_t row = u / blocks;
        const int b = (int)(u - row * blocks), c = b * 128 + 8 * l16;
        const float4* g = reinterpret_cast<const float4*>(a + row * 2 * I + c);
        const float4* p = reinterpret_cast<const float4*>(a + row * 2 * I + I + c);
        const float4 g0 = g[0], g1 = g[1], p0 = p[0], p1 = p[1];
        const float gate[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
        const float up[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fp8_silu(gate[i]) * up[i];
        const float amax = fp8_amax(row16_max(fp8_largest8(v))), factor = fp8_factor(amax);
        if (l16 == 0) s[b * ld + row] = fp8_scale(amax);
        *reinterpret_cast<uint2*>(q + row * I + c) =
            make_uint2(fp8_codes4_by(v[0], v[1], v[2], v[3], factor), fp8_codes4_by(v[4], v[5], v[6], v[7], factor));
    }
}

__device__ __forceinline__ uint16_t out_bits(float f, int dt) {
    return dt == WUSH_DTYPE_F16 ? f32_to_f16_bits(f) : (uint16_t)(f != f ? 0x7fc0u : f32_to_bf16_rne(f));
}

// y of a token: the sum of its experts' rows, in the order of its choices; 8 columns a thread.
// SHARED: rows are fp16 with a power of two for each 64 columns.  4096 x 8 rows of 4096: 55 us, 5.5 TB/s, with four rows in
// flight (one: 78).
template <bool SHARED>
__global__ __launch_bounds__(256) void moe_sum_kernel(const void* __restrict__ o, const float* __restrict__ os,
                                                      const int* __restrict__ pos, const float* __restrict__ weights,
                                                      uint16_t* __restrict__ y, int dt, int64_t T, int k, int H) {
    const int units = H >> 3;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = at / units;
    if (t >= T) return;
    const int c = (int)(at - t * units) * 8;
    float v[8] = {};
    constexpr int kAhead = 4;                    // rows in flight
    for (int j0 = 0; j0 < k; j0 += kAhead) {
        int r[kAhead];
        float w[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t j = t * k + min(j0 + u, k - 1);
            r[u] = j0 + u < k ? pos[j] : -1;
            w[u] = weights[j];
        }
        if constexpr (SHARED) {
            uint4 h[kAhead];
            float by[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t row = max(r[u], 0);
                by[u] = os[row * ((H + 63) >> 6) + (c >> 6)];
                h[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(o) + row * H + c);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (r[u] < 0) continue;
                float f[8];
                fp8_unpack8<WUSH_DTYPE_F16>(h[u], f);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(w[u] * by[u], f[i], v[i]);
            }
        } else {
            float4 f[kAhead][2];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(o) + (int64_t)max(r[u], 0) * H + c);
                f[u][0] = p[0], f[u][1] = p[1];
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (r[u] < 0) continue;
                const float g[8] = {f[u][0].x, f[u][0].y, f[u][0].z, f[u][0].w, f[u][1].x, f[u][1].y, f[u][1].z, f[u][1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(w[u], g[i], v[i]);
            }
        }
    }
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = out_bits(v[2 * i], dt) | (uint32_t)out_bits(v[2 * i + 1], dt) << 16;
    uint16_t* p = y + t * H + c;
    if ((reinterpret_cast<uintptr_t>(y) & 15u) == 0) *reinterpret_cast<uint4*>(p) = make_uint4(out[0], out[1], out[2], out[3]);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(out[i >> 1] >> (16 * (i & 1)));
}

// ------------------------------------------------------------ sizes of a call
// Tokens go through in runs of at most kRunPairs pairs: the workspace does not grow beyond that,
// and offsets of rows of x and h within a run stay below 2^32.
constexpr int64_t kRunPairs = 65536;

struct ExpertsPlan {
    int64_t tokens, pairs;                       // of a run
    bool few, fused, shared, once;               // see experts_plan
    int tile_rows, most_tiles;
    size_t xq, xs, row_of, pos, tiles, ntiles, a, hq, hs, o, os, bytes;
};

// Three ways.
// A few tokens: dot products that read an expert's weights for each choice (fp8_gemv.hip).
// Fused: tiles of 64 or 128 x 256, one after another (gemm_fp8_runs.hip), whose epilogue makes the hidden codes.  Experts'
// rows are fp32 for fp16, and for bf16 fp16 with shared powers of two, 2^-12 of a value where y's own rounding is up to 2^-8 of it.
// Otherwise (few rows an expert, and few workgroups of the other kind): tiles of 32 x 64, and intermediate rows in fp32.
// Both take the gate and up products on the fp16 matrix instruction, which cuts none, at half the e4m3 one's rate and with the codes
// widened first.  The e4m3 instruction cuts small products next to large ones, at 2^-13 of the largest of 8: where a
// channel in a hundred is twenty times the others that turns 3 in 1000 of the hidden codes to the other side of a half, 1.1e-3 to
// 2.1e-3 of the output, as much as all of bf16's rounding (1.7e-3) and ten times fp16's (4096 tokens, 8 of 128 experts of
// 4096 x 1024, bf16: 764 us for 1015; 51 tokens 184 for 190).  The down products are cut: 4e-5 of the output.
// us, bf16, by tokens, three ways (dots, 32, 64 rows): 64 experts of 2048 x 1408, 6 choices: 4: 43, 49, 45;
// 8: 62, 60, 67; 64: -, 92, 100; 256: -, 167, 124; 1024: -, 430, 203.  8 of 4096 x
// 1792, 2 choices: 4: 30, 40, 56; 8: 43, 43, 58; 48: -, 53, 60; 256: -, 111, 70; 512: -, 173, 93.
// Fused from 12 rows an expert on, or where the gate and up projections have 640 workgroups' columns, two and a half for each CU:
// over nine layers (8 experts of 4096 x 14336 to 256 of 2048 x 512) and 1/4 to 16 rows an expert, both types, 1.6% behind
// the faster on average; by rows alone 2.5%.  4 and 8 rows, 64 rows' time over 32's: 256 of 2048 x 512 0.92, 0.84; 128 of
// 4096 x 1024 1.00, 0.98; 8 of 4096 x 1792 1.29, 1.33.
// 64 or 128 rows: over eight layers of those and 24 to 128 rows an expert, both types, a border of 80 is 0.7% behind the faster
// on average with all choices here (56: 1.7%; 72 and 96: 0.9%; 112: 1.5%), and with half of them here as well, which the host
// does not see, 1.4% (96: 1.2%).  64 rows' time over 128's at 56, 80 and 96: bf16 0.91, 1.00, 1.03, fp16 0.94, 0.96, 1.02; at 80
// with half of the choices here 0.92, 0.93.
ExpertsPlan experts_plan(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int dtype) {
    ExpertsPlan p = {};
    // us: every choice reads its expert's weights; tiles read each expert once that some choice meets, after some launches
    const double each = 3.0 * (double)H * (double)I / 6.5e6, met = (double)E * (1.0 - std::pow(1.0 - (k < E ? (double)k / (double)E : 1.0), (double)T));
    if ((p.few = fp8_experts_gemv_shape(T, k, H, I) && 9.0 + (double)(T * k) * each < 22.0 + 1.05 * met * each)) {
        p.tokens = T;
        p.bytes = (size_t)(T * k) * I * 4;       // h
        return p;
    }
    int64_t most = kRunPairs / k;
    if (most * H > 0x7fffffffLL) most = 0x7fffffffLL / H;
    if (most * k * I > 0x7fffffffLL) most = 0x7fffffffLL / (k * I);
    p.tokens = T < most ? T : most;
    p.pairs = p.tokens * k;
    const double rows = (double)p.pairs / (double)E;
    p.fused = rows > 12 || met * (double)(I / 128) >= 640;
    p.shared = p.fused && dtype == WUSH_DTYPE_BF16;
    p.tile_rows = !p.fused ? kFp8RowsTile : rows <= 80 ? 64 : 128;
    p.once = rows <= 30;                         // mostly one tile an expert
    p.most_tiles = (int)(p.pairs / p.tile_rows + (p.pairs < E ? p.pairs : E));
    auto take = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += (n + 255) & ~(size_t)255;
        return at;
    };
    p.xq = take((size_t)p.tokens * H);
    p.xs = take((size_t)p.tokens * ((H + 127) / 128) * 4);
    p.row_of = take((size_t)p.pairs * 4);
    p.pos = take((size_t)p.pairs * 4);
    p.tiles = take((size_t)p.most_tiles * 16);
    p.ntiles = take(4);
    p.a = take(p.fused ? 0 : (size_t)p.pairs * 2 * I * 4);
    p.hq = take((size_t)p.pairs * I);
    p.hs = take((size_t)p.pairs * (I / 128) * 4);
    p.o = take((size_t)p.pairs * H * (p.shared ? 2 : 4));
    p.os = take(p.shared ? (size_t)p.pairs * ((H + 63) / 64) * 4 : 0);
    return p;
}

bool experts_sizes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
    return T >= 0 && T <= (1 << 26) && k >= 1 && k <= 64 && E >= 1 && E <= kMostExperts && H > 0 && H % 16 == 0 &&
           H <= WUSH_FP8_MAX_K && I > 0 && I % 128 == 0 && I <= WUSH_FP8_MAX_K;
}

}  // namespace
}  // namespace wush

extern "C" {

int wush_moe_route(const void* logits, int dtype, int64_t row_stride, const float* bias, int64_t rows, int64_t experts,
                   const wush_moe_choice* choice, float* weights, int32_t* ids, hipStream_t stream) {
    WUSH_REQUIRE(choice && rows >= 0 && rows <= 0x7fffffffLL && experts >= 1 && experts <= WUSH_MOE_MAX_EXPERTS);
    const wush_moe_choice& c = *choice;
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16 || dtype == WUSH_DTYPE_F32);
    WUSH_REQUIRE(c.groups >= 1 && c.groups <= 64 && experts % c.groups == 0 && c.keep_groups >= 1 && c.keep_groups <= c.groups);
    const int64_t size = experts / c.groups;
    WUSH_REQUIRE(c.k >= 1 && c.k <= WUSH_MOE_MAX_CHOICES && c.k <= c.keep_groups * size);
    WUSH_REQUIRE((c.group_best == 1 || c.group_best == 2) && c.group_best <= size);
    WUSH_REQUIRE(c.scale - c.scale == 0.0f);
    if (rows == 0) return (int)hipSuccess;
    WUSH_REQUIRE(logits && weights && ids && (rows == 1 || row_stride >= 0));
    WUSH_REQUIRE(((uintptr_t)logits & (dtype == WUSH_DTYPE_F32 ? 3u : 1u)) == 0 &&
                 (((uintptr_t)bias | (uintptr_t)weights | (uintptr_t)ids) & 3u) == 0);
    wush::RouteArgs a;
    a.logits = logits;
    a.stride = rows == 1 ? 0 : row_stride;
    a.bias = bias;
    a.weights = weights;
    a.ids = ids;
    a.rows = rows;
    a.E = (int)experts;
    a.k = c.k;
    a.groups = c.groups;
    a.size = (int)size;
    a.keep = c.keep_groups;
    a.best = c.group_best;
    a.lanes = 64;
    a.shift = 6;
    while (a.lanes * c.groups > 64) {
        a.lanes >>= 1;
        --a.shift;
    }
    a.dtype = dtype;
    a.sigmoid = c.sigmoid != 0;
    a.renorm = c.renorm != 0;
    a.scale = c.scale;
    return wush::launch_route(a, stream);
}

size_t wush_moe_experts_fp8_workspace_bytes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int dtype) {
    if (!wush::experts_sizes(T, k, E, H, I) || T == 0) return 0;
    return wush::experts_plan(T, k, E, H, I, dtype).bytes;
}

int wush_moe_experts_fp8_plan(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int dtype, int32_t plan[4]) {
    WUSH_REQUIRE(plan && T > 0 && wush::experts_sizes(T, k, E, H, I));
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    const wush::ExpertsPlan p = wush::experts_plan(T, k, E, H, I, dtype);
    plan[0] = p.few ? WUSH_MOE_DOT : p.fused ? WUSH_MOE_FUSED : WUSH_MOE_ROWS;
    plan[1] = p.tile_rows;
    plan[2] = p.once;
    plan[3] = (int32_t)p.tokens;
    return (int)hipSuccess;
}

int wush_moe_experts_fp8(const void* x, int dtype, int64_t row_stride, const float* weights, const int32_t* ids,
                         const uint8_t* w_up, const float* s_up, const uint8_t* w_down, const float* s_down, void* y,
                         int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
    WUSH_REQUIRE(wush::experts_sizes(T, k, E, H, I));
    WUSH_REQUIRE(dtype == WUSH_DTYPE_BF16 || dtype == WUSH_DTYPE_F16);
    if (T == 0) return (int)hipSuccess;
    const wush::ExpertsPlan p = wush::experts_plan(T, k, E, H, I, dtype);
    WUSH_REQUIRE(x && weights && ids && w_up && s_up && w_down && s_down && y && workspace && workspace_bytes >= p.bytes);
    WUSH_REQUIRE((((uintptr_t)x | (uintptr_t)w_up | (uintptr_t)w_down | (uintptr_t)workspace) & 15u) == 0 && ((uintptr_t)y & 1u) == 0);
    WUSH_REQUIRE((((uintptr_t)weights | (uintptr_t)ids | (uintptr_t)s_up | (uintptr_t)s_down) & 3u) == 0);
    WUSH_REQUIRE(T == 1 || (row_stride >= 0 && row_stride % 8 == 0));
    if (T == 1) row_stride = 0;
    if (p.few) {
        const wush::Fp8Experts a = {x, row_stride, weights, ids, w_up, w_down, s_up, s_down, static_cast<float*>(workspace), y, dtype,
                                    (int)T, (int)k, (int)E, (int)H, (int)I};
        return wush::launch_fp8_experts_gemv(a, stream);
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const uint16_t* px = static_cast<const uint16_t*>(x);
    uint16_t* py = static_cast<uint16_t*>(y);
    int* row_of = reinterpret_cast<int*>(ws + p.row_of);
    int* pos = reinterpret_cast<int*>(ws + p.pos);
    int4* tiles = reinterpret_cast<int4*>(ws + p.tiles);
    int* ntiles = reinterpret_cast<int*>(ws + p.ntiles);
    float* a = reinterpret_cast<float*>(ws + p.a);
    float* hs = reinterpret_cast<float*>(ws + p.hs);
    float* os = reinterpret_cast<float*>(ws + p.os);
    for (int64_t t = 0; t < T; t += p.tokens) {
        const int64_t n = T - t < p.tokens ? T - t : p.tokens;
        const int P = (int)(n * k);
        const wush::Fp8QuantGrid qg = wush::fp8_quant_grid(n, H);
        const wush::BeginArgs b = {ids + t * k, P, (int)k, (int)E, p.tile_rows, row_of, pos, ntiles, tiles, px + t * row_stride,
                                   ws + p.xq, reinterpret_cast<float*>(ws + p.xs), n, row_stride, (int)H,
                                   (P + wush::kSortPairs - 1) / wush::kSortPairs, (int)qg.x, (int)qg.y};
        int st = wush::launch_begin(b, dtype, qg.rows, stream);
        if (st) return st;
        wush::Fp8Gemm g = {};
        g.x = ws + p.xq;
        g.xs = reinterpret_cast<float*>(ws + p.xs);
        g.ldx = n;
        g.w = w_up;
        g.ws = s_up;
        g.out = wush::kOutF32;
        g.M = P;
        g.N = (int)(2 * I);
        g.K = (int)H;
        g.splits = 1;
        g.tiles = tiles;
        g.ntiles = ntiles;
        g.row_of = row_of;
        g.most_tiles = p.most_tiles;
        g.once = p.once;
        g.act = p.fused;
        g.wide = 1;
        g.y = p.fused ? static_cast<void*>(ws + p.hq) : a;
        g.hs = hs;
        g.ldh = p.pairs;
        st = p.fused ? wush::launch_gemm_fp8_runs(g, p.tile_rows, stream) : wush::launch_gemm_fp8_rows(g, stream);
        if (st) return st;
        if (!p.fused) {
            const int64_t blocks = ((int64_t)P * (I / 128) + 15) / 16;
            wush::moe_act_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(a, ws + p.hq, hs, (int)I, p.pairs, tiles, ntiles);
            if ((st = (int)hipGetLastError())) return st;
        }
        g.x = ws + p.hq;
        g.xs = hs;
        g.ldx = p.pairs;
        g.w = w_down;
        g.ws = s_down;
        g.y = ws + p.o;
        g.N = (int)H;
        g.K = (int)I;
        g.row_of = nullptr;
        g.act = g.wide = 0;
        g.shared = p.shared;
        g.hs = os;
        st = p.fused ? wush::launch_gemm_fp8_runs(g, p.tile_rows, stream) : wush::launch_gemm_fp8_rows(g, stream);
        if (st) return st;
        const unsigned grid = (unsigned)((n * (H / 8) + 255) / 256);
        if (p.shared) wush::moe_sum_kernel<true><<<grid, 256, 0, stream>>>(ws + p.o, os, pos, weights + t * k, py + t * H, dtype, n, (int)k, (int)H);
        else wush::moe_sum_kernel<false><<<grid, 256, 0, stream>>>(ws + p.o, nullptr, pos, weights + t * k, py + t * H, dtype, n, (int)k, (int)H);
        if ((st = (int)hipGetLastError())) return st;
    }
    return (int)hipSuccess;
}

}  // extern "C"
