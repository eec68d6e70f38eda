// bindings.cpp -- the my_int4._C drop-in: the reference's 16 pybind11 ops
// (csrc/bindings.cpp:28-68) with the same names, argument names, argument
// meaning, output dtypes/shapes and TORCH_CHECK error behaviour.  Each op
// validates and allocates with torch on the input's device, takes torch's
// current HIP stream, and calls the C ABI of libwush_int4.so
// (include/wush_int4.h).  No computation happens here.  Behind them, the 8-bit
// operators that the reference lacks (quant_int8_token, w8a8_*, kv8_*).
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <cmath>
#include <optional>
#include <vector>

#include "wush_int4.h"

namespace {

hipStream_t current_stream(const torch::Tensor& t) {
    return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void check_status(int st, const char* op) {
    TORCH_CHECK(st == 0, "my_int4._C.", op, ": ", wush_error_string(st));
}

template <typename T>
T* ptr(const torch::Tensor& t) {
    return reinterpret_cast<T*>(t.data_ptr());
}

c10::SmallVector<int64_t, 6> with_last(const torch::Tensor& t, int64_t last) {
    c10::SmallVector<int64_t, 6> s(t.sizes().begin(), t.sizes().end());
    s.back() = last;
    return s;
}

// Uninitialized contiguous tensor on t's device, straight from the caching
// allocator: every op here writes its outputs whole.  torch::empty goes
// through the dispatcher, 1.7 us a tensor against 3.3 us for a kernel launch;
// with it and views of flat outputs an eager M=1 K=N=4096 layer step (two
// launches) took 11.6 us of host time, without 8.2.  empty_cuda is not one of
// torch's documented interfaces, and dispatch modes do not see what it allocates.
torch::Tensor new_tensor(c10::IntArrayRef sizes, at::ScalarType dtype, const torch::Tensor& t) {
    return torch::Tensor(at::detail::empty_cuda(sizes, dtype, t.device(), std::nullopt));
}

// t as (rows, last), without a dispatched reshape where it is that already.
torch::Tensor as_rows(const torch::Tensor& t, int64_t last) {
    if (t.dim() == 2 && last > 0 && t.size(1) == last) return t;
    return t.reshape({-1, last});
}

// quant_int4 (csrc/quant_int4.cu:109-134).  Also accepts fp16/fp32 input,
// which my_int4/rtn_int4.py:36 quantizes the same way.
std::vector<torch::Tensor> quant_int4(torch::Tensor x) {
    TORCH_CHECK(x.is_cuda() && x.is_contiguous(), "x must be contiguous CUDA tensor");
    const auto dt = x.scalar_type();
    TORCH_CHECK(dt == torch::kBFloat16 || dt == torch::kHalf || dt == torch::kFloat32,
                "x must be bf16 (fp16 and fp32 are also accepted)");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) % 32 == 0, "last dim must be multiple of 32");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t n_groups = x.numel() / 32;
    auto q = new_tensor(with_last(x, x.size(-1) / 2), torch::kUInt8, x);
    auto s = new_tensor(with_last(x, x.size(-1) / 32), torch::kBFloat16, x);
    const int code = dt == torch::kBFloat16 ? WUSH_DTYPE_BF16 : (dt == torch::kHalf ? WUSH_DTYPE_F16 : WUSH_DTYPE_F32);
    check_status(wush_quant_int4(x.data_ptr(), code, ptr<uint8_t>(q), ptr<uint16_t>(s), n_groups,
                                 current_stream(x)),
                 "quant_int4");
    return {q, s};
}

// fused_transform_quant_int4 and its variants (csrc/fused_tq_int4.cu:87-118,
// fused_tq_smallm.cu:89-121, fused_tq_v3.cu:109-140, fused_tq_wmma.cu:131-162):
// one bit-exact implementation serves all four names.
std::vector<torch::Tensor> fused_tq_impl(torch::Tensor x, torch::Tensor t, bool need_rows) {
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && t.is_cuda() && t.is_contiguous(),
                "x/t must be contiguous CUDA tensors");
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16 && t.scalar_type() == torch::kBFloat16,
                "x/t must be bf16");
    TORCH_CHECK(x.dim() >= 1, "x must have a last dimension");
    const int64_t K = x.size(-1);
    const int64_t C = K / 32;
    TORCH_CHECK(K % 32 == 0 && t.dim() == 3 && t.size(0) == C && t.size(1) == 32 && t.size(2) == 32,
                "T must be (K/32, 32, 32)");
    const int64_t rows = K ? x.numel() / K : 0;
    if (need_rows) TORCH_CHECK(rows >= 1, "rows must be >= 1");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    auto q = new_tensor(with_last(x, K / 2), torch::kUInt8, x);
    auto s = new_tensor(with_last(x, C), torch::kBFloat16, x);
    check_status(wush_fused_tq(ptr<uint16_t>(x), ptr<uint16_t>(t), ptr<uint8_t>(q), ptr<uint16_t>(s),
                               rows, K, current_stream(x)),
                 "fused_transform_quant_int4");
    return {q, s};
}

std::vector<torch::Tensor> fused_transform_quant_int4(torch::Tensor x, torch::Tensor t) {
    return fused_tq_impl(x, t, false);
}
std::vector<torch::Tensor> fused_transform_quant_int4_smallm(torch::Tensor x, torch::Tensor t) {
    return fused_tq_impl(x, t, true);
}
std::vector<torch::Tensor> fused_transform_quant_int4_v3(torch::Tensor x, torch::Tensor t) {
    return fused_tq_impl(x, t, false);
}
std::vector<torch::Tensor> fused_transform_quant_int4_wmma(torch::Tensor x, torch::Tensor t) {
    return fused_tq_impl(x, t, false);
}

// Common checks of the packed GEMM operands (csrc/gemm_s4.cu:323-338).
void check_packed(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq,
                  const torch::Tensor& ws) {
    TORCH_CHECK(xq.is_cuda() && wq.is_cuda(), "tensors must be CUDA");
    TORCH_CHECK(xq.scalar_type() == torch::kUInt8 && wq.scalar_type() == torch::kUInt8,
                "packed tensors must be uint8");
    TORCH_CHECK(xs.scalar_type() == torch::kBFloat16 && ws.scalar_type() == torch::kBFloat16,
                "scales must be bf16");
    TORCH_CHECK(xq.is_contiguous() && xs.is_contiguous() && wq.is_contiguous() && ws.is_contiguous(),
                "tensors must be contiguous");
    TORCH_CHECK(xs.is_cuda() && ws.is_cuda(), "tensors must be CUDA");
}

// Which kernel family computes a product with M activation rows.  Both give
// the same math (exact int32 group dots folded in fp32).  Measured on MI355X
// with the weights streamed from HBM: the dot8 streaming GEMV
// (wush_gemv_int4) is faster at M <= 4 on every shape and at every M <= 8 on
// the Llama-70B FFN weights (K=8192 N=57344 M=8: 51.8 vs 55.4 us); the
// K-split int8-MFMA streaming GEMM (wush_gemm_s4) is faster at 5 <= M <= 8
// when N <= 24576 (K=N=4096 M=8: 5.8 vs 7.2 us; K=N=8192 M=8: 11.9 vs
// 13.3 us; K=4096 N=24576 M=8: 14.3 vs 15.0 us).  Which shapes the GEMV
// takes at all (its LDS staging limit, and the K-split kernel's shapes) is
// the library's rule, which its build-time tuning macros change, so it is
// asked, not restated here.
bool gemv_preferred(int64_t M, int64_t N, int64_t K) {
    return wush_gemv_int4_supported(M, N, K) != 0 && (M <= 4 || N > 32768);
}

// The product where the workspace of its plan does not fit the free memory:
// the same plan over fewer rows at a time, so that the result's bits do not
// depend on the memory that happens to be free.  Out of memory only if the
// workspace of 64 rows does not fit either.
torch::Tensor product_by_rows(const torch::Tensor& xq2, const torch::Tensor& xs2, const torch::Tensor& wq,
                              const torch::Tensor& ws, torch::Tensor y, int64_t M, int64_t N, int64_t K,
                              const char* op) {
    for (int64_t rows = (M + 63) / 64 * 64;; rows = (rows / 2 + 63) / 64 * 64) {
        const size_t wsb = wush_gemm_s4_rows_workspace_bytes(ptr<uint8_t>(xq2), ptr<uint16_t>(xs2), ptr<uint8_t>(wq),
                                                             ptr<uint16_t>(ws), M, N, K, rows);
        torch::Tensor work;
        try {
            if (wsb) work = new_tensor({(int64_t)wsb}, torch::kUInt8, xq2);
        } catch (const c10::OutOfMemoryError&) {
            if (rows <= 64) throw;
            continue;
        }
        check_status(wush_gemm_s4_rows(ptr<uint8_t>(xq2), ptr<uint16_t>(xs2), ptr<uint8_t>(wq), ptr<uint16_t>(ws),
                                       ptr<uint16_t>(y), M, N, K, rows, wsb ? work.data_ptr() : nullptr, wsb,
                                       current_stream(xq2)),
                     op);
        return y;
    }
}

// Shared product launch: y (M, N) fp16 = group-scaled product, in `sizes`
// (default (M, N)).
torch::Tensor product_2d(const torch::Tensor& xq2, const torch::Tensor& xs2, const torch::Tensor& wq,
                         const torch::Tensor& ws, int64_t K, const char* op, c10::IntArrayRef sizes = {}) {
    const int64_t M = xq2.size(0), N = wq.size(0);
    // the legacy ops' own checks leave the scale tensors' row counts open
    TORCH_CHECK(xs2.numel() >= M * (K / 32) && ws.numel() >= N * (K / 32), "K mismatch: fewer scales than groups");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(xq2.device());
    const int64_t mn[2] = {M, N};
    auto y = new_tensor(sizes.empty() ? c10::IntArrayRef(mn, 2) : sizes, torch::kHalf, xq2);
    if (gemv_preferred(M, N, K)) {
        check_status(wush_gemv_int4(ptr<uint8_t>(xq2), ptr<uint16_t>(xs2), ptr<uint8_t>(wq), ptr<uint16_t>(ws),
                                    ptr<uint16_t>(y), M, N, K, current_stream(xq2)),
                     op);
        return y;
    }
    const size_t wsb = wush_gemm_s4_best_workspace_bytes(M, N, K);
    torch::Tensor work;
    if (wsb) {
        try {
            work = new_tensor({(int64_t)wsb}, torch::kUInt8, xq2);
        } catch (const c10::OutOfMemoryError&) {
            return product_by_rows(xq2, xs2, wq, ws, y, M, N, K, op);
        }
    }
    check_status(wush_gemm_s4(ptr<uint8_t>(xq2), ptr<uint16_t>(xs2), ptr<uint8_t>(wq), ptr<uint16_t>(ws),
                              ptr<uint16_t>(y), M, N, K, wsb ? work.data_ptr() : nullptr, wsb,
                              current_stream(xq2)),
                 op);
    return y;
}

// w4a4_gemm_s4 (csrc/gemm_s4.cu:320-379): y (M, N) fp16, K % 64 == 0.
torch::Tensor w4a4_gemm_s4(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 64 == 0, "K must be multiple of 64");
    auto xq2 = as_rows(xq, K2);
    auto xs2 = as_rows(xs, G);
    TORCH_CHECK(wq.dim() == 2 && wq.size(1) == K2 && ws.size(-1) == G && ws.numel() == wq.size(0) * G,
                "K mismatch");
    TORCH_CHECK(xs2.size(0) == xq2.size(0), "K mismatch");
    return product_2d(xq2, xs2, wq, ws, K, "w4a4_gemm_s4");
}

// w4a4_gemm (csrc/gemm_int4.cu:89-130): y keeps xq's leading dims, (..., N).
torch::Tensor w4a4_gemm(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    TORCH_CHECK(wq.dim() == 2, "w must be 2D (N, K/2)");
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 32 == 0 && wq.size(1) == K2 && ws.size(-1) == G && xs.size(-1) == G,
                "K mismatch between x/w tensors");
    auto xq2 = xq.view({-1, K2});
    auto xs2 = xs.reshape({-1, G});
    auto y = product_2d(xq2, xs2, wq, ws, K, "w4a4_gemm");
    return y.view(with_last(xq, wq.size(0)));
}

// w4a4_gemm_v1 (csrc/gemm_wmma.cu:128-172): y (M, N).
torch::Tensor w4a4_gemm_v1(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 32 == 0 && wq.dim() == 2 && wq.size(1) == K2 && ws.size(-1) == G, "K mismatch");
    return product_2d(as_rows(xq, K2), as_rows(xs, G), wq, ws, K, "w4a4_gemm_v1");
}

// w4a4_gemm_v2 (csrc/gemm_wmma2.cu:141-181): y (M, N), K % 64 == 0.
torch::Tensor w4a4_gemm_v2(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 64 == 0, "K must be multiple of 64");
    TORCH_CHECK(wq.dim() == 2 && wq.size(1) == K2 && ws.size(-1) == G, "K mismatch");
    return product_2d(as_rows(xq, K2), as_rows(xs, G), wq, ws, K, "w4a4_gemm_v2");
}

// w4a4_gemv (csrc/gemv_int4.cu:191-223): single row, y (N,) fp16.
torch::Tensor w4a4_gemv(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    TORCH_CHECK(xq.dim() <= 2 && xq.numel() == xq.size(-1), "gemv expects a single row");
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 32 == 0 && wq.dim() == 2 && wq.size(1) == K2 && ws.size(-1) == G && xs.numel() == G,
                "K mismatch");
    const int64_t n[1] = {wq.size(0)};
    auto row = [](const torch::Tensor& t, int64_t last) {
        return t.dim() == 2 && t.size(0) == 1 && t.size(1) == last ? t : t.reshape({1, last});
    };
    return product_2d(row(xq, K2), row(xs, G), wq, ws, K, "w4a4_gemv", c10::IntArrayRef(n, 1));
}

// w4a4_gemv_multi (csrc/gemv_int4.cu:145-189): 1 <= M <= 8, y (M, N) fp16.
torch::Tensor w4a4_gemv_multi(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws) {
    check_packed(xq, xs, wq, ws);
    const int64_t K2 = xq.size(-1);
    const int64_t K = K2 * 2, G = K / 32;
    auto xq2 = as_rows(xq, K2);
    auto xs2 = as_rows(xs, G);
    const int64_t M = xq2.size(0);
    TORCH_CHECK(M >= 1 && M <= 8, "gemv_multi expects 1<=M<=8");
    TORCH_CHECK(K % 32 == 0 && wq.dim() == 2 && wq.size(1) == K2 && ws.size(-1) == G && xs2.size(0) == M,
                "K mismatch");
    return product_2d(xq2, xs2, wq, ws, K, "w4a4_gemv_multi");
}

// s4_atom_selftest (csrc/gemm_s4.cu:74-82): c (8, 8) int32 = a (8, 32) @ b (32, 8).
torch::Tensor s4_atom_selftest(torch::Tensor a, torch::Tensor b) {
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && a.is_contiguous() && b.is_contiguous(),
                "a/b must be contiguous CUDA tensors");
    TORCH_CHECK(a.scalar_type() == torch::kInt8 && b.scalar_type() == torch::kInt8, "a/b must be int8");
    TORCH_CHECK(a.numel() == 256 && b.numel() == 256, "a must be (8, 32) and b (32, 8)");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(a.device());
    auto c = torch::zeros({8, 8}, torch::dtype(torch::kInt32).device(a.device()));
    check_status(wush_mfma_selftest(ptr<int8_t>(a), ptr<int8_t>(b), ptr<int32_t>(c), current_stream(a)),
                 "s4_atom_selftest");
    return c;
}

// quant_int4_tensor_scale (csrc/fast_path.cu:42-59): flat (numel/2) codes,
// inverse scale (float)(1.0 / scale) computed in double like the reference.
torch::Tensor quant_int4_tensor_scale(torch::Tensor x, double scale) {
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.scalar_type() == torch::kBFloat16,
                "x must be contiguous CUDA bf16");
    TORCH_CHECK(x.numel() % 32 == 0, "numel must be multiple of 32");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    auto q = new_tensor({x.numel() / 2}, torch::kUInt8, x);
    const float inv = (float)(1.0 / scale);
    check_status(wush_quant_int4_tensor_scale(ptr<uint16_t>(x), ptr<uint8_t>(q), x.numel(), inv, nullptr,
                                              current_stream(x)),
                 "quant_int4_tensor_scale");
    return q;
}

// quant_int4_tensor_scale_dev (csrc/fast_path.cu:92-109).
torch::Tensor quant_int4_tensor_scale_dev(torch::Tensor x, torch::Tensor inv_scale) {
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.scalar_type() == torch::kBFloat16,
                "x must be contiguous CUDA bf16");
    TORCH_CHECK(x.numel() % 32 == 0, "numel must be multiple of 32");
    TORCH_CHECK(inv_scale.is_cuda() && inv_scale.scalar_type() == torch::kFloat32 &&
                    inv_scale.is_contiguous() && inv_scale.numel() == 1,
                "inv_scale must be 1-elem contiguous fp32 CUDA tensor");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    auto q = new_tensor({x.numel() / 2}, torch::kUInt8, x);
    check_status(wush_quant_int4_tensor_scale(ptr<uint16_t>(x), ptr<uint8_t>(q), x.numel(), 0.0f,
                                              ptr<float>(inv_scale), current_stream(x)),
                 "quant_int4_tensor_scale_dev");
    return q;
}

// w4a4_gemm_cutlass / _dev (csrc/gemm_cutlass_int4.cu:132-188): K from wq,
// xq 1-D or 2-D, y (M, N) fp16 = alpha * xq @ wq^T.
torch::Tensor gemm_tensor_scale_impl(torch::Tensor xq, torch::Tensor wq, double alpha,
                                     const torch::Tensor* alpha_dev, const char* op) {
    TORCH_CHECK(xq.is_cuda() && wq.is_cuda(), "tensors must be CUDA");
    TORCH_CHECK(xq.scalar_type() == torch::kUInt8 && wq.scalar_type() == torch::kUInt8,
                "packed tensors must be uint8");
    TORCH_CHECK(xq.is_contiguous() && wq.is_contiguous(), "tensors must be contiguous");
    TORCH_CHECK(wq.dim() == 2, "w must be 2D (N, K/2)");
    const int64_t K2 = wq.size(1);
    TORCH_CHECK(K2 > 0, "K must be positive");
    const int64_t M = xq.numel() / K2;
    TORCH_CHECK(M * K2 == xq.numel(), "xq numel must equal M*K/2 (K from wq)");
    TORCH_CHECK((2 * K2) % 32 == 0, "K must be a multiple of 32");
    TORCH_CHECK(2 * K2 <= WUSH_TENSOR_SCALE_MAX_K, "K must be <= ", WUSH_TENSOR_SCALE_MAX_K,
                " (the per-tensor GEMM's int32 accumulator holds 256 * sum(qx * qw))");
    const int64_t N = wq.size(0);
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(xq.device());
    auto y = new_tensor({M, N}, torch::kHalf, xq);
    check_status(wush_gemm_s4_tensor_scale(ptr<uint8_t>(xq), ptr<uint8_t>(wq), ptr<uint16_t>(y), M, N,
                                           2 * K2, (float)alpha,
                                           alpha_dev ? ptr<float>(*alpha_dev) : nullptr, current_stream(xq)),
                 op);
    return y;
}

torch::Tensor w4a4_gemm_cutlass(torch::Tensor xq, torch::Tensor wq, double alpha) {
    return gemm_tensor_scale_impl(xq, wq, alpha, nullptr, "w4a4_gemm_cutlass");
}

torch::Tensor w4a4_gemm_cutlass_dev(torch::Tensor xq, torch::Tensor wq, torch::Tensor alpha) {
    TORCH_CHECK(alpha.is_cuda() && alpha.scalar_type() == torch::kFloat32 && alpha.is_contiguous() &&
                    alpha.numel() == 1,
                "alpha must be 1-elem contiguous fp32 CUDA tensor");
    return gemm_tensor_scale_impl(xq, wq, 0.0, &alpha, "w4a4_gemm_cutlass_dev");
}

// ------------------------------------------------------------- 8-bit operators
int half_code(at::ScalarType dt, const char* name) {
    TORCH_CHECK(dt == torch::kBFloat16 || dt == torch::kHalf, name, " must be bf16 or fp16, got ", dt);
    return dt == torch::kBFloat16 ? WUSH_DTYPE_BF16 : WUSH_DTYPE_F16;
}

void check_gpu(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}

void check_int8(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == torch::kInt8 && t.is_contiguous(), name, " must be contiguous int8");
}

void check_f32(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == torch::kFloat32 && t.is_contiguous(), name, " must be contiguous fp32");
}

bool aligned16(const torch::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

// x as rows of its last dimension that the kernels can read with 16-byte
// loads: x itself where its rows lie evenly apart, else a contiguous copy.
torch::Tensor token_rows(const torch::Tensor& x, int64_t& rows, int64_t& stride) {
    const int64_t K = x.size(-1);
    rows = K ? x.numel() / K : 0;
    if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= K && x.stride(0) % 8 == 0 && aligned16(x)) {
        stride = x.stride(0);
        return x;
    }
    stride = K;
    return x.is_contiguous() && aligned16(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}

int64_t check_w8(const torch::Tensor& x, const torch::Tensor& wq, const torch::Tensor& ws) {
    check_gpu(wq, "wq", x);
    check_gpu(ws, "ws", x);
    check_int8(wq, "wq");
    check_f32(ws, "ws");
    TORCH_CHECK(x.dim() >= 1 && wq.dim() == 2, "x must have a last dimension and wq be 2D (N, K)");
    const int64_t K = wq.size(1);
    TORCH_CHECK(x.size(-1) == K, "K mismatch: x has ", x.size(-1), " columns, wq ", K);
    TORCH_CHECK(ws.numel() == wq.size(0), "ws must hold one scale per row of wq");
    TORCH_CHECK(K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K, "K must be a multiple of 16 and at most ", WUSH_W8A8_MAX_K);
    TORCH_CHECK(aligned16(wq), "wq must be 16-byte aligned");
    return K;
}

torch::Tensor bytes_like(size_t n, const torch::Tensor& t) {
    return n ? new_tensor({(int64_t)n}, torch::kUInt8, t) : torch::Tensor();
}

std::vector<torch::Tensor> quant_int8_token(torch::Tensor x) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dt = half_code(x.scalar_type(), "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 16 == 0 && x.size(-1) <= WUSH_W8A8_MAX_K,
                "last dim must be a multiple of 16 and at most ", WUSH_W8A8_MAX_K);
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t K = x.size(-1);
    int64_t rows, stride;
    const auto xr = token_rows(x, rows, stride);
    auto q = new_tensor(x.sizes(), torch::kInt8, x);
    auto s = new_tensor(x.sizes().slice(0, x.dim() - 1), torch::kFloat32, x);
    check_status(wush_quant_int8_token(xr.data_ptr(), dt, ptr<int8_t>(q), ptr<float>(s), rows, K, stride, current_stream(x)),
                 "quant_int8_token");
    return {q, s};
}

torch::Tensor w8a8_gemm(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws, at::ScalarType dtype) {
    TORCH_CHECK(xq.is_cuda(), "xq must be a CUDA tensor");
    const int dt = half_code(dtype, "dtype");
    const int64_t K = check_w8(xq, wq, ws);
    check_gpu(xs, "xs", xq);
    check_int8(xq, "xq");
    check_f32(xs, "xs");
    const int64_t M = xq.numel() / K, N = wq.size(0);
    TORCH_CHECK(xs.numel() == M, "xs must hold one scale per row of xq");
    TORCH_CHECK(aligned16(xq), "xq must be 16-byte aligned");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(xq.device());
    auto y = new_tensor(with_last(xq, N), dtype, xq);
    const size_t wsb = wush_gemm_w8a8_workspace_bytes(M, N, K);
    auto work = bytes_like(wsb, xq);
    check_status(wush_gemm_w8a8(ptr<int8_t>(xq), ptr<float>(xs), ptr<int8_t>(wq), ptr<float>(ws), y.data_ptr(), dt, M, N, K,
                                wsb ? work.data_ptr() : nullptr, wsb, current_stream(xq)),
                 "w8a8_gemm");
    return y;
}

torch::Tensor w8a8_linear(torch::Tensor x, torch::Tensor wq, torch::Tensor ws) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int dt = half_code(x.scalar_type(), "x");
    const int64_t K = check_w8(x, wq, ws), N = wq.size(0);
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    int64_t M, stride;
    const auto xr = token_rows(x, M, stride);
    auto y = new_tensor(with_last(x, N), x.scalar_type(), x);
    const size_t wsb = wush_linear_w8a8_workspace_bytes(M, N, K);
    auto work = bytes_like(wsb, x);
    check_status(wush_linear_w8a8(xr.data_ptr(), stride, ptr<int8_t>(wq), ptr<float>(ws), y.data_ptr(), dt, M, N, K,
                                  wsb ? work.data_ptr() : nullptr, wsb, current_stream(x)),
                 "w8a8_linear");
    return y;
}

wush_kv8_cache kv8_cache(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ks, const torch::Tensor& vs,
                         const torch::Tensor& like) {
    check_gpu(k, "k_cache", like);
    check_gpu(v, "v_cache", like);
    check_gpu(ks, "k_scale", like);
    check_gpu(vs, "v_scale", like);
    check_int8(k, "k_cache");
    check_int8(v, "v_cache");
    check_f32(ks, "k_scale");
    check_f32(vs, "v_scale");
    TORCH_CHECK(k.dim() == 4 && v.dim() == 4, "k_cache must be (pages, heads, page_size, head_dim), v_cache (pages, heads, head_dim, page_size)");
    const int64_t P = k.size(0), H = k.size(1), S = k.size(2), D = k.size(3);
    TORCH_CHECK(v.size(0) == P && v.size(1) == H && v.size(2) == D && v.size(3) == S,
                "v_cache must be (pages, heads, head_dim, page_size) of k_cache's sizes");
    TORCH_CHECK(ks.numel() == P * H && vs.numel() == P * H, "k_scale and v_scale must be (pages, heads)");
    TORCH_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128, got ", D);
    TORCH_CHECK(S == 16 || S == 32 || S == 64 || S == 128, "page_size must be 16, 32, 64 or 128, got ", S);
    TORCH_CHECK(P > 0 && P <= 0x7fffffff && H > 0 && H <= 65535, "the cache must hold pages and heads");
    TORCH_CHECK(aligned16(k) && aligned16(v), "the cache must be 16-byte aligned");
    return {ptr<int8_t>(k), ptr<int8_t>(v), ptr<float>(ks), ptr<float>(vs), P, (int32_t)H, (int32_t)S, (int32_t)D};
}

void check_int32(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
    check_gpu(t, name, like);
    TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.is_contiguous(), name, " must be contiguous int32");
}

struct Kv8Batch {
    int64_t seqs, tokens, table_stride;
    const int32_t* cu;
};

Kv8Batch kv8_batch(const torch::Tensor& q, const torch::Tensor& table, const torch::Tensor& lens,
                   const std::optional<torch::Tensor>& cu) {
    check_int32(table, "block_table", q);
    check_int32(lens, "seq_lens", q);
    TORCH_CHECK(table.dim() == 2 && lens.dim() == 1 && lens.size(0) == table.size(0),
                "block_table must be (sequences, pages) and seq_lens (sequences)");
    Kv8Batch b{table.size(0), q.size(0), table.size(1), nullptr};
    if (cu.has_value()) {
        check_int32(*cu, "cu_q", q);
        TORCH_CHECK(cu->dim() == 1 && cu->size(0) == b.seqs + 1, "cu_q must be (sequences + 1)");
        b.cu = ptr<int32_t>(*cu);
    } else {
        TORCH_CHECK(b.tokens == b.seqs, "without cu_q there is one new token per sequence: got ", b.tokens, " tokens, ",
                    b.seqs, " sequences");
    }
    return b;
}

// (tokens, heads, D) that the kernels can read: itself, or a contiguous copy
torch::Tensor heads_view(const torch::Tensor& t) {
    const bool ok = t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned16(t);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

torch::Tensor kv8_append(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cos_sin, torch::Tensor k_cache,
                         torch::Tensor v_cache, torch::Tensor k_scale, torch::Tensor v_scale, torch::Tensor block_table,
                         torch::Tensor seq_lens, std::optional<torch::Tensor> cu_q, bool interleaved) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    const int dt = half_code(q.scalar_type(), "q");
    const auto c = kv8_cache(k_cache, v_cache, k_scale, v_scale, q);
    check_gpu(k, "k", q);
    check_gpu(v, "v", q);
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must be of one type");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v must be (tokens, heads, head_dim)");
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(1) == c.heads && k.size(2) == c.head_dim &&
                    q.size(2) == c.head_dim,
                "q, k and v must agree in tokens, and k and v with the cache's heads and head_dim");
    check_gpu(cos_sin, "cos_sin", q);
    check_f32(cos_sin, "cos_sin");
    TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.size(0) > 0 && cos_sin.size(1) % 16 == 0 && cos_sin.size(1) <= c.head_dim,
                "cos_sin must be (positions, rotated channels): a multiple of 16, at most head_dim");
    TORCH_CHECK(aligned16(cos_sin), "cos_sin must be 16-byte aligned");
    const auto b = kv8_batch(q, block_table, seq_lens, cu_q);
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q.device());
    auto out = new_tensor(q.sizes(), q.scalar_type(), q);
    if (b.tokens == 0) return out;
    if (b.seqs == 0) return out.zero_();           // cu_q gives no token to a sequence
    const auto qv = heads_view(q), kv = heads_view(k), vv = heads_view(v);
    const int64_t strides[6] = {qv.stride(0), qv.stride(1), kv.stride(0), kv.stride(1), vv.stride(0), vv.stride(1)};
    check_status(wush_kv8_append(qv.data_ptr(), kv.data_ptr(), vv.data_ptr(), dt, strides, ptr<float>(cos_sin),
                                 cos_sin.size(0), cos_sin.size(1), interleaved, &c, ptr<int32_t>(block_table),
                                 b.table_stride, ptr<int32_t>(seq_lens), b.cu, b.seqs, b.tokens, q.size(1), out.data_ptr(),
                                 current_stream(q)),
                 "kv8_append");
    return out;
}

torch::Tensor kv8_attention(torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor k_scale,
                            torch::Tensor v_scale, torch::Tensor block_table, torch::Tensor seq_lens,
                            std::optional<torch::Tensor> cu_q, std::optional<double> scale, int64_t window, double softcap,
                            int64_t max_len) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    const int dt = half_code(q.scalar_type(), "q");
    const auto c = kv8_cache(k_cache, v_cache, k_scale, v_scale, q);
    TORCH_CHECK(q.dim() == 3 && q.size(2) == c.head_dim, "q must be (tokens, heads, head_dim) of the cache's head_dim");
    TORCH_CHECK(q.size(1) > 0 && q.size(1) % c.heads == 0, "q's heads must be a multiple of the cache's ", c.heads);
    TORCH_CHECK(window >= 0 && max_len >= 0, "window and max_len must not be negative");
    TORCH_CHECK(!scale.has_value() || std::isfinite((float)*scale), "scale must be finite");
    TORCH_CHECK(softcap >= 0.0 && std::isfinite(softcap), "softcap must be finite and not negative");
    const auto b = kv8_batch(q, block_table, seq_lens, cu_q);
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q.device());
    auto out = new_tensor(q.sizes(), q.scalar_type(), q);
    if (b.tokens == 0) return out;
    if (b.seqs == 0) return out.zero_();           // cu_q gives no token to a sequence
    const auto qv = heads_view(q);
    const size_t wsb = wush_kv8_attention_workspace_bytes(&c, b.seqs, b.tokens, b.cu != nullptr, q.size(1), b.table_stride,
                                                          window, max_len);
    auto work = bytes_like(wsb, q);
    check_status(wush_kv8_attention(qv.data_ptr(), dt, qv.stride(0), qv.stride(1), &c, ptr<int32_t>(block_table),
                                    b.table_stride, ptr<int32_t>(seq_lens), b.cu, b.seqs, b.tokens, q.size(1),
                                    scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)c.head_dim), window,
                                    (float)softcap, max_len, out.data_ptr(), wsb ? work.data_ptr() : nullptr, wsb,
                                    current_stream(q)),
                 "kv8_attention");
    return out;
}

std::vector<torch::Tensor> kv8_read(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor k_scale,
                                    torch::Tensor v_scale, torch::Tensor pages, at::ScalarType dtype) {
    TORCH_CHECK(k_cache.is_cuda(), "k_cache must be a CUDA tensor");
    const int dt = half_code(dtype, "dtype");
    const auto c = kv8_cache(k_cache, v_cache, k_scale, v_scale, k_cache);
    check_int32(pages, "pages", k_cache);
    TORCH_CHECK(pages.dim() == 1, "pages must be one-dimensional");
    const at::hip::OptionalHIPGuardMasqueradingAsCUDA guard(k_cache.device());
    const int64_t sizes[4] = {pages.size(0), c.heads, c.page_size, c.head_dim};
    auto k = new_tensor(c10::IntArrayRef(sizes, 4), dtype, k_cache), v = new_tensor(c10::IntArrayRef(sizes, 4), dtype, k_cache);
    check_status(wush_kv8_read(&c, ptr<int32_t>(pages), pages.size(0), dt, k.data_ptr(), v.data_ptr(), current_stream(k_cache)),
                 "kv8_read");
    return {k, v};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "my_int4._C on MI355X: HIP/gfx950 kernels behind the reference op signatures";
    // One-time per-device set-up (launch attributes, occupancy tables) at
    // import, so that no op run inside a HIP graph capture has to do it.
    // Without a GPU this reports hipErrorNoDevice; the ops then report errors
    // themselves when called.
    m.attr("setup_status") = wush_init();
    m.def("quant_int4_tensor_scale", &quant_int4_tensor_scale, "Per-tensor INT4 quantize",
          py::arg("x"), py::arg("scale"));
    m.def("quant_int4_tensor_scale_dev", &quant_int4_tensor_scale_dev,
          "Per-tensor INT4 quantize, inv_scale from a 1-elem fp32 device tensor", py::arg("x"),
          py::arg("inv_scale"));
    m.def("quant_int4", &quant_int4, "INT4 sigma-clip group quantize (G=32, bf16 scale)", py::arg("x"));
    m.def("w4a4_gemm", &w4a4_gemm, "W4A4 group-scaled matmul (y keeps xq's leading dims)", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("w4a4_gemm_v1", &w4a4_gemm_v1, "W4A4 group-scaled matmul", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"));
    m.def("w4a4_gemm_cutlass", &w4a4_gemm_cutlass, "W4A4 per-tensor matmul on int8 MFMA", py::arg("xq"),
          py::arg("wq"), py::arg("alpha"));
    m.def("w4a4_gemm_cutlass_dev", &w4a4_gemm_cutlass_dev,
          "W4A4 per-tensor matmul, alpha from a 1-elem fp32 device tensor", py::arg("xq"), py::arg("wq"),
          py::arg("alpha"));
    m.def("w4a4_gemm_s4", &w4a4_gemm_s4,
          "W4A4 group-scaled matmul: int8 MFMA with exact int32 group dots below prefill sizes, fp16 MFMA on "
          "code*scale operands for prefill (M > 64)",
          py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("s4_atom_selftest", &s4_atom_selftest, "verify the int8 MFMA fragment layout");
    m.def("w4a4_gemv", &w4a4_gemv, "W4A4 INT4 gemv (M=1 decode path)", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"));
    m.def("w4a4_gemv_multi", &w4a4_gemv_multi, "W4A4 INT4 gemv, 1<=M<=8 (batched decode)", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("fused_transform_quant_int4_v3", &fused_transform_quant_int4_v3,
          "Fused WUSH transform + INT4 quantize (bit-exact)", py::arg("x"), py::arg("t"));
    m.def("fused_transform_quant_int4_smallm", &fused_transform_quant_int4_smallm,
          "Fused WUSH transform + INT4 quantize (bit-exact)", py::arg("x"), py::arg("t"));
    m.def("fused_transform_quant_int4", &fused_transform_quant_int4,
          "Fused WUSH transform + INT4 quantize (bit-exact)", py::arg("x"), py::arg("t"));
    m.def("w4a4_gemm_v2", &w4a4_gemm_v2, "W4A4 group-scaled matmul (K % 64 == 0)", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("fused_transform_quant_int4_wmma", &fused_transform_quant_int4_wmma,
          "Fused WUSH transform + INT4 quantize (bit-exact)", py::arg("x"), py::arg("t"));
    m.def("quant_int8_token", &quant_int8_token, "Per-token INT8 quantize: (codes int8, scales fp32)", py::arg("x"));
    m.def("w8a8_gemm", &w8a8_gemm, "W8A8 matmul, scales per token and per output channel", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"), py::arg("dtype") = at::kHalf);
    m.def("w8a8_linear", &w8a8_linear, "quant_int8_token and w8a8_gemm in one call; y of x's type", py::arg("x"),
          py::arg("wq"), py::arg("ws"));
    m.def("kv8_append", &kv8_append, "rotate q and k by position, put k and v into the 8-bit paged cache; returns q rotated",
          py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cos_sin"), py::arg("k_cache"), py::arg("v_cache"),
          py::arg("k_scale"), py::arg("v_scale"), py::arg("block_table"), py::arg("seq_lens"), py::arg("cu_q") = py::none(),
          py::arg("interleaved") = false);
    m.def("kv8_attention", &kv8_attention, "causal attention over the 8-bit paged cache", py::arg("q"), py::arg("k_cache"),
          py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("block_table"), py::arg("seq_lens"),
          py::arg("cu_q") = py::none(), py::arg("scale") = py::none(), py::arg("window") = 0, py::arg("softcap") = 0.0,
          py::arg("max_len") = 0);
    m.def("kv8_read", &kv8_read, "pages of the 8-bit cache as values: (k, v), each (pages, heads, page_size, head_dim)",
          py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("pages"),
          py::arg("dtype") = at::kBFloat16);
    m.def("abi_version", &wush_abi_version, "C ABI version of libwush_int4.so");
}
