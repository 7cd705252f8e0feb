// cudaop_b200._C — the torch extension in front of libb200q.so.
//
// Same conventions as the reference project's extensions (op/grouped_gemm/csrc/ops.cu:8-14,
// op/grouped_gemm/csrc/grouped_gemm.cuh:106-176, op/neuron/csrc/ops.cpp:117-139): functions take and
// return torch::Tensor, validate with TORCH_CHECK_VALUE (CUDA tensor, same device, contiguous, dtype, shape),
// run under a CUDAGuard on the inputs' device, launch on torch's current stream, allocate outputs with
// torch::empty on the inputs' device, and report failures as exceptions.  No kernel lives here: every
// function forwards raw pointers to the C ABI declared in include/b200q.h.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

#include "../../include/b200q.h"

namespace cudaop_b200 {
namespace {

// Numbers go into error messages as ready-made strings: formatting them through an output stream (which is what the
// TORCH_CHECK macros do with non-string arguments) crashed inside the C++ runtime's locale code in this process.
std::string num(int64_t v) { return std::to_string(v); }

void check_cuda_2d(const torch::Tensor& t, const char* name, std::initializer_list<c10::ScalarType> dtypes, int64_t dim = 2)
{
    TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", num(dim), " dimensions, got ", num(t.dim()));
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
    // the rows and columns of a matrix are 32-bit numbers from here on
    if (dim == 2) TORCH_CHECK_VALUE(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX, name, " has too many rows or columns for 32-bit numbers");
    bool ok = false;
    for (auto d : dtypes) ok = ok || t.scalar_type() == d;
    TORCH_CHECK_VALUE(ok, name, " has dtype ", c10::toString(t.scalar_type()), ", which this operator does not take");
}

void same_device(std::initializer_list<const torch::Tensor*> ts)
{
    const auto dev = (*ts.begin())->device();
    for (auto* t : ts) TORCH_CHECK_VALUE(t->device() == dev, "all tensors must be on the same device");
}

void* stream_of(const torch::Tensor& t)
{
    return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void raise_on(int code, const char* what)
{
    TORCH_CHECK(code == 0, what, " failed with cudaError ", num(code), code == 1 ? " (invalid argument)" : "");
    C10_CUDA_KERNEL_LAUNCH_CHECK();
}

constexpr auto kU8 = c10::ScalarType::Byte;
constexpr auto kE4M3 = c10::ScalarType::Float8_e4m3fn;
constexpr auto kBF16 = c10::ScalarType::BFloat16;
constexpr auto kF16 = c10::ScalarType::Half;
constexpr auto kF32 = c10::ScalarType::Float;
constexpr auto kI8 = c10::ScalarType::Char;
constexpr auto kI32 = c10::ScalarType::Int;

torch::Tensor out_like(const torch::Tensor& ref, std::vector<int64_t> shape, c10::ScalarType dt)
{
    return torch::empty(shape, ref.options().dtype(dt));
}

}  // namespace

torch::Tensor gemm_fp8(torch::Tensor a, torch::Tensor b, double scale_a, double scale_b)
{
    check_cuda_2d(a, "a", {kU8, kE4M3}); check_cuda_2d(b, "b", {kU8, kE4M3}); same_device({&a, &b});
    TORCH_CHECK_VALUE(a.size(1) == b.size(1), "inner dimensions differ: ", num(a.size(1)), " vs ", num(b.size(1)));
    const c10::cuda::CUDAGuard guard(a.device());
    auto c = out_like(a, {a.size(0), b.size(0)}, kBF16);
    raise_on(b200q_gemm_fp8(a.data_ptr(), b.data_ptr(), c.data_ptr(), (int)a.size(0), (int)b.size(0), (int)a.size(1),
                            (float)scale_a, (float)scale_b, stream_of(a)), "b200q_gemm_fp8");
    return c;
}

torch::Tensor gemm_i8(torch::Tensor a, torch::Tensor b, c10::optional<torch::Tensor> c)
{
    check_cuda_2d(a, "a", {kI8}); check_cuda_2d(b, "b", {kI8}); same_device({&a, &b});
    TORCH_CHECK_VALUE(a.size(1) == b.size(1), "inner dimensions differ: ", num(a.size(1)), " vs ", num(b.size(1)));
    const void* cin = nullptr;
    if (c.has_value()) {
        check_cuda_2d(*c, "c", {kI32}); same_device({&a, &*c});
        TORCH_CHECK_VALUE(c->size(0) == a.size(0) && c->size(1) == b.size(0), "c must be [M, N]");
        cin = c->data_ptr();
    }
    const c10::cuda::CUDAGuard guard(a.device());
    auto d = out_like(a, {a.size(0), b.size(0)}, kI32);
    raise_on(b200q_gemm_i8(a.data_ptr(), b.data_ptr(), cin, d.data_ptr(), (int)a.size(0), (int)b.size(0), (int)a.size(1), stream_of(a)),
             "b200q_gemm_i8");
    return d;
}

torch::Tensor gmm_fp8(torch::Tensor a, torch::Tensor a_scale, torch::Tensor b, torch::Tensor b_scale, torch::Tensor batch_sizes)
{
    check_cuda_2d(a, "a", {kU8, kE4M3}); check_cuda_2d(b, "b", {kU8, kE4M3}, 3);
    check_cuda_2d(a_scale, "a_scale", {kF32}, 1); check_cuda_2d(b_scale, "b_scale", {kF32}, 2);
    same_device({&a, &a_scale, &b, &b_scale});
    const int64_t T = a.size(0), K = a.size(1), E = b.size(0), N = b.size(1);
    TORCH_CHECK_VALUE(b.size(2) == K && a_scale.numel() == T && b_scale.size(0) == E && b_scale.size(1) == N, "shape mismatch");
    TORCH_CHECK_VALUE(batch_sizes.dim() == 1 && batch_sizes.numel() == E && batch_sizes.scalar_type() == c10::ScalarType::Long,
                      "batch_sizes must be a 1-D int64 tensor with one entry per expert");
    const c10::cuda::CUDAGuard guard(a.device());
    // the reference passes batch_sizes on the CPU (op/grouped_gemm/csrc/grouped_gemm.cuh:106-143); the kernel reads it on the device
    auto bs = batch_sizes.is_cuda() ? batch_sizes.contiguous() : batch_sizes.to(a.device(), /*non_blocking=*/false).contiguous();
    auto c = torch::zeros({T, N}, a.options().dtype(kBF16));
    raise_on(b200q_gmm_fp8(a.data_ptr(), a_scale.data_ptr<float>(), b.data_ptr(), b_scale.data_ptr<float>(),
                           reinterpret_cast<const long long*>(bs.data_ptr<int64_t>()), c.data_ptr(), (int)T, (int)N, (int)K, (int)E,
                           stream_of(a)), "b200q_gmm_fp8");
    return c;
}

torch::Tensor gemm_fp8_rowcol(torch::Tensor a, torch::Tensor b, torch::Tensor row_scale, torch::Tensor col_scale, bool out_f32)
{
    check_cuda_2d(a, "a", {kU8, kE4M3}); check_cuda_2d(b, "b", {kU8, kE4M3});
    check_cuda_2d(row_scale, "row_scale", {kF32}, 1); check_cuda_2d(col_scale, "col_scale", {kF32}, 1);
    same_device({&a, &b, &row_scale, &col_scale});
    TORCH_CHECK_VALUE(a.size(1) == b.size(1) && row_scale.numel() == a.size(0) && col_scale.numel() == b.size(0), "shape mismatch");
    const c10::cuda::CUDAGuard guard(a.device());
    auto c = out_like(a, {a.size(0), b.size(0)}, out_f32 ? kF32 : kBF16);
    raise_on(b200q_gemm_fp8_rowcol(a.data_ptr(), b.data_ptr(), c.data_ptr(), (int)a.size(0), (int)b.size(0), (int)a.size(1),
                                   row_scale.data_ptr<float>(), col_scale.data_ptr<float>(), out_f32 ? 1 : 0, stream_of(a)),
             "b200q_gemm_fp8_rowcol");
    return c;
}

torch::Tensor gemm_fp8_swiglu(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor row_scale,
                              torch::Tensor gate_scale, torch::Tensor up_scale)
{
    check_cuda_2d(x, "x", {kU8, kE4M3}); check_cuda_2d(w_gate, "w_gate", {kU8, kE4M3}); check_cuda_2d(w_up, "w_up", {kU8, kE4M3});
    check_cuda_2d(row_scale, "row_scale", {kF32}, 1); check_cuda_2d(gate_scale, "gate_scale", {kF32}, 1);
    check_cuda_2d(up_scale, "up_scale", {kF32}, 1);
    same_device({&x, &w_gate, &w_up, &row_scale, &gate_scale, &up_scale});
    const int64_t M = x.size(0), K = x.size(1), I = w_gate.size(0);
    TORCH_CHECK_VALUE(w_gate.size(1) == K && w_up.size(0) == I && w_up.size(1) == K && row_scale.numel() == M &&
                gate_scale.numel() == I && up_scale.numel() == I, "shape mismatch");
    const c10::cuda::CUDAGuard guard(x.device());
    auto h = out_like(x, {M, I}, kBF16);
    raise_on(b200q_gemm_fp8_swiglu(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), h.data_ptr(), (int)M, (int)I, (int)K,
                                   row_scale.data_ptr<float>(), gate_scale.data_ptr<float>(), up_scale.data_ptr<float>(),
                                   stream_of(x)), "b200q_gemm_fp8_swiglu");
    return h;
}

torch::Tensor gemm_w4a16(torch::Tensor x, torch::Tensor wq, torch::Tensor scales, int64_t group)
{
    check_cuda_2d(x, "x", {kBF16}); check_cuda_2d(wq, "wq", {kU8}); check_cuda_2d(scales, "scales", {kF16});
    same_device({&x, &wq, &scales});
    const int64_t M = x.size(0), K = x.size(1), N = wq.size(0);
    TORCH_CHECK_VALUE(group > 0 && wq.size(1) * 2 == K && K % group == 0 && scales.size(0) == N && scales.size(1) == K / group,
                "shape mismatch");
    const c10::cuda::CUDAGuard guard(x.device());
    auto y = out_like(x, {M, N}, kBF16);
    raise_on(b200q_gemm_w4a16(x.data_ptr(), wq.data_ptr(), scales.data_ptr(), y.data_ptr(), (int)M, (int)N, (int)K, (int)group,
                              stream_of(x)), "b200q_gemm_w4a16");
    return y;
}

torch::Tensor nvfp4_swizzle_sf(torch::Tensor sf, int64_t K)
{
    check_cuda_2d(sf, "sf", {kU8});
    TORCH_CHECK_VALUE(sf.size(1) * 16 == K && K % 64 == 0, "scales must be [rows, K/16] with K % 64 == 0");
    const c10::cuda::CUDAGuard guard(sf.device());
    auto out = out_like(sf, {(int64_t)b200q_nvfp4_sf_bytes((int)sf.size(0), (int)K)}, kU8);
    raise_on(b200q_nvfp4_swizzle_sf(sf.data_ptr(), out.data_ptr(), (int)sf.size(0), (int)K, stream_of(sf)), "b200q_nvfp4_swizzle_sf");
    return out;
}

torch::Tensor gemm_nvfp4(torch::Tensor aq, torch::Tensor sfa, torch::Tensor bq, torch::Tensor sfb, double global_a,
                         double global_b, bool blocked)
{
    check_cuda_2d(aq, "aq", {kU8}); check_cuda_2d(bq, "bq", {kU8});
    const int64_t M = aq.size(0), N = bq.size(0), K = 2 * aq.size(1);
    TORCH_CHECK_VALUE(aq.size(1) == bq.size(1) && K % 64 == 0, "shape mismatch (K must match and be a multiple of 64)");
    const c10::cuda::CUDAGuard guard(aq.device());
    auto c = out_like(aq, {M, N}, kBF16);
    if (blocked) {
        check_cuda_2d(sfa, "sfa", {kU8}, 1); check_cuda_2d(sfb, "sfb", {kU8}, 1);
        same_device({&aq, &sfa, &bq, &sfb});
        TORCH_CHECK_VALUE(sfa.numel() == (int64_t)b200q_nvfp4_sf_bytes((int)M, (int)K) && sfb.numel() == (int64_t)b200q_nvfp4_sf_bytes((int)N, (int)K),
                    "blocked scale arrays have the wrong size");
        raise_on(b200q_gemm_nvfp4_blocked(aq.data_ptr(), sfa.data_ptr(), bq.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N,
                                          (int)K, (float)global_a, (float)global_b, stream_of(aq)), "b200q_gemm_nvfp4_blocked");
        return c;
    }
    check_cuda_2d(sfa, "sfa", {kU8}); check_cuda_2d(sfb, "sfb", {kU8});
    same_device({&aq, &sfa, &bq, &sfb});
    TORCH_CHECK_VALUE(sfa.size(0) == M && sfa.size(1) == K / 16 && sfb.size(0) == N && sfb.size(1) == K / 16, "shape mismatch");
    auto ws = out_like(aq, {(int64_t)b200q_gemm_nvfp4_workspace_bytes((int)M, (int)N, (int)K)}, kU8);
    raise_on(b200q_gemm_nvfp4(aq.data_ptr(), sfa.data_ptr(), bq.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                              (float)global_a, (float)global_b, ws.data_ptr(), stream_of(aq)), "b200q_gemm_nvfp4");
    return c;
}

torch::Tensor mxfp8_swizzle_sf(torch::Tensor sf, int64_t K)
{
    check_cuda_2d(sf, "sf", {kU8});
    TORCH_CHECK_VALUE(sf.size(1) * 32 == K, "scales must be [rows, K/32]");
    const c10::cuda::CUDAGuard guard(sf.device());
    auto out = out_like(sf, {(int64_t)b200q_mxfp8_sf_bytes((int)sf.size(0), (int)K)}, kU8);
    raise_on(b200q_mxfp8_swizzle_sf(sf.data_ptr(), out.data_ptr(), (int)sf.size(0), (int)K, stream_of(sf)), "b200q_mxfp8_swizzle_sf");
    return out;
}

torch::Tensor gemm_mxfp8(torch::Tensor a, torch::Tensor sfa, torch::Tensor b, torch::Tensor sfb, bool blocked)
{
    check_cuda_2d(a, "a", {kU8, kE4M3}); check_cuda_2d(b, "b", {kU8, kE4M3});
    const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
    TORCH_CHECK_VALUE(b.size(1) == K && K % 32 == 0, "shape mismatch (K must match and be a multiple of 32)");
    const c10::cuda::CUDAGuard guard(a.device());
    auto c = out_like(a, {M, N}, kBF16);
    if (blocked) {
        check_cuda_2d(sfa, "sfa", {kU8}, 1); check_cuda_2d(sfb, "sfb", {kU8}, 1);
        same_device({&a, &sfa, &b, &sfb});
        TORCH_CHECK_VALUE(sfa.numel() == (int64_t)b200q_mxfp8_sf_bytes((int)M, (int)K) && sfb.numel() == (int64_t)b200q_mxfp8_sf_bytes((int)N, (int)K),
                          "blocked scale arrays have the wrong size");
        raise_on(b200q_gemm_mxfp8_blocked(a.data_ptr(), sfa.data_ptr(), b.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                                          stream_of(a)), "b200q_gemm_mxfp8_blocked");
        return c;
    }
    check_cuda_2d(sfa, "sfa", {kU8}); check_cuda_2d(sfb, "sfb", {kU8});
    same_device({&a, &sfa, &b, &sfb});
    TORCH_CHECK_VALUE(sfa.size(0) == M && sfa.size(1) == K / 32 && sfb.size(0) == N && sfb.size(1) == K / 32, "shape mismatch");
    auto ws = out_like(a, {(int64_t)b200q_gemm_mxfp8_workspace_bytes((int)M, (int)N, (int)K)}, kU8);
    raise_on(b200q_gemm_mxfp8(a.data_ptr(), sfa.data_ptr(), b.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                              ws.data_ptr(), stream_of(a)), "b200q_gemm_mxfp8");
    return c;
}

torch::Tensor gemm_mxfp4(torch::Tensor aq, torch::Tensor sfa, torch::Tensor bq, torch::Tensor sfb, bool blocked)
{
    check_cuda_2d(aq, "aq", {kU8}); check_cuda_2d(bq, "bq", {kU8});
    const int64_t M = aq.size(0), N = bq.size(0), K = 2 * aq.size(1);
    TORCH_CHECK_VALUE(aq.size(1) == bq.size(1) && K % 32 == 0, "shape mismatch (K must match and be a multiple of 32)");
    TORCH_CHECK_VALUE(K <= INT32_MAX, "K is too large for a 32-bit number");
    const c10::cuda::CUDAGuard guard(aq.device());
    auto c = out_like(aq, {M, N}, kBF16);
    if (blocked) {
        check_cuda_2d(sfa, "sfa", {kU8}, 1); check_cuda_2d(sfb, "sfb", {kU8}, 1);
        same_device({&aq, &sfa, &bq, &sfb});
        TORCH_CHECK_VALUE(sfa.numel() == (int64_t)b200q_mxfp8_sf_bytes((int)M, (int)K) && sfb.numel() == (int64_t)b200q_mxfp8_sf_bytes((int)N, (int)K),
                          "blocked scale arrays have the wrong size");
        raise_on(b200q_gemm_mxfp4_blocked(aq.data_ptr(), sfa.data_ptr(), bq.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                                          stream_of(aq)), "b200q_gemm_mxfp4_blocked");
        return c;
    }
    check_cuda_2d(sfa, "sfa", {kU8}); check_cuda_2d(sfb, "sfb", {kU8});
    same_device({&aq, &sfa, &bq, &sfb});
    TORCH_CHECK_VALUE(sfa.size(0) == M && sfa.size(1) == K / 32 && sfb.size(0) == N && sfb.size(1) == K / 32, "shape mismatch");
    auto ws = out_like(aq, {(int64_t)b200q_gemm_mxfp4_workspace_bytes((int)M, (int)N, (int)K)}, kU8);
    raise_on(b200q_gemm_mxfp4(aq.data_ptr(), sfa.data_ptr(), bq.data_ptr(), sfb.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                              ws.data_ptr(), stream_of(aq)), "b200q_gemm_mxfp4");
    return c;
}

torch::Tensor gemm_sparse_fp8(torch::Tensor a_comp, torch::Tensor a_meta, torch::Tensor b, double scale_a, double scale_b)
{
    check_cuda_2d(a_comp, "a_comp", {kU8, kE4M3}); check_cuda_2d(a_meta, "a_meta", {kU8}); check_cuda_2d(b, "b", {kU8, kE4M3});
    same_device({&a_comp, &a_meta, &b});
    const int64_t M = a_comp.size(0), N = b.size(0), K = b.size(1);
    TORCH_CHECK_VALUE(a_comp.size(1) * 2 == K && a_meta.size(0) == M && a_meta.size(1) == K / 8, "shape mismatch");
    const c10::cuda::CUDAGuard guard(b.device());
    auto c = out_like(b, {M, N}, kBF16);
    raise_on(b200q_gemm_sp24_fp8(a_comp.data_ptr(), a_meta.data_ptr(), b.data_ptr(), c.data_ptr(), (int)M, (int)N, (int)K,
                                 (float)scale_a, (float)scale_b, stream_of(b)), "b200q_gemm_sp24_fp8");
    return c;
}

std::tuple<torch::Tensor, torch::Tensor> quant_rows_e4m3(torch::Tensor x)
{
    check_cuda_2d(x, "x", {kBF16});
    const c10::cuda::CUDAGuard guard(x.device());
    auto q = out_like(x, {x.size(0), x.size(1)}, kU8);
    auto s = out_like(x, {x.size(0)}, kF32);
    raise_on(b200q_quant_rows_e4m3(x.data_ptr(), q.data_ptr(), s.data_ptr<float>(), (int)x.size(0), (int)x.size(1), stream_of(x)),
             "b200q_quant_rows_e4m3");
    return {q, s};
}

std::tuple<torch::Tensor, torch::Tensor> quant_rows_nvfp4(torch::Tensor x, double global_scale)
{
    check_cuda_2d(x, "x", {kBF16});
    TORCH_CHECK_VALUE(x.size(1) % 64 == 0, "the row length must be a multiple of 64");
    TORCH_CHECK_VALUE(global_scale > 0.0, "global_scale must be positive");
    const c10::cuda::CUDAGuard guard(x.device());
    auto q = out_like(x, {x.size(0), x.size(1) / 2}, kU8);
    auto sf = out_like(x, {(int64_t)b200q_nvfp4_sf_bytes((int)x.size(0), (int)x.size(1))}, kU8);
    raise_on(b200q_quant_rows_nvfp4(x.data_ptr(), q.data_ptr(), sf.data_ptr(), (int)x.size(0), (int)x.size(1), (float)global_scale,
                                    stream_of(x)), "b200q_quant_rows_nvfp4");
    return {q, sf};
}

std::tuple<torch::Tensor, torch::Tensor> quant_rows_mxfp4(torch::Tensor x)
{
    check_cuda_2d(x, "x", {kBF16});
    TORCH_CHECK_VALUE(x.size(1) % 32 == 0, "the row length must be a multiple of 32");
    const c10::cuda::CUDAGuard guard(x.device());
    auto q = out_like(x, {x.size(0), x.size(1) / 2}, kU8);
    auto sf = out_like(x, {(int64_t)b200q_mxfp8_sf_bytes((int)x.size(0), (int)x.size(1))}, kU8);
    raise_on(b200q_quant_rows_mxfp4(x.data_ptr(), q.data_ptr(), sf.data_ptr(), (int)x.size(0), (int)x.size(1), stream_of(x)),
             "b200q_quant_rows_mxfp4");
    return {q, sf};
}

// ---------------------------------------------------------------------------------------------- paged cache

struct CacheArgs {
    int pages, kv_heads, page, dim, fp8;
    const float *ks, *vs;
};

void same_place(const torch::Tensor& ref, const torch::Tensor& t, const char* name)
{
    TORCH_CHECK_VALUE(t.device() == ref.device(), name, " must be on the same device as the cache");
}

// [pages, kv_heads, page_size, head_dim] in bf16, or in E4M3 with fp32 scales [pages, kv_heads, page_size]
CacheArgs check_cache(const torch::Tensor& kc, const torch::Tensor& vc, const c10::optional<torch::Tensor>& ks,
                      const c10::optional<torch::Tensor>& vs)
{
    check_cuda_2d(kc, "k_cache", {kBF16, kU8, kE4M3}, 4); check_cuda_2d(vc, "v_cache", {kBF16, kU8, kE4M3}, 4);
    same_place(kc, vc, "v_cache");
    TORCH_CHECK_VALUE(kc.scalar_type() == vc.scalar_type() && kc.sizes() == vc.sizes(), "k_cache and v_cache must have the same dtype and shape");
    CacheArgs c{};
    const int64_t page = kc.size(2), dim = kc.size(3);
    TORCH_CHECK_VALUE(kc.size(0) > 0 && kc.size(1) > 0, "the cache is empty");
    TORCH_CHECK_VALUE(page == 16 || page == 32 || page == 64 || page == 128, "page_size must be 16, 32, 64 or 128, got ", num(page));
    TORCH_CHECK_VALUE(dim == 64 || dim == 128, "head_dim must be 64 or 128, got ", num(dim));
    TORCH_CHECK_VALUE(kc.size(0) <= (INT32_MAX - 4096) / (kc.size(1) * page), "the cache has too many rows for 32-bit row numbers");
    c.pages = (int)kc.size(0); c.kv_heads = (int)kc.size(1); c.page = (int)page; c.dim = (int)dim;
    c.fp8 = kc.scalar_type() != kBF16;
    TORCH_CHECK_VALUE(ks.has_value() == (bool)c.fp8 && vs.has_value() == (bool)c.fp8,
                      "k_scale and v_scale belong to an E4M3 cache, and to no other");
    if (c.fp8) {
        check_cuda_2d(*ks, "k_scale", {kF32}, 3); check_cuda_2d(*vs, "v_scale", {kF32}, 3);
        same_place(kc, *ks, "k_scale"); same_place(kc, *vs, "v_scale");
        TORCH_CHECK_VALUE(ks->sizes() == kc.sizes().slice(0, 3) && vs->sizes() == kc.sizes().slice(0, 3),
                          "the scales must be [pages, kv_heads, page_size]");
        c.ks = ks->data_ptr<float>(); c.vs = vs->data_ptr<float>();
    }
    return c;
}

// rows [tokens, heads, dim] in bf16 that may be slices of a wider tensor: the last dimension contiguous, the others any
// multiple of 16 bytes apart
void check_rows(const torch::Tensor& t, const char* name, const torch::Tensor& kc)
{
    TORCH_CHECK_VALUE(t.dim() == 3, name, " must have 3 dimensions, got ", num(t.dim()));
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
    same_place(kc, t, name);
    TORCH_CHECK_VALUE(t.scalar_type() == kBF16, name, " has dtype ", c10::toString(t.scalar_type()), ", which this operator does not take");
    TORCH_CHECK_VALUE(t.size(2) == kc.size(3), name, " must have the cache's head_dim");
    TORCH_CHECK_VALUE(t.size(2) == 1 || t.stride(2) == 1, "the last dimension of ", name, " must be contiguous");
    TORCH_CHECK_VALUE(t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                      "the rows of ", name, " must start on 16-byte boundaries");
}

void check_index(const torch::Tensor& t, const char* name, c10::ScalarType dt, int64_t dim, const torch::Tensor& kc)
{
    check_cuda_2d(t, name, {dt}, dim);
    same_place(kc, t, name);
}

// A table without columns has no page for any token, as one whose page numbers are all -1.
torch::Tensor with_a_column(const torch::Tensor& page_table)
{
    return page_table.size(1) > 0 ? page_table : torch::full({page_table.size(0), 1}, -1, page_table.options());
}

void paged_cache_write(torch::Tensor k, torch::Tensor v, torch::Tensor slots, torch::Tensor k_cache, torch::Tensor v_cache,
                       c10::optional<torch::Tensor> k_scale, c10::optional<torch::Tensor> v_scale)
{
    const CacheArgs c = check_cache(k_cache, v_cache, k_scale, v_scale);
    check_rows(k, "k", k_cache); check_rows(v, "v", k_cache);
    TORCH_CHECK_VALUE(k.size(1) == c.kv_heads && v.sizes() == k.sizes(), "k and v must be [tokens, kv_heads, head_dim]");
    check_index(slots, "slots", c10::ScalarType::Long, 1, k_cache);
    TORCH_CHECK_VALUE(slots.numel() == k.size(0), "slots must have one entry per token");
    TORCH_CHECK_VALUE(k.size(0) <= INT32_MAX - 4096, "too many tokens");
    if (k.size(0) == 0) return;
    const c10::cuda::CUDAGuard guard(k_cache.device());
    raise_on(b200q_paged_cache_write(k.data_ptr(), v.data_ptr(), reinterpret_cast<const long long*>(slots.data_ptr<int64_t>()), k_cache.data_ptr(),
                                     v_cache.data_ptr(), const_cast<float*>(c.ks), const_cast<float*>(c.vs), (int)k.size(0), c.kv_heads, c.dim,
                                     k.stride(0), v.stride(0), k.stride(1), v.stride(1), c.pages, c.page, c.fp8, stream_of(k_cache)),
             "b200q_paged_cache_write");
}

std::tuple<torch::Tensor, torch::Tensor> paged_cache_read(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor page_table,
                                                          torch::Tensor cu_kv, int64_t total, c10::optional<torch::Tensor> k_scale,
                                                          c10::optional<torch::Tensor> v_scale, c10::optional<torch::Tensor> k_out,
                                                          c10::optional<torch::Tensor> v_out)
{
    const CacheArgs c = check_cache(k_cache, v_cache, k_scale, v_scale);
    check_index(page_table, "page_table", kI32, 2, k_cache); check_index(cu_kv, "cu_kv", kI32, 1, k_cache);
    const int64_t seqs = page_table.size(0);
    TORCH_CHECK_VALUE(cu_kv.numel() == seqs + 1, "cu_kv must have one entry per sequence and one more");
    TORCH_CHECK_VALUE(seqs <= INT32_MAX - 4096 && page_table.size(1) <= INT32_MAX - 4096, "page_table is too large");
    TORCH_CHECK_VALUE(total >= 0 && total <= INT32_MAX - 4096, "total must not be negative, nor pass 32 bits");
    TORCH_CHECK_VALUE(k_out.has_value() == v_out.has_value(), "k_out and v_out go together");
    const c10::cuda::CUDAGuard guard(k_cache.device());
    torch::Tensor k, v;
    if (k_out.has_value()) {
        check_cuda_2d(*k_out, "k_out", {kBF16}, 3); check_cuda_2d(*v_out, "v_out", {kBF16}, 3);
        same_place(k_cache, *k_out, "k_out"); same_place(k_cache, *v_out, "v_out");
        TORCH_CHECK_VALUE(k_out->size(0) == total && k_out->size(1) == c.kv_heads && k_out->size(2) == c.dim && v_out->sizes() == k_out->sizes(),
                          "k_out and v_out must be [total, kv_heads, head_dim]");
        k = *k_out; v = *v_out;
    } else {
        k = out_like(k_cache, {total, c.kv_heads, c.dim}, kBF16);
        v = out_like(k_cache, {total, c.kv_heads, c.dim}, kBF16);
    }
    if (total == 0) return {k, v};
    if (seqs == 0) {                                               // every row is one of no sequence
        if (!k_out.has_value()) { k.zero_(); v.zero_(); }
        return {k, v};
    }
    page_table = with_a_column(page_table);
    raise_on(b200q_paged_cache_read(k_cache.data_ptr(), v_cache.data_ptr(), c.ks, c.vs, page_table.data_ptr<int>(), cu_kv.data_ptr<int>(),
                                    k.data_ptr(), v.data_ptr(), (int)seqs, (int)total, c.kv_heads, c.dim, (int)page_table.size(1), c.pages, c.page,
                                    c.fp8, !k_out.has_value(), stream_of(k_cache)), "b200q_paged_cache_read");
    return {k, v};
}

std::tuple<torch::Tensor, c10::optional<torch::Tensor>> paged_attention(
    torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor page_table, torch::Tensor cu_q, torch::Tensor kv_lens,
    int64_t max_q, c10::optional<torch::Tensor> k_scale, c10::optional<torch::Tensor> v_scale, double scale, bool causal, int64_t window,
    bool return_lse, c10::optional<torch::Tensor> out)
{
    const CacheArgs c = check_cache(k_cache, v_cache, k_scale, v_scale);
    check_rows(q, "q", k_cache);
    const int64_t tokens = q.size(0), heads = q.size(1), seqs = kv_lens.numel();
    TORCH_CHECK_VALUE(heads > 0 && heads % c.kv_heads == 0, "the heads of q must be a multiple of the cache's kv_heads");
    check_index(page_table, "page_table", kI32, 2, k_cache); check_index(cu_q, "cu_q", kI32, 1, k_cache);
    check_index(kv_lens, "kv_lens", kI32, 1, k_cache);
    TORCH_CHECK_VALUE(page_table.size(0) == seqs && cu_q.numel() == seqs + 1, "page_table, cu_q and kv_lens must agree on the number of sequences");
    TORCH_CHECK_VALUE(seqs <= 8192, "at most 8192 sequences, got ", num(seqs));
    TORCH_CHECK_VALUE(max_q > 0, "max_q must be positive");
    TORCH_CHECK_VALUE(window >= 0 && (window == 0 || causal), "window must not be negative, and needs causal");
    TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
    TORCH_CHECK_VALUE(tokens * heads <= INT32_MAX - 4096 && page_table.size(1) <= (INT32_MAX - 4096) / c.page,
                      "sizes pass 32 bits");
    const c10::cuda::CUDAGuard guard(k_cache.device());
    const bool given = out.has_value();
    torch::Tensor o;
    if (given) {
        check_cuda_2d(*out, "out", {kBF16}, 3);
        same_place(k_cache, *out, "out");
        TORCH_CHECK_VALUE(out->sizes() == q.sizes(), "out must have the shape of q");
        o = *out;
    } else {
        o = out_like(k_cache, {tokens, heads, c.dim}, kBF16);
    }
    c10::optional<torch::Tensor> lse;
    if (return_lse) lse = given ? torch::full({tokens, heads}, -INFINITY, k_cache.options().dtype(kF32)) : out_like(k_cache, {tokens, heads}, kF32);
    if (tokens == 0) return {o, lse};
    if (seqs == 0) {                                               // every row is one of no sequence
        if (!given) o.zero_();
        if (return_lse) lse->fill_(-INFINITY);
        return {o, lse};
    }
    page_table = with_a_column(page_table);
    auto ws = out_like(k_cache, {(int64_t)b200q_paged_attention_workspace_bytes(c.dim)}, kU8);
    raise_on(b200q_paged_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), c.ks, c.vs, page_table.data_ptr<int>(),
                                   cu_q.data_ptr<int>(), kv_lens.data_ptr<int>(), o.data_ptr(), lse.has_value() ? lse->data_ptr<float>() : nullptr,
                                   (int)seqs, (int)tokens, (int)heads, c.kv_heads, c.dim, q.stride(0), q.stride(1),
                                   (int)std::min<int64_t>(max_q, tokens), (int)page_table.size(1), c.pages, c.page, c.fp8, (float)scale, causal,
                                   (int)std::min<int64_t>(window, INT32_MAX), !given, ws.data_ptr(), stream_of(k_cache)),
             "b200q_paged_attention");
    return {o, lse};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("gemm_fp8", &gemm_fp8, "FP8 E4M3 GEMM, per-tensor scales, bf16 out");
    m.def("gemm_i8", &gemm_i8, "exact INT8 GEMM with int32 accumulation", pybind11::arg("a"), pybind11::arg("b"), pybind11::arg("c") = pybind11::none());
    m.def("gmm_fp8", &gmm_fp8, "grouped (ragged-M) FP8 GEMM");
    m.def("gemm_fp8_rowcol", &gemm_fp8_rowcol, "FP8 E4M3 GEMM, per-row x per-column scales");
    m.def("gemm_fp8_swiglu", &gemm_fp8_swiglu, "fused gate/up projection + SwiGLU on FP8 operands");
    m.def("gemm_w4a16", &gemm_w4a16, "INT4 weight-only GEMM, bf16 activations");
    m.def("nvfp4_swizzle_sf", &nvfp4_swizzle_sf, "row-major UE4M3 scales -> blocked layout");
    m.def("gemm_nvfp4", &gemm_nvfp4, "NVFP4 block-scaled GEMM");
    m.def("mxfp8_swizzle_sf", &mxfp8_swizzle_sf, "row-major UE8M0 scales -> blocked layout");
    m.def("gemm_mxfp8", &gemm_mxfp8, "MXFP8 block-scaled GEMM");
    m.def("gemm_mxfp4", &gemm_mxfp4, "MXFP4 block-scaled GEMM");
    m.def("gemm_sparse_fp8", &gemm_sparse_fp8, "2:4-sparse FP8 GEMM");
    m.def("quant_rows_e4m3", &quant_rows_e4m3, "bf16 rows -> E4M3 + per-row fp32 scale");
    m.def("quant_rows_nvfp4", &quant_rows_nvfp4, "bf16 rows -> packed E2M1 + blocked UE4M3 scales");
    m.def("quant_rows_mxfp4", &quant_rows_mxfp4, "bf16 rows -> packed E2M1 + blocked UE8M0 scales");
    m.def("paged_cache_write", &paged_cache_write, "new tokens' keys and values into a paged cache");
    m.def("paged_cache_read", &paged_cache_read, "sequences of a paged cache back to bf16");
    m.def("paged_attention", &paged_attention, "attention of a chunk of new tokens over a paged cache");
}

}  // namespace cudaop_b200
