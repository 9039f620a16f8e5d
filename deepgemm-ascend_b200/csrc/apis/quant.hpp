// The quantisers in front of the GEMM (deep_gemm/quant_ops.py holds the same in Python): the reference's
// third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py:411-449 and the plain cast.
#pragma once

#include <c10/cuda/CUDAGuard.h>

#include "common.hpp"
#include "gemm.hpp"
#include "runtime.hpp"

namespace dg_host {

inline std::pair<torch::Tensor, torch::Tensor> quantise_fp8(const torch::Tensor& x, int64_t hidden, bool swiglu,
                                                            const std::optional<torch::Tensor>& topk_weights,
                                                            const std::optional<torch::Tensor>& psum,
                                                            const std::optional<double>& clamp_value, int64_t expert_alignment) {
    const int64_t tokens = x.size(0), cols = (hidden / 32 + 1) / 2;
    auto out = torch::empty({tokens, hidden}, x.options().dtype(torch::kFloat8_e4m3fn));
    auto out_sf = torch::empty_strided({tokens, cols}, {1, std::max<int64_t>(tokens, 1)}, x.options().dtype(torch::kInt16));
    if (tokens != 0) {
        if (topk_weights.has_value())
            host_assert(topk_weights->scalar_type() == torch::kFloat32 && topk_weights->is_contiguous() && topk_weights->numel() == tokens,
                        "topk_weights must be a contiguous float32 tensor with one weight per token");
        if (psum.has_value())
            host_assert(psum->scalar_type() == torch::kInt32 && psum->dim() == 1 && psum->is_contiguous() && psum->device() == x.device(),
                        "psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x");
        check(dg_quant_fp8_launch(x.data_ptr(), (uint64_t)x.stride(0), (uint32_t)tokens, (uint32_t)hidden, swiglu ? 1 : 0,
                                  topk_weights.has_value() ? static_cast<const float*>(topk_weights->data_ptr()) : nullptr,
                                  psum.has_value() ? static_cast<const int32_t*>(psum->data_ptr()) : nullptr,
                                  psum.has_value() ? (uint32_t)psum->numel() : 0u, (uint32_t)expert_alignment,
                                  clamp_value.has_value() ? 1 : 0, (float)clamp_value.value_or(0.0), out.data_ptr(), (uint64_t)out.stride(0),
                                  static_cast<int16_t*>(out_sf.data_ptr()), (uint64_t)tokens, stream_of(x)));
    }
    return {out, out_sf};
}

// Microscaled 4-bit values. The pair that is made goes into the GEMMs as it is: K-major codes [.., rows, cols / 2] with scales
// [.., rows, ceil(cols / 64)] whose rows are contiguous, or MN-major codes (K runs down the rows) with scales [.., ceil(rows / 64), cols].
inline TensorPair cast_to_fp4(const torch::Tensor& x, const std::optional<torch::Tensor>& psum, int64_t expert_alignment, bool mn_major) {
    host_assert(x.is_cuda() && (x.dim() == 2 || x.dim() == 3) && x.stride(-1) == 1 &&
                (x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kFloat32),
                "x must be a row-major 2-D or 3-D BF16 or FP32 tensor on a CUDA device");
    const int64_t groups = x.dim() == 3 ? x.size(0) : 1, rows = x.size(-2), cols = x.size(-1);
    host_assert(cols % 32 == 0, "the row length of x must be a multiple of 32");
    host_assert(groups <= INT32_MAX && rows <= INT32_MAX && cols <= INT32_MAX, "x is too large");
    if (psum.has_value()) {
        host_assert(psum->scalar_type() == torch::kInt32 && psum->dim() == 1 && psum->is_contiguous() && psum->device() == x.device(),
                    "psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x");
        // (an empty tensor has no address, and the C ABI takes a null pointer for no layout)
        host_assert(psum->numel() > 0, "psum_num_tokens_per_expert must hold an expert");
        host_assert(x.dim() == 2, "a psum layout needs a 2-D x");
        host_assert(expert_alignment > 0 && expert_alignment <= INT32_MAX && expert_alignment % (mn_major ? 64 : 32) == 0,
                    "expert_alignment must be a positive multiple of 32 (64 when mn_major)");
    }
    const c10::cuda::CUDAGuard guard(x.device());
    auto shape = x.sizes().vec();
    shape.back() = cols / 2;
    auto out = empty_on(shape, torch::kInt8, x);
    const int64_t k64 = ceil_div(mn_major ? rows : cols, 64), run = mn_major ? cols : rows;
    auto sf_shape = x.sizes().vec();
    (mn_major ? sf_shape[sf_shape.size() - 2] : sf_shape.back()) = k64;
    auto sf = mn_major ? empty_on(sf_shape, torch::kInt16, x) : empty_scales(sf_shape, x);
    if (x.numel() != 0)
        check(dg_quant_fp4_launch(x.data_ptr(), x.scalar_type() == torch::kFloat32, rows > 1 ? (uint64_t)x.stride(-2) : (uint64_t)cols,
                                  groups > 1 ? (uint64_t)x.stride(0) : 0, (uint32_t)groups, (uint32_t)rows, (uint32_t)cols, mn_major,
                                  psum.has_value() ? static_cast<const int32_t*>(psum->data_ptr()) : nullptr,
                                  psum.has_value() ? (uint32_t)psum->numel() : 0u, (uint32_t)expert_alignment, out.data_ptr(), (uint64_t)(cols / 2),
                                  (uint64_t)(rows * (cols / 2)), static_cast<int16_t*>(sf.data_ptr()), (uint64_t)run, (uint64_t)(k64 * run), stream_of(x)));
    return {out, sf};
}

inline torch::Tensor cast_from_fp4(const TensorPair& x, const torch::Dtype& out_dtype, bool mn_major) {
    const auto& [codes, sf] = x;
    host_assert(codes.is_cuda() && (codes.dim() == 2 || codes.dim() == 3) && codes.scalar_type() == kPackedFp4 && codes.stride(-1) == 1,
                "x must be a row-major 2-D or 3-D tensor of packed FP4 on a CUDA device, with its scales");
    host_assert(out_dtype == torch::kBFloat16 || out_dtype == torch::kFloat32, "out_dtype must be bf16 or fp32");
    const int64_t groups = codes.dim() == 3 ? codes.size(0) : 1, rows = codes.size(-2), cols = codes.size(-1) * 2;
    host_assert(cols % 32 == 0, "the row length of x must be a multiple of 32");
    host_assert(groups <= INT32_MAX && rows <= INT32_MAX && cols <= INT32_MAX, "x is too large");
    const int64_t k64 = ceil_div(mn_major ? rows : cols, 64), run = mn_major ? cols : rows;
    host_assert(sf.scalar_type() == torch::kInt16 && sf.device() == codes.device() && sf.dim() == codes.dim() && (sf.dim() == 2 || sf.size(0) == groups) &&
                sf.size(mn_major ? -2 : -1) == k64 && sf.size(mn_major ? -1 : -2) == run,
                "the scales must be packed int16 on the device of x, one byte for each 32 values along K");
    host_assert(sf.stride(mn_major ? -1 : -2) == 1 || run <= 1, "the scales must be contiguous along MN");
    const c10::cuda::CUDAGuard guard(codes.device());
    auto shape = codes.sizes().vec();
    shape.back() = cols;
    auto out = empty_on(shape, out_dtype, codes);
    if (out.numel() != 0)
        check(dg_dequant_fp4_launch(codes.data_ptr(), rows > 1 ? (uint64_t)codes.stride(-2) : (uint64_t)(cols / 2), groups > 1 ? (uint64_t)codes.stride(0) : 0,
                                    static_cast<const int16_t*>(sf.data_ptr()), k64 > 1 ? (uint64_t)sf.stride(mn_major ? -2 : -1) : (uint64_t)run,
                                    groups > 1 ? (uint64_t)sf.stride(0) : 0, (uint32_t)groups, (uint32_t)rows, (uint32_t)cols, mn_major,
                                    out.data_ptr(), out_dtype == torch::kFloat32, (uint64_t)cols, (uint64_t)(rows * cols), stream_of(codes)));
    return out;
}

inline void register_quant_apis(py::module_& m) {
    m.def("swiglu_apply_weight_to_fp8", [](const torch::Tensor& x, const std::optional<torch::Tensor>& topk_weights,
                                           const std::optional<torch::Tensor>& psum, const std::optional<double>& clamp_value,
                                           int64_t expert_alignment) {
        host_assert(x.dim() == 2 && x.is_contiguous() && x.scalar_type() == torch::kBFloat16, "x must be a contiguous 2-D BF16 tensor");
        host_assert(x.size(1) % 256 == 0, "the row length of x must be a multiple of 256");
        return quantise_fp8(x, x.size(1) / 2, true, topk_weights, psum, clamp_value, expert_alignment);
    }, py::arg("x"), py::arg("topk_weights") = std::nullopt, py::arg("psum_num_tokens_per_expert") = std::nullopt,
       py::arg("clamp_value") = std::nullopt, py::arg("expert_alignment") = 128);
    m.def("cast_to_fp4", &cast_to_fp4, py::arg("x"), py::arg("psum_num_tokens_per_expert") = std::nullopt, py::arg("expert_alignment") = kMkAlignment,
          py::arg("mn_major") = false);
    m.def("cast_from_fp4", &cast_from_fp4, py::arg("x"), py::arg("out_dtype") = torch::kBFloat16, py::arg("mn_major") = false);
    m.def("cast_to_fp8", [](const torch::Tensor& x, const std::optional<torch::Tensor>& psum, int64_t expert_alignment) {
        host_assert(x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == torch::kBFloat16, "x must be a row-major 2-D BF16 tensor");
        host_assert(x.size(1) % 32 == 0, "the row length of x must be a multiple of 32");
        return quantise_fp8(x, x.size(1), false, std::nullopt, psum, std::nullopt, expert_alignment);
    }, py::arg("x"), py::arg("psum_num_tokens_per_expert") = std::nullopt, py::arg("expert_alignment") = 128);
}

}  // namespace dg_host
