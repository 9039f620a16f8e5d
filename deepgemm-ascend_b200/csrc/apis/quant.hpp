// The quantisers in front of the GEMM (deep_gemm/quant_ops.py holds the same in Python, with the documentation of the entry points): the reference's
// third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py:411-449 and the plain casts; the norm in front of a product; gradients.
#pragma once

#include <c10/cuda/CUDAGuard.h>

#include <variant>

#include "common.hpp"
#include "gemm.hpp"
#include "runtime.hpp"

namespace dg_host {

inline int64_t distance_of_rows(const torch::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }
inline const float* float_ptr(const std::optional<torch::Tensor>& t) { return t.has_value() ? static_cast<const float*>(t->data_ptr()) : nullptr; }
inline const int32_t* int_ptr(const std::optional<torch::Tensor>& t) { return t.has_value() ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; }
inline uint32_t experts_of(const std::optional<torch::Tensor>& psum) { return psum.has_value() ? (uint32_t)psum->numel() : 0u; }
inline bool is_bf16_or_fp32(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32; }

inline void check_row_weights(const std::optional<torch::Tensor>& topk_weights, const std::optional<torch::Tensor>& psum, int64_t tokens, const torch::Tensor& x) {
    if (topk_weights.has_value())
        host_assert(topk_weights->scalar_type() == torch::kFloat32 && topk_weights->is_contiguous() && topk_weights->numel() == tokens &&
                    topk_weights->device() == x.device(), "topk_weights must be a contiguous float32 tensor with one weight per token");
    if (psum.has_value())
        host_assert(psum->scalar_type() == torch::kInt32 && psum->dim() == 1 && psum->is_contiguous() && psum->device() == x.device(),
                    "psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x");
}
// (an empty tensor has no address, and the C ABI takes a null pointer for no layout)
inline void check_psum_layout(const std::optional<torch::Tensor>& psum, int64_t expert_alignment, int64_t multiple) {
    if (!psum.has_value()) return;
    host_assert(psum->numel() > 0, "psum_num_tokens_per_expert must hold an expert");
    host_assert(expert_alignment > 0 && expert_alignment <= INT32_MAX && expert_alignment % multiple == 0,
                multiple == 64 ? "expert_alignment must be a positive multiple of 64" : "expert_alignment must be a positive multiple of 32");
}
inline void check_clamp_value(const std::optional<double>& clamp_value) {
    host_assert(!clamp_value.has_value() || clamp_value.value() >= 0, "clamp_value must not be negative");
}

// `min_amax`: of the plain cast; none takes the reference's constant
inline std::pair<torch::Tensor, torch::Tensor> quantise_fp8(const torch::Tensor& x, int64_t hidden, bool swiglu,
                                                            const std::optional<torch::Tensor>& topk_weights,
                                                            const std::optional<torch::Tensor>& psum,
                                                            const std::optional<double>& clamp_value, int64_t expert_alignment, std::optional<double> min_amax) {
    const int64_t tokens = x.size(0), cols = (hidden / 32 + 1) / 2;
    const c10::cuda::CUDAGuard guard(x.device());
    auto out = empty_on({tokens, hidden}, torch::kFloat8_e4m3fn, x), out_sf = empty_scales({tokens, cols}, x);
    if (tokens != 0) {
        check_row_weights(topk_weights, psum, tokens, x);
        if (min_amax.has_value())
            check(dg_cast_fp8_launch(x.data_ptr(), (uint64_t)distance_of_rows(x), (uint32_t)tokens, (uint32_t)hidden, int_ptr(psum), experts_of(psum),
                                     (uint32_t)expert_alignment, (float)min_amax.value(), out.data_ptr(), (uint64_t)hidden,
                                     static_cast<int16_t*>(out_sf.data_ptr()), (uint64_t)tokens, stream_of(x)));
        else
            check(dg_quant_fp8_launch(x.data_ptr(), (uint64_t)x.stride(0), (uint32_t)tokens, (uint32_t)hidden, swiglu ? 1 : 0, float_ptr(topk_weights),
                                      int_ptr(psum), experts_of(psum), (uint32_t)expert_alignment,
                                      clamp_value.has_value() ? 1 : 0, (float)clamp_value.value_or(0.0), out.data_ptr(), (uint64_t)out.stride(0),
                                      static_cast<int16_t*>(out_sf.data_ptr()), (uint64_t)tokens, stream_of(x)));
    }
    return {out, out_sf};
}

// int16 [rows, cols], consecutive rows contiguous
inline bool is_scales(const torch::Tensor& sf, int64_t rows, int64_t cols) {
    return sf.scalar_type() == torch::kInt16 && sf.dim() == 2 && sf.size(0) == rows && sf.size(1) == cols && (sf.stride(0) == 1 || rows <= 1) &&
           (cols <= 1 || sf.stride(1) >= rows);
}
inline uint64_t scale_stride(const torch::Tensor& sf) { return (uint64_t)(sf.size(1) > 1 ? sf.stride(1) : sf.size(0)); }
inline void check_fp8_out(const TensorPair& out, const torch::Tensor& x, int64_t width) {
    const auto& [q, sf] = out;
    host_assert(q.scalar_type() == torch::kFloat8_e4m3fn && q.device() == x.device() && q.dim() == 2 && q.size(0) == x.size(0) && q.size(1) == width && q.stride(1) == 1 &&
                distance_of_rows(q) >= width && sf.device() == x.device() && is_scales(sf, x.size(0), ceil_div(width, 64)),
                "out must hold E4M3 rows on the device of x and their int16 scales, one element for 64 channels of each row, contiguous along the rows");
}

inline std::pair<TensorPair, TensorPair> swiglu_with_checkpoint(const torch::Tensor& x, const std::optional<torch::Tensor>& topk_weights,
                                                                const std::optional<torch::Tensor>& psum, const std::optional<double>& clamp_value,
                                                                int64_t expert_alignment, const std::optional<std::pair<TensorPair, TensorPair>>& out_in) {
    host_assert(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == torch::kBFloat16, "x must be a row-major 2-D BF16 tensor on a CUDA device");
    host_assert(x.size(1) % 256 == 0, "the row length of x must be a multiple of 256");
    host_assert(x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX, "x is too large");
    const int64_t tokens = x.size(0), hidden = x.size(1) / 2;
    check_row_weights(topk_weights, psum, tokens, x);
    check_psum_layout(psum, expert_alignment, 32);
    check_clamp_value(clamp_value);
    const c10::cuda::CUDAGuard guard(x.device());
    std::pair<TensorPair, TensorPair> out;
    if (out_in.has_value()) {
        out = out_in.value();
    } else {
        out.first = {empty_on({tokens, hidden}, torch::kFloat8_e4m3fn, x), empty_scales({tokens, hidden / 64}, x)};
        out.second = {empty_on({tokens, 2 * hidden}, torch::kFloat8_e4m3fn, x), empty_scales({tokens, hidden / 32}, x)};
    }
    check_fp8_out(out.first, x, hidden);
    check_fp8_out(out.second, x, 2 * hidden);
    const auto& [q, sf] = out.first;
    const auto& [kept, kept_sf] = out.second;
    if (x.numel() != 0)
        check(dg_swiglu_checkpoint_launch(x.data_ptr(), (uint64_t)distance_of_rows(x), (uint32_t)tokens, (uint32_t)hidden, float_ptr(topk_weights), int_ptr(psum),
                                          experts_of(psum), (uint32_t)expert_alignment, clamp_value.has_value() ? 1 : 0, (float)clamp_value.value_or(0.0),
                                          q.data_ptr(), (uint64_t)distance_of_rows(q), static_cast<int16_t*>(sf.data_ptr()), scale_stride(sf),
                                          kept.data_ptr(), (uint64_t)distance_of_rows(kept), static_cast<int16_t*>(kept_sf.data_ptr()), scale_stride(kept_sf), stream_of(x)));
    return out;
}

// An operand in 16 bits, or codes with their scales.
using Operand = std::variant<torch::Tensor, TensorPair>;
struct Split {
    torch::Tensor x, sf;
    bool is_pair;
    explicit Split(const Operand& o) : is_pair(o.index() == 1) {
        if (is_pair) std::tie(x, sf) = std::get<1>(o);
        else x = std::get<0>(o);
    }
    const int16_t* sf_ptr() const { return is_pair ? static_cast<const int16_t*>(sf.data_ptr()) : nullptr; }
};

inline std::pair<torch::Tensor, std::optional<torch::Tensor>> swiglu_grad(const torch::Tensor& grad_out, const Operand& x_in, const std::optional<torch::Tensor>& topk_weights,
                                                                          const std::optional<torch::Tensor>& psum, const std::optional<double>& clamp_value,
                                                                          int64_t expert_alignment, const std::optional<torch::Tensor>& out_in, bool zero_padding) {
    const Split in(x_in);
    const auto& x = in.x;
    host_assert(grad_out.is_cuda() && grad_out.dim() == 2 && grad_out.stride(1) == 1 && grad_out.scalar_type() == torch::kBFloat16,
                "grad_out must be a row-major 2-D BF16 tensor on a CUDA device");
    const int64_t tokens = grad_out.size(0), hidden = grad_out.size(1);
    host_assert(hidden % 128 == 0, "the row length of grad_out must be a multiple of 128");
    host_assert(tokens <= INT32_MAX && 2 * hidden <= INT32_MAX, "grad_out is too large");
    host_assert(x.device() == grad_out.device() && x.dim() == 2 && x.size(0) == tokens && x.size(1) == 2 * hidden && x.stride(1) == 1 &&
                x.scalar_type() == (in.is_pair ? torch::kFloat8_e4m3fn : torch::kBFloat16),
                "x must be a row-major [tokens, 2 * hidden] tensor on the device of grad_out: BF16, or E4M3 with its scales");
    if (in.is_pair)
        host_assert(in.sf.device() == x.device() && is_scales(in.sf, tokens, hidden / 32),
                    "the scales of x must be int16, one element for 64 channels of each row, contiguous along the rows");
    check_row_weights(topk_weights, psum, tokens, x);
    check_psum_layout(psum, expert_alignment, 32);
    check_clamp_value(clamp_value);
    const c10::cuda::CUDAGuard guard(x.device());
    if (out_in.has_value())
        host_assert(out_in->scalar_type() == torch::kBFloat16 && out_in->device() == x.device() && out_in->dim() == 2 && out_in->size(0) == tokens &&
                    out_in->size(1) == 2 * hidden && out_in->stride(1) == 1 && distance_of_rows(out_in.value()) >= 2 * hidden,
                    "out must be a row-major [tokens, 2 * hidden] BF16 tensor on the device of grad_out");
    const auto out = out_in.has_value() ? out_in.value() : empty_on({tokens, 2 * hidden}, torch::kBFloat16, x);
    std::optional<torch::Tensor> grad_weights;
    if (topk_weights.has_value()) grad_weights = empty_on(topk_weights->sizes(), torch::kFloat32, x);
    const uint64_t nbytes = topk_weights.has_value() ? dg_swiglu_grad_scratch_bytes((uint32_t)tokens, (uint32_t)hidden) : 0;
    const auto scratch = nbytes ? empty_on({(int64_t)nbytes}, torch::kUInt8, x) : torch::Tensor();
    if (x.numel() != 0)
        check(dg_swiglu_grad_launch(grad_out.data_ptr(), (uint64_t)distance_of_rows(grad_out), x.data_ptr(), (uint64_t)distance_of_rows(x), in.sf_ptr(),
                                    in.is_pair ? scale_stride(in.sf) : 0, (uint32_t)tokens, (uint32_t)hidden, float_ptr(topk_weights), int_ptr(psum), experts_of(psum),
                                    (uint32_t)expert_alignment, clamp_value.has_value() ? 1 : 0, (float)clamp_value.value_or(0.0), out.data_ptr(),
                                    (uint64_t)distance_of_rows(out), grad_weights.has_value() ? static_cast<float*>(grad_weights->data_ptr()) : nullptr, zero_padding,
                                    nbytes ? scratch.data_ptr() : nullptr, nbytes, stream_of(x)));
    else if (grad_weights.has_value())
        grad_weights->zero_();
    return {out, grad_weights};
}

// `run`: the scales' length along MN
inline void check_packed_scales(const torch::Tensor& x, const torch::Tensor& sf, int64_t groups, int64_t run, int64_t k64, bool mn_major) {
    host_assert(sf.scalar_type() == torch::kInt16 && sf.device() == x.device() && sf.dim() == x.dim() && (sf.dim() == 2 || sf.size(0) == groups) &&
                sf.size(mn_major ? -2 : -1) == k64 && sf.size(mn_major ? -1 : -2) == run,
                "the scales must be packed int16 on the device of x, one byte for each 32 values along K");
    host_assert(sf.stride(mn_major ? -1 : -2) == 1 || run <= 1, "the scales must be contiguous along MN");
}

inline TensorPair cast_to_fp8(const Operand& x_in, const std::optional<torch::Tensor>& psum, int64_t expert_alignment, bool mn_major, double min_amax) {
    const Split in(x_in);
    const auto& x = in.x;
    if (!mn_major) {
        host_assert(!in.is_pair && x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == torch::kBFloat16,
                    "x must be a row-major 2-D BF16 tensor on a CUDA device");
        host_assert(x.size(1) % 32 == 0, "the row length of x must be a multiple of 32");
        return quantise_fp8(x, x.size(1), false, std::nullopt, psum, std::nullopt, expert_alignment, min_amax);
    }
    host_assert(x.is_cuda() && (x.dim() == 2 || x.dim() == 3) && x.stride(-1) == 1 && x.scalar_type() == (in.is_pair ? torch::kFloat8_e4m3fn : torch::kBFloat16),
                "x must be a row-major 2-D or 3-D tensor on a CUDA device: BF16, or E4M3 with its scales");
    const int64_t groups = x.dim() == 3 ? x.size(0) : 1, rows = x.size(-2), cols = x.size(-1), k64 = ceil_div(rows, 64);
    host_assert(cols % 32 == 0, "the row length of x must be a multiple of 32");
    host_assert(groups <= INT32_MAX && rows <= INT32_MAX && cols <= INT32_MAX, "x is too large");
    if (in.is_pair) check_packed_scales(x, in.sf, groups, rows, ceil_div(cols, 64), false);
    check_row_weights(std::nullopt, psum, rows, x);
    check_psum_layout(psum, expert_alignment, 64);
    host_assert(!psum.has_value() || x.dim() == 2, "a psum layout needs a 2-D x");
    const c10::cuda::CUDAGuard guard(x.device());
    auto out = empty_on(x.sizes(), torch::kFloat8_e4m3fn, x);
    auto sf_shape = x.sizes().vec();
    sf_shape[sf_shape.size() - 2] = k64;
    auto sf = empty_on(sf_shape, torch::kInt16, x);
    if (x.numel() != 0)
        check(dg_quant_fp8_mn_launch(x.data_ptr(), (uint64_t)(rows > 1 ? x.stride(-2) : cols), groups > 1 ? (uint64_t)x.stride(0) : 0, in.sf_ptr(),
                                     in.is_pair ? (uint64_t)(cols > 64 ? in.sf.stride(-1) : rows) : 0, in.is_pair && groups > 1 ? (uint64_t)in.sf.stride(0) : 0,
                                     (uint32_t)groups, (uint32_t)rows, (uint32_t)cols, int_ptr(psum), experts_of(psum), (uint32_t)expert_alignment, (float)min_amax,
                                     out.data_ptr(), (uint64_t)cols, (uint64_t)(rows * cols), static_cast<int16_t*>(sf.data_ptr()), (uint64_t)cols, (uint64_t)(k64 * cols),
                                     stream_of(x)));
    return {out, sf};
}

inline torch::Tensor cast_from_fp8(const TensorPair& x, const torch::Dtype& out_dtype, bool mn_major) {
    const auto& [codes, sf] = x;
    host_assert(codes.is_cuda() && (codes.dim() == 2 || codes.dim() == 3) && codes.scalar_type() == torch::kFloat8_e4m3fn && codes.stride(-1) == 1,
                "x must be a row-major 2-D or 3-D E4M3 tensor on a CUDA device, with its scales");
    host_assert(out_dtype == torch::kBFloat16 || out_dtype == torch::kFloat32, "out_dtype must be bf16 or fp32");
    const int64_t groups = codes.dim() == 3 ? codes.size(0) : 1, rows = codes.size(-2), cols = codes.size(-1);
    host_assert(cols % 32 == 0, "the row length of x must be a multiple of 32");
    host_assert(groups <= INT32_MAX && rows <= INT32_MAX && cols <= INT32_MAX, "x is too large");
    const int64_t k64 = ceil_div(mn_major ? rows : cols, 64), run = mn_major ? cols : rows;
    check_packed_scales(codes, sf, groups, run, k64, mn_major);
    const c10::cuda::CUDAGuard guard(codes.device());
    auto out = empty_on(codes.sizes(), out_dtype, codes);
    if (out.numel() != 0)
        check(dg_dequant_fp8_launch(codes.data_ptr(), (uint64_t)(rows > 1 ? codes.stride(-2) : cols), groups > 1 ? (uint64_t)codes.stride(0) : 0,
                                    static_cast<const int16_t*>(sf.data_ptr()), (uint64_t)(k64 > 1 ? sf.stride(mn_major ? -2 : -1) : run),
                                    groups > 1 ? (uint64_t)sf.stride(0) : 0, (uint32_t)groups, (uint32_t)rows, (uint32_t)cols, mn_major, out.data_ptr(),
                                    out_dtype == torch::kFloat32, (uint64_t)cols, (uint64_t)(rows * cols), stream_of(codes)));
    return out;
}

inline void check_norm(const torch::Tensor& x, const torch::Tensor& weight) {
    host_assert(x.size(1) > 0 && x.size(1) % 32 == 0 && x.size(1) <= 16384, "the row length must be a multiple of 32, at most 16384");
    host_assert(x.size(0) <= INT32_MAX, "there are too many tokens");
    host_assert(weight.device() == x.device() && is_bf16_or_fp32(weight) && weight.dim() == 1 && weight.size(0) == x.size(1) && weight.is_contiguous(),
                "weight must be a contiguous BF16 or FP32 vector of the row length, on the device of the rows");
}
// `apart`: rows that are written must not lie on one another
inline void check_like(const std::optional<torch::Tensor>& t, const torch::Tensor& x, bool apart, const char* what) {
    if (t.has_value())
        host_assert(t->scalar_type() == x.scalar_type() && t->device() == x.device() && t->sizes() == x.sizes() && t->stride(1) == 1 &&
                    (!apart || distance_of_rows(t.value()) >= x.size(1)), what);
}

inline std::tuple<TensorPair, std::optional<torch::Tensor>, torch::Tensor, torch::Tensor> rms_norm_to_fp8(
        const torch::Tensor& x, const torch::Tensor& weight, const std::optional<torch::Tensor>& residual, double eps, bool with_rows,
        const std::optional<torch::Tensor>& out_h) {
    host_assert(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && is_bf16_or_fp32(x), "x must be a row-major 2-D BF16 or FP32 tensor on a CUDA device");
    check_norm(x, weight);
    check_like(residual, x, false, "residual must be row-major, of the type, the shape and the device of x");
    check_like(out_h, x, true, "out_h must be row-major, of the type, the shape and the device of x");
    host_assert(!out_h.has_value() || residual.has_value(), "out_h needs a residual");
    const int64_t tokens = x.size(0), hidden = x.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t cols = ceil_div(hidden, 64);
    SharedAllocation small(SharedAllocation::room(tokens * cols * 2) + SharedAllocation::room(tokens * 4), x);
    const auto q = empty_on({tokens, hidden}, torch::kFloat8_e4m3fn, x);
    const auto sf = small.take({tokens, cols}, {1, std::max<int64_t>(tokens, 1)}, torch::kInt16), rstd = small.take({tokens}, {1}, torch::kFloat32);
    std::optional<torch::Tensor> rows;
    if (with_rows) rows = empty_on({tokens, hidden}, torch::kBFloat16, x);
    auto h = !residual.has_value() ? x : out_h.has_value() ? out_h.value() : empty_on({tokens, hidden}, x.scalar_type(), x);
    if (tokens != 0)
        check(dg_rms_norm_fp8_launch(x.data_ptr(), x.scalar_type() == torch::kFloat32, (uint64_t)distance_of_rows(x), residual.has_value() ? residual->data_ptr() : nullptr,
                                     residual.has_value() ? (uint64_t)distance_of_rows(residual.value()) : 0, h.data_ptr(), (uint64_t)distance_of_rows(h),
                                     weight.data_ptr(), weight.scalar_type() == torch::kFloat32, (float)eps, (uint32_t)tokens, (uint32_t)hidden, q.data_ptr(),
                                     (uint64_t)hidden, static_cast<int16_t*>(sf.data_ptr()), (uint64_t)tokens, with_rows ? rows->data_ptr() : nullptr, (uint64_t)hidden,
                                     static_cast<float*>(rstd.data_ptr()), stream_of(x)));
    return {{q, sf}, rows, h, rstd};
}

inline TensorPair rms_norm_grad(const torch::Tensor& grad_out, const torch::Tensor& h, const torch::Tensor& weight, const torch::Tensor& rstd,
                                const std::optional<torch::Tensor>& grad_h, const std::optional<torch::Tensor>& out_in) {
    host_assert(h.is_cuda() && h.dim() == 2 && h.stride(1) == 1 && is_bf16_or_fp32(h), "h must be a row-major 2-D BF16 or FP32 tensor on a CUDA device");
    check_norm(h, weight);
    host_assert(grad_out.device() == h.device() && grad_out.sizes() == h.sizes() && grad_out.stride(1) == 1 &&
                (grad_out.scalar_type() == h.scalar_type() || grad_out.scalar_type() == torch::kBFloat16),
                "grad_out must be row-major, of the shape and the device of h, BF16 or of the type of h");
    host_assert(rstd.device() == h.device() && rstd.scalar_type() == torch::kFloat32 && rstd.dim() == 1 && rstd.size(0) == h.size(0) && rstd.is_contiguous(),
                "rstd must be a contiguous float32 vector with one value per token, on the device of h");
    check_like(grad_h, h, false, "grad_h must be row-major, of the type, the shape and the device of h");
    check_like(out_in, h, true, "out must be row-major, of the type, the shape and the device of h");
    const int64_t tokens = h.size(0), hidden = h.size(1);
    const c10::cuda::CUDAGuard guard(h.device());
    const auto out = out_in.has_value() ? out_in.value() : empty_on(h.sizes(), h.scalar_type(), h);
    const uint64_t nbytes = dg_rms_norm_grad_scratch_bytes((uint32_t)tokens, (uint32_t)hidden);
    const auto grad_weight = empty_on({hidden}, torch::kFloat32, h), scratch = empty_on({(int64_t)nbytes}, torch::kUInt8, h);
    check(dg_rms_norm_grad_launch(grad_out.data_ptr(), grad_out.scalar_type() == torch::kFloat32, (uint64_t)distance_of_rows(grad_out), h.data_ptr(),
                                  h.scalar_type() == torch::kFloat32, (uint64_t)distance_of_rows(h), weight.data_ptr(), weight.scalar_type() == torch::kFloat32,
                                  static_cast<const float*>(rstd.data_ptr()), grad_h.has_value() ? grad_h->data_ptr() : nullptr,
                                  grad_h.has_value() ? (uint64_t)distance_of_rows(grad_h.value()) : 0, (uint32_t)tokens, (uint32_t)hidden, out.data_ptr(),
                                  (uint64_t)distance_of_rows(out), static_cast<float*>(grad_weight.data_ptr()), scratch.data_ptr(), nbytes, stream_of(h)));
    return {out, grad_weight};
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

// A function of a tensor and of a pair, the tensor first: as one function of a variant its calls take a third of a microsecond more.
template <class Make, class... Args> void define_for_operands(py::module_& m, const char* name, Make make, const Args&... args) {
    m.def(name, make(torch::Tensor()), args...);
    m.def(name, make(TensorPair()), args...);
}

inline void register_quant_apis(py::module_& m) {
    m.def("swiglu_apply_weight_to_fp8", [](const torch::Tensor& x, const std::optional<torch::Tensor>& topk_weights,
                                           const std::optional<torch::Tensor>& psum, const std::optional<double>& clamp_value,
                                           int64_t expert_alignment) {
        host_assert(x.is_cuda() && x.dim() == 2 && x.is_contiguous() && x.scalar_type() == torch::kBFloat16, "x must be a contiguous 2-D BF16 tensor on a CUDA device");
        host_assert(x.size(1) % 256 == 0, "the row length of x must be a multiple of 256");
        return quantise_fp8(x, x.size(1) / 2, true, topk_weights, psum, clamp_value, expert_alignment, std::nullopt);
    }, py::arg("x"), py::arg("topk_weights") = std::nullopt, py::arg("psum_num_tokens_per_expert") = std::nullopt,
       py::arg("clamp_value") = std::nullopt, py::arg("expert_alignment") = 128);
    m.def("swiglu_apply_weight_to_fp8_with_checkpoint", &swiglu_with_checkpoint, py::arg("x"), py::arg("topk_weights") = std::nullopt,
          py::arg("psum_num_tokens_per_expert") = std::nullopt, py::arg("clamp_value") = std::nullopt, py::arg("expert_alignment") = 128, py::arg("out") = std::nullopt);
    define_for_operands(m, "swiglu_apply_weight_grad", [](auto operand) {
        return [](const torch::Tensor& grad_out, const decltype(operand)& x, const std::optional<torch::Tensor>& topk_weights, const std::optional<torch::Tensor>& psum,
                  const std::optional<double>& clamp_value, int64_t expert_alignment, const std::optional<torch::Tensor>& out, bool zero_padding) {
            return swiglu_grad(grad_out, x, topk_weights, psum, clamp_value, expert_alignment, out, zero_padding);
        };
    }, py::arg("grad_out"), py::arg("x"), py::arg("topk_weights") = std::nullopt, py::arg("psum_num_tokens_per_expert") = std::nullopt,
       py::arg("clamp_value") = std::nullopt, py::arg("expert_alignment") = 128, py::arg("out") = std::nullopt, py::arg("zero_padding") = false);
    m.def("cast_to_fp4", &cast_to_fp4, py::arg("x"), py::arg("psum_num_tokens_per_expert") = std::nullopt, py::arg("expert_alignment") = kMkAlignment,
          py::arg("mn_major") = false);
    m.def("cast_from_fp4", &cast_from_fp4, py::arg("x"), py::arg("out_dtype") = torch::kBFloat16, py::arg("mn_major") = false);
    define_for_operands(m, "cast_to_fp8", [](auto operand) {
        return [](const decltype(operand)& x, const std::optional<torch::Tensor>& psum, int64_t expert_alignment, bool mn_major, double min_amax) {
            return cast_to_fp8(x, psum, expert_alignment, mn_major, min_amax);
        };
    }, py::arg("x"), py::arg("psum_num_tokens_per_expert") = std::nullopt, py::arg("expert_alignment") = 128, py::arg("mn_major") = false, py::arg("min_amax") = 1e-4);
    m.def("cast_from_fp8", &cast_from_fp8, py::arg("x"), py::arg("out_dtype") = torch::kBFloat16, py::arg("mn_major") = false);
    m.def("rms_norm_to_fp8", &rms_norm_to_fp8, py::arg("x"), py::arg("weight"), py::arg("residual") = std::nullopt, py::arg("eps") = 1e-6, py::arg("with_rows") = false,
          py::arg("out_h") = std::nullopt);
    m.def("rms_norm_grad", &rms_norm_grad, py::arg("grad_out"), py::arg("h"), py::arg("weight"), py::arg("rstd"), py::arg("grad_h") = std::nullopt,
          py::arg("out") = std::nullopt);
}

}  // namespace dg_host
