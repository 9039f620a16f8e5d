// From the router's choices to the rows of a grouped layout and back (deep_gemm/moe_ops.py holds the same in Python, with the
// documentation of the entry points).
#pragma once

#include <c10/cuda/CUDAGuard.h>

#include "common.hpp"
#include "gemm.hpp"
#include "runtime.hpp"

namespace dg_host {

using MoePlan = std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>;

// What moe_sort has made, checked against the device of the rows and the number of tokens.
struct MoeRows {
    const torch::Tensor &layout, &token_rows, &row_choices;
    int64_t tokens, topk, experts, max_m, rows;

    MoeRows(const MoePlan& plan, const torch::Tensor& x, int64_t num_tokens)
        : layout(std::get<0>(plan)), token_rows(std::get<1>(plan)), row_choices(std::get<2>(plan)) {
        for (const auto* t : {&layout, &token_rows, &row_choices})
            host_assert(t->scalar_type() == torch::kInt32 && t->is_contiguous() && t->device() == x.device(),
                        "plan must hold the three contiguous int32 tensors of moe_sort, on the device of the rows");
        host_assert(layout.dim() == 1 && token_rows.dim() == 2 && (row_choices.dim() == 1 || (row_choices.dim() == 2 && row_choices.size(0) == layout.size(0))),
                    "plan must hold the three tensors of moe_sort: layout, token_rows, row_choices");
        tokens = token_rows.size(0); topk = token_rows.size(1); experts = layout.size(0);
        max_m = row_choices.dim() == 2 ? row_choices.size(1) : 0;
        rows = row_choices.numel();
        host_assert(tokens <= INT32_MAX && topk <= INT32_MAX && token_rows.numel() <= INT32_MAX && rows <= INT32_MAX, "plan is too large");
        host_assert(num_tokens < 0 || tokens == num_tokens, "plan was made for another number of tokens");
    }
    std::vector<int64_t> shape(int64_t last) const {
        return row_choices.dim() == 2 ? std::vector<int64_t>{experts, max_m, last} : std::vector<int64_t>{rows, last};
    }
    const int32_t* token_rows_ptr() const { return static_cast<const int32_t*>(token_rows.data_ptr()); }
    const int32_t* row_choices_ptr() const { return static_cast<const int32_t*>(row_choices.data_ptr()); }
    const int32_t* layout_ptr() const { return static_cast<const int32_t*>(layout.data_ptr()); }
    // Distance between the rows of a tensor of the grouped layout; `what` is the message where its rows do not lie at one distance
    // (or lie on one another).
    int64_t check_rows(const torch::Tensor& t, const char* what) const {
        const auto want = shape(t.dim() > 0 ? t.size(-1) : 0);
        host_assert(t.sizes() == at::IntArrayRef(want) && t.stride(-1) == 1, what);
        const int64_t per_group = row_choices.dim() == 2 ? max_m : rows;
        const int64_t stride = per_group > 1 ? t.stride(-2) : row_choices.dim() == 2 && experts > 1 ? t.stride(0) : t.size(-1);
        host_assert(stride >= t.size(-1) && (t.dim() == 2 || experts <= 1 || t.stride(0) == stride * max_m), what);
        return stride;
    }
};

inline bool bf16_or_fp32(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32; }
inline int64_t stride_of_rows(const torch::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }
inline void check_tokens(const torch::Tensor& x, const char* what) {
    host_assert(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && bf16_or_fp32(x), what);
}
inline void check_alignment(int64_t expert_alignment) {
    host_assert(expert_alignment > 0 && expert_alignment <= INT32_MAX, "expert_alignment must be positive");
}
inline void check_weights(const torch::Tensor& w, const MoeRows& plan) {
    host_assert(w.scalar_type() == torch::kFloat32 && w.is_contiguous() && w.device() == plan.token_rows.device() && w.sizes() == plan.token_rows.sizes(),
                "topk_weights must be a contiguous float32 tensor with one weight per choice, on the device of the rows");
}

inline void check_router(const torch::Tensor& logits, int64_t topk, const std::string& scoring) {
    host_assert(logits.is_cuda() && logits.dim() == 2 && bf16_or_fp32(logits) && (logits.stride(1) == 1 || logits.size(1) == 1),
                "logits must be a row-major 2-D BF16 or FP32 tensor on a CUDA device");
    host_assert(scoring == "softmax" || scoring == "sigmoid", "scoring must be 'softmax' or 'sigmoid'");
    const int64_t experts = logits.size(1);
    host_assert(experts > 0 && experts <= 1024, "the number of experts must be between 1 and 1024");
    host_assert(topk > 0 && topk <= std::min<int64_t>(32, experts), "topk must be between 1 and 32, and at most the number of experts");
    host_assert(logits.size(0) <= INT32_MAX, "there are too many tokens");
}

inline TensorPair moe_route(const torch::Tensor& logits, int64_t topk, const std::string& scoring, const std::optional<torch::Tensor>& bias, int64_t num_groups,
                            int64_t topk_groups, int64_t group_best, bool renormalize, double scale) {
    check_router(logits, topk, scoring);
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    if (bias.has_value())
        host_assert(bias->scalar_type() == torch::kFloat32 && bias->is_contiguous() && bias->dim() == 1 && bias->size(0) == experts && bias->device() == logits.device(),
                    "bias must be a contiguous float32 vector with one value per expert, on the device of logits");
    host_assert(num_groups > 0 && num_groups <= 32 && experts % num_groups == 0, "num_groups must be between 1 and 32 and divide the number of experts");
    host_assert(topk_groups > 0 && topk_groups <= num_groups, "topk_groups must be between 1 and num_groups");
    host_assert(group_best == 1 || group_best == 2, "group_best must be 1 or 2");
    host_assert(topk <= experts / num_groups * topk_groups, "the groups that are taken hold fewer experts than topk");
    const c10::cuda::CUDAGuard guard(logits.device());
    SharedAllocation both(2 * SharedAllocation::room(tokens * topk * 4), logits);
    const auto idx = both.take({tokens, topk}, {topk, 1}, torch::kInt32), weights = both.take({tokens, topk}, {topk, 1}, torch::kFloat32);
    if (tokens != 0)
        check(dg_moe_route_launch(logits.data_ptr(), logits.scalar_type() == torch::kFloat32, (uint64_t)stride_of_rows(logits), (uint32_t)tokens, (uint32_t)experts,
                                  (uint32_t)topk, scoring == "sigmoid", bias.has_value() ? static_cast<const float*>(bias->data_ptr()) : nullptr, (uint32_t)num_groups,
                                  (uint32_t)topk_groups, (uint32_t)group_best, renormalize, (float)scale, static_cast<int32_t*>(idx.data_ptr()),
                                  static_cast<float*>(weights.data_ptr()), stream_of(logits)));
    return {idx, weights};
}

inline torch::Tensor moe_route_grad(const torch::Tensor& grad_weights, const torch::Tensor& logits, const torch::Tensor& topk_idx, const std::string& scoring,
                                    bool renormalize, double scale, const std::optional<torch::Tensor>& out_in) {
    host_assert(topk_idx.dim() == 2 && (topk_idx.scalar_type() == torch::kInt32 || topk_idx.scalar_type() == torch::kInt64) && topk_idx.is_contiguous() &&
                topk_idx.device() == logits.device() && topk_idx.size(0) == logits.size(0),
                "topk_idx must be a contiguous int32 or int64 [tokens, topk] tensor on the device of logits");
    check_router(logits, topk_idx.size(1), scoring);
    host_assert(grad_weights.scalar_type() == torch::kFloat32 && grad_weights.is_contiguous() && grad_weights.device() == logits.device() &&
                grad_weights.sizes() == topk_idx.sizes(), "grad_weights must be a contiguous float32 tensor with one value per choice, on the device of logits");
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    const c10::cuda::CUDAGuard guard(logits.device());
    if (out_in.has_value())
        host_assert(out_in->scalar_type() == logits.scalar_type() && out_in->device() == logits.device() && out_in->sizes() == logits.sizes() &&
                    (out_in->stride(1) == 1 || experts == 1) && stride_of_rows(out_in.value()) >= experts,
                    "out must be row-major, of the type, the shape and the device of logits");
    const auto out = out_in.has_value() ? out_in.value() : empty_on({tokens, experts}, logits.scalar_type(), logits);
    if (tokens != 0)
        check(dg_moe_route_grad_launch(static_cast<const float*>(grad_weights.data_ptr()), logits.data_ptr(), logits.scalar_type() == torch::kFloat32,
                                       (uint64_t)stride_of_rows(logits), (uint32_t)tokens, (uint32_t)experts, topk_idx.data_ptr(),
                                       topk_idx.scalar_type() == torch::kInt64, (uint32_t)topk_idx.size(1), scoring == "sigmoid", renormalize, (float)scale,
                                       out.data_ptr(), (uint64_t)stride_of_rows(out), stream_of(logits)));
    return out;
}

inline MoePlan moe_sort(const torch::Tensor& topk_idx, int64_t num_experts, int64_t expert_alignment, const std::optional<int64_t>& max_m) {
    host_assert(topk_idx.is_cuda() && topk_idx.dim() == 2 && topk_idx.is_contiguous() &&
                (topk_idx.scalar_type() == torch::kInt64 || topk_idx.scalar_type() == torch::kInt32),
                "topk_idx must be a contiguous 2-D int32 or int64 tensor on a CUDA device");
    host_assert(num_experts > 0 && num_experts <= 1024, "num_experts must be between 1 and 1024");
    host_assert(!max_m.has_value() || (max_m.value() > 0 && max_m.value() <= INT32_MAX), "max_m must be positive");
    check_alignment(expert_alignment);
    host_assert(topk_idx.numel() <= INT32_MAX, "topk_idx is too large");
    const int64_t slots = max_m.value_or(0);
    const int64_t rows = slots ? num_experts * slots : (int64_t)dg_moe_num_rows((uint32_t)topk_idx.numel(), (uint32_t)num_experts, (uint32_t)expert_alignment);
    host_assert(rows <= INT32_MAX, "the layout has too many rows");
    const c10::cuda::CUDAGuard guard(topk_idx.device());
    // one allocation for the three (about a microsecond of host time each; to torch they are no views, but keeping one keeps all); every part
    // starts on 16 bytes
    const int64_t part[3] = {num_experts, topk_idx.numel(), rows};
    int64_t offset = 0;
    const auto buffer = empty_on({align_up(part[0], 4) + align_up(part[1], 4) + part[2]}, torch::kInt32, topk_idx);
    const auto take = [&](int k, at::IntArrayRef sizes) {
        auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
        t.unsafeGetTensorImpl()->set_storage_offset(offset);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        offset += align_up(part[k], 4);
        return t;
    };
    const auto layout = take(0, {num_experts}), token_rows = take(1, topk_idx.sizes());
    const auto row_choices = slots ? take(2, {num_experts, slots}) : take(2, {rows});
    check(dg_moe_sort_launch(topk_idx.data_ptr(), topk_idx.scalar_type() == torch::kInt64, (uint32_t)topk_idx.size(0), (uint32_t)topk_idx.size(1),
                             (uint32_t)num_experts, (uint32_t)expert_alignment, (uint32_t)slots, static_cast<int32_t*>(layout.data_ptr()),
                             static_cast<int32_t*>(token_rows.data_ptr()), static_cast<int32_t*>(row_choices.data_ptr()), (uint64_t)rows, stream_of(topk_idx)));
    return {layout, token_rows, row_choices};
}

inline torch::Tensor moe_dispatch(const torch::Tensor& x, const MoePlan& plan_in, const std::optional<torch::Tensor>& out_in, bool zero_padding,
                                  int64_t expert_alignment) {
    check_tokens(x, "x must be a row-major 2-D BF16 or FP32 tensor on a CUDA device");
    const MoeRows plan(plan_in, x, x.size(0));
    check_alignment(expert_alignment);
    const c10::cuda::CUDAGuard guard(x.device());
    if (out_in.has_value()) host_assert(out_in->scalar_type() == x.scalar_type() && out_in->device() == x.device() && out_in->size(-1) == x.size(1),
                                        "out must have the type, the device and the row length of x");
    const auto out = out_in.has_value() ? out_in.value() : empty_on(plan.shape(x.size(1)), x.scalar_type(), x);
    const int64_t stride = plan.check_rows(out, "out must hold a row for each of the layout's, at one distance"), es = x.element_size();
    check(dg_moe_dispatch_launch(x.data_ptr(), (uint64_t)(stride_of_rows(x) * es), (uint32_t)plan.tokens, (uint32_t)plan.topk, (uint64_t)(x.size(1) * es),
                                 plan.token_rows_ptr(), plan.row_choices_ptr(), (uint64_t)plan.rows, out.data_ptr(), (uint64_t)(stride * es), plan.layout_ptr(),
                                 (uint32_t)plan.experts, (uint32_t)expert_alignment, (uint32_t)plan.max_m, zero_padding, stream_of(x)));
    return out;
}

inline TensorPair moe_dispatch_to_fp8(const torch::Tensor& x, const MoePlan& plan_in, const std::optional<TensorPair>& out_in) {
    host_assert(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == torch::kBFloat16, "x must be a row-major 2-D BF16 tensor on a CUDA device");
    host_assert(x.size(1) % 32 == 0, "the row length of x must be a multiple of 32");
    host_assert(x.size(1) <= INT32_MAX, "x is too large");
    const MoeRows plan(plan_in, x, x.size(0));
    const int64_t hidden = x.size(1), cols = ceil_div(hidden, 64), per_group = plan.max_m ? plan.max_m : plan.rows;
    const c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor out, sf;
    if (out_in.has_value()) {
        std::tie(out, sf) = out_in.value();
        host_assert(out.scalar_type() == torch::kFloat8_e4m3fn && out.device() == x.device() && out.size(-1) == hidden,
                    "out must be an E4M3 tensor of the row length and the device of x, with its scales");
        host_assert(sf.scalar_type() == torch::kInt16 && sf.device() == x.device() && sf.sizes() == at::IntArrayRef(plan.shape(cols)) &&
                    (sf.stride(-2) == 1 || per_group <= 1) && (cols <= 1 || sf.stride(-1) >= per_group) &&
                    (sf.dim() == 2 || plan.experts <= 1 || sf.stride(0) >= (cols > 1 ? (cols - 1) * sf.stride(-1) : 0) + per_group),
                    "the scales of out must be int16, one element for 64 channels of each row, contiguous along the rows");
    } else {
        out = empty_on(plan.shape(hidden), torch::kFloat8_e4m3fn, x);
        sf = empty_scales(plan.shape(cols), x);
    }
    const int64_t stride = plan.check_rows(out, "out must hold a row for each of the layout's, at one distance");
    const uint64_t nbytes = dg_moe_dispatch_fp8_scratch_bytes((uint32_t)plan.tokens, (uint32_t)hidden);
    const auto scratch = nbytes ? empty_on({(int64_t)nbytes}, torch::kUInt8, x) : torch::Tensor();
    check(dg_moe_dispatch_fp8_launch(x.data_ptr(), (uint64_t)stride_of_rows(x), (uint32_t)plan.tokens, (uint32_t)plan.topk, (uint32_t)hidden,
                                     plan.token_rows_ptr(), plan.row_choices_ptr(), (uint64_t)plan.rows,
                                     out.data_ptr(), (uint64_t)stride, static_cast<int16_t*>(sf.data_ptr()),
                                     (uint64_t)(cols > 1 ? sf.stride(-1) : per_group), sf.dim() == 3 && plan.experts > 1 ? (uint64_t)sf.stride(0) : 0,
                                     (uint32_t)per_group, nbytes ? scratch.data_ptr() : nullptr, nbytes, stream_of(x)));
    return {out, sf};
}

inline torch::Tensor moe_combine(const torch::Tensor& rows, const MoePlan& plan_in, const std::optional<torch::Tensor>& topk_weights,
                                 const std::optional<torch::Tensor>& out_in) {
    host_assert(rows.is_cuda() && (rows.dim() == 2 || rows.dim() == 3) && bf16_or_fp32(rows), "rows must be a 2-D or 3-D BF16 or FP32 tensor on a CUDA device");
    const MoeRows plan(plan_in, rows, -1);
    const int64_t stride = plan.check_rows(rows, "rows must hold a row for each of the layout's, at one distance"), hidden = rows.size(-1);
    host_assert(hidden <= INT32_MAX, "rows are too long");
    if (topk_weights.has_value()) check_weights(topk_weights.value(), plan);
    const c10::cuda::CUDAGuard guard(rows.device());
    if (out_in.has_value())
        host_assert(out_in->scalar_type() == rows.scalar_type() && out_in->device() == rows.device() && out_in->dim() == 2 && out_in->size(0) == plan.tokens &&
                    out_in->size(1) == hidden && out_in->stride(1) == 1 && stride_of_rows(out_in.value()) >= hidden,
                    "out must be a row-major [tokens, hidden] tensor of the type and the device of rows");
    const auto out = out_in.has_value() ? out_in.value() : empty_on({plan.tokens, hidden}, rows.scalar_type(), rows);
    check(dg_moe_combine_launch(rows.data_ptr(), rows.scalar_type() == torch::kFloat32, (uint64_t)stride, (uint64_t)plan.rows, (uint32_t)hidden, plan.token_rows_ptr(),
                                (uint32_t)plan.tokens, (uint32_t)plan.topk, topk_weights.has_value() ? static_cast<const float*>(topk_weights->data_ptr()) : nullptr,
                                out.data_ptr(), (uint64_t)stride_of_rows(out), stream_of(rows)));
    return out;
}

inline TensorPair moe_combine_grad(const torch::Tensor& grad_out, const torch::Tensor& rows, const MoePlan& plan_in, const torch::Tensor& topk_weights,
                                   const std::optional<torch::Tensor>& out_in, bool zero_padding, int64_t expert_alignment) {
    check_tokens(grad_out, "grad_out must be a row-major 2-D BF16 or FP32 tensor on a CUDA device");
    const MoeRows plan(plan_in, grad_out, grad_out.size(0));
    const int64_t hidden = grad_out.size(1);
    host_assert(rows.scalar_type() == grad_out.scalar_type() && rows.device() == grad_out.device() && rows.size(-1) == hidden,
                "rows must have the type, the device and the row length of grad_out");
    const int64_t stride = plan.check_rows(rows, "rows must hold a row for each of the layout's, at one distance");
    host_assert(hidden <= INT32_MAX, "rows are too long");
    check_weights(topk_weights, plan);
    check_alignment(expert_alignment);
    const c10::cuda::CUDAGuard guard(grad_out.device());
    if (out_in.has_value())
        host_assert(out_in->scalar_type() == rows.scalar_type() && out_in->device() == rows.device() && out_in->size(-1) == hidden,
                    "out must have the type, the device and the row length of rows");
    const auto out = out_in.has_value() ? out_in.value() : empty_on(plan.shape(hidden), rows.scalar_type(), rows);
    const int64_t out_stride = plan.check_rows(out, "out must hold a row for each of the layout's, at one distance");
    const auto grad_weights = empty_on(topk_weights.sizes(), topk_weights.scalar_type(), topk_weights);
    check(dg_moe_combine_grad_launch(grad_out.data_ptr(), rows.scalar_type() == torch::kFloat32, (uint64_t)stride_of_rows(grad_out), rows.data_ptr(), (uint64_t)stride,
                                     (uint64_t)plan.rows, (uint32_t)hidden, plan.token_rows_ptr(), plan.row_choices_ptr(), (uint32_t)plan.tokens,
                                     (uint32_t)plan.topk, static_cast<const float*>(topk_weights.data_ptr()), out.data_ptr(), (uint64_t)out_stride,
                                     static_cast<float*>(grad_weights.data_ptr()), plan.layout_ptr(), (uint32_t)plan.experts, (uint32_t)expert_alignment,
                                     (uint32_t)plan.max_m, zero_padding, stream_of(grad_out)));
    return {out, grad_weights};
}

inline void register_moe_apis(py::module_& m) {
    m.def("moe_route", &moe_route, py::arg("logits"), py::arg("topk"), py::arg("scoring") = "softmax", py::arg("bias") = std::nullopt, py::arg("num_groups") = 1,
          py::arg("topk_groups") = 1, py::arg("group_best") = 2, py::arg("renormalize") = false, py::arg("scale") = 1.0);
    m.def("moe_route_grad", &moe_route_grad, py::arg("grad_weights"), py::arg("logits"), py::arg("topk_idx"), py::arg("scoring") = "softmax",
          py::arg("renormalize") = false, py::arg("scale") = 1.0, py::arg("out") = std::nullopt);
    m.def("moe_sort", &moe_sort, py::arg("topk_idx"), py::arg("num_experts"), py::arg("expert_alignment") = kMkAlignment, py::arg("max_m") = std::nullopt);
    m.def("moe_dispatch", &moe_dispatch, py::arg("x"), py::arg("plan"), py::arg("out") = std::nullopt, py::arg("zero_padding") = false,
          py::arg("expert_alignment") = kMkAlignment);
    m.def("moe_dispatch_to_fp8", &moe_dispatch_to_fp8, py::arg("x"), py::arg("plan"), py::arg("out") = std::nullopt);
    m.def("moe_combine", &moe_combine, py::arg("rows"), py::arg("plan"), py::arg("topk_weights") = std::nullopt, py::arg("out") = std::nullopt);
    m.def("moe_combine_grad", &moe_combine_grad, py::arg("grad_out"), py::arg("rows"), py::arg("plan"), py::arg("topk_weights"), py::arg("out") = std::nullopt,
          py::arg("zero_padding") = false, py::arg("expert_alignment") = kMkAlignment);
}

}  // namespace dg_host
