// From the router's choices to the rows of a grouped layout and back: what stands in front of and behind the m-grouped GEMMs.
//
// With T tokens of k choices each, i = t k + j the index of a choice and e_i its expert, the row of a choice is
//     row(i) = start(e_i) + #{i' < i : e_i' = e_i}
// with start(g) the sum of the earlier groups' sizes, each rounded up to the alignment (psum layout), or g * max_m (masked layout,
// where what comes after max_m rows is dropped). The order inside a group is that of the choices, so results do not depend on timing.
//     dispatch   rows[row(t,j)] = x[t]                        (copied, or quantised to E4M3 + UE8M0 per 32)
//     combine    out[t] = sum_j w[t,j] rows[row(t,j)]         (FP32 sums in the order of j, one rounding)
//     gradient   drows[row(t,j)] = w[t,j] dout[t],  dw[t,j] = <rows[row(t,j)], dout[t]>
// A choice without a row (an expert of another rank, or dropped) takes part in none of them; its dw is 0. Every row has one writer,
// so there are no atomics. Everything but the sort is bound by HBM: each token's row and each expert row moves once.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

// ---------------------------------------------------------------------------------------------------------- sort
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortMaxExperts = 1024, kSortMaxCluster = 8;

struct SortArgs {
    const void* idx;                                    // [n] int32 or int64
    int32_t *layout, *token_rows, *row_choices;         // [experts], [n], [rows]
    uint32_t n, experts, alignment, max_m, rows;
    uint32_t segment;                                   // choices of a warp, a multiple of 32
    uint32_t warps;                                     // warps of a CTA that hold choices
};

template <typename T>
__device__ __forceinline__ uint32_t expert_of(const SortArgs& a, uint32_t i, uint32_t end) {
    if (i >= end) return 0xffffffffu;
    T e;
    if constexpr (sizeof(T) == 8) asm volatile("ld.global.s64 %0, [%1];" : "=l"(e) : "l"(static_cast<const T*>(a.idx) + i));
    else asm volatile("ld.global.s32 %0, [%1];" : "=r"(e) : "l"(static_cast<const T*>(a.idx) + i));
    return e >= 0 && e < (T)a.experts ? (uint32_t)e : 0xffffffffu;
}

// A stable counting sort in one launch: one CTA, or a cluster whose CTAs exchange their counts through distributed shared memory.
// Every warp owns a run of choices and a row of counters of its own (no atomics): it counts, the counters become offsets (over the
// warps of the CTA, the CTAs of the cluster, and the experts with their alignment), and it walks its run a second time to hand
// out rows. Within 32 choices the order is that of the lanes (match).
template <typename T>
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const SortArgs a) {
    extern __shared__ uint32_t smem[];
    uint32_t* const counts = smem;                                      // [warps][experts]
    uint32_t* const totals = smem + a.warps * a.experts;                // [experts]: of this CTA
    uint32_t* const bases = totals + a.experts;                         // [experts]: row of this CTA's first choice
    __shared__ uint32_t scan[kSortWarps];
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t cta = blockIdx.x, ctas = gridDim.x;
    for (uint32_t i = tid; i < a.warps * a.experts; i += kSortThreads) counts[i] = 0;
    griddep_wait();
    griddep_launch_dependents();
    // no row holds a choice until the second pass says so (the barrier in between orders the writes)
    for (uint32_t i = cta * kSortThreads + tid; i < a.rows; i += ctas * kSortThreads) a.row_choices[i] = -1;
    __syncthreads();
    const uint32_t first = min(a.n, (cta * a.warps + warp) * a.segment), last = warp < a.warps ? min(a.n, first + a.segment) : first;
    uint32_t* const mine = counts + warp * a.experts;
    for (uint32_t i0 = first; i0 < last; i0 += 32) {
        const uint32_t e = expert_of<T>(a, i0 + lane, last);
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        if (e != 0xffffffffu && lane == (uint32_t)__ffs(peers) - 1) mine[e] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    uint32_t total = 0;
    if (tid < a.experts) {
        for (uint32_t w = 0; w < a.warps; ++w) {
            const uint32_t c = counts[w * a.experts + tid];
            counts[w * a.experts + tid] = total;
            total += c;
        }
        totals[tid] = total;
    }
    uint32_t before = 0;
    if (ctas > 1) {
        cluster_arrive();
        cluster_wait();
        if (tid < a.experts) {
            total = 0;
            const uint32_t at = smem_u32(totals + tid);
            for (uint32_t r = 0; r < ctas; ++r) {
                uint32_t c;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(mapa_shared(at, r)) : "memory");
                before += r < cta ? c : 0u;
                total += c;
            }
        }
        cluster_arrive();
    }
    // exclusive sum over the experts' sizes
    const uint32_t size = tid >= a.experts ? 0u : a.max_m ? a.max_m : (total + a.alignment - 1) / a.alignment * a.alignment;
    uint32_t start = size;
    #pragma unroll
    for (uint32_t d = 1; d < 32; d *= 2) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, start, d);
        if (lane >= d) start += up;
    }
    if (lane == 31) scan[warp] = start;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = scan[lane];
        #pragma unroll
        for (uint32_t d = 1; d < 32; d *= 2) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += up;
        }
        scan[lane] = s;
    }
    __syncthreads();
    start = start - size + (warp == 0 ? 0u : scan[warp - 1]);
    if (tid < a.experts) {
        bases[tid] = start + before;
        if (cta == 0) a.layout[tid] = (int32_t)(a.max_m ? min(total, a.max_m) : start + total);
    }
    __syncthreads();
    for (uint32_t i0 = first; i0 < last; i0 += 32) {
        const uint32_t i = i0 + lane, e = expert_of<T>(a, i, last);
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        uint32_t row = 0xffffffffu;
        if (e != 0xffffffffu) {
            row = bases[e] + mine[e] + __popc(peers & ((1u << lane) - 1u));
            if (a.max_m && row >= (e + 1) * a.max_m) row = 0xffffffffu;
        }
        __syncwarp();
        if (e != 0xffffffffu && lane == (uint32_t)__ffs(peers) - 1) mine[e] += __popc(peers);
        __syncwarp();
        if (i < last) a.token_rows[i] = (int32_t)row;
        if (row < a.rows) a.row_choices[row] = (int32_t)i;
    }
    if (ctas > 1) cluster_wait();                       // the others have read this CTA's totals
}

// -------------------------------------------------------------------------------------------------- rows and layouts
// What the other kernels know of the layout.
struct RowsArgs {
    const int32_t* token_rows;                          // [tokens][topk]
    const int32_t* layout; uint32_t experts, alignment, max_m;     // of the padding, where it is to be zeroed
    uint32_t tokens, topk, rows;
};

// Zeros in the padding row that `item` stands for: items [0, alignment) (psum) or [0, max_m) (masked) belong to the first group, and
// so on. One warp a row, `units` pieces of 16 bytes.
__device__ __forceinline__ void zero_padding_row(const RowsArgs& a, uint64_t item, uint8_t* out, uint64_t stride, uint32_t units, uint32_t lane) {
    const uint32_t span = a.max_m ? a.max_m : a.alignment, g = (uint32_t)(item / span), r = (uint32_t)(item - (uint64_t)g * span);
    if (g >= a.experts) return;
    const uint32_t p = ld_global_u32(a.layout + g);
    const uint64_t row = a.max_m ? (uint64_t)g * a.max_m + r : (uint64_t)p + r;
    if (a.max_m ? r < p : row >= ((uint64_t)p + a.alignment - 1) / a.alignment * a.alignment) return;
    if (row >= a.rows) return;
    for (uint32_t u = lane; u < units; u += 32) *reinterpret_cast<uint4*>(out + row * stride + (uint64_t)u * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// -------------------------------------------------------------------------------------------------- dispatch
constexpr uint32_t kMoeThreads = 256, kMoeWarps = kMoeThreads / 32;
constexpr uint32_t kCopyUnits = 4;                      // pieces of 16 bytes that a lane of the copy holds

struct DispatchArgs {
    RowsArgs r;
    const uint8_t* x; uint64_t x_stride;                // bytes
    uint8_t* out; uint64_t out_stride;                  // bytes
    uint32_t units, chunks;                             // of 16 bytes in a row; warps a row takes
    uint64_t token_items, items;                        // warps that copy, and with those that zero the padding
    uint8_t* sf; uint64_t sf_col_stride, sf_group_stride;          // E4M3 only: bytes between scale columns and groups
    uint32_t sf_rows, hidden;                                      // rows of a group of scales
};

// A warp takes 32 x kCopyUnits pieces of a token's row, reads them once and writes them to the rows of all its choices.
__global__ void __launch_bounds__(kMoeThreads) moe_dispatch_kernel(const DispatchArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint64_t item = (uint64_t)blockIdx.x * kMoeWarps + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.token_items) {
        if (item < a.items) zero_padding_row(a.r, item - a.token_items, a.out, a.out_stride, a.units, lane);
        return;
    }
    const uint32_t token = (uint32_t)(item / a.chunks), u0 = (uint32_t)(item - (uint64_t)token * a.chunks) * 32 * kCopyUnits + lane;
    uint4 v[kCopyUnits];
    #pragma unroll
    for (uint32_t k = 0; k < kCopyUnits; ++k)
        if (u0 + k * 32 < a.units) v[k] = ld_stream_v4(a.x + token * a.x_stride + (uint64_t)(u0 + k * 32) * 16);
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
        const uint32_t mine = j0 + lane < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j0 + lane) : 0xffffffffu;
        for (uint32_t j = 0; j < min(32u, a.r.topk - j0); ++j) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, j);
            if (row >= a.r.rows) continue;
            #pragma unroll
            for (uint32_t k = 0; k < kCopyUnits; ++k)
                if (u0 + k * 32 < a.units) *reinterpret_cast<uint4*>(a.out + row * a.out_stride + (uint64_t)(u0 + k * 32) * 16) = v[k];
        }
    }
}

// The same with a quantisation on the way: a warp takes 256 channels of a token, eight to a lane, four lanes to a block of 32.
__global__ void __launch_bounds__(kMoeThreads) moe_dispatch_fp8_kernel(const DispatchArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint64_t item = (uint64_t)blockIdx.x * kMoeWarps + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.token_items) return;
    const uint32_t token = (uint32_t)(item / a.chunks), c0 = (uint32_t)(item - (uint64_t)token * a.chunks) * 256, c = c0 + lane * 8;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (c < a.hidden) raw = ld_stream_v4(a.x + token * a.x_stride + (uint64_t)c * 2);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float v[8], amax = 0.f;
    #pragma unroll
    for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
    #pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t e = e4m3_scale_byte(amax);
    const uint2 q = e4m3_pack8(v, e);
    // scale column lane % 4 of this tile: the bytes of blocks 2 (lane % 4) and 2 (lane % 4) + 1 (zero behind the last one)
    const uint32_t byte = c < a.hidden ? e : 0u, col = lane % 4;
    const uint32_t pair = __shfl_sync(0xffffffffu, byte, col * 8) | (__shfl_sync(0xffffffffu, byte, col * 8 + 4) << 8);
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
        const uint32_t mine = j0 + lane < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j0 + lane) : 0xffffffffu;
        const uint32_t some = min(32u, a.r.topk - j0);
        for (uint32_t j = 0; j < some; ++j) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, j);
            if (row < a.r.rows && c < a.hidden) *reinterpret_cast<uint2*>(a.out + row * a.out_stride + c) = q;
        }
        // eight rows' scales at a time, four columns each
        for (uint32_t j = 0; j < some; j += 8) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, min(31u, j + lane / 4));
            if (j + lane / 4 < some && row < a.r.rows && c0 + col * 64 < a.hidden) {
                const uint32_t g = row / a.sf_rows;
                *reinterpret_cast<uint16_t*>(a.sf + g * a.sf_group_stride + (uint64_t)(c0 / 64 + col) * a.sf_col_stride + (uint64_t)(row - g * a.sf_rows) * 2) = (uint16_t)pair;
            }
        }
    }
}

// -------------------------------------------------------------------------------------------------- combine
struct CombineArgs {
    RowsArgs r;
    const uint8_t* y; uint64_t y_stride;                // [rows], bytes
    const float* w;                                     // [tokens][topk] or nullptr
    uint8_t* out; uint64_t out_stride;
    uint32_t units, chunks;
    uint64_t items;
};

// 16 bytes as FP32 values, and back.
template <typename T> struct Unit;
template <> struct Unit<__nv_bfloat16> {
    static constexpr int kValues = 8;
    static __device__ __forceinline__ void values(const uint4& q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        uint32_t w[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Unit<float> {
    static constexpr int kValues = 4;
    static __device__ __forceinline__ void values(const uint4& q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};

// A warp takes 32 pieces of 16 bytes of a token's result; eight rows are on their way at once.
template <typename T>
__global__ void __launch_bounds__(kMoeThreads) moe_combine_kernel(const CombineArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint64_t item = (uint64_t)blockIdx.x * kMoeWarps + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.items) return;
    const uint32_t token = (uint32_t)(item / a.chunks), u = (uint32_t)(item - (uint64_t)token * a.chunks) * 32 + lane;
    float sum[Unit<T>::kValues] = {};
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 8) {
        const uint32_t at = j0 + lane % 8;
        const uint32_t mine = at < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + at) : 0xffffffffu;
        const float weight = a.w != nullptr && at < a.r.topk ? __uint_as_float(ld_global_u32(a.w + (uint64_t)token * a.r.topk + at)) : 1.0f;
        uint4 q[8];
        #pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, j);
            if (row < a.r.rows && u < a.units) q[j] = ld_stream_v4(a.y + row * a.y_stride + (uint64_t)u * 16);
        }
        #pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, j);
            const float w = __shfl_sync(0xffffffffu, weight, j);
            if (row < a.r.rows && u < a.units) {
                float v[Unit<T>::kValues];
                Unit<T>::values(q[j], v);
                #pragma unroll
                for (int k = 0; k < Unit<T>::kValues; ++k) sum[k] = fmaf(w, v[k], sum[k]);
            }
        }
    }
    if (u < a.units) *reinterpret_cast<uint4*>(a.out + token * a.out_stride + (uint64_t)u * 16) = Unit<T>::pack(sum);
}

// -------------------------------------------------------------------------------------------------- gradient of the combine
struct CombineGradArgs {
    RowsArgs r;
    const uint8_t* g; uint64_t g_stride;                // gradient of the result, [tokens]
    const uint8_t* y; uint64_t y_stride;
    const float* w;
    uint8_t* dy; uint64_t dy_stride;
    float* dw;                                          // [tokens][topk]
    uint32_t units;
};

// One CTA a token: its gradient is read once and multiplied with eight rows at a time; the products with the rows are summed over the
// CTA. The CTAs behind the last token zero the padding.
template <typename T>
__global__ void __launch_bounds__(kMoeThreads) moe_combine_grad_kernel(const CombineGradArgs a) {
    __shared__ float partial[kMoeWarps][8];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, token = blockIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.r.tokens) {
        zero_padding_row(a.r, (uint64_t)(token - a.r.tokens) * kMoeWarps + warp, a.dy, a.dy_stride, a.units, lane);
        return;
    }
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 8) {
        uint32_t row[8];
        float weight[8], dot[8];
        #pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const bool is = j0 + j < a.r.topk;
            row[j] = is ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j0 + j) : 0xffffffffu;
            weight[j] = is ? __uint_as_float(ld_global_u32(a.w + (uint64_t)token * a.r.topk + j0 + j)) : 0.f;
            dot[j] = 0.f;
        }
        for (uint32_t u = threadIdx.x; u < a.units; u += kMoeThreads) {
            uint4 q[8];
            const uint4 gq = ld_global_v4(a.g + token * a.g_stride + (uint64_t)u * 16);
            #pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (row[j] < a.r.rows) q[j] = ld_stream_v4(a.y + row[j] * a.y_stride + (uint64_t)u * 16);
            float g[Unit<T>::kValues];
            Unit<T>::values(gq, g);
            #pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                if (row[j] >= a.r.rows) continue;
                float v[Unit<T>::kValues], d[Unit<T>::kValues];
                Unit<T>::values(q[j], v);
                #pragma unroll
                for (int k = 0; k < Unit<T>::kValues; ++k) {
                    dot[j] = fmaf(v[k], g[k], dot[j]);
                    d[k] = weight[j] * g[k];
                }
                *reinterpret_cast<uint4*>(a.dy + row[j] * a.dy_stride + (uint64_t)u * 16) = Unit<T>::pack(d);
            }
        }
        #pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            #pragma unroll
            for (uint32_t d = 16; d > 0; d /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
            if (lane == 0) partial[warp][j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < 8 && j0 + threadIdx.x < a.r.topk) {
            float s = 0.f;
            #pragma unroll
            for (uint32_t w = 0; w < kMoeWarps; ++w) s += partial[w][threadIdx.x];
            a.dw[(uint64_t)token * a.r.topk + j0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
}

}  // namespace dg

using namespace dg;

extern "C" uint64_t dg_moe_num_rows(uint32_t choices, uint32_t num_experts, uint32_t alignment) {
    const uint64_t used = choices < num_experts ? choices : num_experts;
    return used == 0 || alignment == 0 ? 0 : (uint64_t)alignment * (used + (choices - used) / alignment);
}

extern "C" int dg_moe_sort_launch(const void* topk_idx, int idx_is_int64, uint32_t tokens, uint32_t topk, uint32_t num_experts, uint32_t alignment,
                                  uint32_t max_m, int32_t* layout, int32_t* token_rows, int32_t* row_choices, uint64_t num_rows, void* stream) {
    DG_CHECK_ARG(num_experts > 0 && num_experts <= kSortMaxExperts, "moe_sort: the number of experts must be between 1 and %u", kSortMaxExperts);
    DG_CHECK_ARG((uint64_t)tokens * topk <= 0x7fffffffull, "moe_sort: too many choices");
    const uint32_t n = tokens * topk;
    DG_CHECK_ARG(layout != nullptr && (n == 0 || (topk_idx != nullptr && token_rows != nullptr)) && (num_rows == 0 || row_choices != nullptr),
                 "moe_sort: null pointer");
    DG_CHECK_ARG(max_m > 0 || alignment > 0, "moe_sort: the alignment must be positive");
    DG_CHECK_ARG(num_rows == (max_m ? (uint64_t)num_experts * max_m : dg_moe_num_rows(n, num_experts, alignment)), "moe_sort: wrong number of rows");
    DG_CHECK_ARG(num_rows <= 0x7fffffffull, "moe_sort: too many rows");
    SortArgs a{};
    a.idx = topk_idx; a.layout = layout; a.token_rows = token_rows; a.row_choices = row_choices;
    a.n = n; a.experts = num_experts; a.alignment = max_m ? 1 : alignment; a.max_m = max_m; a.rows = (uint32_t)num_rows;
    const uint32_t ctas = n <= 4096 && num_rows <= 16384 ? 1 : kSortMaxCluster;
    a.segment = ((n + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) / 32 * 32;
    a.warps = a.segment == 0 ? 0 : (n + a.segment - 1) / a.segment < kSortWarps ? (n + a.segment - 1) / a.segment : kSortWarps;
    const uint32_t smem = (a.warps + 2) * num_experts * 4;
    const void* fn = idx_is_int64 ? (const void*)moe_sort_kernel<int64_t> : (const void*)moe_sort_kernel<int32_t>;
    if (smem > 48 * 1024) DG_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    void* params[] = {&a};
    return launch_overlapped(fn, dim3(ctas), dim3(kSortThreads), params, static_cast<cudaStream_t>(stream), smem, ctas);
}

// Checks of what the other three share; fills `r`.
static int rows_args(RowsArgs& r, const int32_t* token_rows, uint32_t tokens, uint32_t topk, uint64_t num_rows, const int32_t* layout,
                     uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding) {
    DG_CHECK_ARG(token_rows != nullptr || (uint64_t)tokens * topk == 0, "moe: null pointer");
    DG_CHECK_ARG((uint64_t)tokens * topk <= 0x7fffffffull && num_rows <= 0x7fffffffull, "moe: too many choices or rows");
    DG_CHECK_ARG(!zero_padding || (layout != nullptr && num_experts > 0 && (max_m > 0 || alignment > 0)), "moe: zeros in the padding need the layout");
    r.token_rows = token_rows; r.tokens = tokens; r.topk = topk; r.rows = (uint32_t)num_rows;
    r.layout = layout; r.experts = zero_padding ? num_experts : 0; r.alignment = alignment; r.max_m = max_m;
    return DG_OK;
}
static uint64_t padding_items(const RowsArgs& r) { return (uint64_t)r.experts * (r.max_m ? r.max_m : r.alignment); }
static bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride_bytes % 16 == 0; }

extern "C" int dg_moe_dispatch_launch(const void* x, uint64_t x_stride_bytes, uint32_t tokens, uint32_t topk, uint64_t row_bytes,
                                      const int32_t* token_rows, uint64_t num_rows, void* out, uint64_t out_stride_bytes,
                                      const int32_t* layout, uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding, void* stream) {
    if (row_bytes == 0 || num_rows == 0) return DG_OK;
    DG_CHECK_ARG(out != nullptr && (x != nullptr || tokens == 0), "moe_dispatch: null pointer");
    DG_CHECK_ARG(row_bytes % 16 == 0 && aligned16(x, x_stride_bytes) && aligned16(out, out_stride_bytes),
                 "moe_dispatch: rows must start on 16-byte boundaries and hold a multiple of 16 bytes");
    DG_CHECK_ARG(row_bytes / 16 <= 0x7fffffffull, "moe_dispatch: rows too long");
    DispatchArgs a{};
    if (int rc = rows_args(a.r, token_rows, tokens, topk, num_rows, layout, num_experts, alignment, max_m, zero_padding)) return rc;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride_bytes;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride_bytes;
    a.units = (uint32_t)(row_bytes / 16);
    a.chunks = (a.units + 32 * kCopyUnits - 1) / (32 * kCopyUnits);
    a.token_items = (uint64_t)tokens * a.chunks;
    a.items = a.token_items + padding_items(a.r);
    const uint64_t ctas = (a.items + kMoeWarps - 1) / kMoeWarps;
    if (ctas == 0) return DG_OK;
    DG_CHECK_ARG(ctas <= 0x7fffffffull, "moe_dispatch: too many rows");
    void* params[] = {&a};
    return launch_overlapped((const void*)moe_dispatch_kernel, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
}

extern "C" int dg_moe_dispatch_fp8_launch(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t topk, uint32_t hidden,
                                          const int32_t* token_rows, uint64_t num_rows, void* out, uint64_t out_stride,
                                          int16_t* out_sf, uint64_t sf_col_stride, uint64_t sf_group_stride, uint32_t sf_rows, void* stream) {
    if (tokens == 0 || topk == 0 || hidden == 0 || num_rows == 0) return DG_OK;
    DG_CHECK_ARG(x != nullptr && out != nullptr && out_sf != nullptr, "moe_dispatch_fp8: null pointer");
    DG_CHECK_ARG(hidden % 32 == 0, "moe_dispatch_fp8: hidden must be a multiple of 32");
    DG_CHECK_ARG(aligned16(x, x_stride * 2), "moe_dispatch_fp8: input rows must start on 16-byte boundaries");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 7) == 0 && out_stride % 8 == 0, "moe_dispatch_fp8: output rows must start on 8-byte boundaries");
    DG_CHECK_ARG(sf_rows > 0 && sf_col_stride >= sf_rows, "moe_dispatch_fp8: scale column stride smaller than the rows of a group");
    DispatchArgs a{};
    if (int rc = rows_args(a.r, token_rows, tokens, topk, num_rows, nullptr, 0, 0, 0, 0)) return rc;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride;
    a.sf = reinterpret_cast<uint8_t*>(out_sf); a.sf_col_stride = sf_col_stride * 2; a.sf_group_stride = sf_group_stride * 2;
    a.sf_rows = sf_rows; a.hidden = hidden;
    a.chunks = (hidden + 255) / 256;
    a.token_items = (uint64_t)tokens * a.chunks;
    const uint64_t ctas = (a.token_items + kMoeWarps - 1) / kMoeWarps;
    DG_CHECK_ARG(ctas <= 0x7fffffffull, "moe_dispatch_fp8: too many tokens");
    void* params[] = {&a};
    return launch_overlapped((const void*)moe_dispatch_fp8_kernel, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
}

extern "C" int dg_moe_combine_launch(const void* rows, int is_fp32, uint64_t rows_stride, uint64_t num_rows, uint32_t hidden, const int32_t* token_rows,
                                     uint32_t tokens, uint32_t topk, const float* topk_weights, void* out, uint64_t out_stride, void* stream) {
    if (tokens == 0 || hidden == 0) return DG_OK;
    const uint64_t es = is_fp32 ? 4 : 2;
    DG_CHECK_ARG(out != nullptr && (rows != nullptr || num_rows == 0), "moe_combine: null pointer");
    DG_CHECK_ARG(hidden * es % 16 == 0 && aligned16(rows, rows_stride * es) && aligned16(out, out_stride * es),
                 "moe_combine: rows must start on 16-byte boundaries and hold a multiple of 16 bytes");
    CombineArgs a{};
    if (int rc = rows_args(a.r, token_rows, tokens, topk, num_rows, nullptr, 0, 0, 0, 0)) return rc;
    a.y = static_cast<const uint8_t*>(rows); a.y_stride = rows_stride * es;
    a.w = topk_weights;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride * es;
    a.units = (uint32_t)(hidden * es / 16);
    a.chunks = (a.units + 31) / 32;
    a.items = (uint64_t)tokens * a.chunks;
    const uint64_t ctas = (a.items + kMoeWarps - 1) / kMoeWarps;
    DG_CHECK_ARG(ctas <= 0x7fffffffull, "moe_combine: too many tokens");
    const void* fn = is_fp32 ? (const void*)moe_combine_kernel<float> : (const void*)moe_combine_kernel<__nv_bfloat16>;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
}

extern "C" int dg_moe_combine_grad_launch(const void* grad_out, int is_fp32, uint64_t grad_stride, const void* rows, uint64_t rows_stride,
                                          uint64_t num_rows, uint32_t hidden, const int32_t* token_rows, uint32_t tokens, uint32_t topk,
                                          const float* topk_weights, void* grad_rows, uint64_t grad_rows_stride, float* grad_weights,
                                          const int32_t* layout, uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding,
                                          void* stream) {
    if (tokens == 0 && !zero_padding) return DG_OK;
    const uint64_t es = is_fp32 ? 4 : 2;
    DG_CHECK_ARG((tokens == 0 || hidden == 0 || grad_out != nullptr) && (num_rows == 0 || hidden == 0 || (rows != nullptr && grad_rows != nullptr)) &&
                 (tokens == 0 || topk == 0 || (topk_weights != nullptr && grad_weights != nullptr)), "moe_combine_grad: null pointer");
    DG_CHECK_ARG(hidden * es % 16 == 0 && aligned16(grad_out, grad_stride * es) && aligned16(rows, rows_stride * es) &&
                 aligned16(grad_rows, grad_rows_stride * es), "moe_combine_grad: rows must start on 16-byte boundaries and hold a multiple of 16 bytes");
    CombineGradArgs a{};
    if (int rc = rows_args(a.r, token_rows, tokens, topk, num_rows, layout, num_experts, alignment, max_m, zero_padding)) return rc;
    a.g = static_cast<const uint8_t*>(grad_out); a.g_stride = grad_stride * es;
    a.y = static_cast<const uint8_t*>(rows); a.y_stride = rows_stride * es;
    a.w = topk_weights;
    a.dy = static_cast<uint8_t*>(grad_rows); a.dy_stride = grad_rows_stride * es;
    a.dw = grad_weights;
    a.units = (uint32_t)(hidden * es / 16);
    const uint64_t ctas = tokens + (padding_items(a.r) + kMoeWarps - 1) / kMoeWarps;
    if (ctas == 0) return DG_OK;
    DG_CHECK_ARG(ctas <= 0x7fffffffull, "moe_combine_grad: too many rows");
    const void* fn = is_fp32 ? (const void*)moe_combine_grad_kernel<float> : (const void*)moe_combine_grad_kernel<__nv_bfloat16>;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
}
