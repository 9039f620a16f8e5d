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

#include <atomic>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

// ---------------------------------------------------------------------------------------------------------- sort
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortMaxExperts = 1024, kSortMaxCluster = 16, kSortBatch = 8;

struct SortArgs {
    const void* idx;                                    // [n] int32 or int64
    int32_t *layout, *token_rows, *row_choices;         // [experts], [n], [rows]
    uint32_t n, experts, alignment, max_m, rows;
    uint32_t segment;                                   // choices of a warp, a multiple of 32
    uint32_t warps;                                     // warps of a CTA that hold choices
};

// The experts of kBatch runs of 32 choices from `i` on (all loads on their way at once); `experts` stands for none.
template <typename T, uint32_t kBatch>
__device__ __forceinline__ void load_experts(const SortArgs& a, uint32_t i, uint32_t end, uint32_t (&expert)[kBatch]) {
    T e[kBatch];
    #pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) {
        e[k] = -1;
        if (i + k * 32 < end) {
            const T* p = static_cast<const T*>(a.idx) + i + k * 32;
            if constexpr (sizeof(T) == 8) asm volatile("ld.global.s64 %0, [%1];" : "=l"(e[k]) : "l"(p));
            else asm volatile("ld.global.s32 %0, [%1];" : "=r"(e[k]) : "l"(p));
        }
    }
    #pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) expert[k] = e[k] >= 0 && e[k] < (T)a.experts ? (uint32_t)e[k] : a.experts;
}
// The lanes that hold the same expert, bit by bit (a match over 32 lanes takes a turn for every value that occurs: three times as long).
__device__ __forceinline__ uint32_t same_expert(uint32_t e, uint32_t bits) {
    uint32_t peers = 0xffffffffu;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (e >> b) & 1u;
        const uint32_t with = __ballot_sync(0xffffffffu, set);
        peers &= set ? with : ~with;
    }
    return peers;
}

// A stable counting sort in one launch: one CTA, or a cluster whose CTAs exchange their counts through distributed shared memory.
// Every warp owns a run of choices and a row of counters of its own (no atomics): it counts, the counters become offsets (over the
// warps of the CTA, the CTAs of the cluster, and the experts with their alignment), and it walks its run a second time to hand
// out rows. Within 32 choices the order is that of the lanes. Runs that fit kBatch are read once; kBatch is 1 where 32 choices for each
// of a CTA's warps are all (1024 choices: 3.6 us against 4.4 with 8). 131072 choices of 256 experts: 12.2 us with 16 CTAs, 19 with 8; 40 with
// one load at a time and a match for the peers.
template <typename T, uint32_t kBatch>
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const SortArgs a) {
    extern __shared__ uint32_t smem[];
    uint32_t* const counts = smem;                                      // [warps][experts]
    uint32_t* const totals = smem + a.warps * a.experts;                // [experts]: of this CTA
    uint32_t* const bases = totals + a.experts;                         // [experts]: row of this CTA's first choice
    // experts of the batch whose rows a thread hands out (kept here, the loop over them need not be unrolled)
    uint16_t* const held = reinterpret_cast<uint16_t*>(bases + a.experts);      // [kBatch][threads]
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
    uint32_t expert[kBatch];
    for (uint32_t i0 = first; i0 < last; i0 += 32 * kBatch) {
        load_experts<T>(a, i0 + lane, last, expert);
        #pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            if (expert[k] < a.experts) atomicAdd(mine + expert[k], 1u);
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
    const uint32_t bits = 32 - __clz(a.experts);
    for (uint32_t i0 = first; i0 < last; i0 += 32 * kBatch) {
        if (last - first > 32 * kBatch) load_experts<T>(a, i0 + lane, last, expert);
        #pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) held[k * kSortThreads + tid] = (uint16_t)expert[k];
        #pragma unroll 1
        for (uint32_t k = 0; k < kBatch && i0 + k * 32 < last; ++k) {
            const uint32_t i = i0 + k * 32 + lane, e = held[k * kSortThreads + tid], peers = same_expert(e, bits);
            uint32_t row = 0xffffffffu;
            if (e < a.experts) {
                row = bases[e] + mine[e] + __popc(peers & ((1u << lane) - 1u));
                if (a.max_m && row >= (e + 1) * a.max_m) row = 0xffffffffu;
            }
            __syncwarp();
            if (e < a.experts && lane == (uint32_t)__ffs(peers) - 1) mine[e] += __popc(peers);
            __syncwarp();
            if (i < last) a.token_rows[i] = (int32_t)row;
            if (row < a.rows) a.row_choices[row] = (int32_t)i;
        }
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
    uint8_t* scratch;                                              // scale bytes by token, [tokens][scratch_stride], or nullptr
    uint32_t scratch_stride;
    const int32_t* row_choices;                                    // where the scales go through the scratch
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

// The same with a quantisation on the way: a warp takes 256 channels of a token, eight to a lane, four lanes to a block of 32. The
// scales of a row lie num_rows elements apart, and the rows of a token far from one another: written from here, each is a store of two
// bytes with a sector of L2 to itself. That suits a few tokens. For many (65536 rows of 7168: 127 us, 93 without the scales), the
// bytes go to a scratch, by token, and moe_scales_kernel behind this one turns them into runs.
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
        if (a.scratch != nullptr) continue;
        // eight rows' scales at a time, four columns each
        for (uint32_t j = 0; j < some; j += 8) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, min(31u, j + lane / 4));
            if (j + lane / 4 < some && row < a.r.rows && c0 + col * 64 < a.hidden) {
                const uint32_t g = row / a.sf_rows;
                *reinterpret_cast<uint16_t*>(a.sf + g * a.sf_group_stride + (uint64_t)(c0 / 64 + col) * a.sf_col_stride + (uint64_t)(row - g * a.sf_rows) * 2) = (uint16_t)pair;
            }
        }
    }
    if (a.scratch != nullptr && lane < 4 && c0 + col * 64 < a.hidden)
        *reinterpret_cast<uint16_t*>(a.scratch + (uint64_t)token * a.scratch_stride + c0 / 32 + col * 2) = (uint16_t)pair;
}

// Scale bytes by token -> the layout that the GEMM reads. One CTA = 64 rows: their tokens' bytes are read 16 at a time into shared memory
// (rows an odd number of words apart: the columns are read without conflicts), and every scale column of the tile is a run of 128 bytes.
constexpr uint32_t kScaleRows = 64, kScaleChunk = 256;  // rows of a CTA, scale bytes of a row that it holds at a time
__global__ void __launch_bounds__(kMoeThreads) moe_scales_kernel(const DispatchArgs a) {
    __shared__ uint32_t bytes[kScaleRows][kScaleChunk / 4 + 1];
    __shared__ uint32_t token_of[kScaleRows];
    const uint32_t row0 = blockIdx.x * kScaleRows, b0 = blockIdx.y * kScaleChunk, tid = threadIdx.x;
    // (the choices come from in front of the dispatch, whose CTAs have all passed their own wait when this kernel is let in: they may be read
    // before the bytes that it writes are there)
    bool some = false;
    if (tid < kScaleRows) {
        const uint32_t choice = row0 + tid < a.r.rows ? ld_global_u32(a.row_choices + row0 + tid) : 0xffffffffu;
        const uint32_t token = choice / max(a.r.topk, 1u);
        some = (int32_t)choice >= 0 && token < a.r.tokens;
        token_of[tid] = some ? token : 0xffffffffu;
    }
    some = __syncthreads_or(some);
    griddep_wait();
    griddep_launch_dependents();
    if (!some) return;
    const uint32_t words = min(kScaleChunk, a.scratch_stride - b0) / 16;       // pieces of 16 bytes
    for (uint32_t i = tid; i < kScaleRows * words; i += kMoeThreads) {
        const uint32_t r = i / words, w = i - r * words, token = token_of[r];
        if (token == 0xffffffffu) continue;
        const uint4 v = ld_global_v4(a.scratch + (uint64_t)token * a.scratch_stride + b0 + w * 16);
        uint32_t* to = &bytes[r][w * 4];
        to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
    }
    __syncthreads();
    const uint32_t r = tid % kScaleRows, row = row0 + r;
    if (token_of[r] == 0xffffffffu) return;
    const uint32_t g = row / a.sf_rows;
    uint8_t* const to = a.sf + g * a.sf_group_stride + (uint64_t)(row - g * a.sf_rows) * 2;
    const uint32_t cols = (a.hidden + 63) / 64, c0 = b0 / 2;
    for (uint32_t c = tid / kScaleRows; c < kScaleChunk / 2 && c0 + c < cols; c += kMoeThreads / kScaleRows)
        *reinterpret_cast<uint16_t*>(to + (uint64_t)(c0 + c) * a.sf_col_stride) = (uint16_t)(bytes[r][c / 2] >> (c % 2 * 16));
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

constexpr uint32_t kGradThreads = 128, kGradCtas = 6;   // of a CTA; CTAs that an SM has the registers for

// Where the rows of up to eight choices begin. In shared memory: as registers these words left eight
// warps on an SM.
struct GradRows {
    const uint8_t* from[8];
    uint8_t* to[8];
    float weight[8];
    uint32_t choice[8];
};

// kRows rows at a time, kTurns turns of the CTA over the row together: 8 to 10 pieces of 16 bytes on their way, however few rows there are.
template <typename T, int kRows, int kTurns>
__device__ __forceinline__ void grad_rows(const CombineGradArgs& a, const uint8_t* grad, const GradRows& rows, uint32_t n, float (&dot)[kRows]) {
    #pragma unroll
    for (int r = 0; r < kRows; ++r) dot[r] = 0.f;
    for (uint32_t u0 = threadIdx.x; u0 < a.units; u0 += blockDim.x * kTurns) {
        uint4 gq[kTurns], q[kTurns][kRows];
        #pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const uint32_t u = u0 + t * blockDim.x;
            gq[t] = make_uint4(0u, 0u, 0u, 0u);
            if (u < a.units) gq[t] = ld_global_v4(grad + (uint64_t)u * 16);
            #pragma unroll
            for (uint32_t r = 0; r < kRows; ++r)
                if (u < a.units && (kRows <= 2 || r < n)) q[t][r] = ld_stream_v4(rows.from[r] + (uint64_t)u * 16);
        }
        #pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const uint32_t u = u0 + t * blockDim.x;
            float g[Unit<T>::kValues];
            Unit<T>::values(gq[t], g);
            #pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                if (u >= a.units || !(kRows <= 2 || r < n)) continue;
                float v[Unit<T>::kValues], d[Unit<T>::kValues];
                Unit<T>::values(q[t][r], v);
                const float w = rows.weight[r];
                #pragma unroll
                for (int k = 0; k < Unit<T>::kValues; ++k) {
                    dot[r] = fmaf(v[k], g[k], dot[r]);
                    d[k] = w * g[k];
                }
                *reinterpret_cast<uint4*>(rows.to[r] + (uint64_t)u * 16) = Unit<T>::pack(d);
            }
        }
    }
}

// The sums of `dot` over the CTA, of which thread r < n writes the r-th.
template <int kRows>
__device__ __forceinline__ void write_sums(const CombineGradArgs& a, const GradRows& rows, uint32_t n, float (&partial)[kGradThreads / 32][8],
                                           float (&dot)[kRows]) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    #pragma unroll
    for (int r = 0; r < kRows; ++r) {
        #pragma unroll
        for (uint32_t d = 16; d > 0; d /= 2) dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], d);
        if (lane == 0) partial[warp][r] = dot[r];
    }
    __syncthreads();
    if (threadIdx.x < n) {
        float s = 0.f;
        for (uint32_t w = 0; w < blockDim.x / 32; ++w) s += partial[w][threadIdx.x];
        a.dw[rows.choice[threadIdx.x]] = s;
    }
}

// One CTA a token: its gradient is read once and multiplied with the rows of its choices, up to eight at a time, and the products with the
// rows are summed over the CTA. Choices without a row are passed over: a rank that has an eighth of the experts sees one of eight. The
// CTAs behind the last token zero the padding.
template <typename T>
__global__ void __launch_bounds__(kGradThreads, kGradCtas) moe_combine_grad_kernel(const CombineGradArgs a) {
    __shared__ float partial[kGradThreads / 32][8];
    __shared__ GradRows rows;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, token = blockIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.r.tokens) {
        zero_padding_row(a.r, (uint64_t)(token - a.r.tokens) * (blockDim.x / 32) + warp, a.dy, a.dy_stride, a.units, lane);
        return;
    }
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
        const uint32_t choice = token * a.r.topk + j0 + lane;
        const uint32_t row = j0 + lane < a.r.topk ? ld_global_u32(a.r.token_rows + choice) : 0xffffffffu;
        const float weight = warp == 0 && j0 + lane < a.r.topk ? __uint_as_float(ld_global_u32(a.w + choice)) : 0.f;
        uint32_t live = __ballot_sync(0xffffffffu, row < a.r.rows);
        if (warp == 0 && row >= a.r.rows && j0 + lane < a.r.topk) a.dw[choice] = 0.f;
        while (live != 0) {
            const uint32_t n = min(8u, (uint32_t)__popc(live)), rank = __popc(live & ((1u << lane) - 1u));
            const bool taken = ((live >> lane) & 1u) && rank < 8;
            if (warp == 0 && taken) {
                rows.from[rank] = a.y + row * a.y_stride;
                rows.to[rank] = a.dy + row * a.dy_stride;
                rows.weight[rank] = weight;
                rows.choice[rank] = choice;
            }
            live &= ~__ballot_sync(0xffffffffu, taken);
            __syncthreads();
            const uint8_t* grad = a.g + token * a.g_stride;
            if (n > 4) {
                float dot[8];
                grad_rows<T, 8, 1>(a, grad, rows, n, dot);
                write_sums(a, rows, n, partial, dot);
            } else if (n > 2) {
                float dot[4];
                grad_rows<T, 4, 1>(a, grad, rows, n, dot);
                write_sums(a, rows, n, partial, dot);
            } else if (n == 2) {
                float dot[2];
                grad_rows<T, 2, 1>(a, grad, rows, n, dot);
                write_sums(a, rows, n, partial, dot);
            } else {
                float dot[1];
                grad_rows<T, 1, 2>(a, grad, rows, n, dot);
                write_sums(a, rows, n, partial, dot);
            }
        }
    }
}

}  // namespace dg

using namespace dg;

static const void* sort_kernel(bool int64, bool small) {
    return int64 ? small ? (const void*)moe_sort_kernel<int64_t, 1> : (const void*)moe_sort_kernel<int64_t, kSortBatch>
                 : small ? (const void*)moe_sort_kernel<int32_t, 1> : (const void*)moe_sort_kernel<int32_t, kSortBatch>;
}

// CTAs of the sort's cluster on the current device: 16 where it keeps that many together (they have to share a GPC), else the portable 8.
// The first call on a device gives the kernels leave for it, and for the shared memory of the most experts (once and for all: a
// limit set before each launch could be lowered by another thread in between).
static int sort_cluster(uint32_t* out) {
    constexpr int kMaxDevices = 64;
    static std::atomic<uint8_t> known[kMaxDevices];
    int device = 0;
    DG_CHECK_CUDA(cudaGetDevice(&device));
    uint32_t ctas = device < kMaxDevices ? known[device].load(std::memory_order_acquire) : 0;
    if (ctas == 0) {
        const int smem = (int)((kSortWarps + 2) * kSortMaxExperts * 4 + kSortBatch * kSortThreads * 2);
        int fits = 1;
        for (int k = 0; k < 4; ++k) {
            const void* fn = sort_kernel(k & 1, k & 2);
            DG_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            DG_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(kSortMaxCluster);
            cfg.blockDim = dim3(kSortThreads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim = {kSortMaxCluster, 1, 1};
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            DG_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&clusters, fn, &cfg));
            fits = fits && clusters > 0;
        }
        ctas = fits ? kSortMaxCluster : kSortMaxCluster / 2;
        if (device < kMaxDevices) known[device].store((uint8_t)ctas, std::memory_order_release);
    }
    *out = ctas;
    return DG_OK;
}

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
    // One CTA where the cluster's barriers cost more than its other 15 CTAs take off (measured, one CTA against 16: 1024 choices of 32 experts,
    // 8960 rows, 4.0 against 4.6 us; 2048 5.2 against 4.5; 64 of 256 experts, 16384 rows, 3.5 against 3.9; 128, 32768 rows to clear, 4.7
    // against 4.0).
    uint32_t ctas = 1;
    if (int rc = sort_cluster(&ctas)) return rc;
    if (n <= 1024 && num_rows <= 16384) ctas = 1;
    a.segment = ((n + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) / 32 * 32;
    a.warps = a.segment == 0 ? 0 : (n + a.segment - 1) / a.segment < kSortWarps ? (n + a.segment - 1) / a.segment : kSortWarps;
    const bool small = a.segment <= 32;
    const void* fn = sort_kernel(idx_is_int64, small);
    const uint32_t smem = (a.warps + 2) * num_experts * 4 + (small ? 1 : kSortBatch) * kSortThreads * 2;
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
// Bytes that a token's scales take in the scratch, and from how many scale elements on they go through it.
static uint32_t scale_bytes_of(uint32_t hidden) { return (hidden / 32 + 15) / 16 * 16; }
constexpr uint64_t kScatteredScales = 1ull << 18;
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

extern "C" uint64_t dg_moe_dispatch_fp8_scratch_bytes(uint32_t tokens, uint32_t topk, uint32_t hidden) {
    // (see moe_dispatch_fp8_kernel) the second launch costs more than a few scales written one by one
    const uint64_t scales = (uint64_t)tokens * topk * ((hidden + 63) / 64);
    return scales < kScatteredScales ? 0 : (uint64_t)tokens * scale_bytes_of(hidden);
}

extern "C" int dg_moe_dispatch_fp8_launch(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t topk, uint32_t hidden,
                                          const int32_t* token_rows, const int32_t* row_choices, uint64_t num_rows, void* out, uint64_t out_stride,
                                          int16_t* out_sf, uint64_t sf_col_stride, uint64_t sf_group_stride, uint32_t sf_rows,
                                          void* scratch, uint64_t scratch_bytes, void* stream) {
    if (tokens == 0 || topk == 0 || hidden == 0 || num_rows == 0) return DG_OK;
    DG_CHECK_ARG(x != nullptr && out != nullptr && out_sf != nullptr, "moe_dispatch_fp8: null pointer");
    DG_CHECK_ARG(hidden % 32 == 0, "moe_dispatch_fp8: hidden must be a multiple of 32");
    DG_CHECK_ARG(aligned16(x, x_stride * 2), "moe_dispatch_fp8: input rows must start on 16-byte boundaries");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 7) == 0 && out_stride % 8 == 0, "moe_dispatch_fp8: output rows must start on 8-byte boundaries");
    DG_CHECK_ARG(sf_rows > 0 && sf_col_stride >= sf_rows, "moe_dispatch_fp8: scale column stride smaller than the rows of a group");
    DG_CHECK_ARG(scratch == nullptr || (row_choices != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 &&
                                        scratch_bytes >= (uint64_t)tokens * scale_bytes_of(hidden)),
                 "moe_dispatch_fp8: the scratch must be 16-byte aligned, hold dg_moe_dispatch_fp8_scratch_bytes, and come with the rows' choices");
    DispatchArgs a{};
    if (int rc = rows_args(a.r, token_rows, tokens, topk, num_rows, nullptr, 0, 0, 0, 0)) return rc;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride;
    a.sf = reinterpret_cast<uint8_t*>(out_sf); a.sf_col_stride = sf_col_stride * 2; a.sf_group_stride = sf_group_stride * 2;
    a.sf_rows = sf_rows; a.hidden = hidden;
    a.scratch = static_cast<uint8_t*>(scratch); a.scratch_stride = scale_bytes_of(hidden); a.row_choices = row_choices;
    a.chunks = (hidden + 255) / 256;
    a.token_items = (uint64_t)tokens * a.chunks;
    const uint64_t ctas = (a.token_items + kMoeWarps - 1) / kMoeWarps, tiles = (num_rows + kScaleRows - 1) / kScaleRows;
    const uint32_t pieces = (a.scratch_stride + kScaleChunk - 1) / kScaleChunk;
    DG_CHECK_ARG(ctas <= 0x7fffffffull && pieces <= 65535, "moe_dispatch_fp8: too many tokens or channels");
    void* params[] = {&a};
    if (int rc = launch_overlapped((const void*)moe_dispatch_fp8_kernel, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream))) return rc;
    if (scratch == nullptr) return DG_OK;
    return launch_overlapped((const void*)moe_scales_kernel, dim3((uint32_t)tiles, pieces), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
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
    // as few threads as take a row in the same number of turns
    const uint32_t turns = a.units > kGradThreads ? (a.units + kGradThreads - 1) / kGradThreads : 1;
    const uint32_t threads = a.units == 0 ? 32 : ((a.units + turns - 1) / turns + 31) / 32 * 32;
    const uint64_t ctas = tokens + (padding_items(a.r) + threads / 32 - 1) / (threads / 32);
    if (ctas == 0) return DG_OK;
    DG_CHECK_ARG(ctas <= 0x7fffffffull, "moe_combine_grad: too many rows");
    const void* fn = is_fp32 ? (const void*)moe_combine_grad_kernel<float> : (const void*)moe_combine_grad_kernel<__nv_bfloat16>;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)ctas), dim3(threads), params, static_cast<cudaStream_t>(stream));
}
