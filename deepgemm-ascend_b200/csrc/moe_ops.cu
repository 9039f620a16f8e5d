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
// and no result is summed by atomics. Everything but the sort is bound by HBM: each token's row and each expert row moves once.
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
// The lanes that hold the same expert, bit by bit (a match over 32 lanes takes a turn for every value that occurs). The number of bits is
// rounded up to one that is unrolled: as a loop, the rest of it cost as much as the votes.
template <uint32_t kBits>
__device__ __forceinline__ uint32_t same_bits(uint32_t e) {
    uint32_t peers = 0xffffffffu;
    #pragma unroll
    for (uint32_t b = 0; b < kBits; ++b) {
        const bool set = e & (1u << b);
        const uint32_t with = __ballot_sync(0xffffffffu, set);
        peers &= with ^ (set ? 0u : 0xffffffffu);
    }
    return peers;
}
__device__ __forceinline__ uint32_t same_expert(uint32_t e, uint32_t bits) {
    return bits <= 6 ? same_bits<6>(e) : bits <= 9 ? same_bits<9>(e) : same_bits<11>(e);
}

// A stable counting sort in one launch: one CTA, or a cluster whose CTAs exchange their counts through distributed shared memory.
// Every warp owns a run of choices and a row of counters of its own: it counts (in any order, a count does not depend on it), the counters
// become offsets (over the warps of the CTA, the CTAs of the cluster, and the experts with their alignment), and it walks its run a
// second time to hand out rows. Within 32 choices the order is that of the lanes. Runs that fit kBatch are read once; kBatch is 1 where 32 choices for each
// of a CTA's warps are all (1024 choices: 3.5 us against 4.4 with 8). 131072 choices of 256 experts: 11.6 us with 16 CTAs, 19 with 8; 40 with
// one load at a time and a match for the peers. What is left at that size is the second pass, 6 of the 11.6 us: some 150 instructions for 32 choices, half
// of them the votes that find a choice's peers, and one store to a place of its own for every choice, which 16 SMs have to make. (Four clusters that
// count all choices each and share the second pass: 12.4 us; all votes of a batch at once, unrolled: 14.2.)
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
    const uint32_t first = min(a.n, (cta * a.warps + warp) * a.segment), last = warp < a.warps ? min(a.n, first + a.segment) : first;
    uint32_t* const mine = counts + warp * a.experts;
    uint32_t expert[kBatch];
    load_experts<T>(a, first + lane, last, expert);
    // no row holds a choice until the second pass says so (the barriers in between order the writes)
    for (uint32_t i = cta * kSortThreads + tid; i < a.rows; i += ctas * kSortThreads) a.row_choices[i] = -1;
    __syncthreads();
    for (uint32_t i0 = first; i0 < last; i0 += 32 * kBatch) {
        if (i0 > first) load_experts<T>(a, i0 + lane, last, expert);
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
        // (all three barriers follow branches that a number of experts or choices can end inside a warp)
        cluster_arrive_diverged();
        cluster_wait_diverged();
        if (tid < a.experts) {
            // (all on their way at once: one after the other, sixteen of them took 2 us)
            const uint32_t at = smem_u32(totals + tid);
            uint32_t c[kSortMaxCluster];
            #pragma unroll
            for (uint32_t r = 0; r < kSortMaxCluster; ++r) {
                c[r] = 0;
                if (r < ctas) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[r]) : "r"(mapa_shared(at, r)));
            }
            total = 0;
            #pragma unroll
            for (uint32_t r = 0; r < kSortMaxCluster; ++r) {
                before += r < cta ? c[r] : 0u;
                total += c[r];
            }
        }
        cluster_arrive_diverged();
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
    // (every warp takes the same turns, with no choices in those behind its last: 32768 choices 6.5 us, and 8.0 where each ended at its own)
    for (uint32_t at = 0; at < a.segment; at += 32 * kBatch) {
        if (a.segment > 32 * kBatch) load_experts<T>(a, first + at + lane, last, expert);
        #pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) held[k * kSortThreads + tid] = (uint16_t)expert[k];
        const uint32_t turns = min(kBatch, (a.segment - at) / 32);
        #pragma unroll 1
        for (uint32_t k = 0; k < turns; ++k) {
            const uint32_t i = first + at + k * 32 + lane, e = held[k * kSortThreads + tid], peers = same_expert(e, bits);
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
    if (ctas > 1) cluster_wait_diverged();              // the others have read this CTA's totals
}

// -------------------------------------------------------------------------------------------------- rows and layouts
// What the other kernels know of the layout.
struct RowsArgs {
    const int32_t* token_rows;                          // [tokens][topk]
    const int32_t* layout; uint32_t experts, alignment, max_m;     // of the padding, where it is to be zeroed,
    const int32_t* row_choices;                                    // and which rows hold a choice
    uint32_t tokens, topk, rows;
};

// Zeros in the padding row that `item` stands for: items [0, alignment) (psum) or [0, max_m) (masked) belong to the first group, and
// so on. One warp a row, `units` pieces of 16 bytes.
__device__ __forceinline__ void zero_padding_row(const RowsArgs& a, uint32_t item, uint8_t* out, uint64_t stride, uint32_t units, uint32_t lane) {
    const uint32_t span = a.max_m ? a.max_m : a.alignment, g = item / span, r = item - g * span;
    if (g >= a.experts) return;
    const uint32_t p = ld_global_u32(a.layout + g);
    const uint64_t row = a.max_m ? (uint64_t)g * a.max_m + r : (uint64_t)p + r;
    if (a.max_m ? r < p : row >= ((uint64_t)p + a.alignment - 1) / a.alignment * a.alignment) return;
    // (a row that holds a choice is no padding, whatever the alignment says)
    if (row >= a.rows || (int32_t)ld_global_u32(a.row_choices + row) >= 0) return;
    for (uint32_t u = lane; u < units; u += 32) *reinterpret_cast<uint4*>(out + row * stride + (uint64_t)u * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// -------------------------------------------------------------------------------------------------- dispatch
constexpr uint32_t kMoeThreads = 256, kMoeWarps = kMoeThreads / 32;
constexpr uint32_t kCopyUnits = 4;                      // pieces of 16 bytes that a lane of the copy holds
constexpr uint32_t kBusyWarps = 148 * 64;               // warps that fill the device: below them, latency counts and not the work of one

struct DispatchArgs {
    RowsArgs r;
    const uint8_t* x; uint64_t x_stride;                // bytes
    uint8_t* out; uint64_t out_stride;                  // bytes
    uint32_t units, chunks;                             // of 16 bytes in a row; warps a row takes
    uint32_t eager;                                     // read a token's row before it is known whether a choice wants it
    uint32_t token_items, items;                        // warps that copy, and with those that zero the padding
    uint8_t* sf; uint64_t sf_col_stride, sf_group_stride;          // E4M3 only: bytes between scale columns and groups
    uint32_t sf_rows, hidden;                                      // rows of a group of scales
    uint8_t* scratch;                                              // scale bytes by token, [tokens][scratch_stride], or nullptr
    uint32_t scratch_stride;
};

// The rows of a token's first 32 choices, by lanes, and whether there is any (of the first 32: with more it cannot say no).
__device__ __forceinline__ uint32_t rows_of_token(const RowsArgs& a, uint32_t token, uint32_t lane) {
    return lane < a.topk ? ld_global_u32(a.token_rows + (uint64_t)token * a.topk + lane) : 0xffffffffu;
}
__device__ __forceinline__ bool wanted(const RowsArgs& a, uint32_t mine) { return a.topk > 32 || __any_sync(0xffffffffu, mine < a.rows); }

// A warp takes 32 x kCopyUnits pieces of a token's row, reads them once and writes them to the rows of all its choices. Tokens without a
// choice here are not read (a rank with an eighth of the experts, 16384 tokens x 7168: 66 us against 75 when all are), unless there are so
// few tokens that the second round trip to memory is what counts. 4095 tokens x 2048 of 6 choices, with zeros in the padding: 24 us, 6.3 TB/s.
__global__ void __launch_bounds__(kMoeThreads) moe_dispatch_kernel(const DispatchArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t item = blockIdx.x * kMoeWarps + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.token_items) {
        if (item < a.items) zero_padding_row(a.r, item - a.token_items, a.out, a.out_stride, a.units, lane);
        return;
    }
    const uint32_t token = item / a.chunks, u0 = (item - token * a.chunks) * 32 * kCopyUnits + lane;
    uint32_t mine = rows_of_token(a.r, token, lane);
    if (!a.eager && !wanted(a.r, mine)) return;
    uint4 v[kCopyUnits];
    #pragma unroll
    for (uint32_t k = 0; k < kCopyUnits; ++k)
        if (u0 + k * 32 < a.units) v[k] = ld_stream_v4(a.x + token * a.x_stride + (uint64_t)(u0 + k * 32) * 16);
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
        if (j0 > 0) mine = j0 + lane < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j0 + lane) : 0xffffffffu;
        for (uint32_t live = __ballot_sync(0xffffffffu, mine < a.r.rows); live != 0; live &= live - 1) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, __ffs(live) - 1);
            #pragma unroll
            for (uint32_t k = 0; k < kCopyUnits; ++k)
                if (u0 + k * 32 < a.units) *reinterpret_cast<uint4*>(a.out + row * a.out_stride + (uint64_t)(u0 + k * 32) * 16) = v[k];
        }
    }
}

// The same with a quantisation on the way: a warp takes kTiles x 256 channels of a token, eight to a lane, four lanes to a block of 32. The
// scales of a row lie num_rows elements apart, and the rows of a token far from one another: written from here, each is a store of two
// bytes with a sector of L2 to itself. That suits a few tokens. For many (65536 rows of 7168: 127 us, 93 without the scales), the
// bytes go to a scratch, by token, and moe_scales_kernel behind this one turns them into runs: 100 us together, 6.0 TB/s. Two tiles to a
// warp then: with one, 16384 tokens of which a rank has one choice of eight take 98 us, with two 66, with four 78. (A grid of one wave whose
// warps take one piece after the other, the next on its way: 98 us, and 120 instead of 101.)
constexpr uint32_t kFp8Tiles = 2;
template <uint32_t kTiles>
__global__ void __launch_bounds__(kMoeThreads) moe_dispatch_fp8_kernel(const DispatchArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t item = blockIdx.x * kMoeWarps + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.token_items) return;
    const uint32_t token = item / a.chunks, c0 = (item - token * a.chunks) * 256 * kTiles, c = c0 + lane * 8;
    uint32_t mine = rows_of_token(a.r, token, lane);
    if (!a.eager && !wanted(a.r, mine)) return;
    uint4 raw[kTiles];
    #pragma unroll
    for (uint32_t t = 0; t < kTiles; ++t) {
        raw[t] = make_uint4(0u, 0u, 0u, 0u);
        if (c + t * 256 < a.hidden) raw[t] = ld_stream_v4(a.x + token * a.x_stride + (uint64_t)(c + t * 256) * 2);
    }
    // scale column lane % 4 of a tile: the bytes of blocks 2 (lane % 4) and 2 (lane % 4) + 1 (zero behind the last one)
    uint2 q[kTiles];
    uint32_t pair[kTiles];
    const uint32_t col = lane % 4;
    #pragma unroll
    for (uint32_t t = 0; t < kTiles; ++t) {
        const uint32_t w[4] = {raw[t].x, raw[t].y, raw[t].z, raw[t].w};
        float v[8], amax = 0.f;
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
        #pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t e = e4m3_scale_byte(amax), byte = c + t * 256 < a.hidden ? e : 0u;
        q[t] = e4m3_pack8(v, e);
        pair[t] = __shfl_sync(0xffffffffu, byte, col * 8) | (__shfl_sync(0xffffffffu, byte, col * 8 + 4) << 8);
    }
    for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
        if (j0 > 0) mine = j0 + lane < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j0 + lane) : 0xffffffffu;
        const uint32_t live = __ballot_sync(0xffffffffu, mine < a.r.rows);
        for (uint32_t m = live; m != 0; m &= m - 1) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, __ffs(m) - 1);
            #pragma unroll
            for (uint32_t t = 0; t < kTiles; ++t)
                if (c + t * 256 < a.hidden) *reinterpret_cast<uint2*>(a.out + row * a.out_stride + c + t * 256) = q[t];
        }
        if (a.scratch != nullptr) continue;
        // eight rows' scales at a time, four columns each
        for (uint32_t j = 0; j < min(32u, a.r.topk - j0); j += 8) {
            const uint32_t row = __shfl_sync(0xffffffffu, mine, j + lane / 4);
            if (row >= a.r.rows) continue;
            const uint32_t g = row / a.sf_rows;
            uint8_t* const to = a.sf + g * a.sf_group_stride + (uint64_t)(row - g * a.sf_rows) * 2;
            #pragma unroll
            for (uint32_t t = 0; t < kTiles; ++t)
                if (c0 + t * 256 + col * 64 < a.hidden) *reinterpret_cast<uint16_t*>(to + (uint64_t)(c0 / 64 + t * 4 + col) * a.sf_col_stride) = (uint16_t)pair[t];
        }
    }
    if (a.scratch != nullptr) {
        uint32_t mine_pair = pair[0];
        #pragma unroll
        for (uint32_t t = 1; t < kTiles; ++t) mine_pair = lane / 4 == t ? pair[t] : mine_pair;
        if (lane < 4 * kTiles && c0 + lane * 64 < a.hidden)
            *reinterpret_cast<uint16_t*>(a.scratch + (uint64_t)token * a.scratch_stride + c0 / 32 + lane * 2) = (uint16_t)mine_pair;
    }
}

// Scale bytes by token -> the layout that the GEMM reads. One CTA = 64 rows: their tokens' bytes are read 16 at a time into shared memory
// (rows an odd number of words apart: the columns are read without conflicts), and every scale column of the tile is a run of 128 bytes.
constexpr uint32_t kScaleRows = 64, kScaleChunk = 256;  // rows of a CTA, scale bytes of a row that it holds at a time
__global__ void __launch_bounds__(kMoeThreads) moe_scales_kernel(const DispatchArgs a) {
    __shared__ uint32_t bytes[kScaleRows][kScaleChunk / 4 + 1];
    __shared__ uint32_t token_of[kScaleRows];
    const uint32_t row0 = blockIdx.x * kScaleRows, b0 = blockIdx.y * kScaleChunk, tid = threadIdx.x;
    // (the choices come from in front of the dispatch, whose CTAs have all passed their own wait when this kernel is let in, so they are in L2: they
    // may be read from there, but not through L1, which only this kernel's wait brings up to date, before the bytes that the dispatch writes are
    // there. Behind the wait, 8192 x 7168 of 8 choices take 101.9 instead of 101.4 us, 2048 x 7168 of one 14.2 instead of 13.7.)
    bool some = false;
    if (tid < kScaleRows) {
        const uint32_t choice = row0 + tid < a.r.rows ? ld_relaxed_u32(a.r.row_choices + row0 + tid) : 0xffffffffu;
        const uint32_t token = choice / max(a.r.topk, 1u);
        some = (int32_t)choice >= 0 && token < a.r.tokens;
        token_of[tid] = some ? token : 0xffffffffu;
    }
    some = __syncthreads_or(some);
    griddep_wait();
    griddep_launch_dependents();
    if (!some) return;
    // (a thread keeps to its piece of the rows, and its row of the columns: what is left of an index is an addition)
    const uint32_t pieces = min(kScaleChunk, a.scratch_stride - b0) / 16, piece = tid % (kScaleChunk / 16);
    for (uint32_t r = tid / (kScaleChunk / 16); r < kScaleRows && piece < pieces; r += kMoeThreads / (kScaleChunk / 16)) {
        const uint32_t token = token_of[r];
        if (token == 0xffffffffu) continue;
        const uint4 v = ld_global_v4(a.scratch + (uint64_t)token * a.scratch_stride + b0 + piece * 16);
        uint32_t* to = &bytes[r][piece * 4];
        to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
    }
    __syncthreads();
    const uint32_t r = tid % kScaleRows, row = row0 + r;
    if (token_of[r] == 0xffffffffu) return;
    const uint32_t g = row / a.sf_rows, cols = (a.hidden + 63) / 64, c0 = b0 / 2;
    uint32_t word = tid / kScaleRows;                     // two columns
    uint8_t* to = a.sf + g * a.sf_group_stride + (uint64_t)(row - g * a.sf_rows) * 2 + (uint64_t)(c0 + 2 * word) * a.sf_col_stride;
    for (; word < pieces * 4; word += kMoeThreads / kScaleRows, to += 2 * (kMoeThreads / kScaleRows) * a.sf_col_stride) {
        const uint32_t pair = bytes[r][word];
        if (c0 + 2 * word < cols) *reinterpret_cast<uint16_t*>(to) = (uint16_t)pair;
        if (c0 + 2 * word + 1 < cols) *reinterpret_cast<uint16_t*>(to + a.sf_col_stride) = (uint16_t)(pair >> 16);
    }
}

// -------------------------------------------------------------------------------------------------- combine
struct CombineArgs {
    RowsArgs r;
    const uint8_t* y; uint64_t y_stride;                // [rows], bytes
    const float* w;                                     // [tokens][topk] or nullptr
    uint8_t* out; uint64_t out_stride;
    uint32_t units, chunks, turns;                      // pieces of 16 bytes in a row; warps a row takes; pieces of a lane
    uint32_t items;
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

// Up to eight rows with a choice, compacted, and their weights.
struct LiveRows {
    uint32_t row[8];
    float weight[8];
    uint32_t n;
    // The first eight lanes of `live`, which loses them.
    __device__ __forceinline__ LiveRows(uint32_t& live, uint32_t mine, float w) {
        n = min(8u, (uint32_t)__popc(live));
        #pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int from = __ffs(live) - 1;
            row[r] = __shfl_sync(0xffffffffu, mine, from);
            weight[r] = __shfl_sync(0xffffffffu, w, from);
            live &= live - 1;
        }
    }
};

// kRows rows, times their weights, added to kTurns pieces of the result that lie 32 apart.
template <typename T, int kRows, int kTurns>
__device__ __forceinline__ void add_rows(const CombineArgs& a, uint32_t u, const LiveRows& rows, float (&sum)[kTurns][Unit<T>::kValues]) {
    uint4 q[kRows][kTurns];
    #pragma unroll
    for (uint32_t r = 0; r < kRows; ++r)
        #pragma unroll
        for (int t = 0; t < kTurns; ++t)
            if (r < rows.n && u + t * 32 < a.units) q[r][t] = ld_stream_v4(a.y + rows.row[r] * a.y_stride + (uint64_t)(u + t * 32) * 16);
    #pragma unroll
    for (uint32_t r = 0; r < kRows; ++r)
        #pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            if (r >= rows.n || u + t * 32 >= a.units) continue;
            float v[Unit<T>::kValues];
            Unit<T>::values(q[r][t], v);
            #pragma unroll
            for (int k = 0; k < Unit<T>::kValues; ++k) sum[t][k] = fmaf(rows.weight[r], v[k], sum[t][k]);
        }
}
template <typename T, int kTurns>
__device__ __forceinline__ void store_pieces(const CombineArgs& a, uint32_t token, uint32_t u, const float (&sum)[kTurns][Unit<T>::kValues]) {
    #pragma unroll
    for (int t = 0; t < kTurns; ++t)
        if (u + t * 32 < a.units) *reinterpret_cast<uint4*>(a.out + token * a.out_stride + (uint64_t)(u + t * 32) * 16) = Unit<T>::pack(sum[t]);
}

// A warp takes 32 x turns pieces of 16 bytes of a token's result (turns is 1, or kCombineTurns where there are tokens enough): eight pieces of rows
// are on their way at once, of eight rows or of fewer and more turns. 8192 tokens x 7168 of 8 rows each: 164 us, 6.4 TB/s; 16384 tokens of
// which a rank has one row of eight: 186 us with one turn, 86 with four. Seven CTAs of 128 threads, which leaves 72 registers, one too few (4 bytes
// of a thread are in local memory): with eight (64 registers) 167 and 86 us, with five of 256 threads 171 and 97.
constexpr uint32_t kCombineTurns = 4, kCombineThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kCombineThreads, 7) moe_combine_kernel(const CombineArgs a) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t item = blockIdx.x * (kCombineThreads / 32) + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (item >= a.items) return;
    const uint32_t token = item / a.chunks, u = (item - token * a.chunks) * 32 * a.turns + lane;
    const auto row_of = [&](uint32_t j) { return j < a.r.topk ? ld_global_u32(a.r.token_rows + (uint64_t)token * a.r.topk + j) : 0xffffffffu; };
    const auto weight_of = [&](uint32_t j) {
        return a.w != nullptr && j < a.r.topk ? __uint_as_float(ld_global_u32(a.w + (uint64_t)token * a.r.topk + j)) : 1.0f;
    };
    const uint32_t mine = row_of(lane);
    const float weight = weight_of(lane);
    uint32_t live = __ballot_sync(0xffffffffu, mine < a.r.rows);
    LiveRows rows(live, mine, weight);
    if (live != 0 || a.r.topk > 32) {
        // more than eight rows, or so it may be
        for (uint32_t t = 0; t < a.turns; ++t) {
            float sum[1][Unit<T>::kValues] = {};
            for (uint32_t j0 = 0; j0 < a.r.topk; j0 += 32) {
                const uint32_t row = row_of(j0 + lane);
                const float w = weight_of(j0 + lane);
                live = __ballot_sync(0xffffffffu, row < a.r.rows);
                while (live != 0) add_rows<T, 8, 1>(a, u + t * 32, LiveRows(live, row, w), sum);
            }
            store_pieces<T, 1>(a, token, u + t * 32, sum);
        }
    } else if (a.turns == 1 || rows.n > 4) {
        for (uint32_t t = 0; t < a.turns; ++t) {
            float sum[1][Unit<T>::kValues] = {};
            add_rows<T, 8, 1>(a, u + t * 32, rows, sum);
            store_pieces<T, 1>(a, token, u + t * 32, sum);
        }
    } else if (rows.n > 2) {
        for (uint32_t t = 0; t < a.turns; t += 2) {
            float sum[2][Unit<T>::kValues] = {};
            add_rows<T, 4, 2>(a, u + t * 32, rows, sum);
            store_pieces<T, 2>(a, token, u + t * 32, sum);
        }
    } else {
        float sum[kCombineTurns][Unit<T>::kValues] = {};
        add_rows<T, 2, kCombineTurns>(a, u, rows, sum);
        store_pieces<T, kCombineTurns>(a, token, u, sum);
    }
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

// Where the rows of up to eight choices begin. In shared memory: as registers these words left eight warps on an SM (4096 tokens x 7168, 8 rows each:
// 210 us; with three CTAs of 256 threads 160, six of 128 158, eight of 128 161).
struct GradRows {
    const uint8_t* from[8];
    uint8_t* to[8];
    float weight[8];
    uint32_t choice[8];
};

// kRows rows at a time, kTurns turns of the CTA over the row together: what 80 registers hold. (One row: 16384 tokens of which a rank has one choice in
// eight, 123 us with two turns, 127 with one; more turns, or two with two or four rows, spill and cost 5 to 30 %.)
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
    // (the lanes that did not write fill `rows` again: not before these have read it)
    __syncwarp();
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
        zero_padding_row(a.r, (token - a.r.tokens) * (blockDim.x / 32) + warp, a.dy, a.dy_stride, a.units, lane);
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
static int rows_args(RowsArgs& r, const int32_t* token_rows, const int32_t* row_choices, uint32_t tokens, uint32_t topk, uint64_t num_rows,
                     const int32_t* layout, uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding) {
    DG_CHECK_ARG(token_rows != nullptr || (uint64_t)tokens * topk == 0, "moe: null pointer");
    DG_CHECK_ARG((uint64_t)tokens * topk <= 0x7fffffffull && num_rows <= 0x7fffffffull, "moe: too many choices or rows");
    DG_CHECK_ARG(!zero_padding || num_rows == 0 || (layout != nullptr && row_choices != nullptr && num_experts > 0 && (max_m > 0 || alignment > 0)),
                 "moe: zeros in the padding need the layout and the rows' choices");
    r.token_rows = token_rows; r.row_choices = row_choices; r.tokens = tokens; r.topk = topk; r.rows = (uint32_t)num_rows;
    r.layout = layout; r.experts = zero_padding && num_rows > 0 ? num_experts : 0; r.alignment = alignment; r.max_m = max_m;
    return DG_OK;
}
constexpr uint64_t kMaxItems = 0xfffffff0ull;          // warps of a launch, counted in 32 bits (a division by 64 costs more than the rest of an index)
static uint64_t padding_items(const RowsArgs& r) { return (uint64_t)r.experts * (r.max_m ? r.max_m : r.alignment); }
// Bytes that a token's scales take in the scratch, and from how many tokens and scale elements of theirs on they go through it.
static uint32_t scale_bytes_of(uint32_t hidden) { return (hidden / 32 + 15) / 16 * 16; }
constexpr uint32_t kManyTokens = 2048, kManyScales = 1u << 16;
static bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride_bytes % 16 == 0; }

extern "C" int dg_moe_dispatch_launch(const void* x, uint64_t x_stride_bytes, uint32_t tokens, uint32_t topk, uint64_t row_bytes,
                                      const int32_t* token_rows, const int32_t* row_choices, uint64_t num_rows, void* out, uint64_t out_stride_bytes,
                                      const int32_t* layout, uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding, void* stream) {
    if (row_bytes == 0 || num_rows == 0) return DG_OK;
    DG_CHECK_ARG(out != nullptr && (x != nullptr || tokens == 0), "moe_dispatch: null pointer");
    DG_CHECK_ARG(row_bytes % 16 == 0 && aligned16(x, x_stride_bytes) && aligned16(out, out_stride_bytes),
                 "moe_dispatch: rows must start on 16-byte boundaries and hold a multiple of 16 bytes");
    DG_CHECK_ARG(row_bytes / 16 <= 0x7fffffffull, "moe_dispatch: rows too long");
    DispatchArgs a{};
    if (int rc = rows_args(a.r, token_rows, row_choices, tokens, topk, num_rows, layout, num_experts, alignment, max_m, zero_padding)) return rc;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride_bytes;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride_bytes;
    a.units = (uint32_t)(row_bytes / 16);
    a.chunks = (a.units + 32 * kCopyUnits - 1) / (32 * kCopyUnits);
    const uint64_t items = (uint64_t)tokens * a.chunks + padding_items(a.r);
    DG_CHECK_ARG(items <= kMaxItems, "moe_dispatch: too many rows");
    if (items == 0) return DG_OK;
    a.token_items = tokens * a.chunks;
    a.items = (uint32_t)items;
    a.eager = a.token_items < kBusyWarps;
    const uint32_t ctas = (a.items + kMoeWarps - 1) / kMoeWarps;
    void* params[] = {&a};
    return launch_overlapped((const void*)moe_dispatch_kernel, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t dg_moe_dispatch_fp8_scratch_bytes(uint32_t tokens, uint32_t hidden) {
    // Measured, the second launch against scales written one by one, 1024 / 2048 / 4096 tokens: 7168 channels, 8 choices 20.8 / 32.9 / 56.4 against
    // 19.0 / 34.7 / 65.9 us, one choice 10.2 / 14.9 / 24.5 against 8.8 / 15.5 / 29.4, 8 choices of which a rank has one 9.6 / 13.9 / 22.3 against
    // 7.5 / 13.2 / 25.6; 2048 channels, 8 choices 8.0 / 11.2 / 18.7 against 7.1 / 11.7 / 21.2; 512 channels 4.8 / 5.7 / 8.2 against 3.4 / 4.4 / 7.0.
    return tokens < kManyTokens || (uint64_t)tokens * ((hidden + 63) / 64) < kManyScales ? 0 : (uint64_t)tokens * scale_bytes_of(hidden);
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
    if (int rc = rows_args(a.r, token_rows, row_choices, tokens, topk, num_rows, nullptr, 0, 0, 0, 0)) return rc;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride;
    a.sf = reinterpret_cast<uint8_t*>(out_sf); a.sf_col_stride = sf_col_stride * 2; a.sf_group_stride = sf_group_stride * 2;
    a.sf_rows = sf_rows; a.hidden = hidden;
    a.scratch = static_cast<uint8_t*>(scratch); a.scratch_stride = scale_bytes_of(hidden);
    // (many tokens, many stores: more bytes in each)
    const uint32_t tiles_of_warp = scratch == nullptr ? 1 : kFp8Tiles;
    a.chunks = (hidden + 256 * tiles_of_warp - 1) / (256 * tiles_of_warp);
    const uint64_t items = (uint64_t)tokens * a.chunks;
    a.token_items = (uint32_t)items;
    a.eager = items < kBusyWarps;
    const uint64_t ctas = (items + kMoeWarps - 1) / kMoeWarps, tiles = (num_rows + kScaleRows - 1) / kScaleRows;
    const uint32_t pieces = (a.scratch_stride + kScaleChunk - 1) / kScaleChunk;
    DG_CHECK_ARG(items <= kMaxItems && pieces <= 65535, "moe_dispatch_fp8: too many tokens or channels");
    void* params[] = {&a};
    const void* fn = tiles_of_warp == 1 ? (const void*)moe_dispatch_fp8_kernel<1> : (const void*)moe_dispatch_fp8_kernel<kFp8Tiles>;
    if (int rc = launch_overlapped(fn, dim3((uint32_t)ctas), dim3(kMoeThreads), params, static_cast<cudaStream_t>(stream))) return rc;
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
    if (int rc = rows_args(a.r, token_rows, nullptr, tokens, topk, num_rows, nullptr, 0, 0, 0, 0)) return rc;
    a.y = static_cast<const uint8_t*>(rows); a.y_stride = rows_stride * es;
    a.w = topk_weights;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride * es;
    a.units = (uint32_t)(hidden * es / 16);
    a.turns = (uint64_t)tokens * ((a.units + 31) / 32) < kBusyWarps ? 1 : kCombineTurns;
    a.chunks = (a.units + 32 * a.turns - 1) / (32 * a.turns);
    const uint64_t items = (uint64_t)tokens * a.chunks;
    DG_CHECK_ARG(items <= kMaxItems, "moe_combine: too many tokens");
    a.items = (uint32_t)items;
    const uint32_t ctas = (a.items + kCombineThreads / 32 - 1) / (kCombineThreads / 32);
    const void* fn = is_fp32 ? (const void*)moe_combine_kernel<float> : (const void*)moe_combine_kernel<__nv_bfloat16>;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)ctas), dim3(kCombineThreads), params, static_cast<cudaStream_t>(stream));
}

extern "C" int dg_moe_combine_grad_launch(const void* grad_out, int is_fp32, uint64_t grad_stride, const void* rows, uint64_t rows_stride,
                                          uint64_t num_rows, uint32_t hidden, const int32_t* token_rows, const int32_t* row_choices,
                                          uint32_t tokens, uint32_t topk, const float* topk_weights, void* grad_rows, uint64_t grad_rows_stride, float* grad_weights,
                                          const int32_t* layout, uint32_t num_experts, uint32_t alignment, uint32_t max_m, int zero_padding,
                                          void* stream) {
    if (tokens == 0 && !zero_padding) return DG_OK;
    const uint64_t es = is_fp32 ? 4 : 2;
    DG_CHECK_ARG((tokens == 0 || hidden == 0 || grad_out != nullptr) && (num_rows == 0 || hidden == 0 || (rows != nullptr && grad_rows != nullptr)) &&
                 (tokens == 0 || topk == 0 || (topk_weights != nullptr && grad_weights != nullptr)), "moe_combine_grad: null pointer");
    DG_CHECK_ARG(hidden * es % 16 == 0 && aligned16(grad_out, grad_stride * es) && aligned16(rows, rows_stride * es) &&
                 aligned16(grad_rows, grad_rows_stride * es), "moe_combine_grad: rows must start on 16-byte boundaries and hold a multiple of 16 bytes");
    CombineGradArgs a{};
    if (int rc = rows_args(a.r, token_rows, row_choices, tokens, topk, num_rows, layout, num_experts, alignment, max_m, zero_padding)) return rc;
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
    DG_CHECK_ARG(ctas <= 0x7fffffffull && padding_items(a.r) <= kMaxItems, "moe_combine_grad: too many rows");
    const void* fn = is_fp32 ? (const void*)moe_combine_grad_kernel<float> : (const void*)moe_combine_grad_kernel<__nv_bfloat16>;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)ctas), dim3(threads), params, static_cast<cudaStream_t>(stream));
}
