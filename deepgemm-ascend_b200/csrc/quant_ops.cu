// The step in front of a block-scaled GEMM: BF16 activations -> E4M3 with one UE8M0 scale per 32 channels, the scales
// written straight into the layout the GEMM reads (int16 [tokens, ceil(H/64)], token-major columns), so that no
// scale-factor relayout runs between the producer and the GEMM. Optionally with SwiGLU in front
// (out = silu(x[:, :H]) * x[:, H:] * weight), which is the operator between the two expert GEMMs of an MoE layer.
//
// Follows third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py of the reference: clamp (:156-161), SiLU = x / (1 + e^-x)
// (:162-165; here with the fast exponential and the hardware reciprocal, each within 2 ulp of the exact operation: a value
// on a rounding boundary of E4M3 may land on the neighbouring code, and the exact division cost a third of the run time), scale = 2^ceil(log2(max(amax, 1e-4) / 448)) from the bit pattern (:80-90), values times the
// inverse scale rounded to E4M3 (:250-252), packed scales transposed per group of 32 tokens (:104-125), tokens in
// the padding of a psum layout skipped (:263-268).
//
// HBM-bound: 4 H bytes read and H + H/32 bytes written per token (2 H + H + H/32 without SwiGLU). With a checkpoint the input itself is written in 8 bits
// too, as the plain cast would write it: 2 H + H/16 bytes instead of the 6 H that a cast of its own would move.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kTokenGroup = 32;         // tokens per CTA: one 64-byte run of every scale column
constexpr uint32_t kQuantThreads = 256;      // 8 warps, 4 tokens each
constexpr uint32_t kTileChannels = 256;      // channels per CTA: eight per lane, eight 32-channel blocks, four scale columns
constexpr uint32_t kWarpTokens = kTokenGroup / (kQuantThreads / 32);

struct QuantArgs {
    const __nv_bfloat16* x; uint64_t x_stride;          // [tokens, (swiglu ? 2 : 1) * hidden], elements
    uint8_t* out; uint64_t out_stride;                  // [tokens, hidden] E4M3
    uint8_t* out_sf; uint64_t sf_col_stride;            // int16 [ceil(hidden/64)][sf_col_stride] seen as bytes, 2 per token
    const float* weights;                               // [tokens] or nullptr
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t tokens, hidden;
    float clamp, floor; uint32_t has_clamp;
    uint8_t* kept; uint64_t kept_stride;                // [tokens, 2 * hidden] E4M3
    uint8_t* kept_sf; uint64_t kept_sf_col_stride;      // int16 [hidden/32][kept_sf_col_stride] seen as bytes
};

// One CTA = 32 tokens x 256 channels. A warp takes four tokens and issues the loads of all of them (4 or 8 x 16 bytes per
// lane) before it uses the first. Cutting the channels as well as the tokens is what gives a decoding step its parallelism:
// a CTA that ran through the whole row left 64 tokens x 7168 channels to two CTAs. Bound by HBM for many tokens, by one
// round trip to memory and the launch for few. Measured back to back: 64 x 7168 25.8 -> 1.7 us, 4096 x 7168 31 -> 12.6 us
// (7.1 TB/s), 68495 x 7168 237 -> 214 us (6.9 TB/s); SwiGLU 4096 x 2048 15.0 -> 7.9 us, 68495 x 2048 118 -> 106 us.
template <bool kSwiglu>
__global__ void __launch_bounds__(kQuantThreads) quant_fp8_kernel(const QuantArgs a) {
    __shared__ __align__(8) uint8_t sf_smem[kTokenGroup][kTileChannels / 32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t tiles_c = (a.hidden + kTileChannels - 1) / kTileChannels;
    const uint32_t tg = blockIdx.x / tiles_c, c0 = (blockIdx.x - tg * tiles_c) * kTileChannels;
    const uint32_t token_base = tg * kTokenGroup;
    // (may have been scheduled while the kernel that writes x is still running)
    griddep_wait();
    griddep_launch_dependents();
    uint32_t valid_end = min(a.tokens, token_base + kTokenGroup);
    if (a.psum != nullptr) valid_end = min(valid_end, max(group_end_of(a.psum, a.num_experts, a.alignment, token_base, lane).valid, token_base));
    if (valid_end <= token_base) return;                  // the whole group is padding (uniform over the CTA)

    const uint32_t c = c0 + lane * 8, t0 = token_base + warp * kWarpTokens;
    uint4 left[kWarpTokens], right[kSwiglu ? kWarpTokens : 1];
    float weight[kSwiglu ? kWarpTokens : 1];
    #pragma unroll
    for (uint32_t i = 0; i < kWarpTokens; ++i) {
        left[i] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kSwiglu) { right[i] = left[i]; weight[i] = 1.0f; }
        if (t0 + i < valid_end && c < a.hidden) {
            const __nv_bfloat16* row = a.x + (uint64_t)(t0 + i) * a.x_stride + c;
            left[i] = ld_stream_v4(row);
            if constexpr (kSwiglu) {
                right[i] = ld_stream_v4(row + a.hidden);
                if (a.weights) weight[i] = __uint_as_float(ld_stream_u32(a.weights + t0 + i));
            }
        }
    }
    #pragma unroll
    for (uint32_t i = 0; i < kWarpTokens; ++i) {
        const uint32_t lw[4] = {left[i].x, left[i].y, left[i].z, left[i].w};
        float v[8];
        if constexpr (kSwiglu) {
            const uint32_t rw[4] = {right[i].x, right[i].y, right[i].z, right[i].w};
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                float xl[2] = {bf16_lo(lw[j]), bf16_hi(lw[j])}, xr[2] = {bf16_lo(rw[j]), bf16_hi(rw[j])};
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (a.has_clamp) {
                        xl[k] = fminf(xl[k], a.clamp);
                        xr[k] = fmaxf(fminf(xr[k], a.clamp), -a.clamp);
                    }
                    const float silu = __fdividef(xl[k], 1.0f + __expf(-xl[k]));
                    float y = silu * xr[k];
                    if (a.weights) y *= weight[i];
                    v[j * 2 + k] = y;
                }
            }
        } else {
            #pragma unroll
            for (int j = 0; j < 4; ++j) { v[j * 2] = bf16_lo(lw[j]); v[j * 2 + 1] = bf16_hi(lw[j]); }
        }
        float amax = 0.f;
        #pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t e = e4m3_scale_byte(amax, a.floor);
        if (t0 + i < valid_end && c < a.hidden)
            *reinterpret_cast<uint2*>(a.out + (uint64_t)(t0 + i) * a.out_stride + c) = e4m3_pack8(v, e);
        // (the second block of a last, half-used scale column is zero)
        if ((lane & 3u) == 0) sf_smem[warp * kWarpTokens + i][lane / 4] = c < a.hidden ? (uint8_t)e : (uint8_t)0;
    }
    __syncthreads();
    // scale column j (int16 = channels [64 j, 64 j + 64)) of the valid tokens: one contiguous run of 2-byte elements
    const uint32_t col = threadIdx.x / kTokenGroup, tl = threadIdx.x % kTokenGroup;
    if (col < kTileChannels / 64 && c0 + col * 64 < a.hidden && tl < valid_end - token_base) {
        const uint16_t pair = *reinterpret_cast<const uint16_t*>(&sf_smem[tl][col * 2]);
        *reinterpret_cast<uint16_t*>(a.out_sf + ((uint64_t)(c0 / 64 + col) * a.sf_col_stride + token_base + tl) * 2) = pair;
    }
}

// SwiGLU with a checkpoint. A warp takes four tokens x 256 channels and shares nothing with others, so that small CTAs come and go by themselves: the scales of a
// block's four tokens are collected by shuffles and written in one store of eight bytes where the column starts on a boundary of that. HBM-bound, 4 H bytes read and
// 3 H (1 + 1/32) written: 65536 x 2048 152 us, 6.3 TB/s (the bytes alone 145 at the rate of a copy; 173 in a long row of passes, which draws the power cap). Inside the
// kernel above, whose CTAs share 32 tokens' scales, it took 190.
constexpr uint32_t kKeepThreads = 128, kKeepTokens = kWarpTokens * kKeepThreads / 32;
__device__ __forceinline__ uint32_t cast_piece(const Pair (&v)[4], float floor, uint2& codes) {
    float amax = 0.f;
    #pragma unroll
    for (int j = 0; j < 4; ++j) amax = larger_magnitude(amax, v[j]);
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t e = e4m3_scale_byte(amax, floor);
    codes = e4m3_pack8(v, e);
    return e;
}
__global__ void __launch_bounds__(kKeepThreads, 8) swiglu_checkpoint_kernel(const QuantArgs a) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t tiles_c = (a.hidden + kTileChannels - 1) / kTileChannels;
    const uint32_t tg = blockIdx.x / tiles_c, c = (blockIdx.x - tg * tiles_c) * kTileChannels + lane * 8;
    const uint32_t token_base = tg * kKeepTokens, t0 = token_base + warp * kWarpTokens;
    griddep_wait();
    griddep_launch_dependents();
    // (asked for before it is known which rows hold a value)
    uint4 left[kWarpTokens], right[kWarpTokens];
    float weight[kWarpTokens];
    const bool inside = c < a.hidden;
    const __nv_bfloat16* row = a.x + (uint64_t)t0 * a.x_stride + c;
    #pragma unroll
    for (uint32_t i = 0; i < kWarpTokens; ++i, row += a.x_stride) {
        left[i] = right[i] = make_uint4(0u, 0u, 0u, 0u);
        weight[i] = 1.0f;
        if (t0 + i >= a.tokens) continue;
        if (inside) {
            left[i] = ld_stream_v4(row);
            right[i] = ld_stream_v4(row + a.hidden);
        }
        if (a.weights) weight[i] = __uint_as_float(ld_global_u32(a.weights + t0 + i));
    }
    uint32_t valid_end = min(a.tokens, token_base + kKeepTokens);
    if (a.psum != nullptr) valid_end = min(valid_end, group_end_of(a.psum, a.num_experts, a.alignment, token_base, lane).valid);
    if (t0 >= valid_end) return;                          // (the same for the whole warp)
    uint32_t bytes[3] = {};                               // scales of the result, of the left half, of the right one: a byte a token
    #pragma unroll
    for (uint32_t i = 0; i < kWarpTokens; ++i) {
        const uint32_t lw[4] = {left[i].x, left[i].y, left[i].z, left[i].w}, rw[4] = {right[i].x, right[i].y, right[i].z, right[i].w};
        // The numbers of the kernel above, two at a time: with its instructions one by one the arithmetic takes longer than the bytes (65536 x 2048 rows 182
        // against 161 us).
        Pair l[4], r[4], y[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            l[j] = Pair(bf16_lo(lw[j]), bf16_hi(lw[j]));
            r[j] = Pair(bf16_lo(rw[j]), bf16_hi(rw[j]));
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            Pair xl = l[j], xr = r[j];
            float v0, v1;
            if (a.has_clamp) {
                xl.get(v0, v1);
                xl = Pair(fminf(v0, a.clamp), fminf(v1, a.clamp));
                xr.get(v0, v1);
                xr = Pair(fmaxf(fminf(v0, a.clamp), -a.clamp), fmaxf(fminf(v1, a.clamp), -a.clamp));
            }
            (xl * Pair(-kLog2E)).get(v0, v1);
            (Pair(fast_exp2(v0), fast_exp2(v1)) + Pair(1.0f)).get(v0, v1);
            y[j] = xl * Pair(fast_reciprocal(v0), fast_reciprocal(v1)) * xr;
            if (a.weights) y[j] = y[j] * Pair(weight[i]);
        }
        uint2 codes[3];
        bytes[0] |= cast_piece(y, a.floor, codes[0]) << (8 * i);
        bytes[1] |= cast_piece(l, a.floor, codes[1]) << (8 * i);
        bytes[2] |= cast_piece(r, a.floor, codes[2]) << (8 * i);
        if (t0 + i < valid_end && inside) {
            *reinterpret_cast<uint2*>(a.out + (uint64_t)(t0 + i) * a.out_stride + c) = codes[0];
            uint8_t* to = a.kept + (uint64_t)(t0 + i) * a.kept_stride + c;
            *reinterpret_cast<uint2*>(to) = codes[1];
            *reinterpret_cast<uint2*>(to + a.hidden) = codes[2];
        }
    }
    // Lane 0 of eight has the even block's bytes, lane 4 the odd one's. (hidden is a multiple of 64: no column is half used or holds blocks of both halves)
    #pragma unroll
    for (uint32_t k = 0; k < 3; ++k) {
        const uint32_t odd = __shfl_down_sync(0xffffffffu, bytes[k], 4);
        if (lane % 8 != 0 || !inside) continue;
        const uint64_t stride = k == 0 ? a.sf_col_stride : a.kept_sf_col_stride;
        uint8_t* to = (k == 0 ? a.out_sf : a.kept_sf) + ((uint64_t)((k == 2 ? a.hidden + c : c) / 64) * stride + t0) * 2;
        const uint2 pairs = make_uint2(__byte_perm(bytes[k], odd, 0x5140), __byte_perm(bytes[k], odd, 0x7362));
        if (t0 + kWarpTokens <= valid_end && reinterpret_cast<uintptr_t>(to) % 8 == 0) {
            *reinterpret_cast<uint2*>(to) = pairs;
        } else {
            #pragma unroll
            for (uint32_t i = 0; i < kWarpTokens; ++i)
                if (t0 + i < valid_end) reinterpret_cast<uint16_t*>(to)[i] = (uint16_t)((i < 2 ? pairs.x : pairs.y) >> (16 * (i % 2)));
        }
    }
}

}  // namespace dg

using namespace dg;

static int launch_quant_fp8(QuantArgs a, const void* fn, uint32_t tile_tokens, uint32_t threads, void* stream) {
    DG_CHECK_ARG(a.x != nullptr && a.out != nullptr && a.out_sf != nullptr, "quant_fp8: null pointer");
    DG_CHECK_ARG(a.hidden > 0 && a.hidden % 32 == 0, "quant_fp8: hidden must be a multiple of 32");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.x_stride % 8 == 0,
                 "quant_fp8: input rows must start on 16-byte boundaries");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(a.out) & 7) == 0 && a.out_stride % 8 == 0,
                 "quant_fp8: output rows must start on 8-byte boundaries");
    DG_CHECK_ARG(a.sf_col_stride >= a.tokens, "quant_fp8: scale column stride smaller than the token count");
    DG_CHECK_ARG(a.psum == nullptr || (a.num_experts > 0 && a.alignment > 0 && a.alignment % kTokenGroup == 0),
                 "quant_fp8: a psum layout needs experts and an alignment that is a multiple of 32");
    if (a.tokens == 0) return DG_OK;
    if (a.psum == nullptr) a.num_experts = 0;
    const uint64_t tiles = (((uint64_t)a.tokens + tile_tokens - 1) / tile_tokens) * ((a.hidden + kTileChannels - 1) / kTileChannels);
    DG_CHECK_ARG(tiles <= 0x7fffffffull, "quant_fp8: too many tokens");
    void* params[] = {&a};
    return launch_overlapped(fn, dim3((uint32_t)tiles), dim3(threads), params, static_cast<cudaStream_t>(stream));
}

static QuantArgs quant_args(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t hidden, const float* topk_weights, const int32_t* psum, uint32_t num_experts,
                            uint32_t alignment, int has_clamp, float clamp_value, float floor, void* out, uint64_t out_stride, int16_t* out_sf, uint64_t sf_col_stride) {
    QuantArgs a{};
    a.x = static_cast<const __nv_bfloat16*>(x); a.x_stride = x_stride;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride;
    a.out_sf = reinterpret_cast<uint8_t*>(out_sf); a.sf_col_stride = sf_col_stride;
    a.weights = topk_weights; a.psum = psum; a.num_experts = num_experts; a.alignment = alignment;
    a.tokens = tokens; a.hidden = hidden;
    a.clamp = clamp_value; a.has_clamp = has_clamp ? 1u : 0u; a.floor = floor;
    return a;
}

extern "C" int dg_quant_fp8_launch(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t hidden, int swiglu,
                                   const float* topk_weights, const int32_t* psum, uint32_t num_experts, uint32_t alignment,
                                   int has_clamp, float clamp_value, void* out, uint64_t out_stride,
                                   int16_t* out_sf, uint64_t sf_col_stride, void* stream) {
    const QuantArgs a = quant_args(x, x_stride, tokens, hidden, topk_weights, psum, num_experts, alignment, has_clamp, clamp_value, 1e-4f, out, out_stride, out_sf, sf_col_stride);
    return launch_quant_fp8(a, swiglu ? (const void*)quant_fp8_kernel<true> : (const void*)quant_fp8_kernel<false>, kTokenGroup, kQuantThreads, stream);
}

extern "C" int dg_cast_fp8_launch(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t hidden, const int32_t* psum, uint32_t num_experts, uint32_t alignment,
                                  float min_amax, void* out, uint64_t out_stride, int16_t* out_sf, uint64_t sf_col_stride, void* stream) {
    DG_CHECK_ARG(min_amax >= 0.0f && min_amax <= 3.0e38f, "cast_fp8: min_amax must be a finite number that is not negative");
    const QuantArgs a = quant_args(x, x_stride, tokens, hidden, nullptr, psum, num_experts, alignment, 0, 0.0f, min_amax, out, out_stride, out_sf, sf_col_stride);
    return launch_quant_fp8(a, (const void*)quant_fp8_kernel<false>, kTokenGroup, kQuantThreads, stream);
}

extern "C" int dg_swiglu_checkpoint_launch(const void* x, uint64_t x_stride, uint32_t tokens, uint32_t hidden, const float* topk_weights, const int32_t* psum,
                                           uint32_t num_experts, uint32_t alignment, int has_clamp, float clamp_value, void* out, uint64_t out_stride,
                                           int16_t* out_sf, uint64_t sf_col_stride, void* kept, uint64_t kept_stride, int16_t* kept_sf, uint64_t kept_sf_col_stride,
                                           void* stream) {
    QuantArgs a = quant_args(x, x_stride, tokens, hidden, topk_weights, psum, num_experts, alignment, has_clamp, clamp_value, 1e-4f, out, out_stride, out_sf, sf_col_stride);
    if (tokens != 0) {
        DG_CHECK_ARG(kept != nullptr && kept_sf != nullptr, "swiglu_checkpoint: null pointer");
        DG_CHECK_ARG(hidden % 64 == 0, "swiglu_checkpoint: hidden must be a multiple of 64");
        DG_CHECK_ARG((reinterpret_cast<uintptr_t>(kept) | kept_stride) % 8 == 0, "swiglu_checkpoint: rows of the checkpoint must start on 8-byte boundaries");
        DG_CHECK_ARG(kept_sf_col_stride >= tokens, "swiglu_checkpoint: scale column stride smaller than the token count");
    }
    a.kept = static_cast<uint8_t*>(kept); a.kept_stride = kept_stride;
    a.kept_sf = reinterpret_cast<uint8_t*>(kept_sf); a.kept_sf_col_stride = kept_sf_col_stride;
    return launch_quant_fp8(a, (const void*)swiglu_checkpoint_kernel, kKeepTokens, kKeepThreads, stream);
}
