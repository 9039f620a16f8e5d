// The gradient of SwiGLU with a weight per row, from its BF16 input or from the E4M3 checkpoint of it.
//
// Mathematics, per row with weight w (1 where there is none) and the gradient g of the result y = silu(l) r w, l = min(x_l, clamp),
// r = min(max(x_r, -clamp), clamp), p = 1 / (1 + e^-l):
//     dx_l = g w r p (1 + l (1 - p)) where x_l <= clamp (else 0)      dx_r = g w l p where |x_r| <= clamp (else 0)
//     dw = sum over the row of g l p r
// all in FP32 (the fast exponential and reciprocal: p within a few ulp, and not below 2^-126), dx rounded once to BF16.
//
// HBM-bound: 2 H + 2 H + H / 16 bytes read (6 H from BF16) and 4 H written per row; the arithmetic, about 25 instructions a channel, is two thirds of
// that time, so a warp asks for its next 256 channels before it works on those it has.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kGradThreads = 256, kGradTokens = kGradThreads / 32, kGradTile = 256, kMostCtas = 8;
constexpr uint32_t kFewGroups = 148 * 4;                    // groups of rows that give every SM its CTAs

struct SwigluGradArgs {
    const uint8_t* g; uint64_t g_stride;                      // BF16 [tokens, hidden], bytes between rows
    const uint8_t* x; uint64_t x_stride;                      // BF16 or E4M3 [tokens, 2 * hidden]
    const uint8_t* x_sf; uint64_t x_sf_stride;                // int16 [hidden / 32][x_sf_stride / 2] seen as bytes
    uint8_t* dx; uint64_t dx_stride;                          // BF16 [tokens, 2 * hidden]
    const float* weights; float* grad_weights;                // [tokens] or nullptr
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t tokens, hidden, ctas, zero_padding;
    float clamp;
};

__device__ __forceinline__ uint4 pack_bf16(const float (&v)[8]) {
    uint32_t w[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void unpack_bf16(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    #pragma unroll
    for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
}

// Eight channels of a row as they lie in memory: the gradient, and both halves of the input in BF16, or in codes with their scales.
template <bool kFromFp8> struct Tile8;
template <> struct Tile8<false> {
    uint4 g, l, r;
    __device__ __forceinline__ void load(const SwigluGradArgs& a, uint64_t token, uint32_t c) {
        g = ld_stream_v4(a.g + token * a.g_stride + (uint64_t)c * 2);
        const uint8_t* x = a.x + token * a.x_stride + (uint64_t)c * 2;
        l = ld_stream_v4(x);
        r = ld_stream_v4(x + (uint64_t)a.hidden * 2);
    }
    __device__ __forceinline__ void get(float (&lv)[8], float (&rv)[8]) const { unpack_bf16(l, lv); unpack_bf16(r, rv); }
};
template <> struct Tile8<true> {
    uint4 g;
    uint2 l, r;
    uint16_t el, er;
    uint32_t shift;
    __device__ __forceinline__ void load(const SwigluGradArgs& a, uint64_t token, uint32_t c) {
        g = ld_stream_v4(a.g + token * a.g_stride + (uint64_t)c * 2);
        const uint8_t *x = a.x + token * a.x_stride + c, *sf = a.x_sf + (uint64_t)(c / 64) * a.x_sf_stride + token * 2;
        l = ld_stream_v2(x);
        r = ld_stream_v2(x + a.hidden);
        // (the rows of the other warps have theirs in the same sectors: these stay in L1)
        el = ld_global_u16(sf);
        er = ld_global_u16(sf + (uint64_t)(a.hidden / 64) * a.x_sf_stride);
        shift = c / 32 % 2 * 8;
    }
    static __device__ __forceinline__ void values(const uint2& q, float scale, float (&v)[8]) {
        float lo[4], hi[4];
        e4m3_unpack4(q.x, lo);
        e4m3_unpack4(q.y, hi);
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = lo[j] * scale; v[4 + j] = hi[j] * scale; }
    }
    __device__ __forceinline__ void get(float (&lv)[8], float (&rv)[8]) const {
        values(l, ue8m0_float((uint32_t)el >> shift & 0xffu), lv);
        values(r, ue8m0_float((uint32_t)er >> shift & 0xffu), rv);
    }
};

// A warp takes a row. Where there are few rows, the channels are shared by a cluster of CTAs, and their sums for dw meet in the first CTA's
// shared memory, added in the order of the CTAs.
template <bool kFromFp8, bool kClamp>
__global__ void __launch_bounds__(kGradThreads, 4) swiglu_grad_kernel(const SwigluGradArgs a) {
    __shared__ float sums[kMostCtas][kGradTokens];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t part = a.ctas > 1 ? blockIdx.x % a.ctas : 0, token_base = (a.ctas > 1 ? blockIdx.x / a.ctas : blockIdx.x) * kGradTokens, token = token_base + warp;
    // (the other CTAs write to this one's shared memory, which has to be there)
    const bool in_cluster = a.grad_weights != nullptr && a.ctas > 1;
    if (in_cluster) cluster_arrive();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t step = a.ctas * kGradTile;
    uint32_t c = part * kGradTile + lane * 8;
    // (asked for before it is known whether the row holds a value)
    Tile8<kFromFp8> now{}, next{};
    if (token < a.tokens && c < a.hidden) now.load(a, token, c);
    const float weight = a.weights && token < a.tokens ? __uint_as_float(ld_stream_u32(a.weights + token)) : 1.0f;
    bool valid = token < a.tokens, zero = false;
    if (a.psum != nullptr) {
        const GroupEnd end = group_end_of(a.psum, a.num_experts, a.alignment, token_base, lane);
        zero = valid && a.zero_padding && token >= end.valid && token < end.whole;
        valid = token < min(a.tokens, end.valid);
    }
    float dw = 0.0f;
    if (valid) {
        for (; c < a.hidden; c += step) {
            if (c + step < a.hidden) next.load(a, token, c + step);
            float g[8], l[8], r[8];
            unpack_bf16(now.g, g);
            now.get(l, r);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                bool outside_l = false, outside_r = false;
                if constexpr (kClamp) {
                    // (a NaN is on no side of the clamp, and stays one)
                    outside_l = l[j] > a.clamp;
                    outside_r = fabsf(r[j]) > a.clamp;
                    if (outside_l) l[j] = a.clamp;
                    if (outside_r) r[j] = copysignf(a.clamp, r[j]);
                }
                // (the reciprocal of a number beyond 2^126 would be 0, and its product with that an invalid one; 1 - p would lose its bits where p is near 1)
                const float z = fast_exp2(fminf(-kLog2E * l[j], 126.0f)), p = fast_reciprocal(1.0f + z), rest = z * p, silu = l[j] * p;
                const float gs = g[j] * silu, gr = g[j] * r[j] * weight;
                dw = fmaf(gs, r[j], dw);
                l[j] = outside_l ? 0.0f : gr * fmaf(silu, rest, p);
                r[j] = outside_r ? 0.0f : gs * weight;
            }
            uint8_t* to = a.dx + (uint64_t)token * a.dx_stride + (uint64_t)c * 2;
            *reinterpret_cast<uint4*>(to) = pack_bf16(l);
            *reinterpret_cast<uint4*>(to + (uint64_t)a.hidden * 2) = pack_bf16(r);
            now = next;
        }
    } else if (zero) {
        for (; c < a.hidden; c += step) {
            uint8_t* to = a.dx + (uint64_t)token * a.dx_stride + (uint64_t)c * 2;
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(to + (uint64_t)a.hidden * 2) = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    if (a.grad_weights == nullptr) return;                    // (the same for all CTAs)
    __syncwarp();
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) dw += __shfl_xor_sync(0xffffffffu, dw, o);
    // (rows that hold no value have the gradient 0: nothing was added)
    if (!in_cluster) {
        if (lane == 0 && token < a.tokens) a.grad_weights[token] = dw;
        return;
    }
    cluster_wait();
    if (lane == 0) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&sums[part][warp]), 0)), "f"(dw) : "memory");
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (part == 0 && threadIdx.x < kGradTokens && token_base + threadIdx.x < a.tokens) {
        float sum = 0.0f;
        for (uint32_t i = 0; i < a.ctas; ++i) sum += sums[i][threadIdx.x];
        a.grad_weights[token_base + threadIdx.x] = sum;
    }
}

}  // namespace dg

using namespace dg;

extern "C" int dg_swiglu_grad_launch(const void* grad_out, uint64_t grad_stride, const void* x, uint64_t x_stride, const int16_t* x_sf, uint64_t x_sf_col_stride,
                                     uint32_t tokens, uint32_t hidden, const float* topk_weights, const int32_t* psum, uint32_t num_experts, uint32_t alignment,
                                     int has_clamp, float clamp_value, void* grad_x, uint64_t grad_x_stride, float* grad_weights, int zero_padding, void* stream) {
    if (tokens == 0) return DG_OK;
    const bool from_fp8 = x_sf != nullptr;
    const uint64_t es = from_fp8 ? 1 : 2;
    DG_CHECK_ARG(grad_out != nullptr && x != nullptr && grad_x != nullptr, "swiglu_grad: null pointer");
    DG_CHECK_ARG(hidden > 0 && hidden % 64 == 0 && hidden <= 0x3fffffffu, "swiglu_grad: hidden must be a multiple of 64");
    DG_CHECK_ARG(tokens <= 0x7fffffffu, "swiglu_grad: too many tokens");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(grad_out) | grad_stride * 2 | reinterpret_cast<uintptr_t>(grad_x) | grad_x_stride * 2) % 16 == 0 &&
                 (reinterpret_cast<uintptr_t>(x) | x_stride * es) % (from_fp8 ? 8 : 16) == 0,
                 "swiglu_grad: rows must start on 16-byte boundaries (8 for E4M3)");
    DG_CHECK_ARG(!from_fp8 || x_sf_col_stride >= tokens, "swiglu_grad: scale column stride smaller than the token count");
    DG_CHECK_ARG(grad_weights == nullptr || topk_weights != nullptr, "swiglu_grad: a gradient of weights that are not there");
    DG_CHECK_ARG(psum == nullptr || (num_experts > 0 && alignment > 0 && alignment % 32 == 0),
                 "swiglu_grad: a psum layout needs experts and an alignment that is a multiple of 32");
    SwigluGradArgs a{};
    a.g = static_cast<const uint8_t*>(grad_out); a.g_stride = grad_stride * 2;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * es;
    a.x_sf = reinterpret_cast<const uint8_t*>(x_sf); a.x_sf_stride = x_sf_col_stride * 2;
    a.dx = static_cast<uint8_t*>(grad_x); a.dx_stride = grad_x_stride * 2;
    a.weights = topk_weights; a.grad_weights = grad_weights;
    a.psum = psum; a.num_experts = psum ? num_experts : 0; a.alignment = alignment;
    a.tokens = tokens; a.hidden = hidden; a.zero_padding = zero_padding ? 1u : 0u;
    a.clamp = clamp_value;
    const uint32_t tiles = (hidden + kGradTile - 1) / kGradTile, groups = (tokens + kGradTokens - 1) / kGradTokens;
    a.ctas = 1;
    while (a.ctas < kMostCtas && a.ctas < tiles && groups * a.ctas < kFewGroups) a.ctas *= 2;
    void* params[] = {&a};
    const void* fn = has_clamp ? (from_fp8 ? (const void*)swiglu_grad_kernel<true, true> : (const void*)swiglu_grad_kernel<false, true>)
                               : (from_fp8 ? (const void*)swiglu_grad_kernel<true, false> : (const void*)swiglu_grad_kernel<false, false>);
    return launch_overlapped(fn, dim3(groups * a.ctas), dim3(kGradThreads), params, static_cast<cudaStream_t>(stream), 0, grad_weights ? a.ctas : 1);
}
