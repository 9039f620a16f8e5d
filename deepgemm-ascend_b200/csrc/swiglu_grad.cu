// The gradient of SwiGLU with a weight per row, from its BF16 input or from the E4M3 checkpoint of it.
//
// Mathematics, per row with weight w (1 where there is none) and the gradient g of the result y = silu(l) r w, l = min(x_l, clamp),
// r = min(max(x_r, -clamp), clamp), p = 1 / (1 + e^-l):
//     dx_l = g w r p (1 + l (1 - p)) where x_l <= clamp (else 0)      dx_r = g w l p where |x_r| <= clamp (else 0)
//     dw = sum over the row of g l p r
// all in FP32 (the fast exponential and the hardware reciprocal of the forward pass), dx rounded once to BF16.
//
// A cluster of CTAs shares 32 rows: each takes every n-th tile of 256 channels, a warp four rows, a lane eight channels, and the sums for dw meet
// in the first CTA's shared memory, added in the order of the CTAs. HBM-bound: 2 H + 2 H + H / 16 bytes read (6 H from BF16) and 4 H written per row.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kGradThreads = 256, kGradTokens = 32, kGradTile = 256, kGradWarpTokens = 4, kMostCtas = 8;

struct SwigluGradArgs {
    const uint8_t* g; uint64_t g_stride;                      // BF16 [tokens, hidden], bytes between rows
    const uint8_t* x; uint64_t x_stride;                      // BF16 or E4M3 [tokens, 2 * hidden]
    const uint8_t* x_sf; uint64_t x_sf_stride;                // int16 [hidden / 32][x_sf_stride / 2] seen as bytes
    uint8_t* dx; uint64_t dx_stride;                          // BF16 [tokens, 2 * hidden]
    const float* weights; float* grad_weights;                // [tokens] or nullptr
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t tokens, hidden, ctas, zero_padding;
    float clamp; uint32_t has_clamp;
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

// Eight values of the input as they lie in memory: BF16, or codes with their scale.
template <bool kFromFp8> struct Input8;
template <> struct Input8<false> {
    uint4 q;
    __device__ __forceinline__ void clear() { q = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void load(const SwigluGradArgs& a, uint64_t token, uint32_t c) { q = ld_stream_v4(a.x + token * a.x_stride + (uint64_t)c * 2); }
    __device__ __forceinline__ void get(float (&v)[8]) const { unpack_bf16(q, v); }
};
template <> struct Input8<true> {
    uint2 q;
    uint32_t e;
    __device__ __forceinline__ void clear() { q = make_uint2(0u, 0u); e = 127u; }
    __device__ __forceinline__ void load(const SwigluGradArgs& a, uint64_t token, uint32_t c) {
        q = ld_stream_v2(a.x + token * a.x_stride + c);
        // (the other rows of the 32 have theirs in the same sectors: these stay in L1)
        e = ld_global_u16(a.x_sf + (uint64_t)(c / 64) * a.x_sf_stride + token * 2) >> (c / 32 % 2 * 8) & 0xffu;
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const float scale = ue8m0_float(e);
        float lo[4], hi[4];
        e4m3_unpack4(q.x, lo);
        e4m3_unpack4(q.y, hi);
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = lo[j] * scale; v[4 + j] = hi[j] * scale; }
    }
};

template <bool kFromFp8>
__global__ void __launch_bounds__(kGradThreads) swiglu_grad_kernel(const SwigluGradArgs a) {
    __shared__ float sums[kMostCtas][kGradTokens];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t part = blockIdx.x % a.ctas, token_base = blockIdx.x / a.ctas * kGradTokens;
    // (the other CTAs write to this one's shared memory, which has to be there)
    const bool in_cluster = a.grad_weights != nullptr && a.ctas > 1;
    if (in_cluster) cluster_arrive();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t write_end = min(a.tokens, token_base + kGradTokens);
    uint32_t valid_end = write_end, zero_end = token_base;
    if (a.psum != nullptr) {
        const GroupEnd end = group_end_of(a.psum, a.num_experts, a.alignment, token_base, lane);
        valid_end = min(write_end, max(end.valid, token_base));
        zero_end = a.zero_padding ? min(write_end, max(end.whole, token_base)) : token_base;
    }
    const uint32_t t0 = token_base + warp * kGradWarpTokens;
    float weight[kGradWarpTokens], dw[kGradWarpTokens];
    #pragma unroll
    for (uint32_t i = 0; i < kGradWarpTokens; ++i) {
        dw[i] = 0.0f;
        weight[i] = a.weights && t0 + i < valid_end ? __uint_as_float(ld_stream_u32(a.weights + t0 + i)) : 1.0f;
    }
    for (uint32_t c = part * kGradTile + lane * 8; c < a.hidden; c += a.ctas * kGradTile) {
        uint4 g[kGradWarpTokens];
        Input8<kFromFp8> left[kGradWarpTokens], right[kGradWarpTokens];
        #pragma unroll
        for (uint32_t i = 0; i < kGradWarpTokens; ++i) {
            if (t0 + i >= valid_end) continue;
            g[i] = ld_stream_v4(a.g + (uint64_t)(t0 + i) * a.g_stride + (uint64_t)c * 2);
            left[i].load(a, t0 + i, c);
            right[i].load(a, t0 + i, a.hidden + c);
        }
        #pragma unroll
        for (uint32_t i = 0; i < kGradWarpTokens; ++i) {
            uint8_t* to = a.dx + (uint64_t)(t0 + i) * a.dx_stride + (uint64_t)c * 2;
            if (t0 + i >= valid_end) {
                if (t0 + i < zero_end) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(to + (uint64_t)a.hidden * 2) = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            float gv[8], xl[8], xr[8];
            unpack_bf16(g[i], gv);
            left[i].get(xl);
            right[i].get(xr);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                // (a NaN is on no side of the clamp, and stays one)
                const bool outside_l = a.has_clamp && xl[j] > a.clamp, outside_r = a.has_clamp && fabsf(xr[j]) > a.clamp;
                const float l = outside_l ? a.clamp : xl[j], r = outside_r ? copysignf(a.clamp, xr[j]) : xr[j];
                // (by e^-|l|: the reciprocal of a number beyond 2^126 would be 0, and 1 - p would lose its bits where p is near 1)
                const float z = __expf(-fabsf(l)), near = __fdividef(1.0f, 1.0f + z), far = z * near;
                const float p = l < 0.0f ? far : near, rest = l < 0.0f ? near : far, silu = l * p, gw = gv[j] * weight[i];
                dw[i] = fmaf(gv[j] * silu, r, dw[i]);
                xl[j] = outside_l ? 0.0f : gw * r * fmaf(silu, rest, p);
                xr[j] = outside_r ? 0.0f : gw * silu;
            }
            *reinterpret_cast<uint4*>(to) = pack_bf16(xl);
            *reinterpret_cast<uint4*>(to + (uint64_t)a.hidden * 2) = pack_bf16(xr);
        }
    }
    if (a.grad_weights == nullptr) return;                    // (the same for all CTAs)
    __syncwarp();
    if (in_cluster) cluster_wait();
    #pragma unroll
    for (uint32_t i = 0; i < kGradWarpTokens; ++i) {
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        if (lane == i) {
            const uint32_t at = smem_u32(&sums[part][warp * kGradWarpTokens + i]);
            if (in_cluster) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(at, 0)), "f"(dw[i]) : "memory");
            else sums[0][warp * kGradWarpTokens + i] = dw[i];
        }
    }
    if (in_cluster) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (part != 0) return;
    } else {
        __syncthreads();
    }
    if (threadIdx.x < kGradTokens && token_base + threadIdx.x < write_end) {
        float sum = 0.0f;
        for (uint32_t i = 0; i < a.ctas; ++i) sum += sums[i][threadIdx.x];
        // (rows that hold no value have the gradient 0: nothing was added)
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
    DG_CHECK_ARG(psum == nullptr || (num_experts > 0 && alignment > 0 && alignment % kGradTokens == 0),
                 "swiglu_grad: a psum layout needs experts and an alignment that is a multiple of 32");
    SwigluGradArgs a{};
    a.g = static_cast<const uint8_t*>(grad_out); a.g_stride = grad_stride * 2;
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * es;
    a.x_sf = reinterpret_cast<const uint8_t*>(x_sf); a.x_sf_stride = x_sf_col_stride * 2;
    a.dx = static_cast<uint8_t*>(grad_x); a.dx_stride = grad_x_stride * 2;
    a.weights = topk_weights; a.grad_weights = grad_weights;
    a.psum = psum; a.num_experts = psum ? num_experts : 0; a.alignment = alignment;
    a.tokens = tokens; a.hidden = hidden; a.zero_padding = zero_padding ? 1u : 0u;
    a.clamp = clamp_value; a.has_clamp = has_clamp ? 1u : 0u;
    const uint32_t tiles = (hidden + kGradTile - 1) / kGradTile;
    a.ctas = tiles < kMostCtas ? tiles : kMostCtas;
    const uint64_t grid = (uint64_t)((tokens + kGradTokens - 1) / kGradTokens) * a.ctas;
    DG_CHECK_ARG(grid <= 0x7fffffffull, "swiglu_grad: too many tokens");
    void* params[] = {&a};
    return launch_overlapped(from_fp8 ? (const void*)swiglu_grad_kernel<true> : (const void*)swiglu_grad_kernel<false>, dim3((uint32_t)grid), dim3(kGradThreads), params,
                             static_cast<cudaStream_t>(stream), 0, grad_weights ? a.ctas : 1);
}
