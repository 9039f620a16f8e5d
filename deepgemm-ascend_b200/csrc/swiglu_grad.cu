// The gradient of SwiGLU with a weight per row, from its BF16 input or from the E4M3 checkpoint of it.
//
// Mathematics, per row with weight w (1 where there is none) and the gradient g of the result y = silu(l) r w, l = min(x_l, clamp),
// r = min(max(x_r, -clamp), clamp), p = 1 / (1 + e^-l):
//     dx_l = g w r p (1 + l (1 - p)) where x_l <= clamp (else 0)      dx_r = g w l p where |x_r| <= clamp (else 0)
//     dw = sum over the row of g l p r
// A NaN is on no side of the clamp here and shows in all three; the forward pass, which takes minima and maxima, makes the clamp of it.
// all in FP32 (the fast exponential and reciprocal: p within a few ulp, and 0 below 2^-126), dx rounded once to BF16.
//
// HBM-bound: 2 H + 2 H + H / 16 bytes read (6 H from BF16) and 4 H written per row; the arithmetic, two channels an instruction, is two thirds of that time.
// 65536 x 2048 from 8 bits 178 us, 6.1 TB/s (the bytes alone 165 at the rate of a copy; 200 in a long row of passes, which draws the power cap), from BF16 212 us, 6.3 TB/s; 77 x 2048
// from BF16 2.7 us, launch and latency, with weights 4.3 (a second launch). At 64 registers it spills 40 bytes from BF16, 24 from 8 bits with a clamp.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kGradThreads = 128, kWarpTokens = 4, kGradTokens = kWarpTokens * kGradThreads / 32, kGradTile = 256;

struct SwigluGradArgs {
    const uint8_t* g; uint64_t g_stride;                      // BF16 [tokens, hidden], bytes between rows
    const uint8_t* x; uint64_t x_stride;                      // BF16 or E4M3 [tokens, 2 * hidden]
    const uint8_t* x_sf; uint64_t x_sf_stride;                // int16 [hidden / 32][x_sf_stride / 2] seen as bytes
    uint8_t* dx; uint64_t dx_stride;                          // BF16 [tokens, 2 * hidden]
    const float* weights;                                     // [tokens] or nullptr
    float* partial;                                           // [tiles][tokens]: sums for dw, or nullptr
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t tokens, hidden, tiles, zero_padding;
    float clamp;
};

// Where a lane's channels of a row lie.
template <bool kFromFp8> struct Cursor {
    const uint8_t *g, *l, *r, *sf;
    uint64_t sf_right;
    uint32_t shift;
    __device__ __forceinline__ Cursor(const SwigluGradArgs& a, uint64_t token, uint32_t c) : shift(c / 32 % 2 * 8) {
        g = a.g + token * a.g_stride + (uint64_t)c * 2;
        l = a.x + token * a.x_stride + (uint64_t)c * (kFromFp8 ? 1 : 2);
        r = l + (uint64_t)a.hidden * (kFromFp8 ? 1 : 2);
        sf = a.x_sf + (uint64_t)(c / 64) * a.x_sf_stride + token * 2;
        sf_right = (uint64_t)(a.hidden / 64) * a.x_sf_stride;
    }
    __device__ __forceinline__ void next_row(const SwigluGradArgs& a) {
        g += a.g_stride;
        l += a.x_stride;
        r += a.x_stride;
        sf += 2;
    }
};
// Eight channels of a row as they lie in memory: the gradient, and both halves of the input in BF16, or in codes with their scales.
template <bool kFromFp8> struct Tile8;
template <> struct Tile8<false> {
    uint4 g, l, r;
    __device__ __forceinline__ void load(const Cursor<false>& at) {
        g = ld_stream_v4(at.g);
        l = ld_stream_v4(at.l);
        r = ld_stream_v4(at.r);
    }
    __device__ __forceinline__ void get(uint32_t, Pair (&lv)[4], Pair (&rv)[4]) const {
        const uint32_t lw[4] = {l.x, l.y, l.z, l.w}, rw[4] = {r.x, r.y, r.z, r.w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) { lv[j] = Pair(bf16_lo(lw[j]), bf16_hi(lw[j])); rv[j] = Pair(bf16_lo(rw[j]), bf16_hi(rw[j])); }
    }
};
template <> struct Tile8<true> {
    uint4 g;
    uint2 l, r;
    uint32_t e;
    __device__ __forceinline__ void load(const Cursor<true>& at) {
        g = ld_stream_v4(at.g);
        l = ld_stream_v2(at.l);
        r = ld_stream_v2(at.r);
        // (the other rows of the tile have theirs in the same sectors: these stay in L1)
        e = ld_global_u16(at.sf) | (uint32_t)ld_global_u16(at.sf + at.sf_right) << 16;
    }
    static __device__ __forceinline__ void values(const uint2& q, float scale, Pair (&v)[4]) {
        float four[4];
        const Pair s(scale);
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            e4m3_unpack4(h ? q.y : q.x, four);
            v[2 * h] = Pair(four[0], four[1]) * s;
            v[2 * h + 1] = Pair(four[2], four[3]) * s;
        }
    }
    // The lowest numbers of BF16 round to codes that stand for -2^128, -inf in FP32: the lowest finite number for it, so that a closed gate is no infinity times 0.
    // As whole numbers -inf is the first one above that; a NaN that the conversion and the product make is a positive one and stays.
    static __device__ __forceinline__ void lowest_for_infinity(Pair (&v)[4]) {
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a, b;
            v[j].get(a, b);
            v[j] = Pair(__uint_as_float(min(__float_as_uint(a), 0xff7fffffu)), __uint_as_float(min(__float_as_uint(b), 0xff7fffffu)));
        }
    }
    __device__ __forceinline__ void get(uint32_t shift, Pair (&lv)[4], Pair (&rv)[4]) const {
        values(l, ue8m0_float(e >> shift & 0xffu), lv);
        values(r, ue8m0_float(e >> (shift + 16) & 0xffu), rv);
        lowest_for_infinity(lv);
        lowest_for_infinity(rv);
    }
};

// One CTA = 16 rows x 256 channels, a warp four rows, a lane eight channels of each: everything a warp reads is asked for at once, and small CTAs that come and go
// overlap better than a loop over the channels does (65536 x 2048 from 8 bits: a warp a row with one to three tiles on their way 209 to 226 us; four rows a
// warp at 80 registers 206, at 64 registers 198 and in CTAs of 128 threads 192; two rows a warp 215). The sums of a row's tiles go to `partial`
// and are added up in the order of the tiles by a second kernel.
template <bool kFromFp8, bool kClamp>
__global__ void __launch_bounds__(kGradThreads, 8) swiglu_grad_kernel(const SwigluGradArgs a) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t token_base = blockIdx.x / a.tiles * kGradTokens, tile = blockIdx.x % a.tiles, c = tile * kGradTile + lane * 8, t0 = token_base + warp * kWarpTokens;
    griddep_wait();
    griddep_launch_dependents();
    // (asked for before it is known which rows hold a value)
    Tile8<kFromFp8> tiles[kWarpTokens]{};
    float weight[kWarpTokens];
    const bool inside = c < a.hidden;
    Cursor<kFromFp8> at(a, t0, c);
    #pragma unroll
    for (uint32_t i = 0; i < kWarpTokens; ++i, at.next_row(a)) {
        weight[i] = 1.0f;
        if (t0 + i >= a.tokens) continue;
        if (inside) tiles[i].load(at);
        if (a.weights) weight[i] = __uint_as_float(ld_global_u32(a.weights + t0 + i));
    }
    uint32_t valid_end = min(a.tokens, token_base + kGradTokens), zero_end = 0;
    if (a.psum != nullptr) {
        const GroupEnd end = group_end_of(a.psum, a.num_experts, a.alignment, token_base, lane);
        zero_end = a.zero_padding ? min(valid_end, end.whole) : 0;
        valid_end = min(valid_end, end.valid);
    }
    uint8_t* to = a.dx + (uint64_t)t0 * a.dx_stride + (uint64_t)c * 2;
    const uint64_t to_right = (uint64_t)a.hidden * 2;
    const Pair one(1.0f), exponent(-kLog2E);
    float dw[kWarpTokens];
    #pragma unroll
    for (uint32_t t = 0; t < kWarpTokens; ++t, to += a.dx_stride) {
        dw[t] = 0.0f;
        if (t0 + t >= valid_end) {
            if (t0 + t < zero_end && inside) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(to + to_right) = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        const uint32_t gw[4] = {tiles[t].g.x, tiles[t].g.y, tiles[t].g.z, tiles[t].g.w};
        const Pair weights(weight[t]);
        Pair l[4], r[4], sum(0.0f);
        tiles[t].get(at.shift, l, r);
        uint32_t dl[4], dr[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            bool outside_l[2] = {}, outside_r[2] = {};
            if constexpr (kClamp) {
                // (a NaN is on no side of it, and stays one)
                float lv[2], rv[2];
                l[j].get(lv[0], lv[1]);
                r[j].get(rv[0], rv[1]);
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    outside_l[i] = lv[i] > a.clamp;
                    outside_r[i] = fabsf(rv[i]) > a.clamp;
                    if (outside_l[i]) lv[i] = a.clamp;
                    if (outside_r[i]) rv[i] = copysignf(a.clamp, rv[i]);
                }
                l[j] = Pair(lv[0], lv[1]);
                r[j] = Pair(rv[0], rv[1]);
            }
            // (beyond 2^126 p is 0, as it has to be for l down to the type's lowest number, and so is any product with it but that of an infinity; 1 - p would
            // lose its bits where p is near 1)
            float z0, z1, x0, x1;
            (l[j] * exponent).get(z0, z1);
            z0 = fast_exp2(z0);
            z1 = fast_exp2(z1);
            (Pair(z0, z1) + one).get(x0, x1);
            const Pair p(fast_reciprocal(x0), fast_reciprocal(x1)), rest = Pair(fminf(z0, 0x1p126f), fminf(z1, 0x1p126f)) * p, silu = l[j] * p, g(bf16_lo(gw[j]), bf16_hi(gw[j]));
            const Pair gs = g * silu;
            sum = fma2(gs, r[j], sum);
            float v[4];
            // (r times the slope first: 0 for a closed gate, whatever r is, where the gradient times r could leave the range)
            (g * weights * (r[j] * fma2(silu, rest, p))).get(v[0], v[1]);
            (gs * weights).get(v[2], v[3]);
            if constexpr (kClamp) {
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (outside_l[i]) v[i] = 0.0f;
                    if (outside_r[i]) v[2 + i] = 0.0f;
                }
            }
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
            dl[j] = *reinterpret_cast<const uint32_t*>(&lo);
            dr[j] = *reinterpret_cast<const uint32_t*>(&hi);
        }
        if (inside) {
            *reinterpret_cast<uint4*>(to) = make_uint4(dl[0], dl[1], dl[2], dl[3]);
            *reinterpret_cast<uint4*>(to + to_right) = make_uint4(dr[0], dr[1], dr[2], dr[3]);
        }
        float other;
        sum.get(dw[t], other);
        dw[t] += other;
    }
    if (a.partial == nullptr) return;
    // (lanes behind the last channel hold zeros; rows without a value have the gradient 0)
    #pragma unroll
    for (uint32_t t = 0; t < kWarpTokens; ++t) {
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) dw[t] += __shfl_xor_sync(0xffffffffu, dw[t], o);
        if (lane == t && t0 + t < a.tokens) a.partial[(uint64_t)tile * a.tokens + t0 + t] = dw[t];
    }
}

constexpr uint32_t kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads) swiglu_grad_sum_kernel(const float* partial, float* out, uint32_t tiles, uint32_t tokens) {
    const uint32_t token = blockIdx.x * kSumThreads + threadIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= tokens) return;
    float sum = 0.0f;
    #pragma unroll 8
    for (uint32_t i = 0; i < tiles; ++i) sum += __uint_as_float(ld_global_u32(partial + (uint64_t)i * tokens + token));
    out[token] = sum;
}

}  // namespace dg

using namespace dg;

// Sums of the tiles, where there is more than one.
extern "C" uint64_t dg_swiglu_grad_scratch_bytes(uint32_t tokens, uint32_t hidden) {
    const uint32_t tiles = (hidden + kGradTile - 1) / kGradTile;
    return tiles > 1 ? (uint64_t)tiles * tokens * 4 : 0;
}

extern "C" int dg_swiglu_grad_launch(const void* grad_out, uint64_t grad_stride, const void* x, uint64_t x_stride, const int16_t* x_sf, uint64_t x_sf_col_stride,
                                     uint32_t tokens, uint32_t hidden, const float* topk_weights, const int32_t* psum, uint32_t num_experts, uint32_t alignment,
                                     int has_clamp, float clamp_value, void* grad_x, uint64_t grad_x_stride, float* grad_weights, int zero_padding, void* scratch, uint64_t scratch_bytes,
                                     void* stream) {
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
    a.weights = topk_weights;
    a.psum = psum; a.num_experts = psum ? num_experts : 0; a.alignment = alignment;
    a.tokens = tokens; a.hidden = hidden; a.zero_padding = zero_padding ? 1u : 0u;
    a.clamp = clamp_value;
    a.tiles = (hidden + kGradTile - 1) / kGradTile;
    const uint64_t grid = (uint64_t)((tokens + kGradTokens - 1) / kGradTokens) * a.tiles;
    DG_CHECK_ARG(grid <= 0x7fffffffull, "swiglu_grad: too many tokens");
    const bool sums = grad_weights != nullptr && a.tiles > 1;
    DG_CHECK_ARG(!sums || (scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 4 == 0 && scratch_bytes >= dg_swiglu_grad_scratch_bytes(tokens, hidden)),
                 "swiglu_grad: scratch is too small");
    a.partial = sums ? static_cast<float*>(scratch) : grad_weights;
    void* params[] = {&a};
    const void* fn = has_clamp ? (from_fp8 ? (const void*)swiglu_grad_kernel<true, true> : (const void*)swiglu_grad_kernel<false, true>)
                               : (from_fp8 ? (const void*)swiglu_grad_kernel<true, false> : (const void*)swiglu_grad_kernel<false, false>);
    if (int rc = launch_overlapped(fn, dim3((uint32_t)grid), dim3(kGradThreads), params, static_cast<cudaStream_t>(stream))) return rc;
    if (!sums) return DG_OK;
    const float* from = a.partial;
    void* sum_params[] = {&from, &grad_weights, &a.tiles, &tokens};
    return launch_overlapped((const void*)swiglu_grad_sum_kernel, dim3((tokens + kSumThreads - 1) / kSumThreads), dim3(kSumThreads), sum_params, static_cast<cudaStream_t>(stream));
}
