// The step between the residual stream and a block-scaled product: h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, written as E4M3 with
// one UE8M0 scale per 32 channels in the layout the GEMM reads (and in BF16 where a router or a dispatch wants it), and its gradient.
//
// h is rounded to its type before the norm sees it: what the residual stream holds is what the gradient is taken at. The sum of squares is held in
// 64 bits, so that 1 / sqrt comes out as the same FP32 number however a row is spread over threads: a token's bits do not depend on how many
// others there are. y = (h * rstd) * weight in FP32, one rounding each, then one to E4M3 (values times the inverse of the scale of quant.cuh, which is
// a power of two) and one to BF16.
//
// HBM-bound: BF16 with a residual 4 H bytes read, 2 H + H + H / 32 written per token (2 H more for the BF16 rows).
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kAll = 0xffffffffu, kMostHidden = 32768;

// Eight channels of a lane as they lie in memory.
template <typename T> struct Piece;
template <> struct Piece<__nv_bfloat16> {
    uint4 q;
    __device__ __forceinline__ void load(const uint8_t* p) { q = ld_stream_v4(p); }
    __device__ __forceinline__ void clear() { q = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t w[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&p);
        }
        q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<uint4*>(p) = q; }
};
template <> struct Piece<float> {
    uint4 q, r;
    __device__ __forceinline__ void load(const uint8_t* p) { q = ld_stream_v4(p); r = ld_stream_v4(p + 16); }
    __device__ __forceinline__ void clear() { q = r = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        q = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        r = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        *reinterpret_cast<uint4*>(p) = q;
        *reinterpret_cast<uint4*>(p + 16) = r;
    }
};
__device__ __forceinline__ void weight_at(const void* weight, uint32_t fp32, uint32_t c, float (&v)[8]) {
    if (fp32) {
        const uint4 q = ld_global_v4(static_cast<const float*>(weight) + c), r = ld_global_v4(static_cast<const float*>(weight) + c + 4);
        const uint32_t w[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
        const uint4 q = ld_global_v4(static_cast<const __nv_bfloat16*>(weight) + c);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
    }
}

// Sums of kRows values over the CTA, in every thread. `partial`: [warps][kRows] of shared memory that nobody reads any more.
template <typename S, uint32_t kRows>
__device__ __forceinline__ void cta_sums(S (&v)[kRows], S* partial) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    #pragma unroll
    for (uint32_t r = 0; r < kRows; ++r)
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[r] += __shfl_xor_sync(kAll, v[r], o);
    if (lane < kRows) {
        S mine = v[0];
        #pragma unroll
        for (uint32_t r = 1; r < kRows; ++r) mine = lane == r ? v[r] : mine;
        partial[warp * kRows + lane] = mine;
    }
    __syncthreads();
    // lane = (a warp, a row); the rows' sums end up in lanes 0 .. kRows - 1
    S sum = 0;
    for (uint32_t at = lane; at < warps * kRows; at += 32) sum += partial[at];
    #pragma unroll
    for (uint32_t o = 16; o >= kRows; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    #pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) v[r] = __shfl_sync(kAll, sum, r);
}

struct NormArgs {
    const uint8_t *x, *residual; uint64_t x_stride, residual_stride;     // bytes between rows
    uint8_t* h; uint64_t h_stride;                                       // nullptr: x is h already
    const void* weight; uint32_t weight_fp32;
    uint8_t* rows; uint64_t rows_stride;                                 // BF16 rows, or nullptr
    uint8_t* out; uint64_t out_stride;                                   // E4M3
    uint8_t* sf; uint64_t sf_col_stride;                                 // bytes between scale columns
    float* rstd;
    uint32_t tokens, hidden;
    float eps;
    double inverse_hidden;
};

// 1 / sqrt(m) as the nearest FP32 number (but for one in 10^8): two steps of Newton's method in 64 bits behind the FP32 instruction, where FP32 holds m.
__device__ __forceinline__ float rsqrt_of(double m) {
    if (m > 0x1p-120 && m < 0x1p120) {
        double y = (double)rsqrtf((float)m);
        y = y * fma(-0.5 * m * y, y, 1.5);
        y = y * fma(-0.5 * m * y, y, 1.5);
        return (float)y;
    }
    return (float)(1.0 / sqrt(m));
}

// A CTA walks tokens at a distance of the grid, a thread kPieces x 8 channels of each. With kAhead the next token is asked for before the sum over
// the CTA: what keeps HBM busy over the barrier.
template <typename T, uint32_t kPieces, bool kAhead>
__global__ void __launch_bounds__(kPieces == 1 ? 1024 : 512, kPieces == 2 ? 2 : 1) rms_norm_fp8_kernel(const NormArgs a) {
    __shared__ double partial[2][32];
    const uint32_t lane = threadIdx.x % 32;
    griddep_wait();
    griddep_launch_dependents();
    Piece<T> x[kPieces], more[kPieces];
    const auto load = [&](uint64_t token) {
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            if (c >= a.hidden) continue;
            x[i].load(a.x + token * a.x_stride + (uint64_t)c * sizeof(T));
            if (a.residual) more[i].load(a.residual + token * a.residual_stride + (uint64_t)c * sizeof(T));
        }
    };
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) { x[i].clear(); more[i].clear(); }
    if (kAhead) load(blockIdx.x);
    uint32_t turn = 0;
    for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x, turn ^= 1) {
        if (!kAhead) load(token);
        Piece<T> h[kPieces];
        double sum[1] = {0.0};
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            float v[8];
            h[i] = x[i];
            if (a.residual) {
                float u[8];
                x[i].get(v);
                more[i].get(u);
                #pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += u[j];
                h[i].set(v);
                if (c < a.hidden) h[i].store(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
            }
            h[i].get(v);
            #pragma unroll
            for (int j = 0; j < 8; ++j) sum[0] = fma((double)v[j], (double)v[j], sum[0]);
        }
        if (kAhead && token + gridDim.x < a.tokens) load(token + gridDim.x);
        // (two sets of shared memory: a warp that is a turn ahead does not write to what another still reads)
        cta_sums<double, 1>(sum, partial[turn]);
        const float rstd = rsqrt_of(fma(sum[0], a.inverse_hidden, (double)a.eps));
        if (threadIdx.x == 0) a.rstd[token] = rstd;
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            float w[8] = {}, v[8], amax = 0.0f;
            if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w);
            h[i].get(v);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = __fmul_rn(__fmul_rn(v[j], rstd), w[j]);
                amax = fmaxf(amax, fabsf(v[j]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 2));
            const uint32_t e = e4m3_scale_byte(amax);
            // (the second block of a last, half-used scale column is zero)
            const uint32_t next = __shfl_down_sync(kAll, c < a.hidden ? e : 0u, 4);
            if (c >= a.hidden) continue;
            *reinterpret_cast<uint2*>(a.out + token * a.out_stride + c) = e4m3_pack8(v, e);
            if (a.rows) {
                Piece<__nv_bfloat16> y;
                y.set(v);
                y.store(a.rows + token * a.rows_stride + (uint64_t)c * 2);
            }
            if (lane % 8 == 0) *reinterpret_cast<uint16_t*>(a.sf + (uint64_t)(c / 64) * a.sf_col_stride + token * 2) = (uint16_t)(e | next << 8);
        }
    }
}

// The gradient. With n = h * rstd, u = g * weight: dx = rstd (u - n mean(u n)) + grad_h, dweight = sum over the tokens of g n. A CTA walks tokens at a
// distance of the grid, holds its channels' part of dweight in registers (FP32) and writes it to `partial` at the end, which a second
// kernel sums in the order of the CTAs: nothing depends on timing.
struct NormGradArgs {
    const uint8_t* g; uint64_t g_stride;                                 // BF16 or FP32 as `h` is, or BF16 beside FP32
    const uint8_t *h, *grad_h; uint64_t h_stride, grad_h_stride;         // bytes between rows; grad_h or nullptr
    const void* weight; uint32_t weight_fp32;
    const float* rstd;
    uint8_t* dx; uint64_t dx_stride;
    float* partial;                                                      // [gridDim.x][hidden]
    uint32_t tokens, hidden;
    float inverse_hidden;
};

template <typename T, typename G, uint32_t kPieces, bool kAhead>
__global__ void __launch_bounds__(kPieces == 1 ? 1024 : 512, kPieces == 2 ? 2 : 1) rms_norm_grad_kernel(const NormGradArgs a) {
    __shared__ float sums[2][32];
    griddep_wait();
    griddep_launch_dependents();
    float w[kPieces][8], dw[kPieces][8];
    Piece<T> h[kPieces], more[kPieces];
    Piece<G> g[kPieces];
    float rstd = 0.0f;
    const auto load = [&](uint64_t token) {
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            if (c >= a.hidden) continue;
            h[i].load(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
            g[i].load(a.g + token * a.g_stride + (uint64_t)c * sizeof(G));
            if (a.grad_h) more[i].load(a.grad_h + token * a.grad_h_stride + (uint64_t)c * sizeof(T));
        }
        rstd = __uint_as_float(ld_global_u32(a.rstd + token));
    };
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) { h[i].clear(); g[i].clear(); more[i].clear(); }
    if (kAhead) load(blockIdx.x);
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
        #pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = dw[i][j] = 0.0f;
        if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w[i]);
    }
    uint32_t turn = 0;
    for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x, turn ^= 1) {
        if (!kAhead) load(token);
        Piece<T> h0[kPieces], more0[kPieces];
        Piece<G> g0[kPieces];
        const float r = rstd;
        float dot[1] = {0.0f};
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            h0[i] = h[i]; more0[i] = more[i]; g0[i] = g[i];
            float n[8], u[8];
            h0[i].get(n);
            g0[i].get(u);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                n[j] *= r;
                dw[i][j] = fmaf(u[j], n[j], dw[i][j]);
                dot[0] = fmaf(u[j] * w[i][j], n[j], dot[0]);
            }
        }
        if (kAhead && token + gridDim.x < a.tokens) load(token + gridDim.x);
        cta_sums<float, 1>(dot, sums[turn]);
        const float mean = dot[0] * a.inverse_hidden;
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            if (c >= a.hidden) continue;
            float n[8], u[8], d[8];
            h0[i].get(n);
            g0[i].get(u);
            more0[i].get(d);
            #pragma unroll
            for (int j = 0; j < 8; ++j) d[j] += r * (u[j] * w[i][j] - n[j] * r * mean);
            Piece<T> out;
            out.set(d);
            out.store(a.dx + token * a.dx_stride + (uint64_t)c * sizeof(T));
        }
    }
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
        if (c >= a.hidden) continue;
        Piece<float> out;
        out.set(dw[i]);
        out.store(reinterpret_cast<uint8_t*>(a.partial + (uint64_t)blockIdx.x * a.hidden + c));
    }
}

// 32 channels a CTA, a warp every 32nd of the parts.
constexpr uint32_t kSumThreads = 1024, kSumChannels = 32;
__global__ void __launch_bounds__(kSumThreads) rms_norm_grad_sum_kernel(const float* partial, float* dw, uint32_t parts, uint32_t hidden) {
    __shared__ float sums[32][kSumChannels];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = blockIdx.x * kSumChannels + lane;
    griddep_wait();
    griddep_launch_dependents();
    float sum = 0.0f;
    #pragma unroll 4
    for (uint32_t p = warp; p < parts; p += 32) sum += __uint_as_float(ld_global_u32(partial + (uint64_t)p * hidden + c));
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp != 0) return;
    #pragma unroll
    for (uint32_t i = 1; i < 32; ++i) sum += sums[i][lane];
    dw[c] = sum;
}

// Threads of a CTA whose threads take `pieces` pieces of a row each.
static uint32_t norm_threads(uint32_t hidden, uint32_t pieces) { return ((hidden / 8 + pieces - 1) / pieces + 31) / 32 * 32; }
// CTAs on the 148 SMs: with up to two pieces a thread has 64 registers, beyond that 128.
static uint32_t norm_ctas(uint32_t tokens, uint32_t hidden, uint32_t pieces) {
    const uint32_t most = 148 * (pieces <= 2 ? 1024 / norm_threads(hidden, pieces) : 1);
    return tokens < most ? tokens : most;
}
// Pieces of a row for a thread: one while the row fits `most` threads, then two where there are such kernels, four, eight.
static uint32_t norm_pieces(uint32_t hidden, uint32_t most, bool two) {
    if (norm_threads(hidden, 1) <= most) return 1;
    return two && norm_threads(hidden, 2) <= 512 ? 2 : norm_threads(hidden, 4) <= 512 ? 4 : 8;
}
static uint32_t norm_grad_parts(uint32_t tokens, uint32_t hidden) { return norm_ctas(tokens, hidden, norm_pieces(hidden, 1024, false)); }

}  // namespace dg

using namespace dg;

static int norm_checks(uint32_t tokens, uint32_t hidden) {
    DG_CHECK_ARG(hidden > 0 && hidden % 32 == 0 && hidden <= kMostHidden, "rms_norm: the row length must be a multiple of 32, at most %u", kMostHidden);
    DG_CHECK_ARG(tokens <= 0x7fffffffu, "rms_norm: too many tokens");
    return DG_OK;
}
static bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) | stride_bytes) % 16 == 0; }

template <typename T>
static const void* norm_kernel(uint32_t pieces) {
    if constexpr (sizeof(T) == 2)
        if (pieces == 2) return (const void*)rms_norm_fp8_kernel<T, 2, true>;
    return pieces == 1 ? (const void*)rms_norm_fp8_kernel<T, 1, true> : pieces == 4 ? (const void*)rms_norm_fp8_kernel<T, 4, false> : (const void*)rms_norm_fp8_kernel<T, 8, false>;
}

extern "C" int dg_rms_norm_fp8_launch(const void* x, int is_fp32, uint64_t x_stride, const void* residual, uint64_t residual_stride, void* h, uint64_t h_stride,
                                      const void* weight, int weight_is_fp32, float eps, uint32_t tokens, uint32_t hidden, void* out, uint64_t out_stride,
                                      int16_t* out_sf, uint64_t sf_col_stride, void* rows, uint64_t rows_stride, float* rstd, void* stream) {
    const uint64_t es = is_fp32 ? 4 : 2;
    if (int rc = norm_checks(tokens, hidden)) return rc;
    if (tokens == 0) return DG_OK;
    DG_CHECK_ARG(x != nullptr && weight != nullptr && out != nullptr && out_sf != nullptr && rstd != nullptr && (residual == nullptr || h != nullptr),
                 "rms_norm: null pointer");
    DG_CHECK_ARG(aligned16(x, x_stride * es) && aligned16(residual, residual_stride * es) && aligned16(h, h_stride * es) && aligned16(rows, rows_stride * 2) && aligned16(weight, 0),
                 "rms_norm: rows and the weight must start on 16-byte boundaries");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(out) | out_stride) % 8 == 0, "rms_norm: output rows must start on 8-byte boundaries");
    DG_CHECK_ARG(sf_col_stride >= tokens, "rms_norm: scale column stride smaller than the token count");
    NormArgs a{};
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * es;
    a.residual = static_cast<const uint8_t*>(residual); a.residual_stride = residual_stride * es;
    a.h = static_cast<uint8_t*>(h); a.h_stride = h_stride * es;
    a.weight = weight; a.weight_fp32 = weight_is_fp32 ? 1u : 0u;
    a.rows = static_cast<uint8_t*>(rows); a.rows_stride = rows_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride;
    a.sf = reinterpret_cast<uint8_t*>(out_sf); a.sf_col_stride = sf_col_stride * 2;
    a.rstd = rstd; a.tokens = tokens; a.hidden = hidden; a.eps = eps;
    a.inverse_hidden = 1.0 / hidden;
    // Few tokens: as many threads as a row has pieces; many of BF16: at most 512, so that two CTAs are on an SM. (FP32 has twice the bytes in each.)
    const uint32_t pieces = norm_pieces(hidden, is_fp32 || tokens <= 148 ? 1024 : 512, !is_fp32);
    void* params[] = {&a};
    return launch_overlapped(is_fp32 ? norm_kernel<float>(pieces) : norm_kernel<__nv_bfloat16>(pieces), dim3(norm_ctas(tokens, hidden, pieces)),
                             dim3(norm_threads(hidden, pieces)), params, static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t dg_rms_norm_grad_scratch_bytes(uint32_t tokens, uint32_t hidden) { return hidden ? (uint64_t)norm_grad_parts(tokens, hidden) * hidden * 4 : 0; }

template <typename T, typename G>
static const void* norm_grad_kernel(uint32_t pieces) {
    return pieces == 1 ? (const void*)rms_norm_grad_kernel<T, G, 1, true> : pieces == 4 ? (const void*)rms_norm_grad_kernel<T, G, 4, false>
                                                                                        : (const void*)rms_norm_grad_kernel<T, G, 8, false>;
}

extern "C" int dg_rms_norm_grad_launch(const void* grad_out, int grad_is_fp32, uint64_t grad_stride, const void* h, int is_fp32, uint64_t h_stride, const void* weight,
                                       int weight_is_fp32, const float* rstd, const void* grad_h, uint64_t grad_h_stride, uint32_t tokens, uint32_t hidden,
                                       void* grad_x, uint64_t grad_x_stride, float* grad_weight, void* scratch, uint64_t scratch_bytes, void* stream) {
    const uint64_t es = is_fp32 ? 4 : 2;
    if (int rc = norm_checks(tokens, hidden)) return rc;
    DG_CHECK_ARG(grad_weight != nullptr, "rms_norm_grad: null pointer");
    if (tokens == 0) {
        DG_CHECK_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)hidden * 4, static_cast<cudaStream_t>(stream)));
        return DG_OK;
    }
    DG_CHECK_ARG(grad_out != nullptr && h != nullptr && weight != nullptr && rstd != nullptr && grad_x != nullptr && scratch != nullptr, "rms_norm_grad: null pointer");
    DG_CHECK_ARG(!grad_is_fp32 || is_fp32, "rms_norm_grad: an FP32 gradient beside BF16 rows");
    DG_CHECK_ARG(aligned16(grad_out, grad_stride * (grad_is_fp32 ? 4 : 2)) && aligned16(h, h_stride * es) && aligned16(grad_h, grad_h_stride * es) &&
                 aligned16(grad_x, grad_x_stride * es) && aligned16(weight, 0) && aligned16(scratch, 0), "rms_norm_grad: rows and the weight must start on 16-byte boundaries");
    DG_CHECK_ARG(scratch_bytes >= dg_rms_norm_grad_scratch_bytes(tokens, hidden), "rms_norm_grad: scratch is too small");
    NormGradArgs a{};
    a.g = static_cast<const uint8_t*>(grad_out); a.g_stride = grad_stride * (grad_is_fp32 ? 4 : 2);
    a.h = static_cast<const uint8_t*>(h); a.h_stride = h_stride * es;
    a.grad_h = static_cast<const uint8_t*>(grad_h); a.grad_h_stride = grad_h_stride * es;
    a.weight = weight; a.weight_fp32 = weight_is_fp32 ? 1u : 0u;
    a.rstd = rstd;
    a.dx = static_cast<uint8_t*>(grad_x); a.dx_stride = grad_x_stride * es;
    a.partial = static_cast<float*>(scratch);
    a.tokens = tokens; a.hidden = hidden;
    a.inverse_hidden = 1.0f / (float)hidden;
    const uint32_t pieces = norm_pieces(hidden, 1024, false);
    uint32_t parts = norm_grad_parts(tokens, hidden);
    const void* fn = !is_fp32 ? norm_grad_kernel<__nv_bfloat16, __nv_bfloat16>(pieces) : grad_is_fp32 ? norm_grad_kernel<float, float>(pieces)
                                                                                                      : norm_grad_kernel<float, __nv_bfloat16>(pieces);
    void* params[] = {&a};
    if (int rc = launch_overlapped(fn, dim3(parts), dim3(norm_threads(hidden, pieces)), params, static_cast<cudaStream_t>(stream))) return rc;
    const float* from = a.partial;
    void* sum_params[] = {&from, &grad_weight, &parts, &hidden};
    return launch_overlapped((const void*)rms_norm_grad_sum_kernel, dim3(hidden / kSumChannels), dim3(kSumThreads), sum_params, static_cast<cudaStream_t>(stream));
}
