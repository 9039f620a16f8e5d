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

constexpr uint32_t kAll = 0xffffffffu, kMostHidden = 16384;

// Eight channels of a lane as they lie in memory.
template <typename T> struct Piece;
template <> struct Piece<__nv_bfloat16> {
    uint4 q;
    __device__ __forceinline__ void load(const uint8_t* p) { q = ld_stream_v4(p); }
    __device__ __forceinline__ void clear() { q = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(Pair (&v)[4]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Pair(bf16_lo(w[j]), bf16_hi(w[j]));
    }
    __device__ __forceinline__ void set(const Pair (&v)[4]) {
        uint32_t w[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            v[j].get(lo, hi);
            const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
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
    __device__ __forceinline__ void get(Pair (&v)[4]) const {
        v[0] = Pair(__uint_as_float(q.x), __uint_as_float(q.y)); v[1] = Pair(__uint_as_float(q.z), __uint_as_float(q.w));
        v[2] = Pair(__uint_as_float(r.x), __uint_as_float(r.y)); v[3] = Pair(__uint_as_float(r.z), __uint_as_float(r.w));
    }
    __device__ __forceinline__ void set(const Pair (&v)[4]) {
        float f[8];
        #pragma unroll
        for (int j = 0; j < 4; ++j) v[j].get(f[2 * j], f[2 * j + 1]);
        q = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        r = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        *reinterpret_cast<uint4*>(p) = q;
        *reinterpret_cast<uint4*>(p + 16) = r;
    }
};
__device__ __forceinline__ void weight_at(const void* weight, uint32_t fp32, uint32_t c, Pair (&v)[4]) {
    if (fp32) {
        Piece<float> p;
        p.q = ld_global_v4(static_cast<const float*>(weight) + c);
        p.r = ld_global_v4(static_cast<const float*>(weight) + c + 4);
        p.get(v);
    } else {
        Piece<__nv_bfloat16> p;
        p.q = ld_global_v4(static_cast<const __nv_bfloat16*>(weight) + c);
        p.get(v);
    }
}

// The sum over a group of `warps` warps, of which `first` is the first, in all its threads. `partial`: a place for each warp of the CTA that nobody reads any more.
template <typename S>
__device__ __forceinline__ S group_sum(S v, S* partial, uint32_t first, uint32_t warps, uint32_t barrier) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if (lane == 0) partial[warp] = v;
    named_bar_sync(barrier, warps * 32);
    v = lane < warps ? partial[first + lane] : (S)0;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
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
template <typename T, uint32_t kPieces, uint32_t kThreads, uint32_t kCtas, bool kAhead>
__global__ void __launch_bounds__(kThreads, kCtas) rms_norm_fp8_kernel(const NormArgs a) {
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
        double sum = 0.0;
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            Pair v[4];
            h[i] = x[i];
            if (a.residual) {
                Pair u[4];
                x[i].get(v);
                more[i].get(u);
                #pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = v[j] + u[j];
                h[i].set(v);
                if (c < a.hidden) h[i].store(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
            }
            h[i].get(v);
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                v[j].get(lo, hi);
                sum = fma((double)lo, (double)lo, sum);
                sum = fma((double)hi, (double)hi, sum);
            }
        }
        if (kAhead && token + gridDim.x < a.tokens) load(token + gridDim.x);
        // (two sets of shared memory: a warp that is a turn ahead does not write to what another still reads)
        sum = group_sum(sum, partial[turn], 0, blockDim.x / 32, 1);
        const float rstd = rsqrt_of(fma(sum, a.inverse_hidden, (double)a.eps));
        if (threadIdx.x == 0) a.rstd[token] = rstd;
        const Pair scale(rstd);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * blockDim.x + threadIdx.x) * 8;
            Pair w[4] = {}, v[4];
            if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w);
            h[i].get(v);
            float amax = 0.0f;
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = v[j] * scale * w[j];
                amax = larger_magnitude(amax, v[j]);
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

// The gradient. With n = h * rstd, u = g * weight: dx = rstd (u - n mean(u n)) + grad_h, dweight = sum over the tokens of g n. A group of a CTA's warps takes
// a token, and walks tokens at a distance of all groups; a thread holds its channels' part of dweight in registers (FP32), the groups of a CTA add theirs up,
// and a second kernel sums the CTAs' in their order: nothing depends on timing.
//
// HBM-bound, and what bounds the walk is the way from a token's loads over its barrier to its stores: with kAhead the next token is asked for in front of the
// barrier.
struct NormGradArgs {
    const uint8_t* g; uint64_t g_stride;                                 // BF16 or FP32 as `h` is, or BF16 beside FP32
    const uint8_t *h, *grad_h; uint64_t h_stride, grad_h_stride;         // bytes between rows; grad_h or nullptr
    const void* weight; uint32_t weight_fp32;
    const float* rstd;
    uint8_t* dx; uint64_t dx_stride;
    float* partial;                                                      // [gridDim.x][hidden]
    uint32_t tokens, hidden;
    uint32_t groups, threads;                                            // of a CTA; of a group
    float inverse_hidden;
};

template <typename T, typename G, uint32_t kPieces, uint32_t kThreads, bool kAhead>
__global__ void __launch_bounds__(kThreads) rms_norm_grad_kernel(const NormGradArgs a) {
    extern __shared__ __align__(16) uint8_t others[];
    __shared__ float sums[2][32];
    const uint32_t group = threadIdx.x / a.threads, t = threadIdx.x - group * a.threads, warps = a.threads / 32;
    const uint64_t stride = (uint64_t)gridDim.x * a.groups, first = (uint64_t)blockIdx.x * a.groups + group;
    griddep_wait();
    griddep_launch_dependents();
    Piece<T> h[kPieces], more[kPieces];
    Piece<G> g[kPieces];
    float rstd = 0.0f;
    const auto load = [&](uint64_t token) {
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * a.threads + t) * 8;
            if (c >= a.hidden) continue;
            h[i].load(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
            g[i].load(a.g + token * a.g_stride + (uint64_t)c * sizeof(G));
            if (a.grad_h) more[i].load(a.grad_h + token * a.grad_h_stride + (uint64_t)c * sizeof(T));
        }
        rstd = __uint_as_float(ld_global_u32(a.rstd + token));
    };
    Pair sum_w[kPieces][4];
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        h[i].clear(); g[i].clear(); more[i].clear();
        #pragma unroll
        for (int j = 0; j < 4; ++j) sum_w[i][j] = Pair(0.0f);
    }
    if (kAhead && first < a.tokens) load(first);
    Pair w[4] = {};                                           // (those of several pieces come from L1 each time)
    const auto weights = [&](uint32_t i) {
        const uint32_t c = (i * a.threads + t) * 8;
        if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w);
    };
    if constexpr (kPieces == 1) weights(0);
    uint32_t turn = 0;
    for (uint64_t token = first; token < a.tokens; token += stride, turn ^= 1) {
        if (!kAhead) load(token);
        Piece<T> h0[kPieces], more0[kPieces];
        Piece<G> g0[kPieces];
        const float r = rstd;
        const Pair scale(r);
        // sum(u n) = rstd sum(u h)
        Pair dots(0.0f);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            h0[i] = h[i]; more0[i] = more[i]; g0[i] = g[i];
            Pair n[4], u[4];
            if constexpr (kPieces > 1) weights(i);
            h0[i].get(n);
            g0[i].get(u);
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                dots = fma2(u[j] * w[j], n[j], dots);
                sum_w[i][j] = fma2(u[j], n[j] * scale, sum_w[i][j]);
            }
        }
        if (kAhead && token + stride < a.tokens) load(token + stride);
        float dot, other;
        dots.get(dot, other);
        // (two sets of sums: a warp that is a turn ahead does not write to what another still reads)
        dot = group_sum(dot + other, sums[turn], group * warps, warps, group + 1);
        // dx = rstd u - h (rstd^3 mean(u h)) + grad_h
        const Pair slope(-(r * r * (r * (dot * a.inverse_hidden))));
        // (what several pieces would hold over the barrier is read again: it lies in L2)
        if constexpr (!kAhead) load(token);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * a.threads + t) * 8;
            if (c >= a.hidden) continue;
            Pair n[4], u[4], d[4];
            if constexpr (kPieces > 1) weights(i);
            if constexpr (!kAhead) { h0[i] = h[i]; g0[i] = g[i]; more0[i] = more[i]; }
            h0[i].get(n);
            g0[i].get(u);
            more0[i].get(d);
            #pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = fma2(n[j], slope, fma2(scale, u[j] * w[j], d[j]));
            h0[i].set(d);
            h0[i].store(a.dx + token * a.dx_stride + (uint64_t)c * sizeof(T));
        }
    }
    float dw[kPieces][8];
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) sum_w[i][j].get(dw[i][2 * j], dw[i][2 * j + 1]);
    if (a.groups > 1) {
        float4* const to = reinterpret_cast<float4*>(others);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i)
            #pragma unroll
            for (uint32_t k = 0; k < 2; ++k)
                if (group > 0) to[((group - 1) * 2 * kPieces + 2 * i + k) * a.threads + t] = make_float4(dw[i][4 * k], dw[i][4 * k + 1], dw[i][4 * k + 2], dw[i][4 * k + 3]);
        __syncthreads();
        if (group > 0) return;
        for (uint32_t o = 0; o + 1 < a.groups; ++o)
            #pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i)
                #pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    const float4 v = to[(o * 2 * kPieces + 2 * i + k) * a.threads + t];
                    dw[i][4 * k] += v.x; dw[i][4 * k + 1] += v.y; dw[i][4 * k + 2] += v.z; dw[i][4 * k + 3] += v.w;
                }
    }
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        const uint32_t c = (i * a.threads + t) * 8;
        if (c >= a.hidden) continue;
        float4* const out = reinterpret_cast<float4*>(a.partial + (uint64_t)blockIdx.x * a.hidden + c);
        out[0] = make_float4(dw[i][0], dw[i][1], dw[i][2], dw[i][3]);
        out[1] = make_float4(dw[i][4], dw[i][5], dw[i][6], dw[i][7]);
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

// How the gradient's kernel is laid over the SMs, one CTA each: one piece of a row a thread where that takes at most 896 threads (512 of FP32), in as many groups
// as fit, else four; as many CTAs as finish together.
struct NormGradShape { uint32_t pieces, threads, groups, parts; };
static NormGradShape norm_grad_shape(uint32_t tokens, uint32_t hidden, bool fp32) {
    const uint32_t most = fp32 ? 512 : 896;
    NormGradShape s{};
    s.pieces = norm_threads(hidden, 1) <= most ? 1 : 4;
    s.threads = norm_threads(hidden, s.pieces);
    s.groups = s.pieces == 4 ? 1 : most / s.threads < 8 ? most / s.threads : 8;
    while (s.groups > 1 && (s.groups - 1) * 148 >= tokens) --s.groups;
    const uint32_t wanted = (tokens + s.groups - 1) / s.groups, turns = (wanted + 147) / 148;
    s.parts = turns ? (wanted + turns - 1) / turns : 0;
    return s;
}

}  // namespace dg

using namespace dg;

static int norm_checks(uint32_t tokens, uint32_t hidden) {
    DG_CHECK_ARG(hidden > 0 && hidden % 32 == 0 && hidden <= kMostHidden, "rms_norm: the row length must be a multiple of 32, at most %u", kMostHidden);
    DG_CHECK_ARG(tokens <= 0x7fffffffu, "rms_norm: too many tokens");
    return DG_OK;
}
static bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) | stride_bytes) % 16 == 0; }

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
    // Few tokens: as many threads as a row has pieces. Many of BF16: half as many, and two CTAs on an SM. (FP32 has twice the bytes in each.)
    const void* fn;
    uint32_t pieces = 1, resident = 1;
    if (norm_threads(hidden, 1) <= (is_fp32 || tokens <= 148 ? 1024 : 448)) {
        resident = 896 / norm_threads(hidden, pieces);
        fn = is_fp32 ? (const void*)rms_norm_fp8_kernel<float, 1, 1024, 1, true> : (const void*)rms_norm_fp8_kernel<__nv_bfloat16, 1, 1024, 1, true>;
    } else if (!is_fp32 && norm_threads(hidden, 2) <= 448) {
        pieces = 2;
        resident = 896 / norm_threads(hidden, pieces);
        fn = (const void*)rms_norm_fp8_kernel<__nv_bfloat16, 2, 448, 2, true>;
    } else {
        pieces = 4;
        fn = is_fp32 ? (const void*)rms_norm_fp8_kernel<float, 4, 512, 1, false> : (const void*)rms_norm_fp8_kernel<__nv_bfloat16, 4, 512, 1, true>;
    }
    resident = resident < 1 ? 1 : resident > 16 ? 16 : resident;
    void* params[] = {&a};
    return launch_overlapped(fn, dim3(tokens < 148 * resident ? tokens : 148 * resident), dim3(norm_threads(hidden, pieces)), params, static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t dg_rms_norm_grad_scratch_bytes(uint32_t tokens, uint32_t hidden) {
    if (hidden == 0) return 0;
    const uint32_t bf16 = norm_grad_shape(tokens, hidden, false).parts, fp32 = norm_grad_shape(tokens, hidden, true).parts;
    return (uint64_t)(bf16 > fp32 ? bf16 : fp32) * hidden * 4;
}

template <typename T, typename G>
static const void* norm_grad_kernel(uint32_t pieces) {
    return pieces == 1 ? (const void*)rms_norm_grad_kernel<T, G, 1, sizeof(T) == 4 ? 512 : 896, true> : (const void*)rms_norm_grad_kernel<T, G, 4, 512, false>;
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
    const NormGradShape shape = norm_grad_shape(tokens, hidden, is_fp32);
    a.groups = shape.groups; a.threads = shape.threads;
    uint32_t parts = shape.parts;
    const void* fn = !is_fp32 ? norm_grad_kernel<__nv_bfloat16, __nv_bfloat16>(shape.pieces) : grad_is_fp32 ? norm_grad_kernel<float, float>(shape.pieces)
                                                                                             : norm_grad_kernel<float, __nv_bfloat16>(shape.pieces);
    void* params[] = {&a};
    if (int rc = launch_overlapped(fn, dim3(parts), dim3(shape.groups * shape.threads), params, static_cast<cudaStream_t>(stream),
                                   (shape.groups - 1) * shape.threads * shape.pieces * 32)) return rc;
    const float* from = a.partial;
    void* sum_params[] = {&from, &grad_weight, &parts, &hidden};
    return launch_overlapped((const void*)rms_norm_grad_sum_kernel, dim3(hidden / kSumChannels), dim3(kSumThreads), sum_params, static_cast<cudaStream_t>(stream));
}
