// The step between the residual stream and a block-scaled product: h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, written as E4M3 with
// one UE8M0 scale per 32 channels in the layout the GEMM reads (and in BF16 where a router or a dispatch wants it), and its gradient.
//
// h is rounded to its type before the norm sees it: what the residual stream holds is what the gradient is taken at. The sum of squares is held in
// 64 bits and made in one order however a row is spread over threads (row_sum): a token's bits do not depend on how many others there are. y = (h * rstd) * weight in FP32, one rounding each, then one to E4M3 (values times the inverse of the scale of quant.cuh, which is
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
// How long a wait for a bulk copy may take. (0: every one gives up at once, for a test of what happens then)
#ifndef DG_NORM_LONGEST_WAIT_NS
#define DG_NORM_LONGEST_WAIT_NS 2000000000ull
#endif
constexpr uint64_t kLongestWaitNs = DG_NORM_LONGEST_WAIT_NS, kLongestDrainNs = 2000000000ull;
constexpr int32_t kStatusTimeoutRows = 108;
// 0, or that a wait gave up: a word of this file's own, which its kernels reach without an argument. dg_device_status reads it.
__device__ int32_t g_norm_status = 0;

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
__device__ __forceinline__ float group_sum(float v, float* partial, uint32_t first, uint32_t warps, uint32_t barrier) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if (lane == 0) partial[warp] = v;
    named_bar_sync(barrier, warps * 32);
    v = lane < warps ? partial[first + lane] : 0.0f;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

// The sum over a group of the sums of squares of a thread's pieces, in an order that depends on the row's length alone: pairs of a piece's lanes, then pairs of
// the places that stand 32 pieces (256 channels) apart, whichever thread holds them. `partial`: as above, kPieces places for each warp.
template <uint32_t kPieces>
__device__ __forceinline__ double row_sum(const double (&of)[kPieces], double* partial, uint32_t first, uint32_t warps, uint32_t barrier) {
    const uint32_t warp = threadIdx.x / 32 - first, lane = threadIdx.x % 32;
    partial += first * kPieces;
    double v;
    if constexpr (kPieces == 1) {
        v = of[0] + __shfl_xor_sync(kAll, of[0], 16);
    } else {
        // (the lower lanes carry on with the first piece, the upper ones with the second)
        v = lane < 16 ? of[0] : of[1];
        v += __shfl_xor_sync(kAll, lane < 16 ? of[1] : of[0], 16);
    }
    #pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if (lane % (32 / kPieces) == 0) partial[lane / (32 / kPieces) * warps + warp] = v;
    named_bar_sync(barrier, warps * 32);
    v = lane < kPieces * warps ? partial[lane] : 0.0;
    if (kPieces > 1 && lane + 32 < kPieces * warps) v += partial[lane + 32];
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
    uint32_t groups, threads, stages;                                    // long rows: of a CTA; of a group; tokens in shared memory
    float eps;
    double inverse_hidden;
};

__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
    if (kLongestWaitNs == 0) return false;
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, parity))
        if (global_timer_ns() - t0 > kLongestWaitNs) return false;
    return true;
}
// A wait gave up: a group takes no more tokens. Its first thread says so and lets the copies that were asked for, `asked` from `stage` on, land (again with a limit)
// before the CTA leaves its shared memory to another. Out of line: no launch that works runs it.
static __device__ __noinline__ void report_and_drain(uint32_t full_at, uint32_t stages, uint32_t stage, uint32_t parity, uint64_t asked) {
    atomicCAS(&g_norm_status, 0, kStatusTimeoutRows);
    const uint64_t t0 = global_timer_ns();
    for (uint64_t i = 0; i < asked; ++i) {
        while (!mbar_try_wait(full_at + stage * 8, parity) && global_timer_ns() - t0 < kLongestDrainNs) {}
        if (++stage == stages) { stage = 0; parity ^= 1; }
    }
}
// How many tokens from `token` on there are, `most` at most.
__device__ __forceinline__ uint64_t tokens_ahead(uint64_t token, uint64_t tokens, uint64_t stride, uint32_t most) { return min((tokens - token + stride - 1) / stride, (uint64_t)most); }

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

// h of a piece, and the sum of its squares.
template <typename T>
__device__ __forceinline__ void add_piece(const NormArgs& a, uint64_t token, uint32_t c, const Piece<T>& x, const Piece<T>& more, Piece<T>& h, double& sum) {
    Pair v[4];
    h = x;
    if (a.residual) {
        Pair u[4];
        x.get(v);
        more.get(u);
        #pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = v[j] + u[j];
        h.set(v);
        if (c < a.hidden) h.store(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
    }
    h.get(v);
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        float lo, hi;
        v[j].get(lo, hi);
        sum = fma((double)lo, (double)lo, sum);
        sum = fma((double)hi, (double)hi, sum);
    }
}
// The norm of a piece and its codes. (All lanes of a warp come here.)
template <typename T>
__device__ __forceinline__ void finish_piece(const NormArgs& a, uint64_t token, uint32_t c, const Piece<T>& h, Pair scale) {
    Pair w[4] = {}, v[4];
    if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w);
    h.get(v);
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
    if (c >= a.hidden) return;
    *reinterpret_cast<uint2*>(a.out + token * a.out_stride + c) = e4m3_pack8(v, e);
    if (a.rows) {
        Piece<__nv_bfloat16> y;
        y.set(v);
        y.store(a.rows + token * a.rows_stride + (uint64_t)c * 2);
    }
    if (c % 64 == 0) *reinterpret_cast<uint16_t*>(a.sf + (uint64_t)(c / 64) * a.sf_col_stride + token * 2) = (uint16_t)(e | next << 8);
}

// Few tokens, short rows and some of the middle: a CTA walks tokens at a distance of the grid, a thread kPieces x 8 channels of each. The next token is asked for before
// the sum over the CTA: what keeps HBM busy over the barrier. 8192 x 7168 of BF16 with a residual and BF16 rows 89 us, 5.9 TB/s, where the bytes alone take 81 at the rate
// of a copy (a CTA for every token took 106, L2 asked for the token behind the next 109). 1 x 7168: 2.4 to 2.7 us, launch and latency.
template <typename T, uint32_t kPieces, uint32_t kThreads, uint32_t kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) rms_norm_fp8_kernel(const NormArgs a) {
    __shared__ double partial[2][kPieces * (kThreads / 32)];
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
    load(blockIdx.x);
    uint32_t turn = 0;
    for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x, turn ^= 1) {
        Piece<T> h[kPieces];
        double sums[kPieces] = {};
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) add_piece(a, token, (i * blockDim.x + threadIdx.x) * 8, x[i], more[i], h[i], sums[i]);
        if (token + gridDim.x < a.tokens) load(token + gridDim.x);
        // (two sets of shared memory: a warp that is a turn ahead does not write to what another still reads)
        const double sum = row_sum(sums, partial[turn], 0, blockDim.x / 32, 1);
        const float rstd = rsqrt_of(fma(sum, a.inverse_hidden, (double)a.eps));
        if (threadIdx.x == 0) a.rstd[token] = rstd;
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) finish_piece(a, token, (i * blockDim.x + threadIdx.x) * 8, h[i], Pair(rstd));
    }
}

// Many tokens, and rows too long for the above: the rows of a token come to shared memory by bulk copies, as many tokens ahead as fit there; a group of a CTA's warps
// takes a token, a thread one piece of it or two. Behind the barrier of the sum nobody reads the rows any more, and the next token takes their place.
constexpr uint32_t kLongThreads = 1024, kLongSmem = 225 * 1024, kLongMostStages = 4, kMostGroups = 8;

__device__ __forceinline__ void take(Piece<__nv_bfloat16>& p, const uint8_t* from) { p.q = *reinterpret_cast<const uint4*>(from); }
__device__ __forceinline__ void take(Piece<float>& p, const uint8_t* from) {
    p.q = *reinterpret_cast<const uint4*>(from);
    p.r = *reinterpret_cast<const uint4*>(from + 16);
}

template <typename T, uint32_t kPieces>
__global__ void __launch_bounds__(kLongThreads) rms_norm_fp8_long_kernel(const NormArgs a) {
    extern __shared__ __align__(16) uint8_t places[];         // of each token: the rows of x and of the residual
    __shared__ double partial[2][kPieces * (kLongThreads / 32)];
    __shared__ __align__(8) uint64_t full[kMostGroups * kLongMostStages];
    __shared__ volatile uint32_t gave_up[2][kMostGroups];     // set in front of the barrier of a turn, read behind it: two sets, as of the sums
    const uint32_t groups = a.groups, group = threadIdx.x / a.threads, t = threadIdx.x - group * a.threads, warps = a.threads / 32;
    const uint64_t stride = (uint64_t)gridDim.x * groups, first = (uint64_t)blockIdx.x * groups + group;
    const uint32_t row = a.hidden * sizeof(T), place = a.residual ? 2 * row : row;
    const uint8_t* const mine = places + group * a.stages * place;
    const uint32_t mine_at = smem_u32(mine), full_at = smem_u32(full + group * a.stages);
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < groups * a.stages; ++s) mbar_init(smem_u32(full + s), 1);
        for (uint32_t g = 0; g < groups; ++g) gave_up[0][g] = gave_up[1][g] = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    __syncthreads();
    griddep_wait();
    griddep_launch_dependents();
    const auto ask = [&](uint64_t token, uint32_t stage) {
        const uint32_t to = mine_at + stage * place, bar = full_at + stage * 8;
        mbar_arrive_expect_tx(bar, place);
        bulk_copy_to_smem(to, a.x + token * a.x_stride, row, bar);
        if (a.residual) bulk_copy_to_smem(to + row, a.residual + token * a.residual_stride, row, bar);
    };
    if (t == 0)
        for (uint32_t s = 0; s < a.stages; ++s)
            if (first + s * stride < a.tokens) ask(first + s * stride, s);
    uint32_t turn = 0, stage = 0, parity = 0;
    for (uint64_t token = first; token < a.tokens; token += stride, turn ^= 1) {
        if (!wait_for(full_at + stage * 8, parity)) gave_up[turn][group] = 1;
        const uint8_t* const from = mine + stage * place;
        Piece<T> h[kPieces];
        double sums[kPieces];
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * a.threads + t) * 8;
            Piece<T> x, more;
            x.clear(); more.clear();
            if (c < a.hidden) {
                take(x, from + c * sizeof(T));
                if (a.residual) take(more, from + row + c * sizeof(T));
            }
            sums[i] = 0.0;
            add_piece(a, token, c, x, more, h[i], sums[i]);
        }
        const double sum = row_sum(sums, partial[turn], group * warps, warps, group + 1);
        if (gave_up[turn][group] != 0) {
            if (t != 0) return;
            report_and_drain(full_at, a.stages, stage, parity, tokens_ahead(token, a.tokens, stride, a.stages));
            for (; token < a.tokens; token += stride) a.rstd[token] = __uint_as_float(0x7fc00000u);
            return;
        }
        if (t == 0 && token + a.stages * stride < a.tokens) ask(token + a.stages * stride, stage);
        const float rstd = rsqrt_of(fma(sum, a.inverse_hidden, (double)a.eps));
        if (t == 0) a.rstd[token] = rstd;
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) finish_piece(a, token, (i * a.threads + t) * 8, h[i], Pair(rstd));
        if (++stage == a.stages) { stage = 0; parity ^= 1; }
    }
}

// The gradient. With n = h * rstd, u = g * weight: dx = rstd (u - n mean(u n)) + grad_h, dweight = sum over the tokens of g n. A group of a CTA's warps takes
// a token, and walks tokens at a distance of all groups; a thread holds its channels' part of dweight in registers (FP32), the groups of a CTA add theirs up,
// and a second kernel sums the CTAs' in their order: nothing depends on timing.
//
// HBM-bound: 8192 x 7168 of BF16 with a gradient of h 79 us, 5.9 TB/s (the bytes alone 72 at the rate of a copy); 1531 x 2048 of FP32 11.4 us, of which the second
// kernel and the launches take 3.
struct NormGradArgs {
    const uint8_t* g; uint64_t g_stride;                                 // BF16 or FP32 as `h` is, or BF16 beside FP32
    const uint8_t *h, *grad_h; uint64_t h_stride, grad_h_stride;         // bytes between rows; grad_h or nullptr
    const void* weight; uint32_t weight_fp32;
    const float* rstd;
    uint8_t* dx; uint64_t dx_stride;
    float* partial;                                                      // [gridDim.x][hidden]
    uint32_t tokens, hidden;
    uint32_t groups, threads, stages;                                    // of a CTA; of a group; tokens in shared memory
    float inverse_hidden;
};

// sum(u n), and a thread's part of dweight. (With n and not with h, whose products with u and whose rstd^2 leave the range of FP32 long before dx does.)
__device__ __forceinline__ void add_dots(const Pair (&h)[4], const Pair (&g)[4], const Pair (&w)[4], Pair scale, Pair& dots, Pair (&sum_w)[4]) {
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Pair n = h[j] * scale;
        dots = fma2(g[j] * w[j], n, dots);
        sum_w[j] = fma2(g[j], n, sum_w[j]);
    }
}
// dx = rstd u - n (rstd mean(u n)) + grad_h, which `d` holds
__device__ __forceinline__ void slope_of(const Pair (&h)[4], const Pair (&g)[4], const Pair (&w)[4], Pair scale, Pair slope, Pair (&d)[4]) {
    #pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = fma2(h[j] * scale, slope, fma2(scale, g[j] * w[j], d[j]));
}
__device__ __forceinline__ void store_part(const NormGradArgs& a, uint32_t c, const float (&dw)[8]) {
    float4* const out = reinterpret_cast<float4*>(a.partial + (uint64_t)blockIdx.x * a.hidden + c);
    out[0] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    out[1] = make_float4(dw[4], dw[5], dw[6], dw[7]);
}

// Short rows: a token in registers, a piece of it a thread. What bounds a walk is the way from a token's loads over its barrier to its stores, so the next token
// is asked for in front of the barrier.
template <typename T, typename G, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads) rms_norm_grad_kernel(const NormGradArgs a) {
    extern __shared__ __align__(16) uint8_t others[];
    __shared__ float sums[2][32];
    const uint32_t group = threadIdx.x / a.threads, t = threadIdx.x - group * a.threads, warps = a.threads / 32, c = t * 8;
    const uint64_t stride = (uint64_t)gridDim.x * a.groups, first = (uint64_t)blockIdx.x * a.groups + group;
    const bool inside = c < a.hidden;
    griddep_wait();
    griddep_launch_dependents();
    Piece<T> h, more;
    Piece<G> g;
    float rstd = 0.0f;
    const auto load = [&](uint64_t token) {
        if (inside) {
            h.load(a.h + token * a.h_stride + (uint64_t)c * sizeof(T));
            g.load(a.g + token * a.g_stride + (uint64_t)c * sizeof(G));
            if (a.grad_h) more.load(a.grad_h + token * a.grad_h_stride + (uint64_t)c * sizeof(T));
        }
        rstd = __uint_as_float(ld_global_u32(a.rstd + token));
    };
    h.clear(); g.clear(); more.clear();
    if (first < a.tokens) load(first);
    Pair w[4] = {}, sum_w[4];
    if (inside) weight_at(a.weight, a.weight_fp32, c, w);
    #pragma unroll
    for (int j = 0; j < 4; ++j) sum_w[j] = Pair(0.0f);
    uint32_t turn = 0;
    for (uint64_t token = first; token < a.tokens; token += stride, turn ^= 1) {
        Piece<T> h0 = h, more0 = more;
        const Piece<G> g0 = g;
        const float r = rstd;
        const Pair scale(r);
        Pair n[4], u[4], dots(0.0f);
        h0.get(n);
        g0.get(u);
        add_dots(n, u, w, scale, dots, sum_w);
        if (token + stride < a.tokens) load(token + stride);
        float dot, other;
        dots.get(dot, other);
        // (two sets of sums: a warp that is a turn ahead does not write to what another still reads)
        dot = group_sum(dot + other, sums[turn], group * warps, warps, group + 1);
        if (!inside) continue;
        Pair d[4];
        h0.get(n);
        g0.get(u);
        more0.get(d);
        slope_of(n, u, w, scale, Pair(-(r * (dot * a.inverse_hidden))), d);
        h0.set(d);
        h0.store(a.dx + token * a.dx_stride + (uint64_t)c * sizeof(T));
    }
    float dw[8];
    #pragma unroll
    for (int j = 0; j < 4; ++j) sum_w[j].get(dw[2 * j], dw[2 * j + 1]);
    if (a.groups > 1) {
        float4* const to = reinterpret_cast<float4*>(others);
        #pragma unroll
        for (uint32_t k = 0; k < 2; ++k)
            if (group > 0) to[((group - 1) * 2 + k) * a.threads + t] = make_float4(dw[4 * k], dw[4 * k + 1], dw[4 * k + 2], dw[4 * k + 3]);
        __syncthreads();
        if (group > 0) return;
        for (uint32_t o = 0; o + 1 < a.groups; ++o)
            #pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
                const float4 v = to[(o * 2 + k) * a.threads + t];
                dw[4 * k] += v.x; dw[4 * k + 1] += v.y; dw[4 * k + 2] += v.z; dw[4 * k + 3] += v.w;
            }
    }
    if (inside) store_part(a, c, dw);
}

// Long rows: tokens come to shared memory by bulk copies that the first thread of a group asks for, as many as fit there (16384 channels of FP32 are 192 KB); a
// thread takes one piece of its group's token or two. Behind the barrier of a sum all threads of a group have read the token in front of it, whose place the
// next one takes.
//
// Longer rows than fit in registers: BF16 16384 195, FP32 8192 159, 16384 332 us of 8192 tokens. (Copies that every thread asks for itself, cp.async, took 120 us for 8192
// channels of BF16, where this takes 86: they are issued by the same warps and wait for room.)
template <typename T, typename G, uint32_t kPieces>
__global__ void __launch_bounds__(kLongThreads) rms_norm_grad_long_kernel(const NormGradArgs a) {
    extern __shared__ __align__(16) uint8_t places[];         // of each token: the rows of h, g and grad_h
    __shared__ float sums[2][32];
    __shared__ __align__(8) uint64_t full[kMostGroups * kLongMostStages];
    __shared__ volatile uint32_t gave_up[2][kMostGroups];     // set in front of the barrier of a turn, read behind it: two sets, as of the sums
    // (rows of two pieces leave no room for a second group)
    const uint32_t groups = kPieces == 1 ? a.groups : 1u, group = kPieces == 1 ? threadIdx.x / a.threads : 0u, t = threadIdx.x - group * a.threads, warps = a.threads / 32;
    const uint64_t stride = (uint64_t)gridDim.x * groups, first = (uint64_t)blockIdx.x * groups + group;
    const uint32_t rows_h = a.hidden * sizeof(T), rows_g = a.hidden * sizeof(G), place = rows_h + rows_g + (a.grad_h ? rows_h : 0u);
    const uint8_t* const mine = places + group * a.stages * place;
    const uint32_t mine_at = smem_u32(mine), full_at = smem_u32(full + group * a.stages);
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < groups * a.stages; ++s) mbar_init(smem_u32(full + s), 1);
        for (uint32_t g = 0; g < groups; ++g) gave_up[0][g] = gave_up[1][g] = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    __syncthreads();
    griddep_wait();
    griddep_launch_dependents();
    const auto ask = [&](uint64_t token, uint32_t stage) {
        const uint32_t to = mine_at + stage * place, bar = full_at + stage * 8;
        mbar_arrive_expect_tx(bar, place);
        bulk_copy_to_smem(to, a.h + token * a.h_stride, rows_h, bar);
        bulk_copy_to_smem(to + rows_h, a.g + token * a.g_stride, rows_g, bar);
        if (a.grad_h) bulk_copy_to_smem(to + rows_h + rows_g, a.grad_h + token * a.grad_h_stride, rows_h, bar);
    };
    if (t == 0)
        for (uint32_t s = 0; s < a.stages; ++s)
            if (first + s * stride < a.tokens) ask(first + s * stride, s);
    Pair w[kPieces][4], sum_w[kPieces][4];
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        const uint32_t c = (i * a.threads + t) * 8;
        #pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = sum_w[i][j] = Pair(0.0f);
        if (c < a.hidden) weight_at(a.weight, a.weight_fp32, c, w[i]);
    }
    float next = first < a.tokens ? __uint_as_float(ld_global_u32(a.rstd + first)) : 0.0f;
    uint32_t turn = 0, stage = 0, before = a.stages - 1, parity = 0;
    bool complete = true;
    for (uint64_t token = first; token < a.tokens; token += stride, turn ^= 1) {
        const float r = next;
        if (token + stride < a.tokens) next = __uint_as_float(ld_global_u32(a.rstd + token + stride));
        if (!wait_for(full_at + stage * 8, parity)) gave_up[turn][group] = 1;
        const Pair scale(r);
        const uint8_t* const from = mine + stage * place;
        Pair dots(0.0f);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * a.threads + t) * 8;
            if (c >= a.hidden) continue;
            Piece<T> h;
            Piece<G> g;
            Pair n[4], u[4];
            take(h, from + c * sizeof(T));
            take(g, from + rows_h + c * sizeof(G));
            h.get(n);
            g.get(u);
            add_dots(n, u, w[i], scale, dots, sum_w[i]);
        }
        float dot, other;
        dots.get(dot, other);
        dot = group_sum(dot + other, sums[turn], group * warps, warps, group + 1);
        if (gave_up[turn][group] != 0) {
            complete = false;
            // (behind the first token, the last stage's next one has not been asked for yet)
            if (t == 0) report_and_drain(full_at, a.stages, stage, parity, tokens_ahead(token, a.tokens, stride, token == first || a.stages == 1 ? a.stages : a.stages - 1));
            __syncwarp();
            break;
        }
        // (all threads are done with the token in front)
        const uint64_t later = token + (a.stages - 1) * stride;
        if (t == 0 && a.stages > 1 && token != first && later < a.tokens) ask(later, before);
        const Pair slope(-(r * (dot * a.inverse_hidden)));
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i) {
            const uint32_t c = (i * a.threads + t) * 8;
            if (c >= a.hidden) continue;
            Piece<T> h, more;
            Piece<G> g;
            Pair n[4], u[4], d[4];
            take(h, from + c * sizeof(T));
            take(g, from + rows_h + c * sizeof(G));
            if (a.grad_h) take(more, from + rows_h + rows_g + c * sizeof(T));
            else more.clear();
            h.get(n);
            g.get(u);
            more.get(d);
            slope_of(n, u, w[i], scale, slope, d);
            h.set(d);
            h.store(a.dx + token * a.dx_stride + (uint64_t)c * sizeof(T));
        }
        if (a.stages == 1) {
            named_bar_sync(group + 1, a.threads);
            if (t == 0 && token + stride < a.tokens) ask(token + stride, 0);
        }
        before = stage;
        if (++stage == a.stages) { stage = 0; parity ^= 1; }
    }
    float dw[kPieces][8];
    #pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!complete) sum_w[i][j] = Pair(__uint_as_float(0x7fc00000u));
            sum_w[i][j].get(dw[i][2 * j], dw[i][2 * j + 1]);
        }
    if (groups > 1) {
        __syncthreads();                                      // (nobody reads a token any more)
        float4* const to = reinterpret_cast<float4*>(places);
        #pragma unroll
        for (uint32_t i = 0; i < kPieces; ++i)
            #pragma unroll
            for (uint32_t k = 0; k < 2; ++k)
                if (group > 0) to[((group - 1) * 2 * kPieces + 2 * i + k) * a.threads + t] = make_float4(dw[i][4 * k], dw[i][4 * k + 1], dw[i][4 * k + 2], dw[i][4 * k + 3]);
        __syncthreads();
        if (group > 0) return;
        for (uint32_t o = 0; o + 1 < groups; ++o)
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
        if (c < a.hidden) store_part(a, c, dw[i]);
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

// How the gradient is laid over the SMs, one CTA each: in as many groups as there are threads for (registers: 896, or 512 of FP32, whose pieces are twice as
// large), as many CTAs as finish together. (With registers for 1024 threads some go to memory: 117 us where 896 took 84.)
//
// In registers or in shared memory goes by the groups that each has threads for. Two or more in registers: these. One: of BF16 registers all the same (their next token needs no
// barrier), but not where shared memory holds two and the walks are long; of FP32 shared memory. In registers / in shared memory, us:
//   BF16, tokens     3616 channels       4096           4608           5120           6144           6656          7168
//    1500                           13.7 / 16.0    14.2 / 17.1    14.9 / 17.7    16.2 / 19.6    17.0 / 21.1    17.6 / 21.6
//    3000          21.2 / 22.2      21.7 / 23.0    22.9 / 28.0    23.7 / 28.5    26.2 / 31.3    28.1 / 34.1
//    4500                           29.8 / 30.3
//    6000          38.8 / 36.2      40.5 / 37.1
//    8192          54.5 / 45.6      58.2 / 46.6    61.8 / 63.6    65.1 / 63.9    72.3 / 70.4    76.0 / 78.0    79.3 / 79.9
//   16384         108.6 / 83.5     112.3 / 84.5   118.1 / 119.3  124.8 / 119.6  138.5 / 133.0  146.6 / 147.3  152.8 / 154.0
//   FP32, tokens     2080 channels       2560           4096
//    1000          12.0 / 9.8       13.8 / 11.2    13.8 / 15.8
//    4500          38.3 / 25.8      45.9 / 29.7    46.9 / 47.2
//    8192          64.7 / 39.8      76.5 / 49.3    82.3 / 77.7
// Two in registers, 8192 tokens: BF16 2048 22.9 / 27.2, 3584 38.6 / 41.3; FP32 2048 42.0 / 40.9, 1531 tokens 11.6 / 12.3.
constexpr uint32_t kLongWalk = 32;                            // turns of one group on every SM
struct NormGradShape { uint32_t threads, groups, pieces, stages, parts, smem; };   // stages: 0 in registers
static NormGradShape norm_grad_shape(uint32_t tokens, uint32_t hidden, bool fp32, uint32_t channel_bytes) {
    NormGradShape s{};
    const uint32_t one = norm_threads(hidden, 1), in_registers = (fp32 ? 512 : 896) / one, in_smem = kLongThreads / one;
    const bool whole = in_registers > 1 || (in_registers == 1 && !fp32 && (in_smem == 1 || tokens <= kLongWalk * 148));
    const uint32_t most = !whole ? kLongThreads : fp32 ? 512 : 896, token = hidden * channel_bytes;
    s.pieces = one <= kLongThreads ? 1 : 2;
    s.threads = norm_threads(hidden, s.pieces);
    s.groups = most / s.threads < kMostGroups ? most / s.threads : kMostGroups;
    while (s.groups > 1 && (s.groups - 1) * 148 >= tokens) --s.groups;
    const uint32_t others = (s.groups - 1) * s.threads * s.pieces * 32;
    if (!whole) {
        const uint32_t fit = kLongSmem / (token * s.groups);
        s.stages = fit < kLongMostStages ? fit : kLongMostStages;
    }
    s.smem = s.stages * s.groups * token > others ? s.stages * s.groups * token : others;
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
// Adds to dg_device_status what these kernels recorded, and forgets it. (The device has been waited for.)
namespace dg {
int take_norm_status(int32_t* status) {
    int32_t code = 0;
    const int32_t none = 0;
    DG_CHECK_CUDA(cudaMemcpyFromSymbol(&code, g_norm_status, sizeof(code)));
    if (code != 0) DG_CHECK_CUDA(cudaMemcpyToSymbol(g_norm_status, &none, sizeof(none)));
    if (*status == 0) *status = code;
    return DG_OK;
}
}  // namespace dg
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
    // In registers / by bulk copies, us of 8192 tokens: BF16 512 10.3 / 11.5, 1024 16.1 / 17.5, 1536 27.1 / 24.2, 2048 32.8 / 29.6, 2560 45.8 / 36.5, 3584 49.8 / 50.9, 4096 53.2 / 53.1,
    // 7168 89.1 / 92.6; FP32 1024 23.6 / 24.0, 2048 52.6 / 46.7, 7168 171 / 158, 8192 187 / 159. Few turns do not pay for the copies' start. Between 1024 and 2000 tokens it goes by
    // how the last turn is filled: BF16 x 2048 of 1024 tokens 6.0 / 4.8, 1300 6.2 / 7.6, 1700 7.9 / 7.8, 2300 10.7 / 8.1; x 2560 of 600 to 1100 about the same, 1300 9.1 / 7.5, 2300 14.3 /
    // 11.7; FP32 x 2048 of 1100 9.5 / 7.3, 1300 9.6 / 10.1, 1700 12.5 / 11.2; x 7168 of 1300 26.4 / 28.5, 2300 45.2 / 45.8. With two pieces a thread, and up to 1024 channels, registers
    // win with any number of tokens: BF16 x 4096 of 1300 8.9 / 12.0, 3000 18.9 / 25.7, 16384 101.8 / 100.7; x 1024 of 1700 4.8 / 5.3, 6000 12.5 / 14.0, 16384 31.0 / 33.8.
    // In registers two pieces a thread and two CTAs on an SM for long rows of BF16 (7168 89 us against 100 with one piece) but for few tokens (1 / 128 x 7168 2.4 / 3.0 us
    // with one piece, 2.7 / 3.2 with two).
    const uint32_t one = norm_threads(hidden, 1);
    const bool two = !is_fp32 && one > 448 && one <= 896 && tokens > 148;
    void* params[] = {&a};
    if (one <= 1024 && (hidden <= 1024 || tokens <= 1024 || two)) {
        const uint32_t threads = two ? norm_threads(hidden, 2) : one, resident = 896 / threads < 1 ? 1 : 896 / threads > 16 ? 16 : 896 / threads;
        return launch_overlapped(two ? (const void*)rms_norm_fp8_kernel<__nv_bfloat16, 2, 448, 2> : is_fp32 ? (const void*)rms_norm_fp8_kernel<float, 1, 1024, 1>
                                                                                              : (const void*)rms_norm_fp8_kernel<__nv_bfloat16, 1, 1024, 1>,
                                 dim3(tokens < 148 * resident ? tokens : 148 * resident), dim3(threads), params, static_cast<cudaStream_t>(stream));
    }
    // (two pieces a thread of BF16: 7168 104 us with one)
    const uint32_t pieces = is_fp32 && one <= kLongThreads ? 1 : 2, token = hidden * (uint32_t)(residual ? 2 * es : es);
    a.threads = norm_threads(hidden, pieces);
    a.groups = kLongThreads / a.threads < kMostGroups ? kLongThreads / a.threads : kMostGroups;
    while (a.groups > 1 && (a.groups - 1) * 148 >= tokens) --a.groups;
    const uint32_t fit = kLongSmem / (token * a.groups), ctas = (tokens + a.groups - 1) / a.groups;
    a.stages = fit < kLongMostStages ? fit : kLongMostStages;
    const void* fn = !is_fp32 ? (const void*)rms_norm_fp8_long_kernel<__nv_bfloat16, 2> : pieces == 1 ? (const void*)rms_norm_fp8_long_kernel<float, 1>
                                                                                                      : (const void*)rms_norm_fp8_long_kernel<float, 2>;
    DG_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLongSmem));
    return launch_overlapped(fn, dim3(ctas < 148 ? ctas : 148), dim3(a.groups * a.threads), params, static_cast<cudaStream_t>(stream), a.groups * a.stages * token);
}

extern "C" uint64_t dg_rms_norm_grad_scratch_bytes(uint32_t tokens, uint32_t hidden) {
    if (hidden == 0) return 0;
    return (uint64_t)(tokens < 148 ? tokens : 148) * hidden * 4;
}

template <typename T, typename G>
static const void* norm_grad_kernel(const NormGradShape& s) {
    return s.stages == 0 ? (const void*)rms_norm_grad_kernel<T, G, sizeof(T) == 4 ? 512 : 896>
         : s.pieces == 1 ? (const void*)rms_norm_grad_long_kernel<T, G, 1> : (const void*)rms_norm_grad_long_kernel<T, G, 2>;
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
    const NormGradShape shape = norm_grad_shape(tokens, hidden, is_fp32, (uint32_t)((grad_h ? 2 * es : es) + (grad_is_fp32 ? 4 : 2)));
    a.groups = shape.groups; a.threads = shape.threads; a.stages = shape.stages;
    uint32_t parts = shape.parts;
    const void* fn = !is_fp32 ? norm_grad_kernel<__nv_bfloat16, __nv_bfloat16>(shape) : grad_is_fp32 ? norm_grad_kernel<float, float>(shape)
                                                                                            : norm_grad_kernel<float, __nv_bfloat16>(shape);
    if (shape.stages > 0) DG_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLongSmem));
    void* params[] = {&a};
    if (int rc = launch_overlapped(fn, dim3(parts), dim3(shape.groups * shape.threads), params, static_cast<cudaStream_t>(stream), shape.smem)) return rc;
    const float* from = a.partial;
    void* sum_params[] = {&from, &grad_weight, &parts, &hidden};
    return launch_overlapped((const void*)rms_norm_grad_sum_kernel, dim3(hidden / kSumChannels), dim3(kSumThreads), sum_params, static_cast<cudaStream_t>(stream));
}
