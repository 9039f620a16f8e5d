// A router's scores -> the experts of every token and their weights, and the gradient of the weights.
//
// Mathematics, per token with logits l and a bias b (0 where there is none): s = softmax(l) or 1 / (1 + e^-l); c = s + b; the score of a
// group of experts is the sum of its one or two largest c; of the `topk_groups` best groups the k largest c are chosen, ties to the
// lowest index; the weights are s, divided by their sum where that is asked for, times `scale`. An expert whose logit or bias is
// -inf is never chosen; where fewer than k are left the rest of the choices is -1 with the weight 0.
//
// Who is chosen is decided by c in 64 bits. FP32 scores come first: their error is bounded (score_error), and only where two of those that
// decide lie closer together than that, the warp does the token again with 64-bit scores. Without a bias the scores' order is that of the
// logits, which decide by themselves then.
//
// One warp a token, nothing shared between warps. A group of experts lies in 32 / num_groups lanes (rounded down to a power of two), so that a
// lane holds experts of one group only and a group that is not taken is dropped by its lanes. A choice is a maximum over the lanes and a
// minimum over the places that hold it: one instruction each for a whole warp (redux).
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kRouteThreads = 128, kAll = 0xffffffffu;
constexpr uint32_t kMostChoices = 32, kMostExperts = 1024, kMostGroups = 32;
constexpr float kLeastSum = 1e-20f;                           // under the weights' sum

struct RouteArgs {
    const uint8_t* logits; uint64_t stride;                   // bytes between rows
    const float* bias;
    void* idx; float* weights;                                // [tokens, topk]
    const float* grad_weights;
    uint8_t* grad_logits; uint64_t grad_stride;
    uint32_t tokens, experts, topk, groups, group_size, topk_groups, lanes_log2;
    uint32_t fp32, idx64, sigmoid, renormalize, best_two, by_logits;
    float scale;
};

template <typename T> __device__ __forceinline__ T warp_sum(T v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
// (NaN counts for nothing here)
__device__ __forceinline__ float warp_max(float v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}

__device__ __forceinline__ float logit_at(const RouteArgs& a, const uint8_t* row, uint32_t e) {
    return __uint_as_float(a.fp32 ? ld_global_u32(row + (uint64_t)e * 4) : (uint32_t)ld_global_u16(row + (uint64_t)e * 2) << 16);
}
__device__ __forceinline__ float bias_at(const RouteArgs& a, uint32_t e) { return a.bias ? __uint_as_float(ld_global_u32(a.bias + e)) : 0.0f; }

// The experts of a lane, and their logits (-inf behind the last).
struct Share { uint32_t first, step, end; };
template <uint32_t kItems>
__device__ __forceinline__ void load_logits(const RouteArgs& a, const uint8_t* row, const Share& of, float (&l)[kItems]) {
    if (a.fp32) {
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) {
            const uint32_t e = of.first + i * of.step;
            l[i] = e < of.end ? __uint_as_float(ld_global_u32(row + (uint64_t)e * 4)) : -CUDART_INF_F;
        }
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) {
            const uint32_t e = of.first + i * of.step;
            l[i] = e < of.end ? __uint_as_float((uint32_t)ld_global_u16(row + (uint64_t)e * 2) << 16) : -CUDART_INF_F;
        }
    }
}

// Largest logit and sum of e^(l - largest) of a softmax. (Where every expert is masked: 0 and 1, which makes every score 0.)
struct Softmax { float top, sum; };
template <uint32_t kItems>
__device__ __forceinline__ Softmax softmax_of(const float (&l)[kItems]) {
    Softmax m{-CUDART_INF_F, 0.0f};
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) m.top = fmaxf(m.top, l[i]);
    m.top = warp_max(m.top);
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) m.sum += expf(l[i] - m.top);
    m.sum = warp_sum(m.sum);
    // (a NaN beside masked experts stays one)
    if (m.top == -CUDART_INF_F) {
        bool bad = false;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) bad |= l[i] != l[i];
        m = __any_sync(kAll, bad) ? Softmax{CUDART_NAN_F, 1.0f} : Softmax{0.0f, 1.0f};
    }
    return m;
}
// (by e^-|l|, so that neither end is lost: scores near 0 keep their bits)
__device__ __forceinline__ float sigmoid_of(float l) {
    const float z = expf(-fabsf(l));
    return __fdiv_rn(l < 0.0f ? z : 1.0f, 1.0f + z);
}
__device__ __forceinline__ float score_of(bool sigmoid, const Softmax& m, float l) { return sigmoid ? sigmoid_of(l) : __fdiv_rn(expf(l - m.top), m.sum); }
// How far an FP32 score c = s + b can be from the exact one; `largest`: the largest s. Sigmoid: the exponential within 2 ulp (2^-22), half an ulp
// for the addition and for the division: s within 2^-21 of its value. Softmax: rounding l - top moves s by less than x e^-x 2^-24 < 2^-25 of the
// largest; the exponential 2 ulp; at most 64 + 5 additions of the sum, 2^-17.8; the division: under 2^-17 of the largest in all. The addition of b is
// within 2^-24 of c, its sum with another score of the group (whose errors the caller doubles) too.
__device__ __forceinline__ float score_error(bool sigmoid, float largest, float c) { return (sigmoid ? 0x1p-21f : 0x1p-17f) * largest + 0x1p-23f * fabsf(c); }

// Whole numbers in the order of the values: NaN above everything (as in torch.topk), 0 for what cannot be chosen.
template <typename T> struct Key;
template <> struct Key<float> {
    using type = uint32_t;
    static __device__ __forceinline__ type of(float v) {
        if (v != v) return 0xffffffffu;
        const uint32_t b = __float_as_uint(v + 0.0f);                     // (-0 is 0)
        return b & 0x80000000u ? ~b : b | 0x80000000u;
    }
    static __device__ __forceinline__ float back(type k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
    static __device__ __forceinline__ type largest(type k) { return __reduce_max_sync(kAll, k); }
};
template <> struct Key<double> {
    using type = uint64_t;
    static __device__ __forceinline__ type of(double v) {
        if (v != v) return ~0ull;
        const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
        return b >> 63 ? ~b : b | 1ull << 63;
    }
    static __device__ __forceinline__ type largest(type k) {
        const uint32_t high = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
        return (uint64_t)high << 32 | __reduce_max_sync(kAll, (uint32_t)(k >> 32) == high ? (uint32_t)k : 0u);
    }
};

// The choice of a token with scores of type T: the expert of choice `lane` (-1: none). Answers whether FP32 scores leave it open.
template <typename T, uint32_t kItems>
__device__ __forceinline__ bool choose(const RouteArgs& a, const uint8_t* row, const Share& of, const float (&l)[kItems], const Softmax& m, uint32_t lane,
                                       int32_t& chosen) {
    using K = typename Key<T>::type;
    constexpr bool kFast = sizeof(T) == 4;
    const bool sigmoid = a.sigmoid != 0, with_scores = !a.by_logits || (a.groups > 1 && a.best_two);
    T total = 1;
    if constexpr (!kFast) {
        if (!sigmoid && with_scores) {
            total = 0;
            #pragma unroll 1
            for (uint32_t i = 0; i < kItems; ++i) {
                const uint32_t e = of.first + i * of.step;
                if (e < of.end) total += exp((double)logit_at(a, row, e) - (double)m.top);
            }
            total = warp_sum(total);
        }
    }
    K key[kItems];
    T best = -CUDART_INF, second = -CUDART_INF;               // of the group's values in this lane
    bool nan = false;
    float largest = 0.0f;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) {
        const uint32_t e = of.first + i * of.step;
        key[i] = 0;
        if (e >= of.end || l[i] == -CUDART_INF_F) continue;
        const float b = bias_at(a, e);
        if (b == -CUDART_INF_F) continue;
        T c = (T)l[i];
        if (with_scores) {
            T s;
            if constexpr (kFast) s = score_of(sigmoid, m, l[i]);
            else s = sigmoid ? 1.0 / (1.0 + exp(-(double)l[i])) : exp((double)l[i] - (double)m.top) / total;
            largest = fmaxf(largest, (float)s);
            c = s + (T)b;
        }
        key[i] = Key<T>::of(a.by_logits ? (T)l[i] : c);
        nan |= c != c;
        if (c > best) { second = best; best = c; }
        else if (c > second) second = c;
    }
    bool open = false;
    if (kFast && with_scores) largest = warp_max(largest);
    if (a.groups > 1) {
        const uint32_t lanes = 1u << a.lanes_log2, group = lane >> a.lanes_log2;
        for (uint32_t o = lanes / 2; o > 0; o >>= 1) {
            const T b = __shfl_xor_sync(kAll, best, o), s = __shfl_xor_sync(kAll, second, o);
            nan |= __shfl_xor_sync(kAll, (int)nan, o) != 0;
            const T lower = best < b ? best : b;
            best = best < b ? b : best;
            second = second < s ? s : second;
            second = second < lower ? lower : second;
        }
        // (a group with a single expert that can be chosen counts that one alone)
        T score = a.best_two && second > (T)-CUDART_INF ? best + second : best;
        if (nan) score = (T)CUDART_NAN;
        const K mine = Key<T>::of(score);
        uint32_t ahead = 0, near = 0;
        for (uint32_t g = 0; g < a.groups; ++g) {
            const T other = __shfl_sync(kAll, score, g << a.lanes_log2);
            const K k = Key<T>::of(other);
            ahead += k > mine || (k == mine && g < group);
            if constexpr (kFast)
                if (with_scores && fabsf(other - score) <= 4.0f * score_error(sigmoid, largest, score)) near |= 1u << g;
        }
        const bool taken = group < a.groups && ahead < a.topk_groups;
        const uint32_t all_taken = __ballot_sync(kAll, taken);
        if (group >= a.groups) near = 0;
        for (; near != 0; near &= near - 1) open |= taken != ((all_taken >> ((__ffs(near) - 1) << a.lanes_log2) & 1u) != 0);
        if (!taken) {
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i) key[i] = 0;
        }
    }
    // One choice after the other; one more says whether the last of them is certain.
    K mine = 0;
    uint32_t place = 0;
    const auto find = [&]() {
        mine = 0;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i)
            if (key[i] > mine) { mine = key[i]; place = of.first + i * of.step; }
    };
    find();
    chosen = -1;
    const bool check = kFast && !a.by_logits;
    K before = 0;
    uint32_t expert_before = 0;
    for (uint32_t k = 0; k < a.topk + (check ? 1u : 0u); ++k) {
        const K top = Key<T>::largest(mine);
        if (top == 0) break;
        const uint32_t e = __reduce_min_sync(kAll, mine == top ? place : 0xffffffffu);
        if (lane == k && k < a.topk) chosen = (int32_t)e;
        if constexpr (kFast) {
            if (check && k > 0) {
                const float here = Key<T>::back(top), there = Key<T>::back(before);
                // (equal logits and biases make a tie in any number of bits)
                if (there - here <= 2.0f * score_error(sigmoid, largest, fmaxf(fabsf(here), fabsf(there))) &&
                    (logit_at(a, row, e) != logit_at(a, row, expert_before) || bias_at(a, e) != bias_at(a, expert_before))) open = true;
            }
            before = top;
            expert_before = e;
        }
        if (mine == top && place == e) {
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i)
                if (of.first + i * of.step == e) key[i] = 0;
            find();
        }
        __syncwarp();
    }
    return __any_sync(kAll, open);
}

template <uint32_t kItems>
__global__ void __launch_bounds__(kRouteThreads) moe_route_kernel(const RouteArgs a) {
    const uint32_t lane = threadIdx.x % 32, token = blockIdx.x * (kRouteThreads / 32) + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.tokens) return;
    const uint8_t* row = a.logits + (uint64_t)token * a.stride;
    const uint32_t group = lane >> a.lanes_log2;
    Share of{group * a.group_size + (lane & ((1u << a.lanes_log2) - 1)), 1u << a.lanes_log2, (group + 1) * a.group_size};
    if (group >= a.groups) of.first = of.end = 0;
    float l[kItems];
    load_logits(a, row, of, l);
    Softmax m{0.0f, 1.0f};
    if (!a.sigmoid) m = softmax_of(l);
    int32_t chosen;
    if (choose<float>(a, row, of, l, m, lane, chosen)) choose<double>(a, row, of, l, m, lane, chosen);
    float w = 0.0f;
    if (chosen >= 0) w = score_of(a.sigmoid != 0, m, logit_at(a, row, (uint32_t)chosen));
    if (a.renormalize) w = __fdiv_rn(w, fmaxf(warp_sum(w), kLeastSum));
    if (lane < a.topk) {
        static_cast<int32_t*>(a.idx)[(uint64_t)token * a.topk + lane] = chosen;
        a.weights[(uint64_t)token * a.topk + lane] = w * a.scale;
    }
}

// The gradient: with A_j from choice j (below), dl_e = sum over the choices of e of A_j, and for a softmax that is not renormalised
// - p_e sum(g p) on every expert. Choices of the same expert add up in their order. Bound by HBM for many tokens: the logits are read once and
// their gradient is written once.
template <uint32_t kItems>
__global__ void __launch_bounds__(kRouteThreads) moe_route_grad_kernel(const RouteArgs a) {
    const uint32_t lane = threadIdx.x % 32, token = blockIdx.x * (kRouteThreads / 32) + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.tokens) return;
    const uint8_t* row = a.logits + (uint64_t)token * a.stride;
    const Share of{lane, 32, a.experts};
    float l[kItems];
    load_logits(a, row, of, l);
    int64_t idx = -1;
    float g = 0.0f;
    if (lane < a.topk) {
        const uint64_t at = (uint64_t)token * a.topk + lane;
        idx = a.idx64 ? *(static_cast<const volatile int64_t*>(a.idx) + at) : (int64_t)(int32_t)ld_global_u32(static_cast<const int32_t*>(a.idx) + at);
        if (idx < 0 || idx >= a.experts) idx = -1;
        if (idx >= 0) g = __uint_as_float(ld_global_u32(a.grad_weights + at)) * a.scale;
    }
    const bool sigmoid = a.sigmoid != 0;
    Softmax m{0.0f, 1.0f};
    if (!sigmoid) m = softmax_of(l);
    const float mine = idx >= 0 ? logit_at(a, row, (uint32_t)idx) : 0.0f;
    const float s = idx >= 0 ? score_of(sigmoid, m, mine) : 0.0f;
    // the slope of log s (for a softmax the other part of it is the sum over all experts): 1 - s would lose its bits where s is near 1
    const float slope = sigmoid ? sigmoid_of(-mine) : 1.0f;
    float from_choice, from_all = 0.0f;
    if (a.renormalize) {
        const float sum = warp_sum(s), q = __fdiv_rn(s, fmaxf(sum, kLeastSum)), dot = warp_sum(idx >= 0 ? g * q : 0.0f);
        from_choice = q * (sum > kLeastSum ? g - dot : g) * slope;
    } else {
        from_choice = g * s * slope;
        if (!sigmoid) from_all = warp_sum(idx >= 0 ? g * s : 0.0f);
    }
    float d[kItems];
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) d[i] = sigmoid || a.renormalize ? 0.0f : -from_all * score_of(false, m, l[i]);
    for (uint32_t j = 0; j < a.topk; ++j) {
        const int32_t e = __shfl_sync(kAll, (int32_t)idx, j);
        const float add = __shfl_sync(kAll, from_choice, j);
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i)
            if ((int32_t)(lane + i * 32) == e) d[i] += add;
    }
    uint8_t* out = a.grad_logits + (uint64_t)token * a.grad_stride;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) {
        const uint32_t e = lane + i * 32;
        if (e >= a.experts) continue;
        if (a.fp32) reinterpret_cast<float*>(out)[e] = d[i];
        else reinterpret_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(d[i]);
    }
}

}  // namespace dg

using namespace dg;

template <template <uint32_t> class Pick> static const void* for_items(uint32_t items) {
    return items <= 1 ? Pick<1>::fn() : items <= 2 ? Pick<2>::fn() : items <= 4 ? Pick<4>::fn() : items <= 8 ? Pick<8>::fn() : items <= 16 ? Pick<16>::fn()
           : items <= 32 ? Pick<32>::fn() : Pick<64>::fn();
}
template <uint32_t kItems> struct Forward { static const void* fn() { return (const void*)moe_route_kernel<kItems>; } };
// (a lane holds every 32nd of at most 1024 experts)
template <uint32_t kItems> struct Backward { static const void* fn() { return (const void*)moe_route_grad_kernel<(kItems < 32 ? kItems : 32)>; } };

static int route_args(RouteArgs& a, const void* logits, int is_fp32, uint64_t stride, uint32_t tokens, uint32_t experts, uint32_t topk, int sigmoid,
                      int renormalize, float scale) {
    DG_CHECK_ARG(experts > 0 && experts <= kMostExperts, "moe_route: the number of experts must be between 1 and %u", kMostExperts);
    DG_CHECK_ARG(topk > 0 && topk <= kMostChoices && topk <= experts, "moe_route: topk must be between 1 and %u, and at most the number of experts", kMostChoices);
    DG_CHECK_ARG(tokens <= 0x7fffffffu, "moe_route: too many tokens");
    DG_CHECK_ARG(tokens == 0 || (logits != nullptr && reinterpret_cast<uintptr_t>(logits) % (is_fp32 ? 4 : 2) == 0), "moe_route: logits must be an aligned pointer");
    a.logits = static_cast<const uint8_t*>(logits); a.stride = stride * (is_fp32 ? 4 : 2);
    a.fp32 = is_fp32 ? 1u : 0u;
    a.tokens = tokens; a.experts = experts; a.topk = topk;
    a.sigmoid = sigmoid ? 1u : 0u; a.renormalize = renormalize ? 1u : 0u;
    a.scale = scale;
    return DG_OK;
}

extern "C" int dg_moe_route_launch(const void* logits, int is_fp32, uint64_t stride, uint32_t tokens, uint32_t experts, uint32_t topk, int sigmoid,
                                   const float* bias, uint32_t num_groups, uint32_t topk_groups, uint32_t group_best, int renormalize, float scale,
                                   int32_t* topk_idx, float* topk_weights, void* stream) {
    RouteArgs a{};
    if (int rc = route_args(a, logits, is_fp32, stride, tokens, experts, topk, sigmoid, renormalize, scale)) return rc;
    DG_CHECK_ARG(num_groups > 0 && num_groups <= kMostGroups && experts % num_groups == 0,
                 "moe_route: the number of groups must be between 1 and %u and divide the number of experts", kMostGroups);
    DG_CHECK_ARG(topk_groups > 0 && topk_groups <= num_groups, "moe_route: topk_groups must be between 1 and the number of groups");
    DG_CHECK_ARG(group_best == 1 || group_best == 2, "moe_route: group_best must be 1 or 2");
    DG_CHECK_ARG(topk <= experts / num_groups * topk_groups, "moe_route: the groups that are taken hold fewer experts than topk");
    if (tokens == 0) return DG_OK;
    DG_CHECK_ARG(topk_idx != nullptr && topk_weights != nullptr, "moe_route: null pointer");
    // (with all groups taken there is nothing to decide between them)
    if (topk_groups == num_groups) num_groups = topk_groups = 1;
    a.bias = bias; a.idx = topk_idx; a.weights = topk_weights;
    a.groups = num_groups; a.group_size = experts / num_groups; a.topk_groups = topk_groups;
    a.best_two = group_best == 2; a.by_logits = bias == nullptr;
    while ((2u << a.lanes_log2) * num_groups <= 32) ++a.lanes_log2;
    const uint32_t items = (a.group_size + (1u << a.lanes_log2) - 1) >> a.lanes_log2;
    void* params[] = {&a};
    return launch_overlapped(for_items<Forward>(items), dim3((tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32)), dim3(kRouteThreads), params,
                             static_cast<cudaStream_t>(stream));
}

extern "C" int dg_moe_route_grad_launch(const float* grad_weights, const void* logits, int is_fp32, uint64_t stride, uint32_t tokens, uint32_t experts,
                                        const void* topk_idx, int idx_is_int64, uint32_t topk, int sigmoid, int renormalize, float scale,
                                        void* grad_logits, uint64_t grad_stride, void* stream) {
    RouteArgs a{};
    if (int rc = route_args(a, logits, is_fp32, stride, tokens, experts, topk, sigmoid, renormalize, scale)) return rc;
    if (tokens == 0) return DG_OK;
    DG_CHECK_ARG(grad_weights != nullptr && topk_idx != nullptr && grad_logits != nullptr, "moe_route_grad: null pointer");
    DG_CHECK_ARG(reinterpret_cast<uintptr_t>(grad_logits) % (is_fp32 ? 4 : 2) == 0, "moe_route_grad: grad_logits must be an aligned pointer");
    a.grad_weights = grad_weights; a.idx = const_cast<void*>(topk_idx); a.idx64 = idx_is_int64 ? 1u : 0u;
    a.grad_logits = static_cast<uint8_t*>(grad_logits); a.grad_stride = grad_stride * (is_fp32 ? 4 : 2);
    void* params[] = {&a};
    return launch_overlapped(for_items<Backward>((experts + 31) / 32), dim3((tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32)), dim3(kRouteThreads), params,
                             static_cast<cudaStream_t>(stream));
}
