// A router's scores -> the experts of every token and their weights, and the gradient of the weights.
//
// Mathematics, per token with logits l and a bias b (0 where there is none): s = softmax(l) or 1 / (1 + e^-l); c = s + b; the score of a
// group of experts is the sum of its one or two largest c; of the `topk_groups` best groups the k largest c are chosen, ties to the
// lowest index; the weights are s, divided by their sum where that is asked for, times `scale`. An expert whose logit or bias is
// -inf is never chosen; where fewer than k are left the rest of the choices is -1 with the weight 0.
//
// Who is chosen is decided by c in 64 bits. A whole number that stands for c within a bound comes first (quick_choice): 21 to 23 bits of its distance from
// the token's largest, above the expert's index, so that a choice is one maximum over the warp (redux) and a lane's next candidate one fused add-and-maximum
// for each expert it holds. Only where two of those that decide lie closer together than the bound, the warp does the token again with 64-bit
// scores (exact_choice), or, where it is known who is chosen and only their order is not, the chosen ones' alone (exact_order). Without a bias the order of the
// scores is that of the logits, which stand for them then.
//
// One warp a token, nothing shared between warps. A group of experts lies in 32 / num_groups lanes (rounded down to a power of two), so that a
// lane holds experts of one group only and a group that is not taken is dropped by its lanes.
//
// Bound by instructions, about 800 of a warp for a token of 256 experts and 8 choices: 16384 tokens (sigmoid, bias, 4 of 8 groups, FP32) 17.1 to 19.9 us by
// the input, where the bytes alone take 2.7; without a bias 19.7, of a softmax without groups 13.4 (BF16, whose logits are often equal, 20.3); 128 tokens 2.6 us, launch and latency. (A maximum of scores and then one of the indices that hold it took 43.6, whole-number keys 24 to 26; all
// 64-bit scores where only the order is open 24 where those of the chosen take 19.) The gradient, 16384 x 256 of a softmax that is not renormalised, 6.5 us, 5.4 TB/s.
// (Every form has a frame of 136 bytes for the arguments of what is out of line; 64 experts a lane, one at a time, spill 76 bytes besides.)
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
    uint32_t tokens, experts, topk, groups, group_size, topk_groups, lanes_log2, index_bits;
    uint32_t fp32, idx64, sigmoid, renormalize, best_two, by_logits;
    uint32_t aligned, bias_aligned;                           // four neighbours can be read (and written) at once
    float scale;
};

template <typename T> __device__ __forceinline__ T warp_sum(T v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
// (NaN counts for nothing here)
__device__ __forceinline__ float redux_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}
__device__ __forceinline__ float redux_min(float v) {
    float m;
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

__device__ __forceinline__ float logit_at(const RouteArgs& a, const uint8_t* row, uint32_t e) {
    return __uint_as_float(a.fp32 ? ld_global_u32(row + (uint64_t)e * 4) : (uint32_t)ld_global_u16(row + (uint64_t)e * 2) << 16);
}
__device__ __forceinline__ float bias_at(const RouteArgs& a, uint32_t e) { return a.bias ? __uint_as_float(ld_global_u32(a.bias + e)) : 0.0f; }

// The experts of a lane, below `end`: runs of kVec neighbours, `step` apart, from `first` on; and their logits (-inf behind the last). Runs of four, all whole, wherever
// the number of experts allows it, whether they can be read at once or not: a token's sums do not depend on where it lies.
template <uint32_t kVec> struct Share {
    uint32_t first, step, end;
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return first + i / kVec * step + i % kVec; }
};
template <uint32_t kVec, uint32_t kItems>
__device__ __forceinline__ void load_logits(const RouteArgs& a, const uint8_t* row, const Share<kVec>& of, float (&l)[kItems]) {
    #pragma unroll
    for (uint32_t i = 0; i < kItems; i += kVec) {
        const uint32_t e = of.at(i);
        #pragma unroll
        for (uint32_t j = 0; j < kVec; ++j) l[i + j] = -CUDART_INF_F;
        if (e >= of.end) continue;
        if (kVec == 4 && a.aligned) {
            if (a.fp32) {
                const uint4 q = ld_global_v4(row + (uint64_t)e * 4);
                l[i] = __uint_as_float(q.x);
                if constexpr (kVec == 4) { l[i + 1] = __uint_as_float(q.y); l[i + 2] = __uint_as_float(q.z); l[i + 3] = __uint_as_float(q.w); }
            } else {
                const uint2 q = ld_global_v2(row + (uint64_t)e * 2);
                l[i] = bf16_lo(q.x);
                if constexpr (kVec == 4) { l[i + 1] = bf16_hi(q.x); l[i + 2] = bf16_lo(q.y); l[i + 3] = bf16_hi(q.y); }
            }
        } else {
            #pragma unroll
            for (uint32_t j = 0; j < kVec; ++j) l[i + j] = logit_at(a, row, e + j);
        }
    }
}

// Largest logit and sum of e^(l - largest) of a softmax, which are left in `z`. (Where every expert is masked: 0 and 1, which makes every score 0.)
struct Softmax { float top, sum; };
template <uint32_t kItems>
__device__ __forceinline__ Softmax softmax_of(const float (&l)[kItems], float (&z)[kItems]) {
    Softmax m{-CUDART_INF_F, 0.0f};
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) m.top = fmaxf(m.top, l[i]);
    m.top = redux_max(m.top);
    if (m.top == -CUDART_INF_F) m.top = 0.0f;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) {
        z[i] = fast_exp2((l[i] - m.top) * kLog2E);
        m.sum += z[i];
    }
    m.sum = warp_sum(m.sum);
    if (m.sum == 0.0f) m.sum = 1.0f;
    return m;
}
// (by e^-|l|, so that neither end is lost: scores near 0 keep their bits)
__device__ __forceinline__ float sigmoid_of(float l) {
    const float z = expf(-fabsf(l));
    return __fdiv_rn(l < 0.0f ? z : 1.0f, 1.0f + z);
}
__device__ __forceinline__ float score_of(bool sigmoid, const Softmax& m, float l) { return sigmoid ? sigmoid_of(l) : __fdiv_rn(expf(l - m.top), m.sum); }
// (a NaN stays one)
__device__ __forceinline__ float divisor_of(float sum) { return sum < kLeastSum ? kLeastSum : sum; }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// (NaN if one of them is)
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The choice of a token, the expert of choice `lane` in `chosen` (-1: none; the one behind the last in lane topk), by whole numbers that stand for c; answers
// whether that decides it, or leaves open the order of these only, or who they are. kScores: scores are looked at (there is a bias, or groups are
// compared by sums); else the logits are c.
//
// How far the c here can be from the exact one. Sigmoid: the product with log2(e) is rounded by 2^-24 of it and the exponential is within 2^-22 of its
// value, which moves s by s (1 - s) (|l| + 4) 2^-24 < 1.3 x 2^-24; the addition and the reciprocal by 2^-24 and 2^-23 of s: 4.3 x 2^-24 in all. Softmax: l - top times log2(e) is within
// 2^-23 of its value x, the exponential 2 ulp more, which moves s by x e^-x 2^-23 + 2^-22 < 2^-21.5 of the largest; the sum likewise, and by
// at most 64 + 5 additions, 2^-17.8: under 2^-17 of the largest in all. The addition of b and the difference from the largest are within 2^-24 of their
// values, and so is the sum of two scores: half that of a group is within the error of a score + 2^-24 (|best| + |second|), however small the sum itself.
enum class Choice { kDecided, kOrderOpen, kOpen };
template <uint32_t kVec, uint32_t kItems, bool kScores>
__device__ __forceinline__ Choice quick_choice(const RouteArgs& a, const uint8_t* row, const Share<kVec>& of, const float (&l)[kItems], const Softmax& m, const float (&z)[kItems], uint32_t lane,
                                             int32_t& chosen) {
    float c[kItems], error = 0.0f;
    bool open = false;
    if constexpr (kScores) {
        float b[kItems] = {};
        if (a.bias) {
            #pragma unroll
            for (uint32_t i = 0; i < kItems; i += kVec) {
                const uint32_t e = of.at(i);
                if (e >= of.end) continue;
                if (kVec == 4 && a.bias_aligned) {
                    const uint4 q = ld_global_v4(a.bias + e);
                    b[i] = __uint_as_float(q.x);
                    if constexpr (kVec == 4) { b[i + 1] = __uint_as_float(q.y); b[i + 2] = __uint_as_float(q.z); b[i + 3] = __uint_as_float(q.w); }
                } else {
                    #pragma unroll
                    for (uint32_t j = 0; j < kVec; ++j) b[i + j] = __uint_as_float(ld_global_u32(a.bias + e + j));
                }
            }
        }
        if (a.sigmoid) {
            error = 0x1.2p-22f;
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i) c[i] = fast_reciprocal(1.0f + fast_exp2(-kLog2E * l[i]));
        } else {
            const float inverse = fast_reciprocal(m.sum);
            float largest = 0.0f;
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i) {
                c[i] = z[i] * inverse;
                largest = fmaxf(largest, c[i]);
            }
            error = 0x1p-17f * redux_max(largest);
        }
        // (-inf where the expert cannot be chosen, whichever of the two says so)
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) c[i] = l[i] == -CUDART_INF_F ? -CUDART_INF_F : c[i] + b[i];
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) c[i] = l[i];
    }
    float top;
    if (a.groups > 1) {
        const uint32_t lanes = 1u << a.lanes_log2, group = lane >> a.lanes_log2;
        // the two largest of the group's values, in pairs
        float best = fmaxf(c[0], c[1]), second = fminf(c[0], c[1]), nan = max3_nan(c[0], c[1], c[1]);
        #pragma unroll
        for (uint32_t i = 2; i < kItems; i += 2) {
            const float high = fmaxf(c[i], c[i + 1]), low = fminf(c[i], c[i + 1]);
            second = max3(second, low, fminf(best, high));
            best = fmaxf(best, high);
            nan = max3_nan(nan, c[i], c[i + 1]);
        }
        open |= nan != nan;
        for (uint32_t o = lanes / 2; o > 0; o >>= 1) {
            const float b = __shfl_xor_sync(kAll, best, o), s = __shfl_xor_sync(kAll, second, o);
            second = max3(second, s, fminf(best, b));
            best = fmaxf(best, b);
        }
        // (a group with a single expert that can be chosen counts that one alone)
        // Half the sum: the largest biases there are do not leave the range.
        const bool two = a.best_two && second > -CUDART_INF_F;
        const float score = two ? fmaf(0.5f, second, 0.5f * best) : a.best_two ? 0.5f * best : best;
        // The groups in their order, ties to the lowest: all lanes of a group hold its score.
        float left = group < a.groups ? score : -CUDART_INF_F;
        bool taken = false;
        for (uint32_t k = 0; k < a.topk_groups; ++k) {
            const float last = redux_max(left);
            if (last == -CUDART_INF_F) break;
            const uint32_t first = __ffs(__ballot_sync(kAll, left == last)) - 1;
            if (group == first >> a.lanes_log2) { taken = true; left = -CUDART_INF_F; }
        }
        // The groups that are taken stand for those of 64 bits where the least that one of them can be is above the most that another one can (1.5 x 2^-23 instead
        // of 2^-24: these sums' own rounding). Scores that are logits are exact.
        if (kScores) {
            const float slack = error + 0x1.8p-23f * fabsf(best) + (two ? 0x1.8p-23f * fabsf(second) : 0.0f);
            const float least = redux_min(taken ? score - slack : CUDART_INF_F), most = redux_max(taken || best == -CUDART_INF_F ? -CUDART_INF_F : score + slack);
            open |= most > -CUDART_INF_F && least <= most;
        }
        if (!taken) {
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i) c[i] = -CUDART_INF_F;
        }
    }
    if (kScores && a.by_logits) {
        error = 0.0f;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) c[i] = c[i] == -CUDART_INF_F ? -CUDART_INF_F : l[i];
    }
    // Distances from the largest in units of a range that ends 2 below it (of logits: at the smallest, or 32 below): what lies further down is not told apart.
    top = max3_nan(c[0], c[1], c[1]);
    #pragma unroll
    for (uint32_t i = 2; i < kItems; i += 2) top = max3_nan(top, c[i], c[i + 1]);
    open |= top != top;
    top = redux_max(top);
    const uint32_t units = (1u << (31 - a.index_bits < 23 ? 31 - a.index_bits : 23)) - 32;
    float range = 2.0f;
    if (!kScores || a.by_logits) {
        float bottom = CUDART_INF_F;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i)
            if (c[i] > -CUDART_INF_F) bottom = fminf(bottom, c[i]);
        range = fmaxf(fminf(top - redux_min(bottom), 32.0f), 0x1p-60f);
    }
    chosen = -1;
    if (top == -CUDART_INF_F) return __any_sync(kAll, open) ? Choice::kOpen : Choice::kDecided;    // (nothing can be chosen, unless by NaN)
    open |= top == CUDART_INF_F;
    const float per_unit = __fdividef((float)units, range), offset = (float)(units + 16);
    const uint32_t mask = (1u << a.index_bits) - 1, code = mask - of.first;
    uint32_t key[kItems], mine = 0;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) {
        // (the conversion gives 0 for what is below the range, -inf and NaN)
        const uint32_t field = __float2uint_rn(fmaf(c[i] - top, per_unit, offset));
        key[i] = (field << a.index_bits) + ((code - (of.at(i) - of.first)) & mask);
        mine = max(mine, key[i]);
    }
    uint32_t held = 0xffffffffu;
    for (uint32_t k = 0; k < a.topk; ++k) {
        const uint32_t m1 = __reduce_max_sync(kAll, mine);
        if (lane == k) held = m1;
        // the largest below it: key - m1 wraps around, and the nearest below has the largest difference
        uint32_t next = 0x80000000u;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) next = __viaddmax_u32(key[i], 0u - m1, next);
        if (mine == m1) mine = next == 0x80000000u ? 0u : next + m1;
    }
    const uint32_t behind = __reduce_max_sync(kAll, mine);
    if (lane == a.topk) held = behind;
    chosen = lane <= a.topk && held >> a.index_bits != 0 ? (int32_t)(mask - (held & mask)) : -1;
    // (below the range, or nothing that can be chosen)
    if (lane < a.topk) open |= held >> a.index_bits == 0;
    // Are neighbours of the order apart by more than their errors, or equal because their logits and biases are? The last choice's neighbour is the one that
    // was not taken; where these two are equal or their order is open, its own neighbour might stand between them.
    uint32_t after = __shfl_down_sync(kAll, held, 1);
    if (lane == a.topk - 1) after = behind;
    const float bound = 2.0f * (error + 0x1p-23f * (fabsf(top) + range)) * per_unit + 3.0f;
    const auto near = [&](uint32_t k, uint32_t below) { return (float)((k >> a.index_bits) - (below >> a.index_bits)) <= bound; };
    bool equal = false, order_open = false;
    if (lane < a.topk && near(held, after)) {
        // (only keys above 0 units stand for an expert)
        if (held >> a.index_bits != 0 && after >> a.index_bits != 0) {
            const uint32_t e = mask - (after & mask);
            equal = logit_at(a, row, (uint32_t)chosen) == logit_at(a, row, e) && bias_at(a, (uint32_t)chosen) == bias_at(a, e);
            order_open = !equal;
        } else {
            open = true;
        }
    }
    if (__any_sync(kAll, order_open || (equal && lane == a.topk - 1))) {
        uint32_t next = 0;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i) next = max(next, key[i] < behind ? key[i] : 0u);
        open |= near(behind, __reduce_max_sync(kAll, next));
    }
    return __any_sync(kAll, open) ? Choice::kOpen : __any_sync(kAll, order_open) ? Choice::kOrderOpen : Choice::kDecided;
}

// The order of the choices and the one behind them, where that alone is open: lane j <= topk knows one of them, and its score in 64 bits (a sigmoid's, which
// needs no sum over the others) takes its place.
__device__ __noinline__ int32_t exact_order(const RouteArgs& a, const uint8_t* row, int32_t mine, uint32_t lane) {
    double c = -CUDART_INF;
    if (mine >= 0) {
        const double l = logit_at(a, row, (uint32_t)mine);
        c = a.by_logits ? l : 1.0 / (1.0 + exp(-l)) + bias_at(a, (uint32_t)mine);
    }
    uint32_t place = 0;
    for (uint32_t k = 0; k <= a.topk; ++k) {
        const double other = __shfl_sync(kAll, c, k);
        const int32_t e = __shfl_sync(kAll, mine, k);
        place += other > c || (other == c && e < mine);
    }
    int32_t chosen = -1;
    for (uint32_t k = 0; k <= a.topk; ++k) {
        const int32_t e = __shfl_sync(kAll, mine, k);
        if (__shfl_sync(kAll, place, k) == lane) chosen = e;
    }
    return chosen;
}

// The same with scores of 64 bits. In the order of whole numbers: NaN above everything (as in torch.topk), 0 for what cannot be chosen.
__device__ __forceinline__ uint64_t key_of(double v) {
    if (v != v) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);           // (-0 is 0)
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint64_t largest_key(uint64_t k) {
    const uint32_t high = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
    return (uint64_t)high << 32 | __reduce_max_sync(kAll, (uint32_t)(k >> 32) == high ? (uint32_t)k : 0u);
}
// (out of line: few tokens come here, and its registers would be everybody's)
template <uint32_t kVec, uint32_t kItems>
__device__ __noinline__ int32_t exact_choice(const RouteArgs& a, const uint8_t* row, const Share<kVec> of, float softmax_top, uint32_t lane) {
    const bool sigmoid = a.sigmoid != 0;
    double total = 1;
    if (!sigmoid) {
        total = 0;
        #pragma unroll 1
        for (uint32_t i = 0; i < kItems; ++i)
            if (of.at(i) < of.end) total += exp((double)logit_at(a, row, of.at(i)) - (double)softmax_top);
        total = warp_sum(total);
    }
    uint64_t key[kItems];
    double best = -CUDART_INF, second = -CUDART_INF;
    bool nan = false;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; ++i) {
        const uint32_t e = of.at(i);
        key[i] = 0;
        if (e >= of.end) continue;
        const double l = logit_at(a, row, e), b = bias_at(a, e);
        if (l == -CUDART_INF || b == -CUDART_INF) continue;
        double c = l;
        if (!a.by_logits || a.best_two) c = (sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - (double)softmax_top) / total) + b;
        key[i] = key_of(a.by_logits ? l : c);
        nan |= c != c;
        if (c > best) { second = best; best = c; }
        else if (c > second) second = c;
    }
    if (a.groups > 1) {
        const uint32_t lanes = 1u << a.lanes_log2, group = lane >> a.lanes_log2;
        for (uint32_t o = lanes / 2; o > 0; o >>= 1) {
            const double b = __shfl_xor_sync(kAll, best, o), s = __shfl_xor_sync(kAll, second, o);
            nan |= __shfl_xor_sync(kAll, (int)nan, o) != 0;
            const double lower = best < b ? best : b;
            best = best < b ? b : best;
            second = second < s ? s : second;
            second = second < lower ? lower : second;
        }
        const uint64_t mine = key_of(nan ? CUDART_NAN : a.best_two && second > -CUDART_INF ? best + second : best);
        uint32_t ahead = 0;
        for (uint32_t g = 0; g < a.groups; ++g) {
            const uint64_t k = __shfl_sync(kAll, mine, g << a.lanes_log2);
            ahead += k > mine || (k == mine && g < group);
        }
        if (group >= a.groups || ahead >= a.topk_groups) {
            #pragma unroll
            for (uint32_t i = 0; i < kItems; ++i) key[i] = 0;
        }
    }
    int32_t chosen = -1;
    for (uint32_t k = 0; k < a.topk; ++k) {
        uint64_t mine = 0;
        uint32_t place = 0;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i)
            if (key[i] > mine) { mine = key[i]; place = of.at(i); }
        const uint64_t top = largest_key(mine);
        if (top == 0) break;
        const uint32_t e = __reduce_min_sync(kAll, mine == top ? place : 0xffffffffu);
        if (lane == k) chosen = (int32_t)e;
        #pragma unroll
        for (uint32_t i = 0; i < kItems; ++i)
            if (of.at(i) == e) key[i] = 0;
    }
    return chosen;
}

template <uint32_t kVec, uint32_t kItems, bool kScores>
__global__ void __launch_bounds__(kRouteThreads) moe_route_kernel(const RouteArgs a) {
    const uint32_t lane = threadIdx.x % 32, token = blockIdx.x * (kRouteThreads / 32) + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.tokens) return;
    const uint8_t* row = a.logits + (uint64_t)token * a.stride;
    const uint32_t group = lane >> a.lanes_log2;
    Share<kVec> of{group * a.group_size + (lane & ((1u << a.lanes_log2) - 1)) * kVec, kVec << a.lanes_log2, (group + 1) * a.group_size};
    if (group >= a.groups) of.first = of.end = 0;
    float l[kItems];
    load_logits(a, row, of, l);
    Softmax m{0.0f, 1.0f};
    float z[kItems];
    if (!a.sigmoid) m = softmax_of(l, z);
    int32_t chosen;
    Choice state = quick_choice<kVec, kItems, kScores>(a, row, of, l, m, z, lane, chosen);
    // (a softmax's scores want its sum in 64 bits, and the 33 of 32 choices more lanes)
    if (state == Choice::kOrderOpen) {
        if ((a.sigmoid || a.by_logits) && a.topk < 32) chosen = exact_order(a, row, chosen, lane);
        else state = Choice::kOpen;
    }
    if (state == Choice::kOpen) chosen = exact_choice<kVec, kItems>(a, row, of, m.top, lane);
    if (lane >= a.topk) chosen = -1;
    float w = 0.0f;
    if (chosen >= 0) w = score_of(a.sigmoid != 0, m, logit_at(a, row, (uint32_t)chosen));
    if (a.renormalize) w = __fdiv_rn(w, divisor_of(warp_sum(w)));
    if (lane < a.topk) {
        static_cast<int32_t*>(a.idx)[(uint64_t)token * a.topk + lane] = chosen;
        a.weights[(uint64_t)token * a.topk + lane] = chosen >= 0 ? w * a.scale : 0.0f;
    }
}

// The gradient: with A_j from choice j (below), dl_e = sum over the choices of e of A_j, and for a softmax that is not renormalised
// - p_e sum(g p) on every expert. A lane writes the latter (or zeros) for its experts, and then lane j what its choice adds up to, over the same: equal
// choices add up in their order. Bound by HBM for many tokens: the logits are read once and their gradient is written once.
template <uint32_t kVec, uint32_t kItems>
__global__ void __launch_bounds__(kRouteThreads) moe_route_grad_kernel(const RouteArgs a) {
    const uint32_t lane = threadIdx.x % 32, token = blockIdx.x * (kRouteThreads / 32) + threadIdx.x / 32;
    griddep_wait();
    griddep_launch_dependents();
    if (token >= a.tokens) return;
    const uint8_t* row = a.logits + (uint64_t)token * a.stride;
    const Share<kVec> of{lane * kVec, 32 * kVec, a.experts};
    const bool sigmoid = a.sigmoid != 0, everywhere = !sigmoid && !a.renormalize;
    float l[kItems];
    if (!sigmoid) load_logits(a, row, of, l);
    int32_t idx = -1;
    float g = 0.0f, mine = 0.0f;
    if (lane < a.topk) {
        const uint64_t at = (uint64_t)token * a.topk + lane;
        const int64_t e = a.idx64 ? *(static_cast<const volatile int64_t*>(a.idx) + at) : (int64_t)(int32_t)ld_global_u32(static_cast<const int32_t*>(a.idx) + at);
        g = __uint_as_float(ld_global_u32(a.grad_weights + at)) * a.scale;
        if (e >= 0 && e < a.experts) {
            idx = (int32_t)e;
            mine = logit_at(a, row, (uint32_t)idx);
        }
    }
    if (idx < 0) g = 0.0f;
    Softmax m{0.0f, 1.0f};
    float z[kItems];
    if (!sigmoid) m = softmax_of(l, z);
    const float s = idx >= 0 ? score_of(sigmoid, m, mine) : 0.0f;
    // the slope of log s (for a softmax the other part of it is the sum over all experts): 1 - s would lose its bits where s is near 1
    const float slope = sigmoid ? sigmoid_of(-mine) : 1.0f;
    float from_choice, from_all = 0.0f;
    if (a.renormalize) {
        const float sum = warp_sum(s), q = __fdiv_rn(s, divisor_of(sum)), dot = warp_sum(g * q);
        from_choice = q * (sum <= kLeastSum ? g : g - dot) * slope;
    } else {
        from_choice = g * s * slope;
        if (!sigmoid) from_all = warp_sum(g * s);
    }
    uint8_t* out = a.grad_logits + (uint64_t)token * a.grad_stride;
    // (the logits may lie where their gradient goes)
    __syncwarp();
    const float each = everywhere ? -from_all * __frcp_rn(m.sum) : 0.0f;
    #pragma unroll
    for (uint32_t i = 0; i < kItems; i += kVec) {
        const uint32_t e = of.at(i);
        if (e >= of.end) continue;
        float d[kVec];
        #pragma unroll
        for (uint32_t j = 0; j < kVec; ++j) d[j] = everywhere ? each * z[i + j] : 0.0f;
        if (kVec == 4 && a.aligned) {
            if (a.fp32) {
                *reinterpret_cast<float4*>(out + (uint64_t)e * 4) = make_float4(d[0], d[kVec / 4], d[kVec / 2], d[kVec - 1]);
            } else {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(d[0], d[kVec / 4]), hi = __floats2bfloat162_rn(d[kVec / 2], d[kVec - 1]);
                *reinterpret_cast<uint2*>(out + (uint64_t)e * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
        } else {
            #pragma unroll
            for (uint32_t j = 0; j < kVec; ++j) {
                if (a.fp32) reinterpret_cast<float*>(out)[e + j] = d[j];
                else reinterpret_cast<__nv_bfloat16*>(out)[e + j] = __float2bfloat16_rn(d[j]);
            }
        }
    }
    const uint32_t same = __match_any_sync(kAll, idx);
    float sum = from_choice;
    if (__any_sync(kAll, idx >= 0 && (same & (same - 1)) != 0)) {
        sum = 0.0f;
        for (uint32_t j = 0; j < a.topk; ++j) {
            const float add = __shfl_sync(kAll, from_choice, j);
            if (same >> j & 1u) sum += add;
        }
    }
    // (behind the stores of the other lanes)
    __syncwarp();
    if (idx >= 0 && (same & ((1u << lane) - 1)) == 0) {
        const float d = (everywhere ? -from_all * s : 0.0f) + sum;
        if (a.fp32) reinterpret_cast<float*>(out)[idx] = d;
        else reinterpret_cast<__nv_bfloat16*>(out)[idx] = __float2bfloat16_rn(d);
    }
}

}  // namespace dg

using namespace dg;

// The instantiation for as many experts as a lane holds. (At most 60 of a forward pass, at least 17 lanes having experts, and 32 of a backward one.)
template <template <uint32_t, uint32_t> class Pick> static const void* for_items(bool vec, uint32_t items) {
    if (vec) return items <= 4 ? Pick<4, 4>::fn() : items <= 8 ? Pick<4, 8>::fn() : items <= 16 ? Pick<4, 16>::fn() : items <= 32 ? Pick<4, 32>::fn() : Pick<4, 64>::fn();
    return items <= 2 ? Pick<1, 2>::fn() : items <= 4 ? Pick<1, 4>::fn() : items <= 8 ? Pick<1, 8>::fn() : items <= 16 ? Pick<1, 16>::fn()
           : items <= 32 ? Pick<1, 32>::fn() : Pick<1, 64>::fn();
}
template <uint32_t kVec, uint32_t kItems> struct ByScores { static const void* fn() { return (const void*)moe_route_kernel<kVec, kItems, true>; } };
template <uint32_t kVec, uint32_t kItems> struct ByLogits { static const void* fn() { return (const void*)moe_route_kernel<kVec, kItems, false>; } };
template <uint32_t kVec, uint32_t kItems> struct Backward { static const void* fn() { return (const void*)moe_route_grad_kernel<kVec, (kItems < 32 ? kItems : 32)>; } };

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
    while ((1u << a.index_bits) < experts) ++a.index_bits;
    const bool vec = a.group_size % 4 == 0;
    a.aligned = vec && (reinterpret_cast<uintptr_t>(logits) | a.stride) % (is_fp32 ? 16 : 8) == 0;
    a.bias_aligned = reinterpret_cast<uintptr_t>(bias) % 16 == 0;
    const uint32_t run = vec ? 4 : 1, items = (a.group_size + (run << a.lanes_log2) - 1) / (run << a.lanes_log2) * run;
    void* params[] = {&a};
    const bool scores = !a.by_logits || (num_groups > 1 && a.best_two);
    return launch_overlapped(scores ? for_items<ByScores>(vec, items) : for_items<ByLogits>(vec, items), dim3((tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32)), dim3(kRouteThreads), params,
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
    const bool vec = experts % 4 == 0;
    a.aligned = vec && (reinterpret_cast<uintptr_t>(logits) | a.stride | reinterpret_cast<uintptr_t>(grad_logits) | a.grad_stride) % (is_fp32 ? 16 : 8) == 0;
    void* params[] = {&a};
    return launch_overlapped(for_items<Backward>(vec, vec ? (experts + 127) / 128 * 4 : (experts + 31) / 32), dim3((tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32)), dim3(kRouteThreads), params,
                             static_cast<cudaStream_t>(stream));
}
