// Microscaled 4-bit operands: BF16 or FP32 values -> packed E2M1 with one UE8M0 scale per 32 values along K, in the layout the
// GEMM reads, and back.
//
// Mathematics: over a block of 32 values, s = the smallest power of two with amax <= 6 s and q = x / s rounded to the nearest of
// {0, 0.5, 1, 1.5, 2, 3, 4, 6} and their negatives, halves to the even code (the hardware conversion); s is a power of two, so
// x / s is exact and that is the only rounding. A block that holds an infinity or a NaN gets the scale byte of NaN.
//
// Two directions, because the contraction of a product runs along the row of a K-major operand and down the rows of an MN-major
// one: blocks of 32 lie along a row (K-major) or down a column (MN-major). Codes are packed in pairs along the row either way,
// as the GEMM wants them.
//
// HBM-bound: n values read (2 or 4 bytes each), n / 2 + n / 32 bytes written, or the reverse.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

struct Fp4Args {
    const uint8_t* x; uint64_t x_stride, x_group_stride;                  // bytes
    uint8_t* codes; uint64_t code_stride, code_group_stride;              // bytes; a row holds cols / 2
    uint8_t* sf; uint64_t sf_stride, sf_group_stride;                     // bytes; K-major: [ceil(cols / 64)][rows], MN-major: [ceil(rows / 64)][cols]
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t rows, cols, tiles_r, tiles_c;
    uint32_t sf_aligned;                                                  // eight scales of an MN-major matrix can be read at once
};

// Eight values of a lane, as they lie in memory: kWords words of one or two values. Magnitudes are compared as bit patterns (infinities
// and NaN come out on top by themselves), BF16 two at a time; so are the products with the inverse scales, which are exact (down to where
// BF16 has subnormals, all of which round to zero). What is saved counts: an MN-major quantiser that turned every BF16 into FP32 first kept
// the SMs at 67 % and HBM at 58 %, and in a long run arithmetic draws on the board's power limit.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
    static constexpr int kWords = 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0u; }
    __device__ __forceinline__ void load(const uint8_t* p) {
        const uint4 q = ld_stream_v4(p);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7fff7fffu; }
    // FP32 bits of column `j` of the magnitudes, factors of the columns of a word from the exponent fields of the inverse scales
    static __device__ __forceinline__ uint32_t bits(const uint32_t (&m)[kWords], int j) { return j % 2 ? m[j / 2] & 0xffff0000u : m[j / 2] << 16; }
    static __device__ __forceinline__ uint32_t factor(const uint32_t (&field)[8], int word) { return field[2 * word] << 7 | field[2 * word + 1] << 23; }
    static __device__ __forceinline__ uint32_t factor(uint32_t field) { return field << 7 | field << 23; }
    __device__ __forceinline__ uint32_t codes(const uint32_t (&f)[kWords]) const {
        float v[8];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t p = mul_bf16x2(w[j], f[j]);
            v[2 * j] = bf16_lo(p);
            v[2 * j + 1] = bf16_hi(p);
        }
        return e2m1_pack8(v);
    }
};
template <> struct Raw8<float> {
    static constexpr int kWords = 8;
    uint32_t w[kWords];
    __device__ __forceinline__ void clear() {
        #pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0u;
    }
    __device__ __forceinline__ void load(const uint8_t* p) {
        const uint4 q = ld_global_v4(p), r = ld_global_v4(p + 16);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
        w[4] = r.x; w[5] = r.y; w[6] = r.z; w[7] = r.w;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7fffffffu; }
    static __device__ __forceinline__ uint32_t bits(const uint32_t (&m)[kWords], int j) { return m[j]; }
    static __device__ __forceinline__ uint32_t factor(const uint32_t (&field)[8], int word) { return field[word] << 23; }
    static __device__ __forceinline__ uint32_t factor(uint32_t field) { return field << 23; }
    __device__ __forceinline__ uint32_t codes(const uint32_t (&f)[kWords]) const {
        float v[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]) * __uint_as_float(f[j]);
        return e2m1_pack8(v);
    }
};

constexpr uint32_t kFp4Threads = 256, kFp4Rows = 32, kFp4Cols = 256;

// K-major: one CTA = 32 rows x 256 columns, a warp takes four rows (all loads issued before the first is used), a lane eight
// columns, four lanes a block. Scales go through shared memory, so that every scale column of the tile is one 64-byte run. Bound by HBM for many
// rows, by the launch for few: 64 x 7168 BF16 2.1 us, 2112 x 7168 FP32 12.4 us (5.5 TB/s, from HBM), 8 x 4096 x 7168 BF16 about 90 us (6.6 TB/s).
template <typename T>
__global__ void __launch_bounds__(kFp4Threads) quant_fp4_kernel(const Fp4Args a) {
    constexpr uint32_t kWarpRows = kFp4Rows / (kFp4Threads / 32);
    __shared__ __align__(8) uint8_t sf_smem[kFp4Rows][kFp4Cols / 32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t group = blockIdx.z;
    const uint32_t row_base = blockIdx.x / a.tiles_c * kFp4Rows, c0 = blockIdx.x % a.tiles_c * kFp4Cols;
    griddep_wait();
    griddep_launch_dependents();
    uint32_t row_end = min(a.rows, row_base + kFp4Rows);
    if (a.psum != nullptr) row_end = min(row_end, group_end_of(a.psum, a.num_experts, a.alignment, row_base, lane).valid);
    if (row_end <= row_base) return;                      // the whole tile is padding (uniform over the CTA)

    const uint32_t c = c0 + lane * 8, r0 = row_base + warp * kWarpRows;
    const uint8_t* x = a.x + group * a.x_group_stride + (uint64_t)r0 * a.x_stride + (uint64_t)c * sizeof(T);
    uint8_t* codes = a.codes + group * a.code_group_stride + (uint64_t)r0 * a.code_stride + c / 2;
    Raw8<T> raw[kWarpRows];
    #pragma unroll
    for (uint32_t i = 0; i < kWarpRows; ++i, x += a.x_stride) {
        raw[i].clear();
        if (r0 + i < row_end && c < a.cols) raw[i].load(x);
    }
    #pragma unroll
    for (uint32_t i = 0; i < kWarpRows; ++i) {
        uint32_t m[Raw8<T>::kWords], f[Raw8<T>::kWords];
        #pragma unroll
        for (int j = 0; j < Raw8<T>::kWords; ++j) {
            m[j] = Raw8<T>::magnitude(raw[i].w[j]);
            if (j > 0) m[0] = Raw8<T>::larger(m[0], m[j]);
        }
        uint32_t amax = sizeof(T) == 2 ? max(Raw8<T>::bits(m, 0), Raw8<T>::bits(m, 1)) : m[0];
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t e = e2m1_scale_byte(amax);
        #pragma unroll
        for (int j = 0; j < Raw8<T>::kWords; ++j) f[j] = Raw8<T>::factor(e2m1_inverse(e));
        if (r0 + i < row_end && c < a.cols) *reinterpret_cast<uint32_t*>(codes) = raw[i].codes(f);
        codes += a.code_stride;
        // (the second block of a last, half-used scale column is zero)
        if ((lane & 3u) == 0) sf_smem[warp * kWarpRows + i][lane / 4] = c < a.cols ? (uint8_t)e : (uint8_t)0;
    }
    __syncthreads();
    const uint32_t col = threadIdx.x / kFp4Rows, r = threadIdx.x % kFp4Rows;
    if (col < kFp4Cols / 64 && c0 + col * 64 < a.cols && r < row_end - row_base)
        *reinterpret_cast<uint16_t*>(a.sf + group * a.sf_group_stride + (uint64_t)(c0 / 64 + col) * a.sf_stride + (uint64_t)(row_base + r) * 2) =
            *reinterpret_cast<const uint16_t*>(&sf_smem[r][col * 2]);
}

// MN-major: one CTA = 64 rows x 256 columns. A warp takes one block of 32 rows x 64 columns: lane = (every fourth row, eight columns), so
// that a row of the warp's tile is a whole 128-byte line of BF16 and the maximum down a column takes two shuffles. The codes go through
// shared memory and out as lines of 128 bytes (written by the lanes as they are, a row of a warp's tile is one sector of 32 bytes, and
// the number of stores bounds the kernel: 114 us against 110 for 8 x 4096 x 7168 BF16); its rows are 40 words apart, which keeps the four rows of a
// store in banks of their own. That size now: 90 us, 6.6 TB/s, since whole tiles check no bounds and BF16 goes two at a time. FP32 holds 64 words
// of a tile in each lane, 96 registers, so two CTAs are on an SM where BF16 has five; with twice the bytes on their way in each that is enough: 8 x 4096 x 7168
// 150 us, 7.1 TB/s (84 % of DRAM's cycles), 4096 x 7168 22.4 us, 2112 x 7168 13.3 (12.1 when K-major).
constexpr uint32_t kFp4StageWords = 40;
template <typename T>
__global__ void __launch_bounds__(kFp4Threads) quant_fp4_mn_kernel(const Fp4Args a) {
    __shared__ __align__(8) uint8_t sf_smem[2][kFp4Cols];
    __shared__ __align__(16) uint32_t stage[64][kFp4StageWords];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t group = blockIdx.z;
    const uint32_t row_base = blockIdx.x / a.tiles_c * 64, c0 = blockIdx.x % a.tiles_c * kFp4Cols;
    const uint32_t half = warp / 4, tc = warp % 4 * 64 + lane % 8 * 8, c = c0 + tc;
    const uint32_t tr = half * 32 + lane / 8, r0 = row_base + tr;
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t write_end = min(a.rows, row_base + 64);
    uint32_t row_end = write_end;
    if (a.psum != nullptr) {
        // (groups start on multiples of 64 rows: a tile lies in one) Rows of the padding count as zeros and are written as zeros
        const GroupEnd end = group_end_of(a.psum, a.num_experts, a.alignment, row_base, lane);
        if (end.whole <= row_base) return;                // behind the last group (uniform over the CTA)
        row_end = min(row_end, end.valid);
    }
    const uint8_t* x = a.x + group * a.x_group_stride + (uint64_t)r0 * a.x_stride + (uint64_t)c * sizeof(T);
    Raw8<T> raw[8];
    if (row_base + 64 <= row_end && c0 + kFp4Cols <= a.cols) {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, x += 4 * a.x_stride) raw[i].load(x);
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, x += 4 * a.x_stride) {
            raw[i].clear();
            if (r0 + i * 4 < row_end && c < a.cols) raw[i].load(x);
        }
    }
    uint32_t m[Raw8<T>::kWords] = {}, f[Raw8<T>::kWords], field[8];
    #pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        #pragma unroll
        for (int j = 0; j < Raw8<T>::kWords; ++j) m[j] = Raw8<T>::larger(m[j], Raw8<T>::magnitude(raw[i].w[j]));
    #pragma unroll
    for (int j = 0; j < Raw8<T>::kWords; ++j) {
        m[j] = Raw8<T>::larger(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        m[j] = Raw8<T>::larger(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    }
    uint32_t bytes[2] = {};
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t e = e2m1_scale_byte(Raw8<T>::bits(m, j));
        field[j] = e2m1_inverse(e);
        bytes[j / 4] |= e << (j % 4 * 8);
    }
    #pragma unroll
    for (int j = 0; j < Raw8<T>::kWords; ++j) f[j] = Raw8<T>::factor(field, j);
    // (blocks behind the last row are zero)
    if (lane < 8) *reinterpret_cast<uint2*>(&sf_smem[half][tc]) = row_base + half * 32 < a.rows ? make_uint2(bytes[0], bytes[1]) : make_uint2(0u, 0u);
    #pragma unroll
    for (uint32_t i = 0; i < 8; ++i) stage[tr + i * 4][tc / 8] = raw[i].codes(f);
    __syncthreads();
    #pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = threadIdx.x / 8 + i * 32, part = threadIdx.x % 8;
        if (row_base + r < write_end && c0 + part * 32 < a.cols)
            *reinterpret_cast<uint4*>(a.codes + group * a.code_group_stride + (uint64_t)(row_base + r) * a.code_stride + (c0 + part * 32) / 2) =
                *reinterpret_cast<const uint4*>(&stage[r][part * 4]);
    }
    if (c0 + threadIdx.x < a.cols)
        *reinterpret_cast<uint16_t*>(a.sf + group * a.sf_group_stride + (uint64_t)(row_base / 64) * a.sf_stride + (uint64_t)(c0 + threadIdx.x) * 2) =
            (uint16_t)(sf_smem[0][threadIdx.x] | ((uint32_t)sf_smem[1][threadIdx.x] << 8));
}

// The way back: code x 2^(byte - 127), in the type of the result (exact, but rounded once where that has subnormals).
template <typename T> struct Out8;
template <> struct Out8<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t scale(uint32_t byte) { return ue8m0_bf16(byte) * 0x10001u; }
    static __device__ __forceinline__ uint32_t scale_pair(uint32_t b0, uint32_t b1) { return ue8m0_bf16(b0) | ue8m0_bf16(b1) << 16; }
    static __device__ __forceinline__ void store(uint8_t* p, uint32_t q, const uint32_t (&s)[4]) {
        uint32_t w[4];
        e2m1_to_bf16(q, w);
        *reinterpret_cast<uint4*>(p) = make_uint4(mul_bf16x2(w[0], s[0]), mul_bf16x2(w[1], s[1]), mul_bf16x2(w[2], s[2]), mul_bf16x2(w[3], s[3]));
    }
};
template <> struct Out8<float> {
    // (the scales are held as BF16 pairs too, which holds every power of two that a byte stands for)
    static __device__ __forceinline__ uint32_t scale(uint32_t byte) { return Out8<__nv_bfloat16>::scale(byte); }
    static __device__ __forceinline__ uint32_t scale_pair(uint32_t b0, uint32_t b1) { return Out8<__nv_bfloat16>::scale_pair(b0, b1); }
    static __device__ __forceinline__ void store(uint8_t* p, uint32_t q, const uint32_t (&s)[4]) {
        uint32_t w[4];
        e2m1_to_bf16(q, w);
        float v[8];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = bf16_lo(w[j]) * bf16_lo(s[j]);
            v[2 * j + 1] = bf16_hi(w[j]) * bf16_hi(s[j]);
        }
        // (one store of 32 bytes: as two, each leaves half of every sector to the other)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                     "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    }
};

// One CTA = 8 kWarpRows rows x 256 columns, a warp kWarpRows (4 or 8) of the rows, a lane eight columns. The scales of a K-major tile come in runs
// down the rows, through shared memory; a warp's rows of an MN-major tile lie in one block, whose scales lie along the columns. Four rows where
// the tiles of eight would not fill the device a few times (with the quantiser in front, 2112 x 7168 FP32: 24.2 against 26.1 us, BF16 14.4 against
// 15.1), else eight (8 x 4096 x 7168 BF16 in a long run, at the board's power limit: 187.8 against 191.3 us).
constexpr uint32_t kFewBackTiles = 148 * 8 * 4;
template <typename T, bool kMnMajor, uint32_t kWarpRows>
__global__ void __launch_bounds__(kFp4Threads) dequant_fp4_kernel(const Fp4Args a, uint8_t* out) {
    constexpr uint32_t kTileRows = kWarpRows * kFp4Threads / 32;
    __shared__ __align__(8) uint8_t sf_smem[kTileRows][kFp4Cols / 32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t group = blockIdx.z;
    const uint32_t row_base = blockIdx.x / a.tiles_c * kTileRows, c0 = blockIdx.x % a.tiles_c * kFp4Cols;
    const uint32_t c = c0 + lane * 8, r0 = row_base + warp * kWarpRows;
    griddep_wait();
    griddep_launch_dependents();
    const bool inside = row_base + kTileRows <= a.rows && c0 + kFp4Cols <= a.cols;
    const uint8_t* codes = a.codes + group * a.code_group_stride + (uint64_t)r0 * a.code_stride + c / 2;
    uint32_t q[kWarpRows];
    if (inside) {
        #pragma unroll
        for (uint32_t i = 0; i < kWarpRows; ++i, codes += a.code_stride) q[i] = ld_stream_u32(codes);
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < kWarpRows; ++i, codes += a.code_stride) q[i] = r0 + i < a.rows && c < a.cols ? ld_stream_u32(codes) : 0u;
    }
    const uint8_t* sf = a.sf + group * a.sf_group_stride;
    uint32_t scale[4];
    if constexpr (kMnMajor) {
        const uint8_t* pairs = sf + (uint64_t)(r0 / 64) * a.sf_stride + (uint64_t)c * 2;
        uint32_t p[4] = {};
        if (c < a.cols && a.sf_aligned) {
            const uint4 v = ld_global_v4(pairs);
            p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
        } else if (c < a.cols) {
            #pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = ld_global_u16(pairs + 4 * j) | (uint32_t)ld_global_u16(pairs + 4 * j + 2) << 16;
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t b = p[j] >> (r0 / 32 % 2 * 8);
            scale[j] = Out8<T>::scale_pair(b & 0xffu, (b >> 16) & 0xffu);
        }
    } else {
        const uint32_t col = threadIdx.x / kTileRows, r = threadIdx.x % kTileRows;
        if (col < kFp4Cols / 64 && c0 + col * 64 < a.cols && row_base + r < a.rows)
            *reinterpret_cast<uint16_t*>(&sf_smem[r][col * 2]) = ld_global_u16(sf + (uint64_t)(c0 / 64 + col) * a.sf_stride + (uint64_t)(row_base + r) * 2);
        __syncthreads();
    }
    uint8_t* to = out + group * a.x_group_stride + (uint64_t)r0 * a.x_stride + (uint64_t)c * sizeof(T);
    #pragma unroll
    for (uint32_t i = 0; i < kWarpRows; ++i, to += a.x_stride) {
        if (!inside && (r0 + i >= a.rows || c >= a.cols)) continue;
        if constexpr (!kMnMajor) scale[0] = scale[1] = scale[2] = scale[3] = Out8<T>::scale(sf_smem[warp * kWarpRows + i][lane / 4]);
        Out8<T>::store(to, q[i], scale);
    }
}

}  // namespace dg

using namespace dg;

// What both directions check: the float side is `x`, strides in elements of each side. `x_bytes`, `code_bytes`: the alignment that the
// kernel's loads and stores need.
static int fp4_args(Fp4Args& a, uint32_t tile_rows, uint32_t x_bytes, uint32_t code_bytes, const void* x, int is_fp32, uint64_t x_stride, uint64_t x_group_stride,
                    uint32_t rows, uint32_t cols, const void* codes, uint64_t code_stride, uint64_t code_group_stride,
                    const int16_t* sf, uint64_t sf_stride, uint64_t sf_group_stride, int mn_major) {
    const uint64_t es = is_fp32 ? 4 : 2;
    DG_CHECK_ARG(x != nullptr && codes != nullptr && sf != nullptr, "fp4: null pointer");
    DG_CHECK_ARG(cols % 32 == 0, "fp4: the row length must be a multiple of 32");
    DG_CHECK_ARG(rows <= 0x7fffffffu && cols <= 0x7fffffffu, "fp4: too many values");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | x_stride * es | x_group_stride * es) % x_bytes == 0,
                 "fp4: rows of values must start on %u-byte boundaries", x_bytes);
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(codes) | code_stride | code_group_stride) % code_bytes == 0,
                 "fp4: rows of codes must start on %u-byte boundaries", code_bytes);
    DG_CHECK_ARG(sf_stride >= (mn_major ? cols : rows), "fp4: scale stride smaller than the rows (columns when MN-major)");
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * es; a.x_group_stride = x_group_stride * es;
    a.codes = static_cast<uint8_t*>(const_cast<void*>(codes)); a.code_stride = code_stride; a.code_group_stride = code_group_stride;
    a.sf = reinterpret_cast<uint8_t*>(const_cast<int16_t*>(sf)); a.sf_stride = sf_stride * 2; a.sf_group_stride = sf_group_stride * 2;
    a.rows = rows; a.cols = cols;
    a.tiles_r = (rows + tile_rows - 1) / tile_rows;
    a.tiles_c = (cols + kFp4Cols - 1) / kFp4Cols;
    a.sf_aligned = (reinterpret_cast<uintptr_t>(sf) | a.sf_stride | a.sf_group_stride) % 16 == 0;
    DG_CHECK_ARG((uint64_t)a.tiles_r * a.tiles_c <= 0x7fffffffull, "fp4: too many values");
    return DG_OK;
}

// One launch for as many matrices as a grid holds. `out`: the float side, where it is written.
static int launch_fp4(const void* fn, Fp4Args a, uint32_t groups, void* out, void* stream) {
    constexpr uint32_t kMostGroups = 65535;
    uint8_t* to = static_cast<uint8_t*>(out);
    void* params[] = {&a, &to};
    for (uint32_t g = 0; g < groups; g += kMostGroups) {
        const dim3 grid(a.tiles_r * a.tiles_c, 1, groups - g < kMostGroups ? groups - g : kMostGroups);
        if (int rc = launch_overlapped(fn, grid, dim3(kFp4Threads), params, static_cast<cudaStream_t>(stream))) return rc;
        a.x += kMostGroups * a.x_group_stride; a.codes += kMostGroups * a.code_group_stride; a.sf += kMostGroups * a.sf_group_stride;
        to += kMostGroups * a.x_group_stride;
    }
    return DG_OK;
}

extern "C" int dg_quant_fp4_launch(const void* x, int x_is_fp32, uint64_t x_stride, uint64_t x_group_stride, uint32_t groups, uint32_t rows,
                                   uint32_t cols, int mn_major, const int32_t* psum, uint32_t num_experts, uint32_t alignment,
                                   void* out, uint64_t out_stride, uint64_t out_group_stride,
                                   int16_t* sf, uint64_t sf_stride, uint64_t sf_group_stride, void* stream) {
    if (groups == 0 || rows == 0 || cols == 0) return DG_OK;
    DG_CHECK_ARG(psum == nullptr || (groups == 1 && num_experts > 0 && alignment > 0 && alignment % (mn_major ? 64u : kFp4Rows) == 0),
                 "quant_fp4: a psum layout needs one matrix, experts, and an alignment that is a multiple of %u", mn_major ? 64u : kFp4Rows);
    Fp4Args a{};
    if (int rc = fp4_args(a, mn_major ? 64 : kFp4Rows, 16, mn_major ? 16 : 4, x, x_is_fp32, x_stride, x_group_stride, rows, cols, out, out_stride,
                          out_group_stride, sf, sf_stride, sf_group_stride, mn_major)) return rc;
    a.psum = psum; a.num_experts = psum ? num_experts : 0; a.alignment = alignment;
    const void* fn = mn_major ? (x_is_fp32 ? (const void*)quant_fp4_mn_kernel<float> : (const void*)quant_fp4_mn_kernel<__nv_bfloat16>)
                              : (x_is_fp32 ? (const void*)quant_fp4_kernel<float> : (const void*)quant_fp4_kernel<__nv_bfloat16>);
    return launch_fp4(fn, a, groups, nullptr, stream);
}

template <uint32_t kWarpRows>
static const void* back_kernel(bool fp32, bool mn_major) {
    return mn_major ? (fp32 ? (const void*)dequant_fp4_kernel<float, true, kWarpRows> : (const void*)dequant_fp4_kernel<__nv_bfloat16, true, kWarpRows>)
                    : (fp32 ? (const void*)dequant_fp4_kernel<float, false, kWarpRows> : (const void*)dequant_fp4_kernel<__nv_bfloat16, false, kWarpRows>);
}

extern "C" int dg_dequant_fp4_launch(const void* codes, uint64_t code_stride, uint64_t code_group_stride, const int16_t* sf, uint64_t sf_stride,
                                     uint64_t sf_group_stride, uint32_t groups, uint32_t rows, uint32_t cols, int mn_major,
                                     void* out, int out_is_fp32, uint64_t out_stride, uint64_t out_group_stride, void* stream) {
    if (groups == 0 || rows == 0 || cols == 0) return DG_OK;
    const bool few = (uint64_t)groups * ((rows + 63) / 64) * ((cols + kFp4Cols - 1) / kFp4Cols) < kFewBackTiles;
    Fp4Args a{};
    if (int rc = fp4_args(a, few ? 32 : 64, out_is_fp32 ? 32 : 16, 4, out, out_is_fp32, out_stride, out_group_stride, rows, cols, codes, code_stride,
                          code_group_stride, sf, sf_stride, sf_group_stride, mn_major)) return rc;
    const void* fn = few ? back_kernel<4>(out_is_fp32, mn_major) : back_kernel<8>(out_is_fp32, mn_major);
    return launch_fp4(fn, a, groups, out, stream);
}
