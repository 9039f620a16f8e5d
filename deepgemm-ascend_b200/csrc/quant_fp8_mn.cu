// E4M3 operands whose contraction runs down the rows (both sides of a weight gradient, the weights of a gradient of the activations), made from BF16 or
// from E4M3 rows with scales along them (what a forward pass has kept in 8 bits), and the way back to BF16 or FP32.
//
// Mathematics: over 32 rows of a column, scale = 2^ceil(log2(max(amax, floor) / 448)) as in quant.cuh, codes = x / scale rounded to E4M3. x is exact
// in FP32 in either form (four significant bits times a power of two), so the rounding to E4M3 is the only one. A block that holds an
// infinity or a NaN gets the scale byte of NaN.
//
// HBM-bound: 2 (or 1 + 1/32) bytes read and 1 + 1/32 written per value. 32768 x 7168 from 8 bits 100 us, 5.0 TB/s (the bytes alone 78 at the rate of a copy: the
// instructions of the conversions fill 63 % of the issue slots); 16384 x 7168 from BF16 54 us, 6.6 TB/s, and back to BF16 56 us, 6.4 TB/s, from
// scales along the rows 54.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "../../include/dg_b200.h"
#include "host_common.h"
#include "ptx.cuh"
#include "quant.cuh"

namespace dg {

constexpr uint32_t kMnThreads = 128, kMnCols = 128, kMnRows = 64;      // a CTA of the quantiser: a thread a column of its scales
constexpr uint32_t kBackThreads = 256, kBackCols = 256, kBackRows = 32; // and of the way back

struct MnArgs {
    const uint8_t* x; uint64_t x_stride, x_group_stride;                  // bytes: BF16, or E4M3 with scales along the rows
    const uint8_t* x_sf; uint64_t x_sf_stride, x_sf_group_stride;         // int16 [ceil(cols / 64)][rows] seen as bytes
    uint8_t* out; uint64_t out_stride, out_group_stride;                  // bytes
    uint8_t* sf; uint64_t sf_stride, sf_group_stride;                     // int16 [ceil(rows / 64)][cols] seen as bytes
    const int32_t* psum; uint32_t num_experts, alignment;
    uint32_t rows, cols, tiles_c;
    float floor; uint32_t least;                                          // the least amax, and the scale byte of it
};

// Eight values in each of a lane's eight rows -> codes and scale bytes, through FP32.
__device__ __forceinline__ void quantise_down(const float (&v)[8][8], float floor, uint2& bytes, uint2 (&codes)[8]) {
    uint32_t e[8];
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        // (as whole numbers: infinities and NaN come out on top)
        uint32_t m = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
        e[j] = m >= 0x7f800000u ? 255u : e4m3_scale_byte(__uint_as_float(m), floor);
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        float s[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = v[i][j] * __uint_as_float((254u - min(e[j], 254u)) << 23);
        codes[i] = e4m3_pack8(s, 127u);
    }
    bytes = make_uint2(e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24, e[4] | e[5] << 8 | e[6] << 16 | e[7] << 24);
}

// BF16 rows, two values at a time: magnitudes are compared as whole numbers, products with the inverse scales are exact.
__device__ __forceinline__ void quantise_down_bf16(const uint4 (&q)[8], float floor, uint2& bytes, uint2 (&codes)[8]) {
    uint32_t m[4] = {}, f[4], e[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        #pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = __vmaxu2(m[j], w[j] & 0x7fff7fffu);
    }
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = __vmaxu2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        m[j] = __vmaxu2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
        const float lo = bf16_lo(m[j]), hi = bf16_hi(m[j]);
        e[2 * j] = (m[j] & 0xffffu) >= 0x7f80u ? 255u : e4m3_scale_byte(lo, floor);
        e[2 * j + 1] = m[j] >= 0x7f800000u ? 255u : e4m3_scale_byte(hi, floor);
        f[j] = (254u - min(e[2 * j], 254u)) << 7 | (254u - min(e[2 * j + 1], 254u)) << 23;
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        float s[8];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t p = mul_bf16x2(w[j], f[j]);
            s[2 * j] = bf16_lo(p);
            s[2 * j + 1] = bf16_hi(p);
        }
        codes[i] = e4m3_pack8(s, 127u);
    }
    bytes = make_uint2(e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24, e[4] | e[5] << 8 | e[6] << 16 | e[7] << 24);
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    const __half2 p = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&p);
}
// The larger magnitude of each half, NaN if one is.
__device__ __forceinline__ uint32_t larger_f16x2(uint32_t m, uint32_t v) {
    const __half2 p = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&v)));
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t pair) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t f16x2_to_e4m3(uint32_t v) {
    return (uint32_t)__nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&v), __NV_SATFINITE, __NV_E4M3);
}

// E4M3 rows through FP16, two values at a time, relative to the largest scale byte of the warp's rows, `top`: the codes are FP16 numbers h, the rows' factors
// 2^(b - top) and the columns' 2^(top - e) powers of two. Exact while the former are 2^-15 or more and the latter lie in 2^-14 .. 2^15; answers whether that is
// so (the same in all lanes), which it is where the magnitudes of a tile's rows and columns lie within a few thousand. The scale bytes of two columns at a
// time: amax <= 448 s = 1.75 x 2^8 s, so with amax = 1.m x 2^x (m of ten bits) s is 2^(x - 8), or twice that where m is above 0.75, which is an addition
// to the bits that carries; `least` is the byte of the least amax.
//
// (Through FP32, which takes every input, 32768 x 7168 takes 173 us, through FP16 100, or 114 where each lane makes its own factors. 40 bytes are spilled.)
//
// Whatever a row or a column has once is made once and handed round: `pair` holds the bytes of row `lane` (of the tile's two blocks), `block` says which of them
// this lane's columns lie in, and of the four words of columns that the lanes of a row share each of the four lanes of a column makes one.
__device__ __forceinline__ bool quantise_down_fp8(const uint2 (&q)[8], uint32_t pair, uint32_t block, uint32_t least, uint32_t lane, uint2& bytes, uint2 (&codes)[8]) {
    const uint32_t b0 = pair & 0xffu, b1 = pair >> 8;
    const uint32_t top = __reduce_max_sync(0xffffffffu, max(b0, b1)), low = __reduce_min_sync(0xffffffffu, min(b0, b1));
    // (from 2^120 on codes stand for numbers beyond FP32, which are infinities there whatever else the tile holds)
    if (top > 246u || low == 0u || top - low > 15u) return false;
    // (2^-15 is a subnormal number of FP16)
    const uint32_t factors = max((15u - (top - b0)) << 10, 0x0200u) | max((15u - (top - b1)) << 10, 0x0200u) << 16, both = block ? 0x3232u : 0x1010u;
    uint32_t h[8][4], m[4] = {};
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t factor = __byte_perm(__shfl_sync(0xffffffffu, factors, i * 4 + lane / 8), 0u, both);
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[i][j] = mul_f16x2(e4m3_to_f16x2((j < 2 ? q[i].x : q[i].y) >> (16 * (j % 2))), factor);
            m[j] = larger_f16x2(m[j], h[i][j]);
        }
    }
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = larger_f16x2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        m[j] = larger_f16x2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    }
    const uint32_t word = lane / 8, mine = word < 2 ? (word == 0 ? m[0] : m[1]) : (word == 2 ? m[2] : m[3]);
    // (the exponent field is x + 15; a subnormal m stands for no more than top - 22, which `least` covers or the factor shows)
    const uint32_t some = __vcmpgtu2(mine, 0u), floor = least * 0x10001u;
    const uint32_t e = (__vmaxs2(__vadd2(((mine + 0x00ff00ffu) >> 10) & 0x003f003fu, ((top - 23u) & 0xffffu) * 0x10001u), floor) & some) | (floor & ~some);
    const uint32_t x = __vsub2(top * 0x10001u, e), x_in = __vmins2(__vmaxs2(x, 0xfff2fff2u), 0x000f000fu);
    // (a column of zeros is one under any factor; a NaN is above all codes)
    const bool fits = ((x ^ x_in) & some) == 0u && __vmaxu2(mine, 0x5f005f00u) == 0x5f005f00u;
    if (!__all_sync(0xffffffffu, fits)) return false;
    const uint32_t f = __vadd2(x_in, 0x000f000fu) << 10, two = __byte_perm(e, 0u, 0x4420);
    uint32_t g[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = __shfl_sync(0xffffffffu, f, j * 8 + lane % 8);
    bytes.x = __byte_perm(__shfl_sync(0xffffffffu, two, lane % 8), __shfl_sync(0xffffffffu, two, 8 + lane % 8), 0x5410);
    bytes.y = __byte_perm(__shfl_sync(0xffffffffu, two, 16 + lane % 8), __shfl_sync(0xffffffffu, two, 24 + lane % 8), 0x5410);
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        codes[i] = make_uint2(f16x2_to_e4m3(mul_f16x2(h[i][0], g[0])) | f16x2_to_e4m3(mul_f16x2(h[i][1], g[1])) << 16,
                              f16x2_to_e4m3(mul_f16x2(h[i][2], g[2])) | f16x2_to_e4m3(mul_f16x2(h[i][3], g[3])) << 16);
    return true;
}

__device__ __forceinline__ void load_raw(uint2& q, const uint8_t* p) { q = ld_stream_v2(p); }
__device__ __forceinline__ void load_raw(uint4& q, const uint8_t* p) { q = ld_stream_v4(p); }

// One CTA = 64 rows x 128 columns, a warp 32 rows x 64 columns: lane = (every fourth row, eight columns), so that the maximum down a column takes
// two shuffles, and a row of the warp's tile is a line of 128 bytes of BF16 or two whole sectors of codes. The 64 columns are one column of the
// scales of an 8-bit input, whose 32 rows are one read of 64 bytes. (32768 x 7168 from 8 bits in CTAs of 256 threads 133 us, of 128 114, before the above.)
template <bool kFromFp8>
__global__ void __launch_bounds__(kMnThreads, 8) quant_fp8_mn_kernel(const MnArgs a) {
    __shared__ __align__(8) uint8_t sf_smem[2][kMnCols];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t group = blockIdx.z;
    const uint32_t row_base = blockIdx.x / a.tiles_c * kMnRows, c0 = blockIdx.x % a.tiles_c * kMnCols;
    const uint32_t half = warp / (kMnCols / 64), tc = warp % (kMnCols / 64) * 64 + lane % 8 * 8, c = c0 + tc;
    const uint32_t warp_col = c0 + tc / 64 * 64, warp_row = row_base + half * 32, r0 = warp_row + lane / 8;
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t write_end = min(a.rows, row_base + kMnRows);
    const uint8_t* x = a.x + group * a.x_group_stride + (uint64_t)r0 * a.x_stride + (uint64_t)c * (kFromFp8 ? 1 : 2);
    // (the same for the whole CTA: no bounds inside) What lies there is asked for before it is known which rows count.
    const bool inside = row_base + kMnRows <= a.rows && c0 + kMnCols <= a.cols;
    using Raw = typename std::conditional<kFromFp8, uint2, uint4>::type;
    Raw q[8];
    uint32_t pair = 0x7f7fu;                                  // scales of this lane's row of the tile
    if (inside) {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, x += 4 * a.x_stride) load_raw(q[i], x);
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, x += 4 * a.x_stride) {
            q[i] = Raw{};
            if (r0 + i * 4 < a.rows && c < a.cols) load_raw(q[i], x);
        }
    }
    if (kFromFp8 && warp_col < a.cols && warp_row + lane < a.rows)
        pair = ld_global_u16(a.x_sf + group * a.x_sf_group_stride + (uint64_t)(warp_col / 64) * a.x_sf_stride + (uint64_t)(warp_row + lane) * 2);
    uint32_t row_end = write_end;
    if (a.psum != nullptr) {
        // (groups start on multiples of 64 rows: a tile lies in one) Rows of the padding count as zeros and are written as zeros
        const GroupEnd end = group_end_of(a.psum, a.num_experts, a.alignment, row_base, lane);
        if (end.whole <= row_base) return;                // behind the last group (uniform over the CTA)
        row_end = min(row_end, end.valid);
        if (row_end < write_end) {
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (r0 + i * 4 >= row_end) q[i] = Raw{};
        }
    }
    uint2 codes[8], bytes;
    if constexpr (kFromFp8) {
        // (rows that do not count are zeros and have no scale: the first row lends them its own; the second half of a last, half-used column is lent the first's)
        const uint32_t lent = __shfl_sync(0xffffffffu, pair, 0), block = c < a.cols ? lane % 8 / 4 : 0u;
        if (warp_row + lane >= row_end) pair = warp_row < row_end ? lent : 0x7f7fu;
        if (warp_col + 32 >= a.cols) pair = (pair & 0xffu) * 0x101u;
        if (!quantise_down_fp8(q, pair, block, a.least, lane, bytes, codes)) {
            float v[8][8];
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t b = __shfl_sync(0xffffffffu, pair, i * 4 + lane / 8) >> (block * 8) & 0xffu;
                const float scale = ue8m0_float(r0 + i * 4 < row_end ? b : 127u);
                float lo[4], hi[4];
                e4m3_unpack4(q[i].x, lo);
                e4m3_unpack4(q[i].y, hi);
                #pragma unroll
                for (int j = 0; j < 4; ++j) { v[i][j] = lo[j] * scale; v[i][4 + j] = hi[j] * scale; }
            }
            quantise_down(v, a.floor, bytes, codes);
        }
    } else {
        quantise_down_bf16(q, a.floor, bytes, codes);
    }
    // (blocks behind the last row are zero)
    if (lane < 8) *reinterpret_cast<uint2*>(&sf_smem[half][tc]) = warp_row < a.rows ? bytes : make_uint2(0u, 0u);
    uint8_t* out = a.out + group * a.out_group_stride + (uint64_t)r0 * a.out_stride + c;
    if (inside) {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, out += 4 * a.out_stride) *reinterpret_cast<uint2*>(out) = codes[i];
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < 8; ++i, out += 4 * a.out_stride)
            if (r0 + i * 4 < write_end && c < a.cols) *reinterpret_cast<uint2*>(out) = codes[i];
    }
    __syncthreads();
    if (c0 + threadIdx.x < a.cols)
        *reinterpret_cast<uint16_t*>(a.sf + group * a.sf_group_stride + (uint64_t)(row_base / 64) * a.sf_stride + (uint64_t)(c0 + threadIdx.x) * 2) =
            (uint16_t)(sf_smem[0][threadIdx.x] | ((uint32_t)sf_smem[1][threadIdx.x] << 8));
}

// The way back: code x 2^(byte - 127), rounded once to BF16 or FP32 (which changes nothing but where those have subnormals). One CTA = 32 rows x 256
// columns, a warp four rows, a lane eight columns. The scales of K-major rows come in runs down the rows, through shared memory; those of an MN-major
// tile lie along the columns. HBM-bound: 2112 x 7168 there and back 13.9 us, where the bytes alone take 14.0 from HBM (the codes between the two stay in L2).
template <typename T, bool kMnMajor>
__global__ void __launch_bounds__(kBackThreads) dequant_fp8_kernel(const MnArgs a) {
    constexpr uint32_t kTileRows = kBackRows, kWarpRows = kTileRows / (kBackThreads / 32);
    __shared__ __align__(8) uint8_t sf_smem[kTileRows][kBackCols / 32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t group = blockIdx.z;
    const uint32_t row_base = blockIdx.x / a.tiles_c * kTileRows, c0 = blockIdx.x % a.tiles_c * kBackCols;
    const uint32_t c = c0 + lane * 8, r0 = row_base + warp * kWarpRows;
    griddep_wait();
    griddep_launch_dependents();
    const uint8_t* x = a.x + group * a.x_group_stride + (uint64_t)r0 * a.x_stride + c;
    uint2 q[kWarpRows];
    #pragma unroll
    for (uint32_t i = 0; i < kWarpRows; ++i, x += a.x_stride) {
        q[i] = make_uint2(0u, 0u);
        if (r0 + i < a.rows && c < a.cols) q[i] = ld_stream_v2(x);
    }
    const uint8_t* sf = a.x_sf + group * a.x_sf_group_stride;
    float scale[8] = {};
    if constexpr (kMnMajor) {
        if (c < a.cols) {
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                scale[j] = ue8m0_float(ld_global_u16(sf + (uint64_t)(r0 / 64) * a.x_sf_stride + (uint64_t)(c + j) * 2) >> (r0 / 32 % 2 * 8) & 0xffu);
        }
    } else {
        const uint32_t col = threadIdx.x / kTileRows, r = threadIdx.x % kTileRows;
        if (col < kBackCols / 64 && c0 + col * 64 < a.cols && row_base + r < a.rows)
            *reinterpret_cast<uint16_t*>(&sf_smem[r][col * 2]) = ld_global_u16(sf + (uint64_t)(c0 / 64 + col) * a.x_sf_stride + (uint64_t)(row_base + r) * 2);
        __syncthreads();
    }
    uint8_t* out = a.out + group * a.out_group_stride + (uint64_t)r0 * a.out_stride + (uint64_t)c * sizeof(T);
    #pragma unroll
    for (uint32_t i = 0; i < kWarpRows; ++i, out += a.out_stride) {
        if (r0 + i >= a.rows || c >= a.cols) continue;
        if constexpr (!kMnMajor) {
            const float s = ue8m0_float(sf_smem[warp * kWarpRows + i][lane / 4]);
            #pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] = s;
        }
        float v[8];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            float four[4];
            e4m3_unpack4(h ? q[i].y : q[i].x, four);
            #pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * h + j] = four[j] * scale[4 * h + j];
        }
        if constexpr (sizeof(T) == 2) {
            uint32_t w[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&p);
            }
            *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            // (one store of 32 bytes: as two, each leaves half of every sector to the other)
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                         "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
        }
    }
}

}  // namespace dg

using namespace dg;

static int mn_checks(uint32_t rows, uint32_t cols, const void* x, const void* x_sf, bool needs_sf, const void* out, const void* sf, bool makes_sf) {
    DG_CHECK_ARG(x != nullptr && out != nullptr && (!needs_sf || x_sf != nullptr) && (!makes_sf || sf != nullptr), "fp8: null pointer");
    DG_CHECK_ARG(cols % 32 == 0, "fp8: the row length must be a multiple of 32");
    DG_CHECK_ARG(rows <= 0x7fffffffu && cols <= 0x7fffffffu, "fp8: too many values");
    return DG_OK;
}

// One launch for as many matrices as a grid holds.
static int launch_mn(const void* fn, MnArgs a, uint32_t tile_rows, uint32_t tile_cols, uint32_t threads, uint32_t groups, void* stream) {
    constexpr uint32_t kMostGroups = 65535;
    a.tiles_c = (a.cols + tile_cols - 1) / tile_cols;
    const uint64_t tiles = (uint64_t)((a.rows + tile_rows - 1) / tile_rows) * a.tiles_c;
    DG_CHECK_ARG(tiles <= 0x7fffffffull, "fp8: too many values");
    void* params[] = {&a};
    for (uint32_t g = 0; g < groups; g += kMostGroups) {
        const dim3 grid((uint32_t)tiles, 1, groups - g < kMostGroups ? groups - g : kMostGroups);
        if (int rc = launch_overlapped(fn, grid, dim3(threads), params, static_cast<cudaStream_t>(stream))) return rc;
        a.x += kMostGroups * a.x_group_stride; a.x_sf += kMostGroups * a.x_sf_group_stride;
        a.out += kMostGroups * a.out_group_stride; a.sf += kMostGroups * a.sf_group_stride;
    }
    return DG_OK;
}

// The scale byte of a block whose largest magnitude is `amax`, as on the device.
static uint32_t least_byte(float amax) {
    const float scaled = amax * (1.0f / 448.0f);
    uint32_t bits;
    memcpy(&bits, &scaled, 4);
    const uint32_t e = (bits + 0x7fffffu) >> 23;
    return e < 1u ? 1u : e;
}

extern "C" int dg_quant_fp8_mn_launch(const void* x, uint64_t x_stride, uint64_t x_group_stride, const int16_t* x_sf, uint64_t x_sf_stride, uint64_t x_sf_group_stride,
                                      uint32_t groups, uint32_t rows, uint32_t cols, const int32_t* psum, uint32_t num_experts, uint32_t alignment, float min_amax,
                                      void* out, uint64_t out_stride, uint64_t out_group_stride, int16_t* sf, uint64_t sf_stride, uint64_t sf_group_stride, void* stream) {
    if (groups == 0 || rows == 0 || cols == 0) return DG_OK;
    const bool from_fp8 = x_sf != nullptr;
    const uint64_t es = from_fp8 ? 1 : 2;
    if (int rc = mn_checks(rows, cols, x, x_sf, false, out, sf, true)) return rc;
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | x_stride * es | x_group_stride * es) % (from_fp8 ? 8 : 16) == 0, "fp8: input rows must start on %d-byte boundaries", from_fp8 ? 8 : 16);
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(out) | out_stride | out_group_stride) % 8 == 0, "fp8: output rows must start on 8-byte boundaries");
    DG_CHECK_ARG(sf_stride >= cols && (!from_fp8 || x_sf_stride >= rows), "fp8: scale stride smaller than the columns (rows of a K-major input)");
    DG_CHECK_ARG(psum == nullptr || (groups == 1 && num_experts > 0 && alignment > 0 && alignment % 64 == 0),
                 "fp8: a psum layout needs one matrix, experts, and an alignment that is a multiple of 64");
    DG_CHECK_ARG(min_amax >= 0.0f && min_amax <= 3.0e38f, "fp8: min_amax must be a finite number that is not negative");
    MnArgs a{};
    a.x = static_cast<const uint8_t*>(x); a.x_stride = x_stride * es; a.x_group_stride = x_group_stride * es;
    a.x_sf = reinterpret_cast<const uint8_t*>(x_sf); a.x_sf_stride = x_sf_stride * 2; a.x_sf_group_stride = x_sf_group_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride; a.out_group_stride = out_group_stride;
    a.sf = reinterpret_cast<uint8_t*>(sf); a.sf_stride = sf_stride * 2; a.sf_group_stride = sf_group_stride * 2;
    a.psum = psum; a.num_experts = psum ? num_experts : 0; a.alignment = alignment;
    a.rows = rows; a.cols = cols; a.floor = min_amax; a.least = least_byte(min_amax);
    return launch_mn(from_fp8 ? (const void*)quant_fp8_mn_kernel<true> : (const void*)quant_fp8_mn_kernel<false>, a, kMnRows, kMnCols, kMnThreads, groups, stream);
}

extern "C" int dg_dequant_fp8_launch(const void* codes, uint64_t code_stride, uint64_t code_group_stride, const int16_t* sf, uint64_t sf_stride, uint64_t sf_group_stride,
                                     uint32_t groups, uint32_t rows, uint32_t cols, int mn_major, void* out, int out_is_fp32, uint64_t out_stride,
                                     uint64_t out_group_stride, void* stream) {
    if (groups == 0 || rows == 0 || cols == 0) return DG_OK;
    const uint64_t es = out_is_fp32 ? 4 : 2;
    if (int rc = mn_checks(rows, cols, codes, sf, true, out, nullptr, false)) return rc;
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(codes) | code_stride | code_group_stride) % 8 == 0, "fp8: rows of codes must start on 8-byte boundaries");
    DG_CHECK_ARG((reinterpret_cast<uintptr_t>(out) | out_stride * es | out_group_stride * es) % (8 * es) == 0, "fp8: output rows must start on %d-byte boundaries", (int)(8 * es));
    DG_CHECK_ARG(sf_stride >= (mn_major ? cols : rows), "fp8: scale stride smaller than the rows (columns when MN-major)");
    MnArgs a{};
    a.x = static_cast<const uint8_t*>(codes); a.x_stride = code_stride; a.x_group_stride = code_group_stride;
    a.x_sf = reinterpret_cast<const uint8_t*>(sf); a.x_sf_stride = sf_stride * 2; a.x_sf_group_stride = sf_group_stride * 2;
    a.out = static_cast<uint8_t*>(out); a.out_stride = out_stride * es; a.out_group_stride = out_group_stride * es;
    a.rows = rows; a.cols = cols;
    const void* fn = mn_major ? (out_is_fp32 ? (const void*)dequant_fp8_kernel<float, true> : (const void*)dequant_fp8_kernel<__nv_bfloat16, true>)
                              : (out_is_fp32 ? (const void*)dequant_fp8_kernel<float, false> : (const void*)dequant_fp8_kernel<__nv_bfloat16, false>);
    return launch_mn(fn, a, kBackRows, kBackCols, kBackThreads, groups, stream);
}
