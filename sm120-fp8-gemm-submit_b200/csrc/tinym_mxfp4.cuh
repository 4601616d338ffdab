// tinym_mxfp4.cuh -- MXFP4 quantisation and its inverse.
//
// A block is 32 consecutive columns of a row.  With amax the block's largest
// magnitude, its scale is 2^e, e = floor(log2(amax)) - 2 clamped to
// [-127, 127] (2 = the exponent of E2M1's largest value 6; a block of zeros
// takes -127), and its elements are E2M1 codes of x * 2^-e, rounded to
// nearest even and saturated at 6 (x * 2^-e lies below 8).  x * 2^-e is exact
// or far below the smallest level, so the only rounding is the one to E2M1.
// A block that holds a NaN or an infinity gets the scale NaN (255) and zero
// codes, so it stays visible in every product.
//
// Layout: two codes per byte, the even column in the low nibble; scale bytes
// in blocks of 128 rows x 4 scales (tinym_b200.h), bytes past the matrix 0.
//
// Both directions are bound by the bytes of the wide side, and close to the
// instruction rate: 8 columns cost 87 instructions to quantise and 60 to
// expand (133 and 94, and a third more time, when each thread worked out its
// own rows and blocks; 8 x 5120 x 6144 BF16 there and back: 308 -> 230 us,
// 85 % of the measured copy).  So a warp takes a run of columns of one row:
// a lane holds 8 consecutive ones (16 bytes of BF16) of each step of 256, four
// lanes a block of 32, 16 lanes the four scales of 128 columns, one 4-byte
// word.  Row and addresses are worked out once per run.
#pragma once

#include <cuda_fp4.h>

#include "tinym_grouped.cuh"
#include "tinym_quant.cuh"

namespace tinym {

constexpr int kMxThreads = 256;
// Steps of 256 columns in a warp's run: 64 bytes in flight per lane.
template <typename T>
constexpr int kMxSteps = sizeof(T) == 2 ? 4 : 2;

struct MxParams {
    int32_t rows, k;          // rows of one matrix, columns
    int32_t row_blocks;       // ceil(rows / 128)
    uint32_t runs;            // batch * rows * ceil(k / run)
    uint32_t pad_words;       // batch * (128 * row_blocks - rows) * ceil(k / 128)
    FastDiv per_row, per_matrix;  // divisors: runs of a row, rows
    FastDiv kc, pad_per_matrix;   // divisors: ceil(k / 128), padding rows
};

// Byte offset of the scale word of 128-column group 0 of row r of matrix b;
// group c lies c * kScaleBlock further.
__device__ __forceinline__ int64_t mx_scale_row(const MxParams& p, uint32_t b, uint32_t r) {
    return (static_cast<int64_t>(b) * p.row_blocks + (r >> 7)) * p.kc.d * kScaleBlock +
           (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// 8 columns as loaded: their largest magnitude as FP32 bits, and their values.
template <typename T>
struct MxVec;
template <>
struct MxVec<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ld_after_wait(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
    // magnitudes compare as integers; NaN above infinity above all
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = 0x7FFF7FFFu;
        const uint32_t t = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
        return max(t & 0xFFFF0000u, t << 16);
    }
    __device__ __forceinline__ void values(float (&f)[8]) const { ActVec<__nv_bfloat16>::unpack(v, f); }
};
template <>
struct MxVec<float> {
    uint4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = ld_after_wait(reinterpret_cast<const uint4*>(p));
        b = ld_after_wait(reinterpret_cast<const uint4*>(p) + 1);
    }
    __device__ __forceinline__ void zero() { a = b = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = 0x7FFFFFFFu;
        return max(max(max(a.x & m, a.y & m), max(a.z & m, a.w & m)),
                   max(max(b.x & m, b.y & m), max(b.z & m, b.w & m)));
    }
    __device__ __forceinline__ void values(float (&f)[8]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    }
};

template <typename T>
__global__ void __launch_bounds__(kMxThreads)
    tinym_mxfp4_quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                uint8_t* __restrict__ scales, const MxParams p) {
    constexpr int kSteps = kMxSteps<T>;
    grid_dependency_wait();  // launched while the kernel before may still run
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * (kMxThreads / 32);
    for (uint32_t run = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); run < p.runs; run += warps) {
        const uint32_t row = p.per_row.div(run);
        const int col = static_cast<int>(run - row * p.per_row.d) * (kSteps * 256) + lane * 8;
        const int64_t at = static_cast<int64_t>(row) * p.k + col;
        MxVec<T> v[kSteps];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            if (col + u * 256 < p.k) v[u].load(x + at + u * 256);
            else v[u].zero();
        }
        const uint32_t b = p.per_matrix.div(row);
        uint8_t* word = scales + mx_scale_row(p, b, row - b * p.per_matrix.d) +
                        static_cast<int64_t>(col >> 7) * kScaleBlock;
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            uint32_t top = v[u].top();
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t ex = top >> 23;  // biased floor(log2(amax)); 0 below the normal range
            const bool bad = ex == 255u;
            const uint32_t byte = bad ? 255u : max(ex, 2u) - 2u;
            const float unit = __uint_as_float((254u - byte) << 23);  // 2^-e (-inf if bad: codes dropped below)
            float f[8];
            v[u].values(f);
            uint32_t packed = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                packed |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(
                              make_float2(f[2 * j] * unit, f[2 * j + 1] * unit), __NV_E2M1, cudaRoundNearest))
                          << (8 * j);
            const bool in = col + u * 256 < p.k;
            if (in) *reinterpret_cast<uint32_t*>(codes + (at + u * 256) / 2) = bad ? 0u : packed;
            // the four scale bytes of 16 lanes as one word (columns past K give 0)
            uint32_t s = in ? byte << (8 * ((lane >> 2) & 3)) : 0u;
            s |= __shfl_xor_sync(0xFFFFFFFFu, s, 4);
            s |= __shfl_xor_sync(0xFFFFFFFFu, s, 8);
            if (in && (lane & 15) == 0) *reinterpret_cast<uint32_t*>(word + u * 2 * kScaleBlock) = s;
        }
    }
    // scale words of the rows that fill up the last block
    for (uint32_t i = blockIdx.x * kMxThreads + threadIdx.x; i < p.pad_words;
         i += gridDim.x * kMxThreads) {
        const uint32_t r = p.kc.div(i);
        const uint32_t b = p.pad_per_matrix.div(r);
        *reinterpret_cast<uint32_t*>(scales + mx_scale_row(p, b, p.rows + (r - b * p.pad_per_matrix.d)) +
                                     static_cast<int64_t>(i - r * p.kc.d) * kScaleBlock) = 0u;
    }
}

// Four E2M1 codes (16 bits) as two words of BF16 pairs: the magnitudes' bytes
// are looked up (a code's three lower bits are a byte selector), the signs are
// bits 3, 7, 11 and 15.
__device__ __forceinline__ void e2m1x4_to_bf16(uint32_t c, uint32_t* lo, uint32_t* hi) {
    const uint32_t sel = c & 0x7777u;
    // 0, 0.5, 1, 1.5 | 2, 3, 4, 6 = 0x0000, 0x3F00, 0x3F80, 0x3FC0 | 0x4000, 0x4040, 0x4080, 0x40C0
    const uint32_t upper = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);
    const uint32_t lower = __byte_perm(0xC0800000u, 0xC0804000u, sel);
    const uint32_t sign = __byte_perm(c << 4, c, 0x5140) & 0x80808080u;
    *lo = __byte_perm(lower, upper | sign, 0x5140);
    *hi = __byte_perm(lower, upper | sign, 0x7362);
}

template <typename T>
__global__ void __launch_bounds__(kMxThreads)
    tinym_mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                  const uint8_t* __restrict__ scales, T* __restrict__ y,
                                  const MxParams p) {
    constexpr int kSteps = kMxSteps<T>;
    grid_dependency_wait();  // launched while the kernel before may still run
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * (kMxThreads / 32);
    for (uint32_t run = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); run < p.runs; run += warps) {
        const uint32_t row = p.per_row.div(run);
        const int col = static_cast<int>(run - row * p.per_row.d) * (kSteps * 256) + lane * 8;
        const int64_t at = static_cast<int64_t>(row) * p.k + col;
        const uint32_t b = p.per_matrix.div(row);
        const uint8_t* byte = scales + mx_scale_row(p, b, row - b * p.per_matrix.d) +
                              static_cast<int64_t>(col >> 7) * kScaleBlock + ((lane >> 2) & 3);
        uint32_t c[kSteps], s[kSteps];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            const bool in = col + u * 256 < p.k;
            c[u] = in ? ld_after_wait(reinterpret_cast<const uint32_t*>(codes + (at + u * 256) / 2)) : 0u;
            s[u] = in ? ld_after_wait(byte + u * 2 * kScaleBlock) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            if (col + u * 256 >= p.k) break;
            uint32_t v[4];
            e2m1x4_to_bf16(c[u], &v[0], &v[1]);
            e2m1x4_to_bf16(c[u] >> 16, &v[2], &v[3]);
            // 2^(s - 127) as BF16: 0 is a subnormal, 255 NaN.  Two significant
            // bits times a power of two: exact down to 2^-128.
            const uint32_t unit = s[u] == 0u ? 0x0040u : (s[u] == 255u ? 0x7FC0u : s[u] << 7);
            if constexpr (sizeof(T) == 2) {
                const uint32_t pair = unit | unit << 16;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[j]),
                                                     *reinterpret_cast<const __nv_bfloat162*>(&pair));
                    v[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(y + at + u * 256) = make_uint4(v[0], v[1], v[2], v[3]);
            } else {
                const float scale = __uint_as_float(unit << 16);
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[2 * j] = __uint_as_float(v[j] << 16) * scale;
                    f[2 * j + 1] = __uint_as_float(v[j] & 0xFFFF0000u) * scale;
                }
                float4* o = reinterpret_cast<float4*>(y + at + u * 256);
                o[0] = make_float4(f[0], f[1], f[2], f[3]);
                o[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
        }
    }
}

}  // namespace tinym
