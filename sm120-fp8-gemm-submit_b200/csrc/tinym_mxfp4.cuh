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
// Both directions are bound by the bytes of the wide side.  A thread holds 8
// columns (16 bytes of BF16), four threads a block of 32, 16 threads the four
// scales of 128 columns, which they write (read) as one 4-byte word.
#pragma once

#include <cuda_fp4.h>

#include "tinym_grouped.cuh"
#include "tinym_quant.cuh"

namespace tinym {

constexpr int kMxThreads = 256;
constexpr int kMxUnroll = 4;  // 128-column groups a 16-thread team loads before it uses the first

struct MxParams {
    int32_t rows, k;          // rows of one matrix, columns
    int32_t row_blocks;       // ceil(rows / 128)
    uint32_t groups;          // batch * rows * ceil(k / 128)
    uint32_t pad_words;       // batch * (128 * row_blocks - rows) * ceil(k / 128)
    FastDiv kc, per_matrix, pad_per_matrix;  // divisors: ceil(k / 128), rows, padding rows
};

// Byte offset of the scale word of 128-column group c of row r of matrix b.
__device__ __forceinline__ int64_t mx_scale_word(const MxParams& p, uint32_t b, uint32_t r,
                                                 uint32_t c) {
    return ((static_cast<int64_t>(b) * p.row_blocks + (r >> 7)) * p.kc.d + c) * kScaleBlock +
           (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

template <typename T>
__device__ __forceinline__ void mx_load8(const T* src, float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        ActVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(src)), f);
    } else {
        float a[4], b[4];
        ActVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(src)), a);
        ActVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(src) + 1), b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = a[i];
            f[4 + i] = b[i];
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kMxThreads)
    tinym_mxfp4_quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                uint8_t* __restrict__ scales, const MxParams p) {
    const uint32_t sub = threadIdx.x & 15;
    const uint32_t team = (blockIdx.x * kMxThreads + threadIdx.x) >> 4;
    const uint32_t teams = (gridDim.x * kMxThreads) >> 4;
    // The two teams of a warp take part in the shuffles together, so the
    // loop bound is the warp's.
    for (uint32_t g0 = team; (g0 & ~1u) < p.groups; g0 += teams * kMxUnroll) {
        float f[kMxUnroll][8];
        uint32_t row[kMxUnroll], col[kMxUnroll];
        bool in[kMxUnroll];
#pragma unroll
        for (int u = 0; u < kMxUnroll; ++u) {
            const uint32_t g = g0 + u * teams;
            row[u] = p.kc.div(g);
            col[u] = (g - row[u] * p.kc.d) * 128 + sub * 8;
            in[u] = g < p.groups && col[u] < static_cast<uint32_t>(p.k);
            if (in[u]) {
                mx_load8(x + static_cast<int64_t>(row[u]) * p.k + col[u], f[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[u][j] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kMxUnroll; ++u) {
            uint32_t top = 0;  // magnitudes compare as integers; NaN above infinity above all
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[u][j]) & 0x7FFFFFFFu);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t ex = top >> 23;  // biased floor(log2(amax)); 0 below the normal range
            const bool bad = ex == 255u;
            const uint32_t byte = bad ? 255u : (ex > 2u ? ex - 2u : 0u);
            const float unit = bad ? 0.0f : __uint_as_float((254u - byte) << 23);  // 2^-e
            uint32_t packed = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = bad ? make_float2(0.0f, 0.0f)
                                     : make_float2(f[u][2 * j] * unit, f[u][2 * j + 1] * unit);
                packed |= static_cast<uint32_t>(
                              __nv_cvt_float2_to_fp4x2(v, __NV_E2M1, cudaRoundNearest))
                          << (8 * j);
            }
            // the team's four scale bytes as one word (columns past K give 0)
            uint32_t word = in[u] ? byte << (8 * (sub >> 2)) : 0u;
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
            if (in[u])
                *reinterpret_cast<uint32_t*>(codes + (static_cast<int64_t>(row[u]) * p.k + col[u]) / 2) =
                    packed;
            if (sub == 0 && g0 + u * teams < p.groups) {
                const uint32_t b = p.per_matrix.div(row[u]);
                *reinterpret_cast<uint32_t*>(
                    scales + mx_scale_word(p, b, row[u] - b * p.per_matrix.d, col[u] >> 7)) = word;
            }
        }
    }
    // scale words of the rows that fill up the last block
    for (uint32_t i = blockIdx.x * kMxThreads + threadIdx.x; i < p.pad_words;
         i += gridDim.x * kMxThreads) {
        const uint32_t r = p.kc.div(i);
        const uint32_t b = p.pad_per_matrix.div(r);
        *reinterpret_cast<uint32_t*>(
            scales + mx_scale_word(p, b, p.rows + (r - b * p.pad_per_matrix.d), i - r * p.kc.d)) = 0u;
    }
}

// 2^(byte - 127) as FP32 (byte 0 is a subnormal, 255 NaN).
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
    return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7FC00000u : byte << 23));
}

template <typename T>
__global__ void __launch_bounds__(kMxThreads)
    tinym_mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                  const uint8_t* __restrict__ scales, T* __restrict__ y,
                                  const MxParams p) {
    const uint32_t sub = threadIdx.x & 15;
    const uint32_t team = (blockIdx.x * kMxThreads + threadIdx.x) >> 4;
    const uint32_t teams = (gridDim.x * kMxThreads) >> 4;
    for (uint32_t g0 = team; g0 < p.groups; g0 += teams * kMxUnroll) {
        uint32_t c[kMxUnroll], s[kMxUnroll];
        int64_t at[kMxUnroll];
        bool in[kMxUnroll];
#pragma unroll
        for (int u = 0; u < kMxUnroll; ++u) {
            const uint32_t g = g0 + u * teams;
            const uint32_t row = p.kc.div(g);
            const uint32_t kc = g - row * p.kc.d;
            const uint32_t col = kc * 128 + sub * 8;
            in[u] = g < p.groups && col < static_cast<uint32_t>(p.k);
            at[u] = static_cast<int64_t>(row) * p.k + col;
            c[u] = s[u] = 0;
            if (in[u]) {
                const uint32_t b = p.per_matrix.div(row);
                c[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + at[u] / 2));
                s[u] = __ldg(scales + mx_scale_word(p, b, row - b * p.per_matrix.d, kc) + (sub >> 2));
            }
        }
#pragma unroll
        for (int u = 0; u < kMxUnroll; ++u) {
            if (!in[u]) continue;
            const float unit = e8m0_to_f32(s[u]);
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(
                    static_cast<__nv_fp4x2_storage_t>((c[u] >> (8 * j)) & 0xFFu), __NV_E2M1);
                const float2 w = __half22float2(__half2(h));
                v[2 * j] = w.x * unit;
                v[2 * j + 1] = w.y * unit;
            }
            if constexpr (sizeof(T) == 2) {
                uint4 o;
                uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    ow[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(y + at[u]) = o;
            } else {
                float4* o = reinterpret_cast<float4*>(y + at[u]);
                o[0] = make_float4(v[0], v[1], v[2], v[3]);
                o[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
}

}  // namespace tinym
