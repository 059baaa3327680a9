// Two-level 4-bit floating point (NVFP4) on the device: quantisation of fp32 / bf16 / fp16 matrices, and back.
//
//   g     one fp32 scale per tensor: the smallest power of two >= amax / 2688, 2688 = 6 * 448 being the largest value
//         the two lower levels reach together (g = 1 when amax = 0)
//   s     one e4m3 scale per 16 elements of a row: nearest e4m3 value of max|x| / (6 g), at most 448
//   code  the nearest e2m1 value of x / (s g), ties to the even code, saturating at 6; 0 where s = 0
// A block that holds an infinity or a NaN gets s = NaN (0x7F) and zero codes, so what is wrong stays visible in every
// product of that row. The last block of a row is filled up with zeros.
//
// g is a power of two on purpose: x / g is then exact, and so is every decision below. A border between two codes
// times s has at most seven bits, so a quotient that is rounded correctly never moves onto a border that the exact
// quotient misses, and fp32 gives the codes that real arithmetic gives. It costs no accuracy: the block scales keep
// their relative precision wherever in their range they lie.
//
// Scales are stored as the block-scaled tensor-core instruction reads them: 512-byte tiles of 128 rows x 4 scales (64
// elements of K), tile (row / 128, k / 64) in row-major order, byte (row % 32) * 16 + (row % 128) / 32 * 4 + j. The
// product then needs no pass of its own over the scales. Rows and scales that only pad a tile are zero.
//
// HBM-bound: 2 (or 4) bytes read and 9/16 written per element.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace pto_b200 {

constexpr int kNvQuantThreads = 256;

enum NvSrc : int { NV_F32 = 0, NV_BF16 = 1, NV_F16 = 2 };

template <int SRC>
struct NvElem {
    using type = float;
};
template <>
struct NvElem<NV_BF16> {
    using type = __nv_bfloat16;
};
template <>
struct NvElem<NV_F16> {
    using type = __half;
};

template <int SRC>
__device__ __forceinline__ float nv_to_float(typename NvElem<SRC>::type v)
{
    if constexpr (SRC == NV_F32) {
        return v;
    } else if constexpr (SRC == NV_BF16) {
        return __bfloat162float(v);
    } else {
        return __half2float(v);
    }
}

template <int SRC>
__device__ __forceinline__ void nv_unpack2(uint32_t w, float& lo, float& hi)
{
    if constexpr (SRC == NV_BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    }
}

// 16 consecutive elements from a 16-byte aligned address, read once.
template <int SRC>
__device__ __forceinline__ void nv_load16(const void* ptr, float (&x)[16])
{
    const uint4* p = static_cast<const uint4*>(ptr);
    if constexpr (SRC == NV_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 v = __ldcs(p + i);
            x[4 * i + 0] = __uint_as_float(v.x);
            x[4 * i + 1] = __uint_as_float(v.y);
            x[4 * i + 2] = __uint_as_float(v.z);
            x[4 * i + 3] = __uint_as_float(v.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = __ldcs(p + i);
            nv_unpack2<SRC>(v.x, x[8 * i + 0], x[8 * i + 1]);
            nv_unpack2<SRC>(v.y, x[8 * i + 2], x[8 * i + 3]);
            nv_unpack2<SRC>(v.z, x[8 * i + 4], x[8 * i + 5]);
            nv_unpack2<SRC>(v.w, x[8 * i + 6], x[8 * i + 7]);
        }
    }
}

// Exponent field of g for a tensor maximum: amax / 2688 rounded up to a power of two, 2688 = 1.3125 * 2^11.
__device__ __forceinline__ uint32_t nv_scale_exponent(float amax)
{
    const uint32_t bits = min(__float_as_uint(amax) & 0x7FFFFFFFu, 0x7F7FFFFFu);
    if (bits == 0u) {
        return 127u;
    }
    const int e = static_cast<int>(bits >> 23) - 11 + ((bits & 0x007FFFFFu) > 0x00280000u ? 1 : 0);
    return static_cast<uint32_t>(max(e, 1));
}

__device__ __forceinline__ float nv_e4m3_to_float(uint32_t code)
{
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

// Eight floats -> eight e2m1 codes in a word, the first in the low nibble.
__device__ __forceinline__ uint32_t nv_cvt_e2m1x8(const float* q)
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}"
        : "=r"(r)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return r;
}

// One block: its e4m3 scale code and its sixteen codes.
__device__ __forceinline__ uint32_t nv_quantize_block(float (&x)[16], float inv_g, uint2& codes)
{
    uint32_t top = 0u; // |x| as bits: the integer order is the value order, infinities and NaN above all numbers
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    }
    codes = make_uint2(0u, 0u);
    if (top >= 0x7F800000u) {
        return 0x7Fu;
    }
    const float y_max = __uint_as_float(top) * inv_g;
    const uint32_t s_code =
        __nv_cvt_float_to_fp8(fminf(__fdiv_rn(y_max, 6.0f), 448.0f), __NV_SATFINITE, __NV_E4M3);
    if (s_code == 0u) {
        return 0u;
    }
    const float s = nv_e4m3_to_float(s_code);
    const float r = __frcp_rn(s);
    if (y_max > 1.0e30f) { // only with a caller's amax far below the data: keeps the quotients finite
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = fminf(fmaxf(x[i] * inv_g, -8192.0f), 8192.0f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] *= inv_g;
        }
    }
    // x / s rounded correctly: a quotient from the reciprocal, then one correction by its exact remainder. (s has four
    // significant bits; the product alone misses ties by one unit and 1/16 of all bf16 quotients are ties.)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float q0 = __fmul_rn(x[i], r);
        const float rem = __fmaf_rn(-q0, s, x[i]);
        x[i] = __fmaf_rn(rem, r, q0);
    }
    codes.x = nv_cvt_e2m1x8(x);
    codes.y = nv_cvt_e2m1x8(x + 8);
    return s_code;
}

// Stores a block's codes and, once per four lanes, the scale word of four consecutive blocks. The four lanes of an
// aligned group hold blocks kb, kb + 1, .. kb + 3 of one row and call this together.
__device__ __forceinline__ void nv_store_block(uint8_t* data, uint8_t* scales, long long ld_data, int rows, int k_blocks,
                                               int k_atoms, int row, int kb, uint32_t s_code, const uint2& codes)
{
    if (row < rows && kb < k_blocks) {
        *reinterpret_cast<uint2*>(data + row * ld_data + static_cast<long long>(kb) * 8) = codes;
    }
    const unsigned mask = 0xFu << (threadIdx.x & 28u);
    uint32_t word = s_code << (8 * (threadIdx.x & 3u));
    word |= __shfl_xor_sync(mask, word, 1);
    word |= __shfl_xor_sync(mask, word, 2);
    if ((threadIdx.x & 3u) == 0u) {
        const long long tile = static_cast<long long>(row >> 7) * k_atoms + (kb >> 2);
        *reinterpret_cast<uint32_t*>(scales + tile * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4) = word;
    }
}

// src: [rows][ld_src]; VEC: rows start on 16-byte boundaries. One thread per block of 16 and step.
template <int SRC, bool VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_quantize_kernel(const void* __restrict__ src, const float* __restrict__ amax, uint8_t* __restrict__ data,
                          uint8_t* __restrict__ scales, float* __restrict__ tensor_scale, int rows, int k,
                          long long ld_src, long long ld_data)
{
    using T = typename NvElem<SRC>::type;
    const int k_blocks = (k + 15) / 16;
    const int k_atoms = (k_blocks + 3) / 4;
    const int row_blocks = k_atoms * 4;                // blocks of a row, padding included
    const long long rows_padded = (static_cast<long long>(rows) + 127) / 128 * 128;
    const long long total = rows_padded * row_blocks;  // a multiple of 4, as the stride is: groups of four stay whole
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    const uint32_t e = nv_scale_exponent(__ldg(amax));
    const float inv_g = __uint_as_float((254u - e) << 23);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *tensor_scale = __uint_as_float(e << 23);
    }
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / row_blocks;
    const int kb_step = static_cast<int>(stride - row_step * row_blocks);
    long long row = i / row_blocks;
    int kb = static_cast<int>(i - row * row_blocks);
    for (; i < total; i += stride) {
        uint32_t s_code = 0u;
        uint2 codes = make_uint2(0u, 0u);
        if (row < rows && kb < k_blocks) {
            float x[16];
            const T* p = static_cast<const T*>(src) + row * ld_src + static_cast<long long>(kb) * 16;
            if (VEC && kb * 16 + 16 <= k) {
                nv_load16<SRC>(p, x);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    x[j] = (kb * 16 + j < k) ? nv_to_float<SRC>(p[j]) : 0.0f;
                }
            }
            s_code = nv_quantize_block(x, inv_g, codes);
        }
        nv_store_block(data, scales, ld_data, rows, k_blocks, k_atoms, static_cast<int>(row), kb, s_code, codes);
        row += row_step;
        kb += kb_step;
        if (kb >= row_blocks) {
            kb -= row_blocks;
            row += 1;
        }
    }
}

// The same of the transpose: blocks run down the columns of src [rows][ld_src], row c of the result is column c of src.
// A thread block takes 256 rows x 64 columns through shared memory; sixteen lanes then hold the sixteen blocks of one
// column, so a column's codes leave as 128 contiguous bytes. 16-row groups are skewed by two words, which puts the
// sixteen lanes (16 rows apart) and the two columns of a warp on different banks.
constexpr int kNvTransRows = 256;
constexpr int kNvTransCols = 64;

template <int SRC>
inline constexpr int kNvTransGroupBytes = 16 * kNvTransCols * static_cast<int>(sizeof(typename NvElem<SRC>::type)) + 8;

template <int SRC, bool VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_quantize_transposed_kernel(const void* __restrict__ src, const float* __restrict__ amax,
                                     uint8_t* __restrict__ data, uint8_t* __restrict__ scales,
                                     float* __restrict__ tensor_scale, int rows, int k, long long ld_src, long long ld_data)
{
    using T = typename NvElem<SRC>::type;
    extern __shared__ uint2 nv_trans_smem[];
    uint8_t* tile = reinterpret_cast<uint8_t*>(nv_trans_smem);
    constexpr int kGroupBytes = kNvTransGroupBytes<SRC>;
    const int k_blocks = (rows + 15) / 16; // the result's rows run over src's rows
    const int k_atoms = (k_blocks + 3) / 4;
    const int row0 = static_cast<int>(blockIdx.x) * kNvTransRows;
    const int col0 = static_cast<int>(blockIdx.y) * kNvTransCols;
    const uint32_t e = nv_scale_exponent(__ldg(amax));
    const float inv_g = __uint_as_float((254u - e) << 23);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        *tensor_scale = __uint_as_float(e << 23);
    }
    const T* base = static_cast<const T*>(src);
    constexpr int kPer16 = 16 / static_cast<int>(sizeof(T));   // elements of a 16-byte load
    constexpr int kLoads = kNvTransCols / kPer16;              // of a row
#pragma unroll 4
    for (int it = threadIdx.x; it < kNvTransRows * kLoads; it += kNvQuantThreads) {
        const int r = it / kLoads;
        const int c = (it % kLoads) * kPer16;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row0 + r < rows) {
            const T* p = base + (row0 + r) * ld_src + col0 + c;
            if (VEC && col0 + c + kPer16 <= k) {
                v = __ldcs(reinterpret_cast<const uint4*>(p));
            } else {
                __align__(16) T part[kPer16];
#pragma unroll
                for (int j = 0; j < kPer16; ++j) {
                    part[j] = (col0 + c + j < k) ? p[j] : static_cast<T>(0.0f);
                }
                v = *reinterpret_cast<const uint4*>(part);
            }
        }
        uint2* dst = reinterpret_cast<uint2*>(tile + (r >> 4) * kGroupBytes +
                                              ((r & 15) * kNvTransCols + c) * static_cast<int>(sizeof(T)));
        dst[0] = make_uint2(v.x, v.y);
        dst[1] = make_uint2(v.z, v.w);
    }
    __syncthreads();
    const int b = threadIdx.x & 15;
    const int kb = row0 / 16 + b;
    if (kb >= k_atoms * 4) { // whole groups of four lanes leave together
        return;
    }
    for (int c = threadIdx.x >> 4; c < kNvTransCols; c += kNvQuantThreads / 16) {
        float x[16];
        const T* col = reinterpret_cast<const T*>(tile + b * kGroupBytes) + c;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            x[j] = nv_to_float<SRC>(col[j * kNvTransCols]);
        }
        uint2 codes;
        const uint32_t s_code = nv_quantize_block(x, inv_g, codes);
        nv_store_block(data, scales, ld_data, k, k_blocks, k_atoms, col0 + c, kb, s_code, codes);
    }
}

// Largest finite |x| of a matrix into *out, which the caller has set to zero. The maximum does not depend on the order.
template <int SRC, bool VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    amax_kernel(const void* __restrict__ src, uint32_t* __restrict__ out, int rows, int k, long long ld_src)
{
    using T = typename NvElem<SRC>::type;
    const int items_per_row = (k + 15) / 16;
    const long long total = static_cast<long long>(rows) * items_per_row;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / items_per_row;
    const int c_step = static_cast<int>(stride - row_step * items_per_row);
    long long row = i / items_per_row;
    int c = static_cast<int>(i - row * items_per_row);
    uint32_t top = 0u;
    for (; i < total; i += stride) {
        const T* p = static_cast<const T*>(src) + row * ld_src + static_cast<long long>(c) * 16;
        float x[16];
        if (VEC && c * 16 + 16 <= k) {
            nv_load16<SRC>(p, x);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[j] = (c * 16 + j < k) ? nv_to_float<SRC>(p[j]) : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t bits = __float_as_uint(x[j]) & 0x7FFFFFFFu;
            top = max(top, bits < 0x7F800000u ? bits : 0u);
        }
        row += row_step;
        c += c_step;
        if (c >= items_per_row) {
            c -= items_per_row;
            row += 1;
        }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    __shared__ uint32_t part[kNvQuantThreads / 32];
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    if (threadIdx.x < kNvQuantThreads / 32) {
        top = __reduce_max_sync((1u << (kNvQuantThreads / 32)) - 1u, part[threadIdx.x]);
        if (threadIdx.x == 0 && top != 0u) {
            atomicMax(out, top);
        }
    }
}

// Two e2m1 codes (a byte) -> two floats.
__device__ __forceinline__ float2 nv_e2m1x2_to_float2(uint32_t byte)
{
    uint32_t h;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "}"
        : "=r"(h)
        : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Back to numbers: (code * s) is exact, one rounding by g (none when g is a power of two), one by the output type.
// One thread per eight elements: four bytes in, 16 or 32 contiguous bytes out.
template <int DST, bool VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales,
                            const float* __restrict__ tensor_scale, void* __restrict__ out, int rows, int k,
                            long long ld_data, long long ld_out)
{
    using T = typename NvElem<DST>::type;
    const int items_per_row = (k + 7) / 8;
    const int k_atoms = (k + 63) / 64;
    const float g = tensor_scale != nullptr ? __ldg(tensor_scale) : 1.0f;
    const long long total = static_cast<long long>(rows) * items_per_row;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / items_per_row;
    const int c_step = static_cast<int>(stride - row_step * items_per_row);
    long long row = i / items_per_row;
    int c = static_cast<int>(i - row * items_per_row);
    for (; i < total; i += stride) {
        const uint32_t codes = __ldcs(reinterpret_cast<const uint32_t*>(data + row * ld_data + static_cast<long long>(c) * 4));
        const int kb = c >> 1;
        const long long tile = (row >> 7) * k_atoms + (kb >> 2);
        const float s = nv_e4m3_to_float(__ldg(scales + tile * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (kb & 3)));
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = nv_e2m1x2_to_float2((codes >> (8 * j)) & 0xFFu);
            v[2 * j] = __fmul_rn(__fmul_rn(f.x, s), g);
            v[2 * j + 1] = __fmul_rn(__fmul_rn(f.y, s), g);
        }
        T* dst = static_cast<T*>(out) + row * ld_out + static_cast<long long>(c) * 8;
        __align__(16) T o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o[j] = static_cast<T>(v[j]);
        }
        if (VEC && c * 8 + 8 <= k) {
            constexpr int kQuads = 8 * static_cast<int>(sizeof(T)) / 16;
#pragma unroll
            for (int j = 0; j < kQuads; ++j) {
                reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(o)[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c * 8 + j < k) {
                    dst[j] = o[j];
                }
            }
        }
        row += row_step;
        c += c_step;
        if (c >= items_per_row) {
            c -= items_per_row;
            row += 1;
        }
    }
}

} // namespace pto_b200
