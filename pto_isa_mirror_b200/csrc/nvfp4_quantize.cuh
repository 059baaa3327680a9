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
// quotient misses, and fp32 gives the codes that real arithmetic gives. It costs up to one binade at the top of e4m3's
// range: blocks that are small beside the tensor's maximum reach the subnormal scales, and zero, up to a factor of two
// earlier. Elsewhere the block scales keep their relative precision.
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

#include "row_elements.cuh"
#include "sm100_ptx.cuh"

namespace pto_b200 {

constexpr int kNvQuantThreads = 256;

// Exponent field of g for a tensor maximum: amax / 2688 rounded up to a power of two, 2688 = 1.3125 * 2^11. An infinity or a
// NaN counts as the largest number.
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

__device__ __forceinline__ uint64_t nv_pair(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ uint64_t nv_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t nv_mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// What every block of a tensor needs of its scale g = 2^(e - 127).
struct NvTensorScale {
    uint32_t e;
    float g, inv_g;
    bool plain; // s g and 1 / (s g) are normal numbers for every block scale s

    __device__ __forceinline__ explicit NvTensorScale(float amax)
    {
        e = nv_scale_exponent(amax);
        g = __uint_as_float(e << 23);
        inv_g = __uint_as_float((254u - e) << 23);
        plain = e >= 24u && e <= 230u;
    }
};

// One block with its largest magnitude `top` (an fp32 pattern): its e4m3 scale code and its sixteen codes.
// x / (s g) is rounded correctly: a quotient from the nearest reciprocal, then one correction by its exact remainder
// (Markstein's theorem). s g has four significant bits; the product with the reciprocal alone misses ties by one unit, and
// 1/16 of all bf16 quotients are ties.
__device__ __forceinline__ uint32_t nv_quantize_block(float (&x)[16], uint32_t top, const NvTensorScale& t, uint2& codes)
{
    codes = make_uint2(0u, 0u);
    if (top >= 0x7F800000u) {
        return 0x7Fu;
    }
    const float y_max = __uint_as_float(top) * t.inv_g;
    constexpr float kSixth = 1.0f / 6.0f;
    const float sixth = __fmul_rn(y_max, kSixth); // corrected as below; a NaN from an infinite y_max ends at 448 too
    const float m = __fmaf_rn(__fmaf_rn(-6.0f, sixth, y_max), kSixth, sixth);
    const uint32_t s_code = __nv_cvt_float_to_fp8(fminf(m, 448.0f), __NV_SATFINITE, __NV_E4M3);
    if (s_code == 0u) {
        return 0u;
    }
    const float s = nv_e4m3_to_float(s_code);
    // 1 / s to the nearest float: an approximation and one step of Newton's iteration. s has four significant bits, so no
    // 1 / s lies near the middle of two floats and the step's error cannot decide.
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = __fmaf_rn(r, __fmaf_rn(-s, r, 1.0f), r);
    if (t.plain && y_max <= 1.0e30f) {
        const float ri = r * t.inv_g, sg = -s * t.g; // powers of two: exact
        const uint64_t ri2 = nv_pair(ri, ri), sg2 = nv_pair(sg, sg);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint64_t v = nv_pair(x[i], x[i + 1]);
            const uint64_t q0 = nv_mul2(v, ri2);
            const uint64_t q = nv_fma2(nv_fma2(q0, sg2, v), ri2, q0);
            asm("mov.b64 {%0, %1}, %2;" : "=f"(x[i]), "=f"(x[i + 1]) : "l"(q));
        }
    } else { // a tensor near either end of fp32's range, or a caller's amax far below the data: one step more, clamped
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = fminf(fmaxf(x[i] * t.inv_g, -8192.0f), 8192.0f);
            const float q0 = __fmul_rn(y, r);
            x[i] = __fmaf_rn(__fmaf_rn(-q0, s, y), r, q0);
        }
    }
    codes.x = nv_cvt_e2m1x8(x);
    codes.y = nv_cvt_e2m1x8(x + 8);
    return s_code;
}

__device__ __forceinline__ uint32_t nv_top(const float (&x)[16])
{
    uint32_t t = 0u; // |x| as bits: the integer order is the value order, infinities and NaN above all numbers
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        t = max(t, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    }
    return t;
}

// Stores a block's codes and, once per four lanes, the scale word of four consecutive blocks. Every lane of the warp calls
// it; the four lanes of an aligned group hold blocks kb .. kb + 3 of one row, or none (row < 0). (With a mask per group
// the shuffles cost a synchronisation each: the address unit was busy 31 % of the time.)
__device__ __forceinline__ void nv_store_block(uint8_t* data, uint8_t* scales, long long ld_data, int rows, int k_blocks,
                                               int k_atoms, int row, int kb, uint32_t s_code, const uint2& codes)
{
    if (row >= 0 && row < rows && kb < k_blocks) {
        *reinterpret_cast<uint2*>(data + row * ld_data + static_cast<long long>(kb) * 8) = codes;
    }
    uint32_t word = s_code << (8 * (threadIdx.x & 3u));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
    if ((threadIdx.x & 3u) == 0u && row >= 0) {
        const long long tile = static_cast<long long>(row >> 7) * k_atoms + (kb >> 2);
        *reinterpret_cast<uint32_t*>(scales + tile * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4) = word;
    }
}

// src: [rows][ld_src]; VEC: rows start on 32- or 16-byte boundaries, 0: on any element. One thread per block of 16 and
// step, two blocks in flight.
constexpr int kNvItems = 2;

template <int SRC, int VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_quantize_kernel(const void* src, const float* amax, uint8_t* data,
                          uint8_t* scales, float* tensor_scale, int rows, int k,
                          long long ld_src, long long ld_data)
{
    using T = typename NvElem<SRC>::type;
    const int k_blocks = (k + 15) / 16;
    const int k_atoms = (k_blocks + 3) / 4;
    const int row_blocks = k_atoms * 4;                // blocks of a row, padding included
    const long long rows_padded = (static_cast<long long>(rows) + 127) / 128 * 128;
    const long long total = rows_padded * row_blocks;  // a multiple of 4, as the stride is: groups of four stay whole
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / row_blocks;
    const int kb_step = static_cast<int>(stride - row_step * row_blocks);
    long long row = i / row_blocks;
    int kb = static_cast<int>(i - row * row_blocks);
    ptx::grid_dependency_wait();
    const float top_of_tensor = nv_ld_common(amax);
    const NvTensorScale t(top_of_tensor);
    if (blockIdx.x == 0 && threadIdx.x == 0) { // a maximum gone wrong stays visible in every number and product
        *tensor_scale = isfinite(top_of_tensor) ? t.g : __uint_as_float(0x7FC00000u);
    }
    while (i - static_cast<int>(threadIdx.x & 31u) < total) { // the warp goes on together
        NvRaw16<SRC> raw[kNvItems];
        int rows_of[kNvItems], kbs[kNvItems];
#pragma unroll
        for (int u = 0; u < kNvItems; ++u) {
            rows_of[u] = i < total ? static_cast<int>(row) : -1;
            kbs[u] = kb;
            raw[u].zero();
            if (i < total && row < rows && kb < k_blocks) {
                const T* p = static_cast<const T*>(src) + row * ld_src + static_cast<long long>(kb) * 16;
                if (VEC != 0 && kb * 16 + 16 <= k) {
                    raw[u].template load<VEC>(p);
                } else {
                    raw[u].load_some(p, k - kb * 16);
                }
            }
            i += stride;
            row += row_step;
            kb += kb_step;
            if (kb >= row_blocks) {
                kb -= row_blocks;
                row += 1;
            }
        }
#pragma unroll
        for (int u = 0; u < kNvItems; ++u) {
            float x[16];
            raw[u].unpack(x);
            uint2 codes;
            const uint32_t s_code = nv_quantize_block(x, raw[u].top(), t, codes);
            nv_store_block(data, scales, ld_data, rows, k_blocks, k_atoms, rows_of[u], kbs[u], s_code, codes);
        }
    }
}

// The same of the transpose: blocks run down the columns of src [rows][ld_src], row c of the result is column c of src.
// A thread takes one column (two for 16-bit types with PAIRS: rows start on 4-byte boundaries) down 64 rows: loads are
// contiguous across the lanes, the codes of its four blocks are one 32-byte sector and their scales one word of a scale
// tile, so nothing is exchanged and nothing goes through shared memory. Columns past k fill the padding with zeros.
// (Through a shared-memory tile of 256 x 64: 118 us for bf16 and 249 us for fp32 on 16384 x 8192.)
template <int SRC, bool PAIRS>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_quantize_transposed_kernel(const void* src, const float* amax,
                                     uint8_t* data, uint8_t* scales,
                                     float* tensor_scale, int rows, int k, long long ld_src, long long ld_data)
{
    using T = typename NvElem<SRC>::type;
    constexpr int kCols = PAIRS ? 2 : 1;
    const int k_atoms = (rows + 63) / 64; // the result's rows run over src's rows
    const int col_items = (k + 127) / 128 * (128 / kCols);
    const long long total = static_cast<long long>(k_atoms) * col_items;
    const bool wide = (reinterpret_cast<uintptr_t>(data) & 31u) == 0 && (ld_data & 31) == 0;
    ptx::grid_dependency_wait();
    const float top_of_tensor = nv_ld_common(amax);
    const NvTensorScale t(top_of_tensor);
    if (blockIdx.x == 0 && threadIdx.x == 0) { // a maximum gone wrong stays visible in every number and product
        *tensor_scale = isfinite(top_of_tensor) ? t.g : __uint_as_float(0x7FC00000u);
    }
    for (long long it = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; it < total;
         it += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int atom = static_cast<int>(it / col_items);
        const int col = static_cast<int>(it - static_cast<long long>(atom) * col_items) * kCols;
        const int row0 = atom * 64;
        const int blocks = min(4, (rows - row0 + 15) / 16);
        const bool full = row0 + 64 <= rows && col + kCols <= k;
        uint2 codes[kCols][4];
        uint32_t word[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            word[c] = 0u;
        }
        const T* p = static_cast<const T*>(src) + static_cast<long long>(row0) * ld_src + col;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float x[kCols][16];
            if (full) { // sixteen loads in flight
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const T* at = p + static_cast<long long>(b * 16 + j) * ld_src;
                    if constexpr (PAIRS) {
                        nv_unpack2<SRC>(nv_ld_word_once(at), x[0][j], x[1][j]);
                    } else {
                        x[0][j] = nv_to_float<SRC>(*at);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        x[c][j] = 0.0f;
                        if (row0 + b * 16 + j < rows && col + c < k) {
                            x[c][j] = nv_to_float<SRC>(p[static_cast<long long>(b * 16 + j) * ld_src + c]);
                        }
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                word[c] |= nv_quantize_block(x[c], nv_top(x[c]), t, codes[c][b]) << (8 * b);
            }
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int out_row = col + c;
            if (out_row < k) {
                uint8_t* dst = data + out_row * ld_data + static_cast<long long>(atom) * 32;
                if (wide && blocks == 4) {
                    nv_st32(dst, make_uint4(codes[c][0].x, codes[c][0].y, codes[c][1].x, codes[c][1].y),
                            make_uint4(codes[c][2].x, codes[c][2].y, codes[c][3].x, codes[c][3].y));
                } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if (b < blocks) {
                            reinterpret_cast<uint2*>(dst)[b] = codes[c][b];
                        }
                    }
                }
            }
            const long long tile = static_cast<long long>(out_row >> 7) * k_atoms + atom;
            *reinterpret_cast<uint32_t*>(scales + tile * 512 + (out_row & 31) * 16 + ((out_row >> 5) & 3) * 4) = word[c];
        }
    }
}

template <int SRC>
__device__ __forceinline__ uint32_t nv_finite_top(const NvRaw16<SRC>& raw)
{
    uint32_t top = raw.top();
    if (top >= 0x7F800000u) { // an infinity or a NaN among them: the others one by one
        float x[16];
        raw.unpack(x);
        top = 0u;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t bits = __float_as_uint(x[j]) & 0x7FFFFFFFu;
            top = max(top, bits < 0x7F800000u ? bits : 0u);
        }
    }
    return top;
}

// Largest finite |x| of a matrix into *out: by a maximum with what the caller has set to zero, or (a single block) stored.
// The maximum does not depend on the order.
constexpr int kAmaxSingleThreads = 1024;
constexpr int kAmaxSingleElems = 65536; // what one block of that many threads is given at most

template <int SRC, int VEC>
__global__ void __launch_bounds__(kAmaxSingleThreads)
    amax_kernel(const void* src, uint32_t* out, int rows, int k, long long ld_src)
{
    using T = typename NvElem<SRC>::type;
    constexpr int kAmaxItems = SRC == NV_F32 ? 2 : 4; // 128 bytes in flight per thread
    const int row_items = (k + 15) / 16;
    const long long total = static_cast<long long>(rows) * row_items;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / row_items;
    const int c_step = static_cast<int>(stride - row_step * row_items);
    long long row = i / row_items;
    int c = static_cast<int>(i - row * row_items);
    uint32_t top = 0u;
    while (i < total) {
        NvRaw16<SRC> raw[kAmaxItems];
#pragma unroll
        for (int u = 0; u < kAmaxItems; ++u) {
            raw[u].zero();
            if (i < total) {
                const T* p = static_cast<const T*>(src) + row * ld_src + static_cast<long long>(c) * 16;
                if (VEC != 0 && c * 16 + 16 <= k) {
                    raw[u].template load<VEC>(p);
                } else {
                    raw[u].load_some(p, k - c * 16);
                }
            }
            i += stride;
            row += row_step;
            c += c_step;
            if (c >= row_items) {
                c -= row_items;
                row += 1;
            }
        }
#pragma unroll
        for (int u = 0; u < kAmaxItems; ++u) {
            top = max(top, nv_finite_top(raw[u]));
        }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    __shared__ uint32_t part[kAmaxSingleThreads / 32];
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        top = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x < blockDim.x / 32 ? part[threadIdx.x] : 0u);
        if (threadIdx.x == 0) {
            if (gridDim.x == 1) {
                *out = top;
            } else if (top != 0u) {
                atomicMax(out, top);
            }
        }
    }
}

// Few rows: the largest magnitude and the codes in one launch. A cluster of up to eight CTAs holds the matrix in registers
// between the two, kNvItems blocks of 16 per thread, and exchanges its maxima over distributed shared memory. The CTAs have
// 256, 512 or 1024 threads, the fewest that hold it, since large ones start and meet slowly: 8x4096 bf16 2.9 us with 256,
// 4.1 with 1024 (2.6 as it is launched now). In two launches / in one: 1x4096 4.4 / 2.8, 8x4096 4.9 / 2.6, 64x4096 7.4 / 4.9.
constexpr int kNvOneCtas = 8;
constexpr int kNvOneBlocks = kNvOneCtas * 1024 * kNvItems; // of 16 elements, a row's filled up to 64

template <int SRC, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS)
    nvfp4_quantize_one_kernel(const void* src, float* amax, uint8_t* data,
                              uint8_t* scales, float* tensor_scale, int rows, int k,
                              long long ld_src, long long ld_data)
{
    using T = typename NvElem<SRC>::type;
    __shared__ __align__(16) uint32_t part[32];
    const int k_blocks = (k + 15) / 16;
    const int k_atoms = (k_blocks + 3) / 4;
    const int row_blocks = k_atoms * 4;
    const int total = rows * row_blocks; // at most 16 THREADS, and a multiple of 4: the groups of nv_store_block stay whole
    const int ctas = static_cast<int>(gridDim.x); // the cluster
    const int first = static_cast<int>(blockIdx.x * THREADS + threadIdx.x);
    ptx::grid_dependency_wait(); // the launch may overlap the end of the one before (programmatic serialisation)
    NvRaw16<SRC> raw[kNvItems];
    int rows_of[kNvItems], kbs[kNvItems];
#pragma unroll
    for (int u = 0; u < kNvItems; ++u) {
        const int i = first + u * ctas * THREADS;
        rows_of[u] = i < total ? i / row_blocks : -1;
        kbs[u] = i < total ? i - rows_of[u] * row_blocks : 0;
        raw[u].zero();
        if (i < total && kbs[u] < k_blocks) {
            const T* p = static_cast<const T*>(src) + rows_of[u] * ld_src + kbs[u] * 16ll;
            if (VEC != 0 && kbs[u] * 16 + 16 <= k) {
                raw[u].template load<VEC>(p);
            } else {
                raw[u].load_some(p, k - kbs[u] * 16);
            }
        }
    }
    // scales of the rows that fill up the last tiles, meanwhile: word w of a tile is row w / 4 + 32 (w % 4)
    if ((rows & 127) != 0) {
        uint32_t* tiles = reinterpret_cast<uint32_t*>(scales + static_cast<long long>(rows >> 7) * k_atoms * 512);
        for (int w = first; w < k_atoms * 128; w += ctas * THREADS) {
            if (((w & 127) >> 2) + 32 * (w & 3) >= (rows & 127)) {
                tiles[w] = 0u;
            }
        }
    }
    uint32_t top = 0u;
#pragma unroll
    for (int u = 0; u < kNvItems; ++u) {
        top = max(top, nv_finite_top(raw[u]));
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    const int lane = static_cast<int>(threadIdx.x & 31u);
    if (lane == 0) {
        part[threadIdx.x >> 5] = top;
    }
    if (threadIdx.x < 32 && threadIdx.x >= THREADS / 32) {
        part[threadIdx.x] = 0u;
    }
    if (ctas > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
        const uint32_t at = ptx::smem_u32(part) + 16u * (lane & 7); // eight lanes read one CTA's 32 maxima
        top = 0u;
#pragma unroll
        for (int r = 0; r < kNvOneCtas; r += 4) {
            if (r + (lane >> 3) < ctas) {
                const float4 v = ptx::ld_shared_cluster_f32x4(ptx::map_to_cta(at, static_cast<uint32_t>(r + (lane >> 3))));
                top = max(max(top, max(__float_as_uint(v.x), __float_as_uint(v.y))),
                          max(__float_as_uint(v.z), __float_as_uint(v.w)));
            }
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        ptx::cluster_arrive(); // has read: the releasing form, behind which no read of another CTA is under way any more
    } else {
        __syncthreads();
        top = __reduce_max_sync(0xFFFFFFFFu, part[lane]);
    }
    const NvTensorScale t(__uint_as_float(top));
    if (first == 0) {
        *amax = __uint_as_float(top);
        *tensor_scale = t.g;
    }
#pragma unroll
    for (int u = 0; u < kNvItems; ++u) {
        float x[16];
        raw[u].unpack(x);
        uint2 codes;
        const uint32_t s_code = nv_quantize_block(x, raw[u].top(), t, codes);
        nv_store_block(data, scales, ld_data, rows, k_blocks, k_atoms, rows_of[u], kbs[u], s_code, codes);
    }
    if (ctas > 1) {
        ptx::cluster_wait(); // no CTA leaves while another reads its maxima
    }
}

// Two e2m1 codes (a byte) -> two halves.
__device__ __forceinline__ __half2 nv_e2m1x2_to_half2(uint32_t byte)
{
    uint32_t h;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "}"
        : "=r"(h)
        : "r"(byte));
    return *reinterpret_cast<const __half2*>(&h);
}

// Back to numbers: code * s is exact in fp16 (six significant bits, at most 2688 and at least 2^-10), then one rounding by
// g (none when g is a power of two) and one by the output type. One thread per 32 bytes of the result - 8 or 16
// elements - two of them in flight. VEC: the result's rows start on 32-byte boundaries.
template <int DST, bool VEC>
__global__ void __launch_bounds__(kNvQuantThreads)
    nvfp4_dequantize_kernel(const uint8_t* data, const uint8_t* scales,
                            const float* tensor_scale, void* out, int rows, int k,
                            long long ld_data, long long ld_out)
{
    using T = typename NvElem<DST>::type;
    constexpr int kElems = 32 / static_cast<int>(sizeof(T));
    constexpr int kWords = kElems / 8;
    const int row_items = (k + kElems - 1) / kElems;
    const int k_atoms = (k + 63) / 64;
    ptx::grid_dependency_wait();
    const float g = tensor_scale != nullptr ? nv_ld_common(tensor_scale) : 1.0f;
    const long long total = static_cast<long long>(rows) * row_items;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / row_items;
    const int c_step = static_cast<int>(stride - row_step * row_items);
    long long row = i / row_items;
    int c = static_cast<int>(i - row * row_items);
    while (i < total) {
        uint32_t codes[kNvItems][kWords], s_code[kNvItems];
        long long rows_of[kNvItems];
        int cs[kNvItems];
#pragma unroll
        for (int u = 0; u < kNvItems; ++u) {
            rows_of[u] = -1;
            if (i < total) {
                rows_of[u] = row;
                cs[u] = c;
                const uint32_t* p = reinterpret_cast<const uint32_t*>(data + row * ld_data) + static_cast<long long>(c) * kWords;
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    codes[u][w] = c * kElems + 8 * w < k ? nv_ld_word_once(p + w) : 0u;
                }
                const int kb = c * kElems / 16;
                const long long tile = (row >> 7) * k_atoms + (kb >> 2);
                s_code[u] = nv_ld_byte(scales + tile * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (kb & 3));
            }
            i += stride;
            row += row_step;
            c += c_step;
            if (c >= row_items) {
                c -= row_items;
                row += 1;
            }
        }
#pragma unroll
        for (int u = 0; u < kNvItems; ++u) {
            if (rows_of[u] < 0) {
                continue;
            }
            const __half_raw sr = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(s_code[u]), __NV_E4M3);
            const __half2 s = __half2half2(*reinterpret_cast<const __half*>(&sr));
            __align__(16) T o[kElems];
#pragma unroll
            for (int j = 0; j < kElems / 2; ++j) {
                const float2 f = __half22float2(__hmul2(nv_e2m1x2_to_half2((codes[u][j / 4] >> (8 * (j & 3))) & 0xFFu), s));
                o[2 * j] = static_cast<T>(__fmul_rn(f.x, g));
                o[2 * j + 1] = static_cast<T>(__fmul_rn(f.y, g));
            }
            T* dst = static_cast<T*>(out) + rows_of[u] * ld_out + static_cast<long long>(cs[u]) * kElems;
            if (VEC && cs[u] * kElems + kElems <= k) {
                nv_st32(dst, reinterpret_cast<const uint4*>(o)[0], reinterpret_cast<const uint4*>(o)[1]);
            } else {
#pragma unroll
                for (int j = 0; j < kElems; ++j) {
                    if (cs[u] * kElems + j < k) {
                        dst[j] = o[j];
                    }
                }
            }
        }
    }
}

} // namespace pto_b200
