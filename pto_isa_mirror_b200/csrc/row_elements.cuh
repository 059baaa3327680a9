// Rows of fp32, bf16 or fp16 elements read sixteen at a time by the quantisers: wide loads, the largest magnitude.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace pto_b200 {

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

// Loads of what an earlier launch may still be writing when this one starts (programmatic serialisation). They stand behind
// ptx::grid_dependency_wait in the program, and have to stay there: as volatile asm, and never through the read-only path
// (.nc, __ldg, or what the compiler makes of a const __restrict__ source), which is for memory that nothing writes while the
// kernel runs.
// One float that every thread of a grid reads: through the first-level cache. (A volatile load passes it by: 2 us more for a
// cast of 4093x2904 and back.)
__device__ __forceinline__ float nv_ld_common(const float* ptr)
{
    float f;
    asm volatile("ld.global.ca.f32 %0, [%1];" : "=f"(f) : "l"(ptr) : "memory");
    return f;
}

__device__ __forceinline__ uint32_t nv_ld_byte(const uint8_t* ptr)
{
    uint32_t b;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(b) : "l"(ptr) : "memory");
    return b;
}

__device__ __forceinline__ uint32_t nv_ld_word_once(const void* ptr)
{
    uint32_t w;
    asm volatile("ld.global.cs.b32 %0, [%1];" : "=r"(w) : "l"(ptr) : "memory");
    return w;
}

__device__ __forceinline__ uint4 nv_ld16_once(const void* ptr)
{
    uint4 a;
    asm volatile("ld.global.cs.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w) : "l"(ptr) : "memory");
    return a;
}

// 32 bytes in one access (32-byte aligned): a warp's accesses are then whole lines. With two of 16 bytes each covers
// half of every sector (dequantising 16384 x 8192 to bf16 took 92 us that way).
__device__ __forceinline__ void nv_ld32(const void* ptr, uint4& a, uint4& b)
{
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(ptr)
                 : "memory");
}

__device__ __forceinline__ void nv_st32(void* ptr, const uint4& a, const uint4& b)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

// 16 consecutive elements, read once, as they lie in memory. VEC: what the address is a multiple of, 32 or 16 bytes.
template <int SRC>
struct NvRaw16 {
    static constexpr int kQuads = SRC == NV_F32 ? 4 : 2;
    uint4 q[kQuads];

    template <int VEC>
    __device__ __forceinline__ void load(const void* ptr)
    {
        if constexpr (VEC == 32) {
#pragma unroll
            for (int i = 0; i < kQuads; i += 2) {
                nv_ld32(static_cast<const uint4*>(ptr) + i, q[i], q[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
                q[i] = nv_ld16_once(static_cast<const uint4*>(ptr) + i);
            }
        }
    }
    __device__ __forceinline__ void load_some(const typename NvElem<SRC>::type* p, int n) // the first n, zeros behind
    {
        __align__(16) typename NvElem<SRC>::type part[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            part[j] = j < n ? p[j] : static_cast<typename NvElem<SRC>::type>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            q[i] = reinterpret_cast<const uint4*>(part)[i];
        }
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            q[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ uint32_t word(int i) const
    {
        const uint4& v = q[i / 4];
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
    __device__ __forceinline__ void unpack(float (&x)[16]) const
    {
#pragma unroll
        for (int i = 0; i < 4 * kQuads; ++i) {
            if constexpr (SRC == NV_F32) {
                x[i] = __uint_as_float(word(i));
            } else {
                nv_unpack2<SRC>(word(i), x[2 * i], x[2 * i + 1]);
            }
        }
    }
    // The largest magnitude as an fp32 pattern; an infinity or a NaN among the values gives a pattern of at least 0x7F800000.
    __device__ __forceinline__ uint32_t top() const
    {
        if constexpr (SRC == NV_F32) {
            uint32_t t = 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                t = max(t, word(i) & 0x7FFFFFFFu);
            }
            return t;
        } else if constexpr (SRC == NV_BF16) {
            __nv_bfloat162 t = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = word(i);
                t = __hmax2_nan(t, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
            }
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&t) & 0x7FFF7FFFu;
            return max(w << 16, w & 0xFFFF0000u);
        } else {
            __half2 t = __floats2half2_rn(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = word(i);
                t = __hmax2_nan(t, __habs2(*reinterpret_cast<const __half2*>(&w)));
            }
            const float2 f = __half22float2(t);
            return max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu);
        }
    }
};

} // namespace pto_b200
