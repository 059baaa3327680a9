// Weight gradient from an activation kept in 8 bits (MXFP8), on sm_100a:
//   dW[n][k] = sum_t dy[t][n] * x[t][k] * 2^(e[t][k/32] - 127)   (+ addend[n][k])
// dy [T][N] bf16 or fp16, x [T][K] e4m3 bytes with one e8m0 scale per 32 elements of a row: the pair the forward pass
// quantised, read as it is. The sum runs over tokens, so both operands lie with their summed index outermost
// ("MN-major"): the tensor core takes them in that order from 128-byte swizzled rows and nothing is transposed.
//
// x becomes 16-bit on the way: every e4m3 value times a power of two is a bf16 value exactly (below 2^-126 in magnitude:
// rounded), and an fp16 value where it lies in fp16's range (above it: infinity, below 2^-14: rounded). So dy meets the numbers the checkpoint stands for, at the 16-bit rate of the tensor core.
//
// Two ways to the same bits. Without scratch memory x is converted tile by tile in shared memory, beside the products
// (SCRATCH = false); every tile of x then is converted once for each 256 columns of dy. With scratch for T x K 16-bit
// values x is converted once, by mx_to_16bit_kernel, and both operands come by TMA (SCRATCH = true): at 16384x8192x8192
// 60 us more traffic, but the products run at nearly the rate of a 16-bit GEMM.
//
// A cluster holds `splits` CTA pairs. A pair owns a 256 (k) x 256 (n) tile, or with splits > 1 its part of the
// tokens of one. x is the 256-row side of the product and each CTA converts its own 128: half as many elements per SM as
// on the 256-column side of a single-CTA tile. Roles per CTA:
//   warp 0, 2    TMA loads of dy and of x
//   warp 1       products (even CTA: cta_group::2)
//   warps 4..19  four groups of four, one warp of each per scheduler; a group converts every fourth stage and keeps the
//                fp32 sums of 64 of the 256 columns
// What limits such a kernel is issue slots, not bandwidth: the converting warps leave few, and a role with its own warp
// runs at some eight cycles per instruction beside them. So a group takes a whole stage at a time (waits and counters
// once per 64 values of a thread), scales are fetched by the threads that use them, and the product warp keeps its
// descriptors in uniform registers (its issue alone took 800 cycles of a stage's 513 before).
//
// Sums: the tensor core adds into its accumulator by cutting off, not by rounding. One accumulator for all tokens would lose
// (measured here, relative, normal numbers / of one sign) 8.8e-6 / 3.5e-5 of 16384 of them and 2.1e-5 / 9.1e-5 of 32768. So
// an accumulator takes kWgFoldStages x 64 = 1024 tokens at most; the converting warps then add it to fp32 sums in their
// registers, with rounding, while the other accumulator fills.
// Relative error of 16384 tokens, and time of 16384x8192x8192 with and without scratch, by tokens per accumulator:
//   2048   6.3e-7 (terms of one sign 2.4e-6)   1456 / 1739 us
//   1024   2.9e-7 (9.5e-7)                     1440 / 1778 us
//    512   1.5e-7 (3.6e-7)                     1470 / 1863 us
//    256   1.1e-7 (1.5e-7)                     1515 / 2595 us
// A plain fp32 matrix product of the same numbers has 5.7e-7 there.
// With splits > 1 the parts are added over distributed shared memory in rank order. No atomics: the result does not
// depend on timing.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "gemm_tile_loop.cuh"
#include "row_elements.cuh"
#include "sm100_ptx.cuh"

namespace pto_b200 {

constexpr int kWgThreads = 640;
constexpr int kWgWorkerWarps = 16;
constexpr int kWgGroups = 4;      // of four converting warps; a group takes every fourth stage
constexpr int kWgStages = 6;      // ring of dy tiles and converted x tiles
constexpr int kWgRawStages = 4;   // ring of x tiles as they come: one place per group
static_assert(kWgRawStages == kWgGroups, "a group reads its own place of the ring of x");
// registers: 96 at launch; the loading and multiplying warps give back what the sums need
constexpr int kWgRegsOthers = 32, kWgRegsWorkers = 112;
static_assert(128 * kWgRegsOthers + 512 * kWgRegsWorkers <= kWgThreads * 96, "register split within the launch's total");
constexpr int kWgStageTokens = 64;
constexpr int kWgFoldStages = 16;
static_assert(kWgFoldStages >= kWgStages + kWgGroups, "an accumulator is read before its second successor needs it");

constexpr int ST_WG_PRODUCER = 31;
constexpr int ST_WG_MMA = 32;
constexpr int ST_WG_WORKER = 33;

enum WgOut : int { WG_OUT_F32 = 0, WG_OUT_BF16 = 1, WG_OUT_F16 = 2 };

struct WgradParams {
    void* out;
    const void* addend;   // of out's type, or null; may be out itself
    const uint8_t* scales;
    long long ld_out, ld_addend, ld_scales;
    int t, n, k;
    int k_tiles, n_tiles, group;
    int stages;           // 64-token stages of T
    int splits;
    uint32_t idesc;
    int* status;
    long long wait_limit;
};

struct WgSmem {
    static constexpr int kDyBytes = kWgStageTokens * 128 * 2; // this CTA's 128 columns of dy: two blocks of 64 columns
    static constexpr int kXBytes = kWgStageTokens * 128 * 2;  // converted x: two blocks of 64 columns
    static constexpr int kRawBytes = kWgStageTokens * 128;
    static constexpr int kXOff = kWgStages * kDyBytes;
    static constexpr int kRawOff = kXOff + kWgStages * kXBytes;
    static constexpr int kBarOff = kRawOff + kWgRawStages * kRawBytes;
    static constexpr int kNumBars = 2 * kWgStages + 2 * kWgRawStages + 4;
    static constexpr int kMiscOff = kBarOff + kNumBars * 8;
    static constexpr int kTotal = kMiscOff + 16 + 1024;
};
static_assert(WgSmem::kTotal <= 227 * 1024, "shared memory of the weight-gradient kernel");
static_assert(256 * 128 * 4 <= WgSmem::kRawOff, "partial sums reuse the ring");

// 2^(e - 127): e = 0 is the subnormal 2^-127, e = 255 a NaN.
__device__ __forceinline__ float wg_scale(uint32_t e)
{
    return __uint_as_float(e == 0u ? 0x00400000u : e == 255u ? 0x7FC00000u : e << 23);
}

__device__ __forceinline__ uint32_t wg_e4m3x2_to_f16x2(uint32_t two)
{
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
    return static_cast<uint32_t>(r.x) | (static_cast<uint32_t>(r.y) << 16);
}

// Sixteen e4m3 bytes times 2^(e - 127) -> sixteen 16-bit values, whatever the bytes and e: through fp32.
template <bool F16>
__device__ __forceinline__ void wg_convert16_any(const uint4& raw, uint32_t e, uint32_t (&o)[8])
{
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const float scale = wg_scale(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t h = wg_e4m3x2_to_f16x2((w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        const float lo = f.x * scale, hi = f.y * scale;
        if constexpr (F16) {
            const __half2 v = __floats2half2_rn(lo, hi);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            // exact but below 2^-126, where it rounds as the short form's multiplication does: which of the two a value meets
            // depends on its neighbours
            const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
}

// The same in the fewest instructions, for the scales and bytes that activations have; wg_needs_any() says where it does
// not hold. One multiplication per two values, exact but for results below the type's normal range, rounded once.
// bf16: the byte's fields are put where bf16 has them, sign | 0000 eeee | mmm 0000, which is the value times 2^-120, and
//       multiplied by 2^(e - 7). High and low bytes are made for four values at a time.
// fp16: the conversion instruction, then 2^(e - 127) as an fp16 number.
template <bool F16>
__device__ __forceinline__ void wg_convert16(const uint4& raw, uint32_t e, uint32_t (&o)[8])
{
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (F16) {
        const float f = __uint_as_float(e << 23);
        const __half2 factor = __floats2half2_rn(f, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t h = wg_e4m3x2_to_f16x2((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu);
            const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h), factor);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    } else {
        const uint32_t f = e * 0x00800080u + 0x3C003C00u; // (e - 7 + 127) << 7, twice
        const __nv_bfloat162 factor = *reinterpret_cast<const __nv_bfloat162*>(&f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t low = (w[i] << 4) & 0xF0F0F0F0u;
            const uint32_t high = ((w[i] >> 4) & 0x07070707u) | (w[i] & 0x80808080u);
            const uint32_t a = __byte_perm(low, high, 0x5140), b = __byte_perm(low, high, 0x7362);
            const __nv_bfloat162 va = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), factor);
            const __nv_bfloat162 vb = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&b), factor);
            o[2 * i] = *reinterpret_cast<const uint32_t*>(&va);
            o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&vb);
        }
    }
}

// Whether wg_convert16 does not hold for some of a thread's pieces: a scale whose factor has no number of the type, or
// (bf16) a NaN among the bytes, 0x7F or 0xFF - the bytes whose top bit an added one flips.
template <bool F16>
__device__ __forceinline__ bool wg_needs_any(const uint4 (&in)[4], const uint32_t (&e)[4])
{
    const uint32_t top = max(max(e[0], e[1]), max(e[2], e[3]));
    if constexpr (F16) {
        const uint32_t low = min(min(e[0], e[1]), min(e[2], e[3]));
        return top > 142u || low < 103u;
    } else {
        uint32_t flips = 0u;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            flips |= (in[h].x + 0x01010101u) ^ in[h].x;
            flips |= (in[h].y + 0x01010101u) ^ in[h].y;
            flips |= (in[h].z + 0x01010101u) ^ in[h].z;
            flips |= (in[h].w + 0x01010101u) ^ in[h].w;
        }
        return top > 134u || (flips & 0x80808080u) != 0u;
    }
}

template <int OUT>
struct WgElem {
    using type = float;
};
template <>
struct WgElem<WG_OUT_BF16> {
    using type = __nv_bfloat16;
};
template <>
struct WgElem<WG_OUT_F16> {
    using type = __half;
};

// x [rows][k] as 16-bit values, contiguous rows on 32-byte boundaries: 16 values per thread and step.
constexpr int kWgConvertThreads = 256;

template <bool F16>
__global__ void __launch_bounds__(kWgConvertThreads) mx_to_16bit_kernel(const uint8_t* data,
                                                                         const uint8_t* scales,
                                                                         uint16_t* out, int rows, int k,
                                                                         long long ld_data, long long ld_scales)
{
    const int row_items = k / 16;
    const long long total = static_cast<long long>(rows) * row_items;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const long long row_step = stride / row_items;
    const int c_step = static_cast<int>(stride - row_step * row_items);
    long long row = i / row_items;
    int c = static_cast<int>(i - row * row_items);
    constexpr int kItems = 4;
    ptx::grid_dependency_wait();
    while (i < total) {
        uint4 in[kItems];
        uint32_t e[kItems];
        long long at[kItems];
#pragma unroll
        for (int u = 0; u < kItems; ++u) {
            at[u] = i < total ? i : -1;
            in[u] = make_uint4(0u, 0u, 0u, 0u);
            e[u] = 127u;
            if (i < total) {
                in[u] = nv_ld16_once(reinterpret_cast<const uint4*>(data + row * ld_data) + c);
                e[u] = nv_ld_byte(scales + row * ld_scales + (c >> 1));
            }
            i += stride;
            row += row_step;
            c += c_step;
            if (c >= row_items) {
                c -= row_items;
                row += 1;
            }
        }
        const bool any = wg_needs_any<F16>(in, e);
#pragma unroll
        for (int u = 0; u < kItems; ++u) {
            uint32_t o[8];
            if (!any) {
                wg_convert16<F16>(in[u], e[u], o);
            } else {
                wg_convert16_any<F16>(in[u], e[u], o);
            }
            if (at[u] >= 0) {
                nv_st32(out + at[u] * 16, make_uint4(o[0], o[1], o[2], o[3]), make_uint4(o[4], o[5], o[6], o[7]));
            }
        }
    }
}

// A tile whose tokens were cut over SPLITS pairs: their partial sums [256 n][128 k] lie at the same place of each CTA's
// shared memory, and CTA `split` of a side adds its share of them in rank order, four k per thread and step. The arrival
// that lets the other CTAs leave comes behind the last step's reads, in the releasing form, behind which no read is under
// way, and in front of that step's stores. By the 512 threads of the converting warps.
template <int SPLITS, int OUT>
__device__ __forceinline__ void wg_add_parts(const WgradParams& p, uint32_t base, int split, int side, int k0, int n0, int thread)
{
    constexpr int kThreads = kWgWorkerWarps * 32;
    constexpr int kSteps = 256 * 32 / SPLITS / kThreads;
    using T = typename WgElem<OUT>::type;
    const int first = split * kSteps * kThreads + thread;
    const int k = k0 + (first & 31) * 4; // of every step
#pragma unroll 1
    for (int j = 0; j < kSteps; ++j) {
        const int i = first + j * kThreads;
        const int n = n0 + (i >> 5);
        const bool mine = k < p.k && n < p.n; // p.k is a multiple of 32
        float4 part[SPLITS];
#pragma unroll
        for (int s = 0; s < SPLITS; ++s) {
            part[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (mine) {
                part[s] = ptx::ld_shared_cluster_f32x4(
                    ptx::map_to_cta(base + 16u * static_cast<uint32_t>(i), static_cast<uint32_t>(2 * s + side)));
            }
        }
        float4 f = part[0];
#pragma unroll
        for (int s = 1; s < SPLITS; ++s) {
            f.x += part[s].x;
            f.y += part[s].y;
            f.z += part[s].z;
            f.w += part[s].w;
        }
        if (j == kSteps - 1) {
            __syncwarp();
            ptx::cluster_arrive();
        }
        if (mine) {
            if (p.addend != nullptr) {
                const T* add = static_cast<const T*>(p.addend) + n * p.ld_addend + k;
                const T v[4] = {add[0], add[1], add[2], add[3]};
                f.x += static_cast<float>(v[0]);
                f.y += static_cast<float>(v[1]);
                f.z += static_cast<float>(v[2]);
                f.w += static_cast<float>(v[3]);
            }
            T* at = static_cast<T*>(p.out) + n * p.ld_out + k;
            at[0] = static_cast<T>(f.x);
            at[1] = static_cast<T>(f.y);
            at[2] = static_cast<T>(f.z);
            at[3] = static_cast<T>(f.w);
        }
    }
}

template <bool F16, int OUT, bool SCRATCH>
__global__ void __launch_bounds__(kWgThreads, 1)
    gemm_wgrad_mx(const __grid_constant__ CUtensorMap tmap_dy, const __grid_constant__ CUtensorMap tmap_x, const WgradParams p)
{
    using L = WgSmem;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff); // even CTA: dy landed, x converted, in both CTAs
    uint64_t* empty_bar = full_bar + kWgStages;                         // each CTA: products have read the stage
    uint64_t* raw_full_bar = empty_bar + kWgStages;                     // each CTA: x landed
    uint64_t* raw_empty_bar = raw_full_bar + kWgRawStages;              // each CTA: x read by the converting warps
    uint64_t* acc_full_bar = raw_empty_bar + kWgRawStages;              // each CTA: an accumulator is finished
    uint64_t* acc_empty_bar = acc_full_bar + 2;                         // even CTA: sixteen warps have read it
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = ptx::cluster_ctarank();
    const uint32_t leader_rank = cta_rank & ~1u;
    const bool leader = (cta_rank == leader_rank);
    const int side = static_cast<int>(cta_rank & 1u);
    const int split = static_cast<int>(cta_rank >> 1);
    const uint16_t pair_mask = static_cast<uint16_t>(3u << leader_rank);
    const int cluster_ctas = 2 * p.splits;
    const int cluster = static_cast<int>(blockIdx.x) / cluster_ctas;
    const int clusters = static_cast<int>(gridDim.x) / cluster_ctas;
    const int tiles = p.k_tiles * p.n_tiles;
    const int first_stage = static_cast<int>(static_cast<long long>(p.stages) * split / p.splits);
    const int last_stage = static_cast<int>(static_cast<long long>(p.stages) * (split + 1) / p.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kWgStages; ++s) {
            // dy's bytes (with SCRATCH x's too), and a converting group in each CTA
            ptx::mbar_init(&full_bar[s], SCRATCH ? 1 : 1 + 2 * (kWgWorkerWarps / kWgGroups));
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < kWgRawStages; ++s) {
            ptx::mbar_init(&raw_full_bar[s], 1);
            ptx::mbar_init(&raw_empty_bar[s], kWgWorkerWarps / kWgGroups);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(&acc_full_bar[a], 1);
            ptx::mbar_init(&acc_empty_bar[a], 2 * kWgWorkerWarps);
        }
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_dy);
        ptx::prefetch_tensormap(&tmap_x);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(tmem_base_slot, kTmemCols);
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive(); // the peer's barriers must exist before anything is signalled across the pair: cluster_wait below
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_base_slot;
    // The set-up may overlap the end of the launch before (programmatic serialisation, 0.4 us); nothing of its is read or
    // overwritten before it has ended.
    ptx::grid_dependency_wait();

    auto tile_of = [&](int tile, int& ki, int& ni) { // grouped raster: a wave of pairs shares few columns of dy and x
        const int group_size = p.group * p.n_tiles;
        const int g = tile / group_size;
        const int first = g * p.group;
        const int rows = min(p.k_tiles - first, p.group);
        const int r = tile - g * group_size;
        ki = first + r % rows;
        ni = r / rows;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWgRegsOthers));
        ptx::cluster_wait();
        if (warp == 0) {
            // ---------------------------------------------------------------- loads of dy (with SCRATCH of x, too)
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = cluster; ok && tile < tiles; tile += clusters) {
                int ki, ni;
                tile_of(tile, ki, ni);
                const int k0 = ki * 256 + side * 128;
                const int n0 = ni * 256 + side * 128;
                for (int st = first_stage; st < last_stage; ++st) {
                    const int token = st * kWgStageTokens;
                    ok = bounded_wait_quiet_warp(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, ST_WG_PRODUCER, p.wait_limit);
                    if (!ok) {
                        break;
                    }
                    if (ptx::elect_one()) {
                        if (leader) {
                            ptx::mbar_arrive_expect_tx(&full_bar[stage], 2u * (L::kDyBytes + (SCRATCH ? L::kXBytes : 0)));
                        }
                        const uint32_t full_addr = ptx::map_to_cta(ptx::smem_u32(&full_bar[stage]), leader_rank);
                        uint8_t* dst = smem + stage * L::kDyBytes;
                        ptx::tma_load_2d_pair(dst, &tmap_dy, full_addr, n0, token);
                        ptx::tma_load_2d_pair(dst + 8192, &tmap_dy, full_addr, n0 + 64, token);
                        if constexpr (SCRATCH) {
                            uint8_t* x = smem + L::kXOff + stage * L::kXBytes;
                            ptx::tma_load_2d_pair(x, &tmap_x, full_addr, k0, token);
                            ptx::tma_load_2d_pair(x + 8192, &tmap_x, full_addr, k0 + 64, token);
                        }
                    }
                    __syncwarp();
                    if (++stage == kWgStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
#pragma unroll 1
            for (int i = 0; ok && i < kWgStages; ++i) { // the even CTA's last signals have come before this CTA may leave
                ok = bounded_wait_quiet_warp(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, ST_WG_PRODUCER, p.wait_limit);
                if (++stage == kWgStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        } else if (warp == 2) {
            // ---------------------------------------------------------------- loads of x, as far ahead as their own ring goes
            if (!SCRATCH && lane == 0) {
                int raw = 0;
                uint32_t phase = 0;
                bool ok = true;
                for (int tile = cluster; ok && tile < tiles; tile += clusters) {
                    int ki, ni;
                    tile_of(tile, ki, ni);
                    const int k0 = ki * 256 + side * 128;
                    for (int st = first_stage; st < last_stage; ++st) {
                        ok = bounded_wait_quiet(&raw_empty_bar[raw], phase ^ 1u, abort_flag, p.status, ST_WG_PRODUCER, p.wait_limit);
                        if (!ok) {
                            break;
                        }
                        ptx::mbar_arrive_expect_tx(&raw_full_bar[raw], L::kRawBytes);
                        ptx::tma_load_2d(smem + L::kRawOff + raw * L::kRawBytes, &tmap_x, &raw_full_bar[raw], k0,
                                         st * kWgStageTokens);
                        if (++raw == kWgRawStages) {
                            raw = 0;
                            phase ^= 1u;
                        }
                    }
                }
            }
        } else if (warp == 1 && leader) {
            // ---------------------------------------------------------------- products (even CTA)
            // The whole warp walks the stages and one elected lane issues, so addresses and descriptors stay in uniform
            // registers: beside the converting warps this warp gets few issue slots, and each instruction it saves counts.
            int stage = 0, acc = 0, in_part = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            const uint64_t x_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kXOff), 8192, 1024, ptx::kSwizzle128B);
            const uint64_t dy_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem), 8192, 1024, ptx::kSwizzle128B);
            const int stages = last_stage - first_stage;
            for (int tile = cluster; ok && tile < tiles; tile += clusters) {
                for (int st = 0; st < stages; ++st) {
                    if (in_part == 0) {
                        ok = bounded_wait_quiet_warp(&acc_empty_bar[acc], acc_phase ^ 1u, abort_flag, p.status, ST_WG_MMA, p.wait_limit);
                        if (!ok) {
                            break;
                        }
                    }
                    ok = bounded_wait_quiet_warp(&full_bar[stage], phase, abort_flag, p.status, ST_WG_MMA, p.wait_limit);
                    if (!ok) {
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const bool last = in_part == kWgFoldStages - 1 || st == stages - 1;
                    if (ptx::elect_one()) {
                        // 16 tokens, 16 rows of 128 bytes, per instruction (descriptor addresses count 16 bytes)
                        const uint64_t x_desc = x_desc0 + static_cast<uint64_t>(stage * (L::kXBytes / 16));
                        const uint64_t dy_desc = dy_desc0 + static_cast<uint64_t>(stage * (L::kDyBytes / 16));
                        ptx::umma_f16_pair(tmem_base + 256u * acc, x_desc, dy_desc, p.idesc, in_part != 0 ? 1u : 0u);
#pragma unroll
                        for (int kk = 1; kk < kWgStageTokens / 16; ++kk) {
                            ptx::umma_f16_pair(tmem_base + 256u * acc, x_desc + kk * 128, dy_desc + kk * 128, p.idesc, 1u);
                        }
                        ptx::umma_commit_pair(&empty_bar[stage], pair_mask);
                        if (last) {
                            ptx::umma_commit_pair(&acc_full_bar[acc], pair_mask);
                        }
                    }
                    __syncwarp();
                    if (++stage == kWgStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    ++in_part;
                    if (last) {
                        in_part = 0;
                        acc ^= 1;
                        acc_phase ^= (acc == 0) ? 1u : 0u;
                    }
                }
            }
            for (int i = 0; ok && i < 2; ++i) { // the other CTA's last signals have come before this one may leave
                ok = bounded_wait_quiet_warp(&acc_empty_bar[acc], acc_phase ^ 1u, abort_flag, p.status, ST_WG_MMA, p.wait_limit);
                acc ^= 1;
                acc_phase ^= (acc == 0) ? 1u : 0u;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWgRegsWorkers));
        // ---------------------------------------------------------------- conversion, sums, stores
        const int group = (warp - 4) >> 2;         // converts stages group, group + 4, ..; keeps the sums of 64 columns (n)
        const int quarter = warp & 3;              // and of these 32 tensor-memory lanes (k)
        // Four 16-byte pieces of x per stage: rows row + 16 h of the tile. Eight lanes read a half of one row and the other
        // half of the next, 128 bytes on different banks; converted, the halves of a row lie in blocks 8 KiB apart with a
        // 128-byte swizzle, where the two rows' pieces are on different banks again.
        const int row = quarter * 4 + (lane >> 4) * 2 + ((lane >> 2) & 1);
        const int piece = (lane & 3) + 4 * (((lane >> 2) ^ (lane >> 3)) & 1);
        const uint32_t line = (piece >> 2) * 8192 + row * 128;
        const uint32_t at0 = line + ((((piece & 3) * 2) ^ (row & 7)) * 16); // row + 16 h has the row's swizzle
        const uint32_t at1 = line + ((((piece & 3) * 2 + 1) ^ (row & 7)) * 16);
        const uint8_t* raw = smem + L::kRawOff + group * L::kRawBytes + row * 128 + piece * 16;
        int stage = group, acc = 0;
        uint32_t phase = 0, raw_phase = 0, acc_phase = 0;
        bool ok = true;
        int first_of_tile = group; // first stage of the tile that this group converts
        const int stages = last_stage - first_stage; // of a tile
        const int parts = (stages + kWgFoldStages - 1) / kWgFoldStages;
        // Block scales come straight from memory, one visit (four stages) ahead of their use: their rows start on any byte,
        // so no TMA, and a thread fetches what its own pieces need. What lies outside takes the nearest scale inside: a
        // column past K is never stored, and a token past T has zeros in dy and x.
        int visit_token = 0;      // first token of the stage whose scales come next
        uint32_t scale_off = 0;
        uint32_t e[4] = {127u, 127u, 127u, 127u};
        auto fetch_scales = [&]() {
            const uint8_t* base = p.scales + visit_token * p.ld_scales;
            if (visit_token + kWgStageTokens <= p.t) {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    e[h] = nv_ld_byte(base + 16 * h * p.ld_scales + scale_off);
                }
            } else if (visit_token < p.t) {
                const int last_row = p.t - 1 - visit_token;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    e[h] = nv_ld_byte(base + (min(row + 16 * h, last_row) - row) * p.ld_scales + scale_off);
                }
            }
            visit_token += kWgGroups * kWgStageTokens;
        };
        auto start_scales = [&](int tile) { // of the first stage that this group converts of a tile
            int ki, ni;
            tile_of(tile, ki, ni);
            const int column = min(ki * 256 + side * 128 + piece * 16, p.k - 1) >> 5;
            scale_off = static_cast<uint32_t>(row * p.ld_scales + column);
            visit_token = (first_stage + first_of_tile) * kWgStageTokens;
            fetch_scales();
        };
        if constexpr (!SCRATCH) {
            start_scales(cluster);
        }
        ptx::cluster_wait();
        for (int tile = cluster; ok && tile < tiles; tile += clusters) {
            int ki, ni;
            tile_of(tile, ki, ni);
            float sum[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) {
                sum[i] = 0.0f;
            }
            int folded = 0;
            for (int st = SCRATCH ? stages : first_of_tile; folded < parts; st += kWgGroups) {
                if (!SCRATCH && st < stages) {
                    const uint32_t e_now[4] = {e[0], e[1], e[2], e[3]};
                    fetch_scales(); // of the next visit; past the tile's last token they are not used
                    ok = bounded_wait_quiet(&raw_full_bar[group], raw_phase, abort_flag, p.status, ST_WG_WORKER, p.wait_limit);
                    uint4 in[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        in[h] = *reinterpret_cast<const uint4*>(raw + h * 16 * 128);
                    }
                    ok = ok && bounded_wait_quiet(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, ST_WG_WORKER, p.wait_limit);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) {
                        break;
                    }
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive(&raw_empty_bar[group]);
                    }
                    uint8_t* dst = smem + L::kXOff + stage * L::kXBytes;
                    if (!__any_sync(0xFFFFFFFFu, wg_needs_any<F16>(in, e_now))) {
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            uint32_t o[8];
                            wg_convert16<F16>(in[h], e_now[h], o);
                            *reinterpret_cast<uint4*>(dst + at0 + h * 16 * 128) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(dst + at1 + h * 16 * 128) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    } else {
#pragma unroll 1
                        for (int h = 0; h < 4; ++h) {
                            uint32_t o[8];
                            wg_convert16_any<F16>(h == 0 ? in[0] : h == 1 ? in[1] : h == 2 ? in[2] : in[3],
                                                  h == 0 ? e_now[0] : h == 1 ? e_now[1] : h == 2 ? e_now[2] : e_now[3], o);
                            *reinterpret_cast<uint4*>(dst + at0 + h * 16 * 128) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(dst + at1 + h * 16 * 128) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive_pair(ptx::map_to_cta(ptx::smem_u32(&full_bar[stage]), leader_rank));
                    }
                    raw_phase ^= 1u;
                    stage += kWgGroups;
                    if (stage >= kWgStages) {
                        stage -= kWgStages;
                        phase ^= 1u;
                    }
                }
                // The oldest finished accumulator joins the sums: behind the last stage, or once this group has had a place
                // in the ring whose last products came after that accumulator's - then nothing is waited for.
                if (st >= stages || st >= (folded + 1) * kWgFoldStages + kWgStages) {
                    ok = bounded_wait_quiet(&acc_full_bar[acc], acc_phase, abort_flag, p.status, ST_WG_WORKER, p.wait_limit);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) {
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t t_row = tmem_base + 256u * acc + 64u * group + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t v[32];
                        ptx::tmem_ld_32x32b_x32(t_row + 32u * q, v);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sum[32 * q + i] += __uint_as_float(v[i]);
                        }
                    }
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive_pair(ptx::map_to_cta(ptx::smem_u32(&acc_empty_bar[acc]), leader_rank));
                    }
                    acc ^= 1;
                    acc_phase ^= (acc == 0) ? 1u : 0u;
                    ++folded;
                }
            }
            if (!ok) {
                break;
            }
            first_of_tile = (first_of_tile - stages % kWgGroups + kWgGroups) % kWgGroups; // stages go round the groups
            if (!SCRATCH && tile + clusters < tiles) {
                start_scales(tile + clusters); // come while this tile is stored
            }
            const int in_tile = quarter * 32 + lane;
            if (p.splits == 1) {
                const int k = ki * 256 + side * 128 + in_tile;
                const int n0 = ni * 256 + group * 64;
                if (k < p.k) {
                    using T = typename WgElem<OUT>::type;
                    T* at = static_cast<T*>(p.out) + n0 * p.ld_out + k;
                    const T* add = static_cast<const T*>(p.addend) + (p.addend != nullptr ? n0 * p.ld_addend + k : 0);
#pragma unroll
                    for (int i0 = 0; i0 < 64; i0 += 16) {
                        if (p.addend != nullptr) { // sixteen reads in flight, before the stores: addend may be out
                            T v[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                v[i] = n0 + i0 + i < p.n ? add[(i0 + i) * p.ld_addend] : static_cast<T>(0.0f);
                            }
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                sum[i0 + i] += static_cast<float>(v[i]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (n0 + i0 + i < p.n) {
                                *at = static_cast<T>(sum[i0 + i]); // one rounding to the output's type
                            }
                            at += p.ld_out;
                        }
                    }
                }
            } else {
                float* part = reinterpret_cast<float*>(smem); // [256 n][128 k]: every load and product of the ring is done
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    part[(group * 64 + i) * 128 + in_tile] = sum[i];
                }
            }
        }
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0) {
        for (int i = 0; i < 2000; ++i) { // copies and products in flight end before shared and tensor memory go away
            __nanosleep(1000);
        }
    }
    // No CTA touches another's tensor memory or barriers any more. Partial sums, where there are some, are in place; without
    // them the arrival orders nothing (the other form waits for the tile's stores).
    if (p.splits > 1) {
        ptx::cluster_arrive();
    } else {
        ptx::cluster_arrive_relaxed();
    }
    ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
    if (p.splits > 1) { // one tile per cluster
        if (warp < 4) { // these have given their registers back
            ptx::cluster_arrive();
        } else {
            int ki, ni;
            tile_of(cluster, ki, ni);
            const uint32_t base = ptx::smem_u32(smem);
            const int thread = static_cast<int>(threadIdx.x) - 128;
            if (p.splits == 2) {
                wg_add_parts<2, OUT>(p, base, split, side, ki * 256 + side * 128, ni * 256, thread);
            } else {
                wg_add_parts<4, OUT>(p, base, split, side, ki * 256 + side * 128, ni * 256, thread);
            }
        }
        ptx::cluster_wait(); // no CTA leaves while another still reads its shared memory
    }
}

} // namespace pto_b200
