// Product of two NVFP4 matrices on sm_100a:
//   C[i][j] = ga gb sum_k (a[i][k] sa[i][k/16]) (b[j][k] sb[j][k/16])  (+ bias[j])
// with e2m1 elements, e4m3 scales and fp32 accumulation: tcgen05.mma kind::mxf4nvf4, which multiplies 64 elements of K
// per instruction and applies a scale per 16 of them from tensor memory. A 128-byte swizzle row holds 256 packed
// elements, so a ring stage is 256 elements of K: four instructions.
//
// Scales come in the 512-byte tiles nvfp4_quantize.cuh describes, which tcgen05.cp moves to tensor memory as they are.
// The last stage of K may hold fewer than four 64-element groups: only those that exist are multiplied, so what stands
// in the scale buffers past them never matters.
//
// The tensor core's fp32 sums cut off instead of rounding. They are not joined in parts: an instruction adds 64 of K at once,
// and products of 4-bit numbers and their scales have few bits. Measured, relative (plain fp32 product of the same numbers):
// K = 16384, normal numbers exact, of one sign 4.9e-8 (7.5e-7); 65536, 2e-9 (3e-9) and 5.9e-7 (3.3e-6); 262144 of one sign
// 7.8e-6.
//
// gemm_nvfp4_2cta: a cluster of two CTAs owns a 256 x 256 tile (many rows). gemm_nvfp4_few_rows: few rows of A, the
// bound is reading B; see there.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "gemm_tile_loop.cuh"
#include "row_elements.cuh"
#include "sm100_ptx.cuh"

namespace pto_b200 {

enum NvOut : int { NV_OUT_F32 = 0, NV_OUT_BF16 = 1, NV_OUT_F16 = 2 };

struct NvGemmParams {
    void* c;
    long long ldc;      // elements
    int m, n;
    int m_tiles, n_tiles, group_m;
    int full_units, units; // pair kernel: whole tiles first, then halves (256 x 128) of the last, partly filled wave's
    int k_stages;       // 256-element stages of K
    int k_atoms;        // 64-element groups of K
    uint32_t idesc;
    uint32_t idesc_half; // pair kernel: of a 256 x 128 half tile
    const float* ga;    // tensor scales, or null for 1
    const float* gb;
    const float* bias;  // n values, or null
    const uint8_t* sfa; // tiled scales
    const uint8_t* sfb;
    int* status;
    long long wait_limit;
    int row_access;     // C's rows start on 32- or 16-byte boundaries, or on any element (0)
};

// status codes of bounded waits that gave up
constexpr int ST_NV_PRODUCER = 21;
constexpr int ST_NV_MMA = 22;
constexpr int ST_NV_EPILOGUE = 23;

constexpr int kNvStageK = 256;       // elements of K per stage
constexpr int kNvAtomBytes = 512;    // scales of 128 rows x 64 elements

__device__ __forceinline__ float nv_alpha(const NvGemmParams& p)
{
    const float a = p.ga != nullptr ? nv_ld_common(p.ga) : 1.0f;
    const float b = p.gb != nullptr ? nv_ld_common(p.gb) : 1.0f;
    return a * b;
}

template <int OUT>
__device__ __forceinline__ uint32_t nv_pack2(float lo, float hi)
{
    if constexpr (OUT == NV_OUT_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// ---------------------------------------------------------------- many rows: CTA pairs, 256 x 256 tiles
//
// Roles per CTA: warp 0 loads (TMA), warp 1 copies scales to tensor memory and multiplies (leader CTA), warps 2..9 store.
// A 256-column accumulator and the scale columns of five stages fill tensor memory, so there is one accumulator: the
// store warps - eight of them, so that a thread owns 128 columns of its row - move it to registers in one go and hand it
// back before they convert and store, and the next tile's products start some hundred cycles after the last one's end
// instead of after its stores.
//
// The issuing warps walk their loops as whole warps and one elected lane issues: addresses and descriptors then stay in
// uniform registers. Measured per 256-element stage: twelve scale copies and four products 513 cycles, which is the
// products' own time; issued by a lane that branched off, 1176, and with the copies on the other CTA still 844.
constexpr int kNvPairStages = 5;
constexpr int kNvPairThreads = 320;
constexpr int kNvStoreWarps = 8; // per CTA

struct NvPairSmem {
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = 128 * 128;
    static constexpr int kSfaBytes = 4 * kNvAtomBytes;
    static constexpr int kSfbBytes = 8 * kNvAtomBytes; // scales of all 256 columns, in both CTAs
    static constexpr int kEpiBufBytes = 32 * 128;
    static constexpr int kAOff = 0;
    static constexpr int kBOff = kNvPairStages * kABytes;
    static constexpr int kEpiOff = kBOff + kNvPairStages * kBBytes;
    static constexpr int kSfaOff = kEpiOff + kNvStoreWarps * kEpiBufBytes;
    static constexpr int kSfbOff = kSfaOff + kNvPairStages * kSfaBytes;
    static constexpr int kBarOff = kSfbOff + kNvPairStages * kSfbBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes; // per CTA, on the leader's barrier
    static constexpr int kNumBars = 2 * kNvPairStages + 2;
    static constexpr int kMiscOff = kBarOff + kNumBars * 8;
    static constexpr int kTotal = kMiscOff + 16 + 1024;
};
static_assert(NvPairSmem::kTotal <= 227 * 1024, "shared memory of the pair kernel");

// A pair's unit of work: a whole 256 x 256 tile, or where the last wave would leave half of the pairs or more without a
// tile, one 256 x 128 half of a tile (2040x8100x8192, 256 tiles on 74 pairs: four waves become three and a half).
struct NvUnit {
    int row, col; // first row and column of C
    bool half;
};

__device__ __forceinline__ NvUnit nv_unit(int u, const NvGemmParams& p)
{
    const bool half = u >= p.full_units;
    const int t = half ? p.full_units + ((u - p.full_units) >> 1) : u;
    const int group_size = p.group_m * p.n_tiles;
    const int g = t / group_size;
    const int first_m = g * p.group_m;
    const int gm = min(p.m_tiles - first_m, p.group_m);
    const int r = t - g * group_size;
    return {(first_m + r % gm) * 256, r / gm * 256 + (half ? ((u - p.full_units) & 1) * 128 : 0), half};
}

template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNvPairThreads)
    gemm_nvfp4_2cta(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_b_half, const __grid_constant__ CUtensorMap tmap_sfa,
                    const __grid_constant__ CUtensorMap tmap_sfb, const NvGemmParams p)
{
    using L = NvPairSmem;
    constexpr int STAGES = kNvPairStages;
    constexpr uint32_t kSfCol0 = 256;       // scale columns of stage s: [256 + 48 s, +16) for A, the next 32 for B
    constexpr uint32_t kSfColsPerStage = 48;
    static_assert(256 + STAGES * 48 <= kTmemCols, "accumulator and scale columns");

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff); // leader: both CTAs' operands and scales landed
    uint64_t* empty_bar = full_bar + STAGES;                            // each CTA
    uint64_t* acc_full_bar = empty_bar + STAGES;                        // each CTA
    uint64_t* acc_empty_bar = acc_full_bar + 1;                         // leader: sixteen store warps
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = ptx::cluster_ctarank();
    const bool leader = (cta_rank == 0);
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        ptx::mbar_init(acc_full_bar, 1);
        ptx::mbar_init(acc_empty_bar, 2 * kNvStoreWarps);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
        ptx::prefetch_tensormap(&tmap_sfa);
        ptx::prefetch_tensormap(&tmap_sfb);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(tmem_base_slot, kTmemCols);
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive(); // the peer's barriers must exist before anything is signalled across the pair
    ptx::cluster_wait();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_base_slot;
    ptx::grid_dependency_wait(); // as in the kernel for few rows

    if (warp == 0) {
        // ---------------------------------------------------------------- loads (both CTAs)
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = pair; ok && u < p.units; u += num_pairs) {
            const NvUnit w = nv_unit(u, p);
            const int row_a = w.row + static_cast<int>(cta_rank) * 128;
            const int row_b = w.col + static_cast<int>(cta_rank) * (w.half ? 64 : 128);
            // scale tiles as rows of 256 bytes, two per 512-byte tile; tiles past the last row read as zero
            const int sfa_row = row_a / 128 * p.k_atoms * 2;
            const int sfb_row = w.col / 128 * p.k_atoms * 2;
            const CUtensorMap* map_b = w.half ? &tmap_b_half : &tmap_b; // of a half tile 64 rows and one tile of scales
            const uint32_t stage_bytes = 2u * L::kStageBytes - (w.half ? L::kBBytes + L::kSfbBytes : 0u);
            for (int ks = 0; ks < p.k_stages; ++ks) {
                ok = bounded_wait_warp(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, ST_NV_PRODUCER, p.wait_limit);
                if (!ok) {
                    break;
                }
                if (ptx::elect_one()) {
                    if (leader) {
                        ptx::mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
                    }
                    const uint32_t full_addr = ptx::map_to_cta(ptx::smem_u32(&full_bar[stage]), 0);
                    uint8_t* sfa = smem + L::kSfaOff + stage * L::kSfaBytes;
                    uint8_t* sfb = smem + L::kSfbOff + stage * L::kSfbBytes;
                    ptx::tma_load_2d_pair(smem + L::kAOff + stage * L::kABytes, &tmap_a, full_addr, ks * 128, row_a);
                    ptx::tma_load_2d_pair(smem + L::kBOff + stage * L::kBBytes, map_b, full_addr, ks * 128, row_b);
                    ptx::tma_load_2d_pair(sfa, &tmap_sfa, full_addr, 0, sfa_row + ks * 8);
                    ptx::tma_load_2d_pair(sfb, &tmap_sfb, full_addr, 0, sfb_row + ks * 8);
                    if (!w.half) {
                        ptx::tma_load_2d_pair(sfb + 4 * kNvAtomBytes, &tmap_sfb, full_addr, 0,
                                              sfb_row + p.k_atoms * 2 + ks * 8);
                    }
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- scale copies and products (leader)
        // cta_group::2 copies the same shared-memory offsets of both CTAs into both CTAs' tensor memory; a thread's copies
        // and products run in order
        if (leader) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            const uint64_t a_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kAOff), 16, 1024, ptx::kSwizzle128B);
            const uint64_t b_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kBOff), 16, 1024, ptx::kSwizzle128B);
            const uint64_t sfa_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kSfaOff), 0, 128, ptx::kSwizzleNone);
            const uint64_t sfb_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kSfbOff), 0, 128, ptx::kSwizzleNone);
            // stages left of all units: the last round of the ring is not handed back, since nobody would wait for that and a
            // signal could reach the other CTA after it has left
            long long left = static_cast<long long>((p.units - pair + num_pairs - 1) / num_pairs) * p.k_stages;
            for (int u = pair; ok && u < p.units; u += num_pairs) {
                ok = bounded_wait_warp(acc_empty_bar, acc_phase ^ 1u, abort_flag, p.status, ST_NV_MMA, p.wait_limit);
                if (!ok) {
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t idesc = u < p.full_units ? p.idesc : p.idesc_half;
                for (int ks = 0; ks < p.k_stages; ++ks) {
                    ok = bounded_wait_warp(&full_bar[stage], phase, abort_flag, p.status, ST_NV_MMA, p.wait_limit);
                    if (!ok) {
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    if (ptx::elect_one()) {
                        // descriptor addresses count 16 bytes
                        const uint64_t a_desc = a_desc0 + static_cast<uint64_t>(stage * (L::kABytes / 16));
                        const uint64_t b_desc = b_desc0 + static_cast<uint64_t>(stage * (L::kBBytes / 16));
                        const uint64_t sfa_desc = sfa_desc0 + static_cast<uint64_t>(stage * (L::kSfaBytes / 16));
                        const uint64_t sfb_desc = sfb_desc0 + static_cast<uint64_t>(stage * (L::kSfbBytes / 16));
                        const uint32_t sf = tmem_base + kSfCol0 + kSfColsPerStage * static_cast<uint32_t>(stage);
                        const int groups = p.k_atoms - 4 * ks; // 64-element groups left
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (g < groups) {
                                ptx::tmem_cp_32x128b_warpx4_pair(sf + 4u * g, sfa_desc + 32 * g);
                                ptx::tmem_cp_32x128b_warpx4_pair(sf + 16u + 8u * g, sfb_desc + 32 * g);
                                // (of a half tile what the buffer last held: its columns are not read)
                                ptx::tmem_cp_32x128b_warpx4_pair(sf + 20u + 8u * g, sfb_desc + 128 + 32 * g);
                            }
                        }
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (g < groups) {
                                ptx::umma_nvf4_pair(tmem_base, a_desc + 2 * g, b_desc + 2 * g, idesc, sf + 4u * g,
                                                    sf + 16u + 8u * g, (ks > 0 || g > 0) ? 1u : 0u);
                            }
                        }
                        if (left > STAGES) {
                            ptx::umma_commit_pair(&empty_bar[stage], 0x3);
                        }
                        if (ks == p.k_stages - 1) {
                            ptx::umma_commit_pair(acc_full_bar, 0x3);
                        }
                    }
                    --left;
                    __syncwarp();
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                acc_phase ^= 1u;
            }
            if (ok) { // the other CTA's last signals have come before this one may leave
                bounded_wait_warp(acc_empty_bar, acc_phase ^ 1u, abort_flag, p.status, ST_NV_MMA, p.wait_limit);
            }
        }
    } else {
        // ---------------------------------------------------------------- stores (both CTAs)
        constexpr bool kOut32 = (OUT == NV_OUT_F32);
        constexpr int kBoxCols = kOut32 ? 32 : 64; // 128 bytes
        constexpr int kBoxes = 128 / kBoxCols;
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2; // which 128 columns
        uint8_t* box = smem + L::kEpiOff + (warp - 2) * L::kEpiBufBytes;
        const float alpha = nv_alpha(p);
        auto finish = [&](uint32_t acc, int col) {
            const float f = __uint_as_float(acc) * alpha;
            float add = -0.0f; // changes no number; as a branch around the sum the 16-bit forms spill
            if (p.bias != nullptr && col < p.n) {
                add = nv_ld_common(p.bias + col);
            }
            return f + add;
        };
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int u = pair; ok && u < p.units; u += num_pairs) {
            const NvUnit w = nv_unit(u, p);
            ok = bounded_wait(acc_full_bar, acc_phase, abort_flag, p.status, ST_NV_EPILOGUE, p.wait_limit);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) {
                break;
            }
            acc_phase ^= 1u;
            ptx::tc_fence_after_sync();
            uint32_t v[4][32];
            const uint32_t t_row = tmem_base + static_cast<uint32_t>(half * 128) + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ptx::tmem_ld_32x32b_x32(t_row + 32u * i, v[i]);
            }
            ptx::tmem_ld_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive_pair(ptx::map_to_cta(ptx::smem_u32(acc_empty_bar), 0));
            }
            const int row0 = w.row + static_cast<int>(cta_rank) * 128 + quarter * 32;
            const int col0 = w.half && half != 0 ? p.n : w.col + half * 128; // a half tile has no second 128 columns
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) { // 128 bytes of this thread's row at a time
                const int bc = col0 + b * kBoxCols;
                if (bc >= p.n || row0 >= p.m) {
                    break;
                }
                uint32_t o[32];
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    if constexpr (kOut32) {
                        o[q] = __float_as_uint(finish(v[b][q], bc + q));
                    } else {
                        const int c = 2 * q;
                        o[q] = nv_pack2<OUT>(finish(v[2 * b + c / 32][c % 32], bc + c), finish(v[2 * b + c / 32][c % 32 + 1], bc + c + 1));
                    }
                }
                if (p.row_access == 32 && bc + kBoxCols <= p.n) {
                    // straight from registers: whole 32-byte sectors, nothing to wait for
                    if (row0 + lane < p.m) {
                        uint8_t* dst = static_cast<uint8_t*>(p.c) + ((row0 + lane) * p.ldc + bc) * (kOut32 ? 4 : 2);
#pragma unroll
                        for (int q = 0; q < 32; q += 8) {
                            nv_st32(dst + q * 4, make_uint4(o[q], o[q + 1], o[q + 2], o[q + 3]),
                                    make_uint4(o[q + 4], o[q + 5], o[q + 6], o[q + 7]));
                        }
                    }
                    continue;
                }
                // other rows through shared memory (128-byte swizzle), so that a warp's stores lie along rows: with half
                // sectors from registers 2040x8100x8192 to fp32 (rows on 16-byte boundaries) took 70 us instead of 60
                uint8_t* line = box + lane * 128;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    *reinterpret_cast<uint4*>(line + ((q ^ (lane & 7)) * 16)) =
                        make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                }
                __syncwarp();
                if (p.row_access != 0 && bc + kBoxCols <= p.n) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = i * 4 + (lane >> 3);
                        if (row0 + r < p.m) {
                            uint8_t* dst = static_cast<uint8_t*>(p.c) + ((row0 + r) * p.ldc + bc) * (kOut32 ? 4 : 2);
                            reinterpret_cast<uint4*>(dst)[lane & 7] =
                                *reinterpret_cast<const uint4*>(box + r * 128 + (((lane & 7) ^ (r & 7)) * 16));
                        }
                    }
                } else {
                    const int rows_here = min(32, p.m - row0);
                    for (int r = 0; r < rows_here; ++r) {
                        const uint8_t* src = box + r * 128;
                        const long long base = (static_cast<long long>(row0) + r) * p.ldc + bc;
                        if constexpr (kOut32) {
                            if (bc + lane < p.n) {
                                static_cast<uint32_t*>(p.c)[base + lane] =
                                    *reinterpret_cast<const uint32_t*>(src + ((lane >> 2) ^ (r & 7)) * 16 + (lane & 3) * 4);
                            }
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int e = h * 32 + lane;
                                if (bc + e < p.n) {
                                    static_cast<uint16_t*>(p.c)[base + e] =
                                        *reinterpret_cast<const uint16_t*>(src + ((e >> 3) ^ (r & 7)) * 16 + (e & 7) * 2);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
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
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ---------------------------------------------------------------- few rows of A
//
// With few rows the product reads B once and does little else, so B takes the instruction's 128-row side (128 columns
// of C per CTA) and the rows of A its N side (BLOCK_T = 16 .. 128 of them): no MMA rows are wasted on rows that are not
// there, and lane = column of C makes the stores of a row contiguous. When the tiles are fewer than the CTAs that fit
// the GPU, a cluster of CTAs shares a tile along K: each keeps fp32 partial sums, which are added over distributed
// shared memory in rank order, so the result does not depend on timing and no workspace is needed.
// Shared memory is kept below half an SM's, so that two CTAs run per SM and one's loads cover the other's start and end.
constexpr int kNvFewThreads = 192;

template <int BLOCK_T>
struct NvFewSmem {
    static constexpr int kWBytes = 128 * 128;      // B: 128 columns of C
    static constexpr int kXBytes = BLOCK_T * 128;  // A: BLOCK_T rows
    static constexpr int kSfBytes = 4 * kNvAtomBytes;
    static constexpr int kStageBytes = kWBytes + kXBytes + 2 * kSfBytes;
    static constexpr int kStages = (111 * 1024) / kStageBytes;
    static constexpr int kXOff = kStages * kWBytes;
    static constexpr int kSfwOff = kXOff + kStages * kXBytes;
    static constexpr int kSfxOff = kSfwOff + kStages * kSfBytes;
    static constexpr int kBarOff = kSfxOff + kStages * kSfBytes;
    static constexpr int kMiscOff = kBarOff + (2 * kStages + 1) * 8;
    static constexpr int kTotal = kMiscOff + 16 + 1024;
    static_assert(BLOCK_T * 128 * 4 <= kBarOff, "partial sums reuse the ring");
    static_assert(kTotal <= 113 * 1024, "two CTAs per SM");
    static constexpr int kSfCol = BLOCK_T < 32 ? 32 : BLOCK_T; // scale columns, 32 per stage, behind the accumulator
    static constexpr int kTmem = 256;                          // half an SM's
    static_assert(kSfCol + 32 * kStages <= kTmem, "accumulator and scale columns");
};

template <int OUT>
__device__ __forceinline__ void nv_store_one(const NvGemmParams& p, long long row, int col, float f)
{
    const long long at = row * p.ldc + col;
    if constexpr (OUT == NV_OUT_F32) {
        static_cast<float*>(p.c)[at] = f;
    } else if constexpr (OUT == NV_OUT_BF16) {
        static_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(f);
    } else {
        static_cast<__half*>(p.c)[at] = __float2half_rn(f);
    }
}

// This CTA's share of a tile whose K was cut over SPLITS CTAs: their partial sums [rows][128] lie at the same place of each
// CTA's shared memory and are added in rank order. Four columns per thread and step, kAtOnce steps at a time, all their reads
// in flight together (a read from another SM takes about a thousand cycles: one value at a time this took 12000 cycles for
// 48 rows, one step at a time 4300). The arrival that lets the other CTAs leave comes behind the last reads, in the releasing
// form, behind which no read is under way any more; it waits for stores, too, so few steps (up to 64 rows, or an eighth of
// 128) keep their sums until then. Sums kept / stored as they come, weights in L2: 1x4096x4096 5.2 / 5.3 us, 256x512x8192
// 8.0 / 8.2; 128x8192x8192, eleven steps, 12.8 / 12.4, 200x4096x8192, six, 12.0 / 11.6.
template <int BLOCK_T, int SPLITS, int OUT>
__device__ __forceinline__ void nv_add_parts(const NvGemmParams& p, uint32_t base, int rank, int ni, int row0, int rows)
{
    constexpr int kSteps = (BLOCK_T * 32 / SPLITS + kNvFewThreads - 1) / kNvFewThreads;
    constexpr int kAtOnce = 8 / SPLITS;
    constexpr int kKept = BLOCK_T <= 64 || SPLITS == 8 ? (kSteps + kAtOnce - 1) / kAtOnce * kAtOnce : kAtOnce;
    const int items = rows * 32;
    const int first = items * rank / SPLITS + static_cast<int>(threadIdx.x);
    const int last = items * (rank + 1) / SPLITS;
    static_assert(kNvFewThreads % 32 == 0, "a thread's steps lie in the same columns");
    const int col = ni * 128 + (first & 31) * 4;
    const float alpha = nv_alpha(p);
    float bias[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        bias[c] = p.bias != nullptr && col + c < p.n ? p.bias[col + c] : 0.0f;
    }
#pragma unroll
    for (int k0 = 0; k0 < kSteps; k0 += kKept) {
        float4 sum[kKept];
#pragma unroll
        for (int g = 0; g < kKept; g += kAtOnce) {
            float4 part[kAtOnce][SPLITS];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int i = first + (k0 + g + u) * kNvFewThreads;
#pragma unroll
                for (int r = 0; r < SPLITS; ++r) {
                    part[u][r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (i < last && col < p.n) { // nothing is read that is not used
                        part[u][r] = ptx::ld_shared_cluster_f32x4(ptx::map_to_cta(base + 16u * static_cast<uint32_t>(i), r));
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                sum[g + u] = part[u][0];
#pragma unroll
                for (int r = 1; r < SPLITS; ++r) {
                    sum[g + u].x += part[u][r].x;
                    sum[g + u].y += part[u][r].y;
                    sum[g + u].z += part[u][r].z;
                    sum[g + u].w += part[u][r].w;
                }
            }
        }
        if (k0 + kKept >= kSteps) {
            __syncwarp();
            ptx::cluster_arrive();
        }
#pragma unroll
        for (int u = 0; u < kKept; ++u) {
            const int i = first + (k0 + u) * kNvFewThreads;
            if (i < last && col < p.n) {
                const long long row = row0 + (i >> 5);
                const float f[4] = {sum[u].x * alpha, sum[u].y * alpha, sum[u].z * alpha, sum[u].w * alpha};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (col + c < p.n) {
                        nv_store_one<OUT>(p, row, col + c, f[c] + bias[c]);
                    }
                }
            }
        }
    }
}

// grid: splits (the cluster) x 128-column tiles x BLOCK_T-row tiles
template <int BLOCK_T, int OUT>
__global__ void __launch_bounds__(kNvFewThreads, 2)
    gemm_nvfp4_few_rows(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                        const NvGemmParams p)
{
    using L = NvFewSmem<BLOCK_T>;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* acc_bar = empty_bar + STAGES;
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int splits = static_cast<int>(gridDim.x);
    const int rank = static_cast<int>(blockIdx.x);
    const int ni = static_cast<int>(blockIdx.y);
    const int ti = static_cast<int>(blockIdx.z);
    const int ks0 = static_cast<int>(static_cast<long long>(p.k_stages) * rank / splits);
    const int ks1 = static_cast<int>(static_cast<long long>(p.k_stages) * (rank + 1) / splits);

    auto load_stage = [&](int ks, int stage) {
        const uint32_t sf_bytes = static_cast<uint32_t>(min(4, p.k_atoms - 4 * ks)) * kNvAtomBytes;
        const size_t at = static_cast<size_t>(ks) * 4 * kNvAtomBytes;
        ptx::mbar_arrive_expect_tx(&full_bar[stage], L::kWBytes + L::kXBytes + 2u * sf_bytes);
        ptx::tma_load_2d(smem + stage * L::kWBytes, &tmap_w, &full_bar[stage], ks * 128, ni * 128);
        ptx::bulk_load_1d(smem + L::kSfwOff + stage * L::kSfBytes,
                          p.sfb + static_cast<size_t>(ni) * p.k_atoms * kNvAtomBytes + at, sf_bytes, &full_bar[stage]);
        ptx::tma_load_2d(smem + L::kXOff + stage * L::kXBytes, &tmap_x, &full_bar[stage], ks * 128, ti * BLOCK_T);
        ptx::bulk_load_1d(smem + L::kSfxOff + stage * L::kSfBytes,
                          p.sfa + static_cast<size_t>(ti) * p.k_atoms * kNvAtomBytes + at, sf_bytes, &full_bar[stage]);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        ptx::mbar_init(acc_bar, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    // The launch may overlap the end of the kernel before it in the stream (programmatic serialisation, 0.6 us of a graph's
    // step): nothing above touches global memory, and here every thread waits until that kernel's writes can be seen.
    ptx::grid_dependency_wait();
    if (threadIdx.x == 0) {
        // the first stages are on their way while tensor memory is set up
        for (int ks = ks0; ks < min(ks1, ks0 + STAGES); ++ks) {
            load_stage(ks, ks - ks0);
        }
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_base_slot, L::kTmem);
        ptx::tmem_relinquish_alloc_permit();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_base_slot;

    if (warp == 0) {
        int stage = 0;
        uint32_t phase = 1; // the first round of the ring is loaded above
        for (int ks = ks0 + STAGES; ks < ks1; ++ks) {
            if (!bounded_wait_warp(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, ST_NV_PRODUCER, p.wait_limit)) {
                break;
            }
            if (ptx::elect_one()) {
                load_stage(ks, stage);
            }
            __syncwarp();
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == 1) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint64_t w_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem), 16, 1024, ptx::kSwizzle128B);
        const uint64_t x_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kXOff), 16, 1024, ptx::kSwizzle128B);
        const uint64_t sfw_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kSfwOff), 0, 128, ptx::kSwizzleNone);
        const uint64_t sfx_desc0 = ptx::make_smem_desc(ptx::smem_u32(smem + L::kSfxOff), 0, 128, ptx::kSwizzleNone);
        for (int ks = ks0; ks < ks1; ++ks) {
            ok = bounded_wait_warp(&full_bar[stage], phase, abort_flag, p.status, ST_NV_MMA, p.wait_limit);
            if (!ok) {
                break;
            }
            ptx::tc_fence_after_sync();
            if (ptx::elect_one()) {
                const uint64_t w_desc = w_desc0 + static_cast<uint64_t>(stage * (L::kWBytes / 16));
                const uint64_t x_desc = x_desc0 + static_cast<uint64_t>(stage * (L::kXBytes / 16));
                const uint64_t sfw_desc = sfw_desc0 + static_cast<uint64_t>(stage * (L::kSfBytes / 16));
                const uint64_t sfx_desc = sfx_desc0 + static_cast<uint64_t>(stage * (L::kSfBytes / 16));
                // every stage has its own scale columns: a copy never meets a product that still reads them
                const uint32_t sf = tmem_base + L::kSfCol + 32u * static_cast<uint32_t>(stage);
                const int groups = p.k_atoms - 4 * ks;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (g < groups) {
                        ptx::tmem_cp_32x128b_warpx4(sf + 4u * g, sfw_desc + 32 * g);
                        ptx::tmem_cp_32x128b_warpx4(sf + 16u + 4u * g, sfx_desc + 32 * g);
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (g < groups) {
                        ptx::umma_nvf4(tmem_base, w_desc + 2 * g, x_desc + 2 * g, p.idesc, sf + 4u * g, sf + 16u + 4u * g,
                                       (ks > ks0 || g > 0) ? 1u : 0u);
                    }
                }
                ptx::umma_commit(&empty_bar[stage]);
                if (ks == ks1 - 1) {
                    ptx::umma_commit(acc_bar);
                }
            }
            __syncwarp();
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else {
        bool ok = bounded_wait(acc_bar, 0, abort_flag, p.status, ST_NV_EPILOGUE, p.wait_limit);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (ok) {
            ptx::tc_fence_after_sync();
            const int quarter = warp & 3;
            const int in_tile = quarter * 32 + lane;
            const int col = ni * 128 + in_tile;
            const float alpha = nv_alpha(p);
            const float bias = (p.bias != nullptr && col < p.n) ? p.bias[col] : 0.0f;
            float* part = reinterpret_cast<float*>(smem); // [BLOCK_T][128]; every load and product of the ring is done
            uint32_t v[32];
#pragma unroll
            for (int c = 0; c < (BLOCK_T + 31) / 32; ++c) {
                const int t0 = ti * BLOCK_T + c * 32;
                if (t0 >= p.m) {
                    break;
                }
                ptx::tmem_ld_32x32b_x32(tmem_base + 32u * c + (static_cast<uint32_t>(quarter * 32) << 16), v);
                ptx::tmem_ld_wait();
                const int valid = min(min(32, BLOCK_T), p.m - t0);
                if (splits == 1) {
                    if (col < p.n) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (i < valid) {
                                nv_store_one<OUT>(p, t0 + i, col, __uint_as_float(v[i]) * alpha + bias);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (i < valid) {
                            part[(c * 32 + i) * 128 + in_tile] = __uint_as_float(v[i]);
                        }
                    }
                }
            }
        }
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0) {
        for (int i = 0; i < 2000; ++i) {
            __nanosleep(1000);
        }
    }
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, L::kTmem);
    }
    if (splits > 1) {
        ptx::cluster_arrive(); // every CTA's partial sums are in its shared memory
        ptx::cluster_wait();
        const int rows = min(BLOCK_T, p.m - ti * BLOCK_T);
        if (splits == 2) {
            nv_add_parts<BLOCK_T, 2, OUT>(p, ptx::smem_u32(smem), rank, ni, ti * BLOCK_T, rows);
        } else if (splits == 4) {
            nv_add_parts<BLOCK_T, 4, OUT>(p, ptx::smem_u32(smem), rank, ni, ti * BLOCK_T, rows);
        } else {
            nv_add_parts<BLOCK_T, 8, OUT>(p, ptx::smem_u32(smem), rank, ni, ti * BLOCK_T, rows);
        }
        ptx::cluster_wait(); // no CTA leaves while another still reads its shared memory: nv_add_parts has arrived
    }
}

} // namespace pto_b200
