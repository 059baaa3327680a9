// C ABI of the operators around activations kept in 8 bits: the quantiser from 16-bit rows and the weight gradient.
#include "capi_shared.cuh"

#include <atomic>
#include <type_traits>

#include "gemm_wgrad_mx.cuh"
#include "mx_quantize.cuh"

namespace pto_b200 {
namespace {

bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) != 0; }

template <int ALG, int SRC, int VEC>
int launch_quantize16(cudaStream_t s, const HostContext& host, const uint8_t* src, uint8_t* data, uint8_t* scales, int rows,
                      int k, long long ld_src, long long ld_data, long long ld_scales)
{
    auto kernel = mx_quantize_e4m3_16bit_kernel<ALG, SRC, VEC>;
    static std::atomic<int> blocks_per_sm[kMaxDevices];
    int per_sm = blocks_per_sm[host.device].load(std::memory_order_relaxed);
    if (per_sm == 0) {
        if (int rc = note_cuda_error(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kQuantThreads, 0),
                                     "mx_quantize occupancy")) {
            return rc;
        }
        per_sm = per_sm > 0 ? per_sm : 1;
        blocks_per_sm[host.device].store(per_sm, std::memory_order_relaxed);
    }
    const long long want = (static_cast<long long>(rows) * (k / 16) + kQuantThreads - 1) / kQuantThreads;
    const long long cap = static_cast<long long>(host.sm_count) * per_sm; // one resident wave
    const int grid = static_cast<int>(want < cap ? want : cap);
    count_launches(1);
    return note_cuda_error(launch_rows(host, kernel, grid, kQuantThreads, s, reinterpret_cast<const uint16_t*>(src), data, scales,
                                              rows, k, ld_src, ld_data, ld_scales),
                           "mx_quantize (16-bit) launch");
}

template <int ALG, int SRC>
int launch_quantize16_any(cudaStream_t s, const HostContext& host, const uint8_t* src, uint8_t* data, uint8_t* scales, int rows,
                          int k, long long ld_src, long long ld_data, long long ld_scales)
{
    return !misaligned(src, 32) && ld_src % 16 == 0
               ? launch_quantize16<ALG, SRC, 32>(s, host, src, data, scales, rows, k, ld_src, ld_data, ld_scales)
               : launch_quantize16<ALG, SRC, 16>(s, host, src, data, scales, rows, k, ld_src, ld_data, ld_scales);
}

// x [t][k] as 16-bit values into scratch memory: one resident wave.
template <bool F16>
int launch_convert(cudaStream_t s, const HostContext& host, const uint8_t* data, long long ld_data, uint8_t* scratch,
                   const WgradParams& p)
{
    auto kernel = mx_to_16bit_kernel<F16>;
    static std::atomic<int> blocks_per_sm[kMaxDevices];
    int per_sm = blocks_per_sm[host.device].load(std::memory_order_relaxed);
    if (per_sm == 0) {
        if (int rc = note_cuda_error(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kWgConvertThreads, 0),
                                     "mx_to_16bit occupancy")) {
            return rc;
        }
        per_sm = per_sm > 0 ? per_sm : 1;
        blocks_per_sm[host.device].store(per_sm, std::memory_order_relaxed);
    }
    const long long want = (static_cast<long long>(p.t) * (p.k / 16) + kWgConvertThreads - 1) / kWgConvertThreads;
    const long long cap = static_cast<long long>(host.sm_count) * per_sm;
    count_launches(1);
    return note_cuda_error(launch_rows(host, kernel, static_cast<int>(want < cap ? want : cap), kWgConvertThreads, s, data, p.scales,
                                              reinterpret_cast<uint16_t*>(scratch), p.t, p.k, ld_data, p.ld_scales),
                           "mx_to_16bit launch");
}

template <bool F16, int OUT, bool SCRATCH>
int launch_wgrad(cudaStream_t stream, const HostContext& host, const uint8_t* dy, const uint8_t* data, long long ld_dy,
                 long long ld_data, uint8_t* scratch, WgradParams p)
{
    auto kernel = gemm_wgrad_mx<F16, OUT, SCRATCH>;
    static std::atomic<int> resident[kMaxDevices][3]; // clusters of 2, 4 and 8 CTAs that the device holds at once
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(kWgThreads, 1, 1);
    cfg.dynamicSmemBytes = WgSmem::kTotal;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters_of[3];
    for (int i = 2; i >= 0; --i) { // [0], looked at last here and first above, is stored last: it says that all are known
        clusters_of[i] = resident[host.device][i].load(std::memory_order_acquire);
    }
    if (clusters_of[0] == 0) {
        if (int rc = note_cuda_error(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, WgSmem::kTotal),
                                     "cudaFuncSetAttribute(wgrad)")) {
            return rc;
        }
        for (int i = 2; i >= 0; --i) {
            attr[0].val.clusterDim.x = 2u << i;
            cfg.gridDim = dim3(2u << i, 1, 1);
            if (int rc = note_cuda_error(cudaOccupancyMaxActiveClusters(&clusters_of[i], kernel, &cfg),
                                         "cudaOccupancyMaxActiveClusters")) {
                return rc;
            }
            clusters_of[i] = clusters_of[i] > 0 ? clusters_of[i] : (i == 0 ? 1 : -1);
            resident[host.device][i].store(clusters_of[i], std::memory_order_release);
        }
    }
    CUtensorMap tdy, tx;
    int rc = encode_map_2d(&tdy, F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy, p.t, p.n, ld_dy * 2,
                           64, kWgStageTokens, true);
    if constexpr (SCRATCH) {
        rc = rc ? rc : launch_convert<F16>(stream, host, data, ld_data, scratch, p);
        rc = rc ? rc : encode_map_2d(&tx, F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, scratch, p.t,
                                     p.k, p.k * 2ll, 64, kWgStageTokens, true);
    } else {
        rc = rc ? rc : encode_map_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, data, p.t, p.k, ld_data, 128, kWgStageTokens, false);
    }
    if (rc) {
        return rc;
    }
    p.k_tiles = (p.k + 255) / 256;
    p.n_tiles = (p.n + 255) / 256;
    p.group = 8;
    p.stages = (p.t + kWgStageTokens - 1) / kWgStageTokens;
    // D fp32 (1 at [4,6)), A and B bf16 (1) or fp16 (0), both with the summed index outermost (bits 15 and 16), 256 x 256
    const uint32_t fmt = F16 ? 0u : 1u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
    // Tokens in parts where that ends sooner: waves of tiles times a part's stages, and what a tile costs besides (filling
    // the rings, the stores, some 16 stages; the parts' exchange another 8). Fewer clusters of eight CTAs fit the device than
    // its SMs would hold - 16 tiles in four parts can take two waves - so the waves go by what the device says it holds.
    const long long tiles = static_cast<long long>(p.k_tiles) * p.n_tiles;
    p.splits = 1;
    long long best = 0;
    for (int i = 0; i < 3; ++i) {
        const int splits = 1 << i;
        if (clusters_of[i] <= 0 || (i > 0 && p.stages < 2 * splits)) {
            continue;
        }
        const long long waves = (tiles + clusters_of[i] - 1) / clusters_of[i];
        const long long cost = waves * ((p.stages + splits - 1) / splits + 16 + (i > 0 ? 8 : 0));
        if (i == 0 || cost < best) {
            best = cost;
            p.splits = splits;
        }
    }
    attr[0].val.clusterDim.x = static_cast<unsigned>(2 * p.splits);
    const long long clusters = p.splits > 1 ? tiles : (tiles < clusters_of[0] ? tiles : clusters_of[0]);
    if (clusters * 2 * p.splits > 0x7FFFFFFFll) {
        return PTO_B200_EINVAL;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(2 * p.splits * clusters), 1, 1);
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; // the kernel waits for what comes before it itself
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    count_launches(1);
    return note_cuda_error(cudaLaunchKernelEx(&cfg, kernel, tdy, tx, p), "gemm_wgrad_mx launch");
}

} // namespace
} // namespace pto_b200

using namespace pto_b200;

extern "C" int pto_b200_mx_quantize_e4m3_src(void* stream, uint8_t* data, uint8_t* scales, const uint8_t* src, int rows, int k,
                                             long long ld_src, long long ld_data, long long ld_scales, int src_dtype,
                                             int scale_alg)
{
    if (src_dtype == PTO_B200_F32) {
        return pto_b200_mx_quantize_e4m3_ex(stream, data, scales, src, rows, k, ld_src, ld_data, ld_scales, scale_alg);
    }
    if (data == nullptr || scales == nullptr || src == nullptr || rows <= 0 || k <= 0 || rows > kMaxExtent || k > kMaxExtent ||
        k % 32 != 0 || ld_src < k ||
        ld_data < k || ld_scales < k / 32) {
        return PTO_B200_EINVAL;
    }
    if ((src_dtype != PTO_B200_BF16 && src_dtype != PTO_B200_F16) ||
        (scale_alg != PTO_B200_SCALE_OCP && scale_alg != PTO_B200_SCALE_NV)) {
        return PTO_B200_EDTYPE;
    }
    if (misaligned(src, 16) || ld_src % 8 != 0 || misaligned(data, 8) || ld_data % 8 != 0) {
        return PTO_B200_EALIGN;
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f16 = src_dtype == PTO_B200_F16, nv = scale_alg == PTO_B200_SCALE_NV;
    auto launch = nv ? (f16 ? launch_quantize16_any<MX_SCALE_NV, NV_F16> : launch_quantize16_any<MX_SCALE_NV, NV_BF16>)
                     : (f16 ? launch_quantize16_any<MX_SCALE_OCP, NV_F16> : launch_quantize16_any<MX_SCALE_OCP, NV_BF16>);
    return launch(s, host, src, data, scales, rows, k, ld_src, ld_data, ld_scales);
}

extern "C" int pto_b200_gemm_wgrad_mx(void* stream, uint8_t* out, const uint8_t* dy, const uint8_t* data, const uint8_t* scales,
                                      const uint8_t* addend, uint8_t* workspace, size_t workspace_bytes, int t, int n, int k,
                                      long long ld_dy, long long ld_data, long long ld_scales, long long ld_out,
                                      long long ld_addend, int dy_dtype, int out_dtype)
{
    if ((dy_dtype != PTO_B200_BF16 && dy_dtype != PTO_B200_F16) ||
        (out_dtype != PTO_B200_F32 && out_dtype != PTO_B200_BF16 && out_dtype != PTO_B200_F16)) {
        return PTO_B200_EDTYPE;
    }
    if (out == nullptr || dy == nullptr || data == nullptr || scales == nullptr || t <= 0 || n <= 0 || k <= 0 || t > kMaxExtent ||
        n > kMaxExtent || k > kMaxExtent || k % 32 != 0 ||
        ld_dy < n || ld_data < k || ld_scales < k / 32 || ld_scales >= (1 << 26) || ld_out < k ||
        (addend != nullptr && ld_addend < k)) { // offsets within a stage's scales are 32-bit
        return PTO_B200_EINVAL;
    }
    const unsigned out_es = out_dtype == PTO_B200_F32 ? 4 : 2;
    if (misaligned(dy, 16) || ld_dy % 8 != 0 || misaligned(data, 16) || ld_data % 16 != 0 || misaligned(out, out_es) ||
        misaligned(addend, out_es)) {
        return PTO_B200_EALIGN;
    }
    if (workspace != nullptr &&
        (misaligned(workspace, 32) || workspace_bytes < static_cast<size_t>(t) * static_cast<size_t>(k) * 2)) {
        return PTO_B200_EWORKSPACE;
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    WgradParams p = {};
    p.out = out;
    p.addend = addend;
    p.scales = scales;
    p.ld_out = ld_out;
    p.ld_addend = ld_addend;
    p.ld_scales = ld_scales;
    p.t = t;
    p.n = n;
    p.k = k;
    p.status = host.status;
    p.wait_limit = host.wait_limit;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f16 = dy_dtype == PTO_B200_F16;
    auto launch = [&](auto scratch) {
        constexpr bool kScratch = decltype(scratch)::value;
        auto of_type = out_dtype == PTO_B200_F32
                           ? (f16 ? launch_wgrad<true, WG_OUT_F32, kScratch> : launch_wgrad<false, WG_OUT_F32, kScratch>)
                       : out_dtype == PTO_B200_BF16
                           ? (f16 ? launch_wgrad<true, WG_OUT_BF16, kScratch> : launch_wgrad<false, WG_OUT_BF16, kScratch>)
                           : (f16 ? launch_wgrad<true, WG_OUT_F16, kScratch> : launch_wgrad<false, WG_OUT_F16, kScratch>);
        return of_type(s, host, dy, data, ld_dy, ld_data, workspace, p);
    };
    return workspace != nullptr ? launch(std::true_type{}) : launch(std::false_type{});
}
