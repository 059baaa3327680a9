// C ABI of the NVFP4 operators: argument checks, tensor maps, choice of kernel, launch.
#include "capi_shared.cuh"

#include <atomic>

#include "gemm_nvfp4.cuh"
#include "nvfp4_quantize.cuh"

namespace pto_b200 {
namespace {

int source_of(int dtype)
{
    return dtype == PTO_B200_F32 ? NV_F32 : dtype == PTO_B200_BF16 ? NV_BF16 : dtype == PTO_B200_F16 ? NV_F16 : -1;
}

int size_of(int src) { return src == NV_F32 ? 4 : 2; }

bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) != 0; }

// Blocks for `items` single-thread items: one resident wave that walks them with a grid stride.
template <auto KERNEL>
int one_wave(long long items, const HostContext& host, int* grid)
{
    static std::atomic<int> blocks_per_sm[kMaxDevices];
    int per_sm = blocks_per_sm[host.device].load(std::memory_order_relaxed);
    if (per_sm == 0) {
        if (int rc = note_cuda_error(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERNEL, kNvQuantThreads, 0),
                                     "nvfp4 occupancy")) {
            return rc;
        }
        per_sm = per_sm > 0 ? per_sm : 1;
        blocks_per_sm[host.device].store(per_sm, std::memory_order_relaxed);
    }
    const long long want = (items + kNvQuantThreads - 1) / kNvQuantThreads;
    const long long cap = static_cast<long long>(host.sm_count) * per_sm;
    *grid = static_cast<int>(want < cap ? want : cap);
    return PTO_B200_OK;
}

template <int SRC, int VEC>
int launch_quantize(cudaStream_t s, const HostContext& host, const void* src, const float* amax, uint8_t* data, uint8_t* scales,
                    float* tensor_scale, int rows, int k, long long ld_src, long long ld_data, bool transpose)
{
    int grid = 0;
    cudaError_t launched;
    if (transpose) {
        // 16-bit columns in pairs where rows start on 4-byte boundaries
        const bool pairs = SRC != NV_F32 && !misaligned(src, 4) && ld_src % 2 == 0;
        const long long items = (static_cast<long long>(rows) + 63) / 64 * ((k + 127) / 128 * (pairs ? 64 : 128));
        if (pairs) {
            constexpr bool kPairs = SRC != NV_F32;
            if (int rc = one_wave<nvfp4_quantize_transposed_kernel<SRC, kPairs>>(items, host, &grid)) {
                return rc;
            }
            launched = launch_rows(host, nvfp4_quantize_transposed_kernel<SRC, kPairs>, grid, kNvQuantThreads, s, src, amax, data,
                                          scales, tensor_scale, rows, k, ld_src, ld_data);
        } else {
            if (int rc = one_wave<nvfp4_quantize_transposed_kernel<SRC, false>>(items, host, &grid)) {
                return rc;
            }
            launched = launch_rows(host, nvfp4_quantize_transposed_kernel<SRC, false>, grid, kNvQuantThreads, s, src, amax, data,
                                          scales, tensor_scale, rows, k, ld_src, ld_data);
        }
    } else {
        const long long items = (static_cast<long long>(rows) + 127) / 128 * 128 * ((k + 63) / 64 * 4);
        if (int rc = one_wave<nvfp4_quantize_kernel<SRC, VEC>>(items, host, &grid)) {
            return rc;
        }
        launched = launch_rows(host, nvfp4_quantize_kernel<SRC, VEC>, grid, kNvQuantThreads, s, src, amax, data, scales,
                                      tensor_scale, rows, k, ld_src, ld_data);
    }
    count_launches(1);
    return note_cuda_error(launched, "nvfp4_quantize launch");
}

template <int SRC, int VEC>
int launch_amax(cudaStream_t s, const HostContext& host, const void* src, float* amax, int rows, int k, long long ld_src)
{
    const long long items = static_cast<long long>(rows) * ((k + 15) / 16);
    if (items * 16 <= kAmaxSingleElems) { // small: one block stores the result, nothing to clear first
        amax_kernel<SRC, VEC>
            <<<1, kAmaxSingleThreads, 0, s>>>(src, reinterpret_cast<uint32_t*>(amax), rows, k, ld_src);
    } else {
        int grid = 0;
        if (int rc = one_wave<amax_kernel<SRC, VEC>>(items, host, &grid)) {
            return rc;
        }
        if (int rc = note_cuda_error(cudaMemsetAsync(amax, 0, sizeof(float), s), "amax memset")) {
            return rc;
        }
        amax_kernel<SRC, VEC>
            <<<grid, kNvQuantThreads, 0, s>>>(src, reinterpret_cast<uint32_t*>(amax), rows, k, ld_src);
    }
    count_launches(1);
    return note_cuda_error(cudaGetLastError(), "amax launch");
}

// Largest magnitude and codes in one launch; total = blocks of 16 in rows filled up to 64 elements, at most kNvOneBlocks.
template <int SRC, int VEC, int THREADS>
int launch_quantize_one_of(cudaStream_t s, const void* src, float* amax, uint8_t* data, uint8_t* scales, float* tensor_scale,
                           int rows, int k, long long ld_src, long long ld_data, int total)
{
    int ctas = 1;
    while (ctas < kNvOneCtas && ctas * THREADS < total) {
        ctas *= 2;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.stream = s;
    cfg.attrs = attr;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; // the kernel waits for what comes before it itself
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    count_launches(1);
    return note_cuda_error(cudaLaunchKernelEx(&cfg, nvfp4_quantize_one_kernel<SRC, VEC, THREADS>, src, amax, data, scales,
                                              tensor_scale, rows, k, ld_src, ld_data),
                           "nvfp4_quantize launch");
}

template <int SRC, int VEC>
int launch_quantize_one(cudaStream_t s, const void* src, float* amax, uint8_t* data, uint8_t* scales, float* tensor_scale,
                        int rows, int k, long long ld_src, long long ld_data, int total)
{
    constexpr int kPerThread = kNvOneCtas * kNvItems;
    return total <= 256 * kPerThread
               ? launch_quantize_one_of<SRC, VEC, 256>(s, src, amax, data, scales, tensor_scale, rows, k, ld_src, ld_data, total)
           : total <= 512 * kPerThread
               ? launch_quantize_one_of<SRC, VEC, 512>(s, src, amax, data, scales, tensor_scale, rows, k, ld_src, ld_data, total)
               : launch_quantize_one_of<SRC, VEC, 1024>(s, src, amax, data, scales, tensor_scale, rows, k, ld_src, ld_data, total);
}

template <int DST, bool VEC>
int launch_dequantize(cudaStream_t s, const HostContext& host, const uint8_t* data, const uint8_t* scales, const float* tensor_scale,
                      void* out, int rows, int k, long long ld_data, long long ld_out)
{
    constexpr int kElems = DST == NV_F32 ? 8 : 16; // per thread
    int grid = 0;
    if (int rc = one_wave<nvfp4_dequantize_kernel<DST, VEC>>(static_cast<long long>(rows) * ((k + kElems - 1) / kElems), host, &grid)) {
        return rc;
    }
    count_launches(1);
    return note_cuda_error(launch_rows(host, nvfp4_dequantize_kernel<DST, VEC>, grid, kNvQuantThreads, s, data, scales, tensor_scale,
                                              out, rows, k, ld_data, ld_out),
                           "nvfp4_dequantize launch");
}

// The widest access that every row of a matrix starts on: 32 or 16 bytes, or 0 for its elements.
int row_access(const void* base, long long pitch_bytes)
{
    return !misaligned(base, 32) && pitch_bytes % 32 == 0 ? 32 : !misaligned(base, 16) && pitch_bytes % 16 == 0 ? 16 : 0;
}

// f<type, access>
#define PTO_NV_TYPES(type, access, f, ...)                                                      \
    ((type) == NV_F32 ? f<NV_F32, access>(__VA_ARGS__)                                          \
                      : (type) == NV_BF16 ? f<NV_BF16, access>(__VA_ARGS__) : f<NV_F16, access>(__VA_ARGS__))
#define PTO_NV_DISPATCH(type, access, f, ...)                                                   \
    ((access) == 32 ? PTO_NV_TYPES(type, 32, f, __VA_ARGS__)                                    \
                    : (access) == 16 ? PTO_NV_TYPES(type, 16, f, __VA_ARGS__) : PTO_NV_TYPES(type, 0, f, __VA_ARGS__))

// Instruction descriptor of kind::mxf4nvf4: e2m1 is 1 in both format fields ([7,10) and [10,12)), N >> 3 at [17,23),
// scale format e4m3 (0) at 23, M >> 7 at [27,29), K = 64 (0) at 31; scale ids 0, since an instruction uses all four
// bytes of a scale column.
uint32_t nv_idesc(int m_inst, int n_inst)
{
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n_inst >> 3) << 17) | (static_cast<uint32_t>(m_inst >> 7) << 27);
}

struct NvProblem {
    const uint8_t* a;
    const uint8_t* b;
    int m, n, k;
    long long lda, ldb; // 4-bit elements
};

template <int OUT>
int launch_nv_pair(cudaStream_t stream, const HostContext& host, const NvProblem& q, NvGemmParams p)
{
    auto kernel = gemm_nvfp4_2cta<OUT>;
    static std::atomic<int> max_clusters[kMaxDevices];
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(kNvPairThreads, 1, 1);
    cfg.dynamicSmemBytes = NvPairSmem::kTotal;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = max_clusters[host.device].load(std::memory_order_acquire);
    if (clusters == 0) {
        if (int rc = note_cuda_error(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NvPairSmem::kTotal),
                                     "cudaFuncSetAttribute(nvfp4 pair)")) {
            return rc;
        }
        cfg.gridDim = dim3(2, 1, 1);
        if (int rc = note_cuda_error(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg), "cudaOccupancyMaxActiveClusters")) {
            return rc;
        }
        clusters = clusters > 0 ? clusters : 1;
        max_clusters[host.device].store(clusters, std::memory_order_release);
    }
    p.m_tiles = (q.m + 255) / 256;
    p.n_tiles = (q.n + 255) / 256;
    p.group_m = 8;
    p.idesc = nv_idesc(256, 256);
    p.idesc_half = nv_idesc(256, 128);
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
    if (tiles > 1 << 29) {
        return PTO_B200_EINVAL;
    }
    const int leftover = static_cast<int>(tiles % clusters);
    const bool halves = leftover > 0 && 2 * leftover <= clusters;
    p.full_units = static_cast<int>(tiles) - (halves ? leftover : 0);
    p.units = static_cast<int>(tiles) + (halves ? leftover : 0);
    CUtensorMap ta, tb, tb_half, tsa, tsb;
    const long long sf_rows_a = (static_cast<long long>(q.m) + 127) / 128 * p.k_atoms * 2;
    const long long sf_rows_b = (static_cast<long long>(q.n) + 127) / 128 * p.k_atoms * 2;
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    int rc = encode_map_2d(&ta, u8, q.a, q.m, q.k / 2, q.lda / 2, 128, 128, true);
    rc = rc ? rc : encode_map_2d(&tb, u8, q.b, q.n, q.k / 2, q.ldb / 2, 128, 128, true);
    rc = rc ? rc : encode_map_2d(&tb_half, u8, q.b, q.n, q.k / 2, q.ldb / 2, 128, 64, true);
    rc = rc ? rc : encode_map_2d(&tsa, u8, p.sfa, sf_rows_a, 256, 256, 256, 8, false);
    rc = rc ? rc : encode_map_2d(&tsb, u8, p.sfb, sf_rows_b, 256, 256, 256, 8, false);
    constexpr int esize = OUT == NV_OUT_F32 ? 4 : 2;
    p.row_access = row_access(p.c, p.ldc * esize);
    if (rc) {
        return rc;
    }
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; // the kernel waits for what comes before it itself
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (p.units < clusters ? p.units : clusters)), 1, 1);
    count_launches(1);
    return note_cuda_error(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tb_half, tsa, tsb, p), "gemm_nvfp4_2cta launch");
}

template <int BLOCK_T, int OUT>
int launch_nv_few(cudaStream_t stream, const HostContext& host, const NvProblem& q, NvGemmParams p)
{
    using L = NvFewSmem<BLOCK_T>;
    auto kernel = gemm_nvfp4_few_rows<BLOCK_T, OUT>;
    static std::atomic<int> attr_done[kMaxDevices];
    if (attr_done[host.device].load(std::memory_order_acquire) == 0) {
        if (int rc = note_cuda_error(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal),
                                     "cudaFuncSetAttribute(nvfp4 few rows)")) {
            return rc;
        }
        attr_done[host.device].store(1, std::memory_order_release);
    }
    p.idesc = nv_idesc(128, BLOCK_T);
    CUtensorMap tw, tx;
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    int rc = encode_map_2d(&tw, u8, q.b, q.n, q.k / 2, q.ldb / 2, 128, 128, true);
    rc = rc ? rc : encode_map_2d(&tx, u8, q.a, q.m, q.k / 2, q.lda / 2, 128, BLOCK_T, true);
    if (rc) {
        return rc;
    }
    const long long n_tiles = (static_cast<long long>(q.n) + 127) / 128;
    const long long t_tiles = (static_cast<long long>(q.m) + BLOCK_T - 1) / BLOCK_T; // both fit a grid: launch_nv sees to it
    // K parts: as many as keep all of them resident at two CTAs per SM, each with four stages of K at least (with two,
    // 128x4096x4096 took 11.9 us instead of 9.9)
    int splits = 1;
    while (splits < 8 && n_tiles * t_tiles * splits * 2 <= 2ll * host.sm_count && p.k_stages >= splits * 8) {
        splits *= 2;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; // the kernel waits for what comes before it itself
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(splits), static_cast<unsigned>(n_tiles), static_cast<unsigned>(t_tiles));
    cfg.blockDim = dim3(kNvFewThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launches(1);
    return note_cuda_error(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p), "gemm_nvfp4_few_rows launch");
}

template <int OUT>
int launch_nv(cudaStream_t stream, const HostContext& host, const NvProblem& q, const NvGemmParams& p)
{
    // More than 128 rows: CTA pairs, unless the tiles are so few that the other kernel cuts K into four parts or more and K
    // is long enough to gain by it (beyond eight 256-element stages). Measured, few rows / pairs, us: 512x8192x8192 (64
    // tiles of 256 x 256) 22.1 / 16.5, 200x8192x4096 (32) 10.5 / 10.0, 200x4096x8192 (16) 11.5 / 14.6, 256x512x8192 (2)
    // 8.0 / 14.4, 144x512x1024 (2, four stages) 7.1 / 6.1. At most 128 rows: half of a pair's rows would be empty,
    // 128x8192x8192 12.4 / 14.9, 48x14336x4096 8.9 / 10.7. More columns than a grid's second axis counts in tiles of 128: pairs.
    const long long tiles256 = ((static_cast<long long>(q.m) + 255) / 256) * ((static_cast<long long>(q.n) + 255) / 256);
    constexpr int kMostFewColumns = 65535 * 128;
    if (q.n > kMostFewColumns || (q.m > 128 && (8 * tiles256 > host.sm_count || p.k_stages <= 8))) {
        return launch_nv_pair<OUT>(stream, host, q, p);
    }
    if (q.m <= 16) {
        return launch_nv_few<16, OUT>(stream, host, q, p);
    }
    if (q.m <= 32) {
        return launch_nv_few<32, OUT>(stream, host, q, p);
    }
    if (q.m <= 64) {
        return launch_nv_few<64, OUT>(stream, host, q, p);
    }
    return launch_nv_few<128, OUT>(stream, host, q, p);
}

int check_quantize(const void* data, const void* scales, const void* tensor_scale, const void* src, const void* amax, int rows,
                   int k, long long ld_src, long long ld_data, int src_dtype, int transpose)
{
    const long long length = transpose ? rows : k; // of the result's rows
    if (data == nullptr || scales == nullptr || tensor_scale == nullptr || src == nullptr || amax == nullptr || rows <= 0 ||
        k <= 0 || rows > kMaxExtent || k > kMaxExtent || ld_src < k || ld_data < (length + 15) / 16 * 8) {
        return PTO_B200_EINVAL;
    }
    const int type = source_of(src_dtype);
    if (type < 0) {
        return PTO_B200_EDTYPE;
    }
    if (misaligned(src, size_of(type)) || misaligned(data, 8) || ld_data % 8 != 0 || misaligned(scales, 4) ||
        misaligned(tensor_scale, 4) || misaligned(amax, 4)) {
        return PTO_B200_EALIGN;
    }
    return tensor_scale == amax ? PTO_B200_EINVAL : PTO_B200_OK; // one block writes the one while others still read the other
}

} // namespace
} // namespace pto_b200

using namespace pto_b200;

extern "C" size_t pto_b200_nvfp4_scale_bytes(int rows, int k)
{
    if (rows <= 0 || k <= 0) {
        return 0;
    }
    return ((static_cast<size_t>(rows) + 127) / 128) * ((static_cast<size_t>(k) + 63) / 64) * kNvAtomBytes;
}

extern "C" int pto_b200_amax(void* stream, float* amax, const uint8_t* src, int rows, int k, long long ld_src, int src_dtype)
{
    if (amax == nullptr || src == nullptr || rows <= 0 || k <= 0 || rows > kMaxExtent ||
        k > kMaxExtent || ld_src < k) {
        return PTO_B200_EINVAL;
    }
    const int type = source_of(src_dtype);
    if (type < 0) {
        return PTO_B200_EDTYPE;
    }
    const int es = size_of(type);
    if (misaligned(src, es) || misaligned(amax, 4)) {
        return PTO_B200_EALIGN;
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    return PTO_NV_DISPATCH(type, row_access(src, ld_src * es), launch_amax, static_cast<cudaStream_t>(stream), host, src, amax, rows, k, ld_src);
}

extern "C" int pto_b200_nvfp4_quantize(void* stream, uint8_t* data, uint8_t* scales, float* tensor_scale, const uint8_t* src,
                                       const float* amax, int rows, int k, long long ld_src, long long ld_data,
                                       int src_dtype, int transpose)
{
    if (int rc = check_quantize(data, scales, tensor_scale, src, amax, rows, k, ld_src, ld_data, src_dtype, transpose)) {
        return rc;
    }
    const int type = source_of(src_dtype);
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    return PTO_NV_DISPATCH(type, row_access(src, ld_src * size_of(type)), launch_quantize, static_cast<cudaStream_t>(stream), host, src, amax, data,
                           scales, tensor_scale, rows, k, ld_src, ld_data, transpose != 0);
}

extern "C" int pto_b200_nvfp4_quantize_dynamic(void* stream, uint8_t* data, uint8_t* scales, float* tensor_scale, float* amax,
                                               const uint8_t* src, int rows, int k, long long ld_src, long long ld_data,
                                               int src_dtype, int transpose)
{
    if (int rc = check_quantize(data, scales, tensor_scale, src, amax, rows, k, ld_src, ld_data, src_dtype, transpose)) {
        return rc;
    }
    const long long total = static_cast<long long>(rows) * ((k + 63LL) / 64 * 4);
    if (transpose || total > kNvOneBlocks) {
        if (int rc = pto_b200_amax(stream, amax, src, rows, k, ld_src, src_dtype)) {
            return rc;
        }
        return pto_b200_nvfp4_quantize(stream, data, scales, tensor_scale, src, amax, rows, k, ld_src, ld_data, src_dtype, transpose);
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    const int type = source_of(src_dtype);
    return PTO_NV_DISPATCH(type, row_access(src, ld_src * size_of(type)), launch_quantize_one, static_cast<cudaStream_t>(stream), src,
                           amax, data, scales, tensor_scale, rows, k, ld_src, ld_data, static_cast<int>(total));
}

extern "C" int pto_b200_nvfp4_dequantize(void* stream, uint8_t* out, const uint8_t* data, const uint8_t* scales,
                                         const float* tensor_scale, int rows, int k, long long ld_data, long long ld_out,
                                         int out_dtype)
{
    if (out == nullptr || data == nullptr || scales == nullptr || rows <= 0 || k <= 0 ||
        rows > kMaxExtent || k > kMaxExtent || ld_data < (static_cast<long long>(k) + 7) / 8 * 4 || ld_out < k) {
        return PTO_B200_EINVAL;
    }
    const int type = source_of(out_dtype);
    if (type < 0) {
        return PTO_B200_EDTYPE;
    }
    const int es = size_of(type);
    if (misaligned(out, es) || misaligned(data, 4) || ld_data % 4 != 0 || misaligned(tensor_scale, 4)) {
        return PTO_B200_EALIGN;
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (row_access(out, ld_out * es) == 32) {
        return PTO_NV_TYPES(type, true, launch_dequantize, s, host, data, scales, tensor_scale, out, rows, k, ld_data, ld_out);
    }
    return PTO_NV_TYPES(type, false, launch_dequantize, s, host, data, scales, tensor_scale, out, rows, k, ld_data, ld_out);
}

extern "C" int pto_b200_gemm_nvfp4(void* stream, uint8_t* out, const uint8_t* src0, const uint8_t* src1, const uint8_t* src2,
                                   const uint8_t* src3, const float* scale_a, const float* scale_b, const float* bias, int m,
                                   int n, int k, long long lda, long long ldb, long long ldc, int out_dtype)
{
    if (out_dtype != PTO_B200_F32 && out_dtype != PTO_B200_BF16 && out_dtype != PTO_B200_F16) {
        return PTO_B200_EDTYPE;
    }
    if (out == nullptr || src0 == nullptr || src1 == nullptr || src2 == nullptr || src3 == nullptr || m <= 0 || n <= 0 ||
        k <= 0 || m > kMaxExtent || n > kMaxExtent || k > kMaxExtent || k % 16 != 0 || lda < k || ldb < k || ldc < n) {
        return PTO_B200_EINVAL;
    }
    if (misaligned(src0, 16) || misaligned(src1, 16) || lda % 32 != 0 || ldb % 32 != 0 || misaligned(src2, 16) ||
        misaligned(src3, 16) || misaligned(out, out_dtype == PTO_B200_F32 ? 4 : 2) || misaligned(scale_a, 4) ||
        misaligned(scale_b, 4) || misaligned(bias, 4)) {
        return PTO_B200_EALIGN;
    }
    HostContext host;
    if (int rc = host_context(&host)) {
        return rc;
    }
    NvGemmParams p = {};
    p.c = out;
    p.ldc = ldc;
    p.m = m;
    p.n = n;
    p.k_atoms = (k + 63) / 64;
    p.k_stages = (p.k_atoms + 3) / 4;
    p.ga = scale_a;
    p.gb = scale_b;
    p.bias = bias;
    p.sfa = src2;
    p.sfb = src3;
    p.status = host.status;
    p.wait_limit = host.wait_limit;
    const NvProblem q{src0, src1, m, n, k, lda, ldb};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (out_dtype) {
        case PTO_B200_F32:
            return launch_nv<NV_OUT_F32>(s, host, q, p);
        case PTO_B200_BF16:
            return launch_nv<NV_OUT_BF16>(s, host, q, p);
        default:
            return launch_nv<NV_OUT_F16>(s, host, q, p);
    }
}
