// What the sources behind the C ABI share on the host side: per-device set-up, tensor maps, error notes, launch counts.
#pragma once
#include "../../include/pto_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

namespace pto_b200 {

constexpr int kMaxDevices = 64;

constexpr int kMaxExtent = 0x7FFFF000; // of a matrix: kernels count past it in steps of a tile

struct HostContext {
    int device;           // ordinal of the current device, below kMaxDevices
    int sm_count;
    int* status;          // device address of the status word the kernels record a given-up wait in
    long long wait_limit; // cycles one bounded wait may take
};

// The current device's context; a PTO_B200 code other than 0 when it is no sm_100 GPU or a CUDA call fails.
int host_context(HostContext* out);

// Records the text of a failed CUDA call for pto_b200_last_cuda_error; PTO_B200_OK or PTO_B200_ECUDA.
int note_cuda_error(cudaError_t e, const char* what);

// Counts kernel launches for pto_b200_launch_count.
void count_launches(int n);

// Launches a one-dimensional grid; a small one may start while the launch before it in the stream ends (programmatic
// serialisation), so the kernel has to call ptx::grid_dependency_wait before it touches global memory. Small: two blocks per
// SM at most. That saves 0.4 us of 2; the NVFP4 cast of 16384x8192 bf16, five blocks per SM, took 84 us that way instead of 75.
template <typename... P, typename... A>
cudaError_t launch_rows(const HostContext& host, void (*kernel)(P...), int grid, int threads, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = grid <= 2 * host.sm_count ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// 2-D map of [rows, cols] elements of `type` with a row pitch in bytes and 128-byte swizzled (or plain) boxes.
int encode_map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, long long cols,
                  long long pitch_bytes, int box_cols, int box_rows, bool swizzle128);

} // namespace pto_b200
