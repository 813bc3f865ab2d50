// What the library's translation units share on the host side: the device's state, launches and tensor maps.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace arc {

// The dynamic part of a decode kernel's shared memory may use the opt-in maximum minus this reserve.
constexpr int kDecodeStaticSmem = 1024;

// Of the current device (arc_sdpa.cu keeps it).
struct HostState {
    uint32_t* fault;  // the status word kernels report to
    int sm_count, smem_optin;
    int device;
    int decode_clusters[9];  // [size]: clusters of decode CTAs the device holds at once
};
constexpr int kMaxDevices = 64;
int host_state(HostState* out);

// Keeps the text of a failing CUDA call for arc_sdpa_last_error(); returns ARC_ERR_CUDA.
int cuda_fail(const char* what, cudaError_t e);

#define ARC_CUDA(call)                                      \
    do {                                                    \
        cudaError_t e_ = (call);                            \
        if (e_ != cudaSuccess) return cuda_fail(#call, e_); \
    } while (0)

// A tensor map of bf16 values, 128-byte swizzle, reads past the end are zero.  strides: bytes, of all dimensions but the first.
int encode_bf16_map(CUtensorMap* tm, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                    const char* what);

void count_launch();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename K>
static cudaError_t opt_in_smem(K kernel, int bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// Launch `kernel` behind the previous kernel of `stream` with programmatic serialization: its CTAs may be scheduled and
// run up to their grid_dependency_wait() while that kernel is still running, which takes the launch latency and the
// prologue off the critical path (2-3 us of a small call).  Every kernel of the library is launched this way, and every
// one of them waits before it touches global memory and only then releases the kernel behind it
// (grid_launch_dependents): so when a kernel may run, everything in front of its predecessor has completed, and no grid
// completes before the one in front of it has.  cluster > 1: in clusters of that many CTAs along x.
template <typename... KArgs, typename... Args>
static cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster,
                                    Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

}  // namespace arc
