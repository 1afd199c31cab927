// Helpers of the C entry points that more than one source file of the library uses.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

namespace gnf4b {

struct DevInfo {
    int sm_count = 0;
    int smem_optin = 0;
    bool ok = false;
};

// records the text gnf4b_last_cuda_error returns; always GNF4B_ECUDA
int cuda_fail(cudaError_t e, const char* what);
// of the current device, looked up once
int device_info(DevInfo* out);

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// cudaFuncSetAttribute is per device and not free; raise a kernel's dynamic shared-memory
// limit only when a launch needs more than was already granted on this device.  One thread at a time: a smaller limit
// set between another thread's larger one and its record would leave a record of more than the kernel has.
inline std::mutex& smem_limit_mutex() {
    static std::mutex mu;
    return mu;
}
template <typename F>
static cudaError_t ensure_smem(F kfn, size_t smem, int* granted /*[64], zero-initialised*/) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    dev &= 63;
    std::lock_guard<std::mutex> lock(smem_limit_mutex());
    if ((int)smem > granted[dev]) {
        e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        granted[dev] = (int)smem;
    }
    return cudaSuccess;
}

// Launch with programmatic stream serialization: the kernel may start while its predecessor in the stream is
// still running and must call pdl_wait() before it touches anything (reads or writes) the predecessor may use.
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl_smem(void (*kfn)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                                   Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kfn, static_cast<KArgs>(args)...);
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kfn)(KArgs...), unsigned grid, unsigned block, cudaStream_t st, Args... args) {
    return launch_pdl_smem(kfn, grid, block, 0, st, args...);
}

}  // namespace gnf4b
