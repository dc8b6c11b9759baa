// Kernel launch helper: every kernel of the library goes through cudaLaunchKernelEx with the programmatic
// stream-serialisation attribute (see pdl_wait() in common.cuh), unless the option `pdl` is 0.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "options.h"

namespace lfm25 {

inline bool pdl_enabled() { return option(kOptPdl) != 0; }

template <typename... Parameters, typename... Arguments>
cudaError_t launch_kernel(void (*kernel)(Parameters...), unsigned int blocks, unsigned int threads, size_t shared_bytes,
                          cudaStream_t stream, unsigned int cluster, Arguments... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = shared_bytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    unsigned int count = 0;
    if (pdl_enabled()) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    if (cluster > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = cluster;
        attributes[count].val.clusterDim.y = 1;
        attributes[count].val.clusterDim.z = 1;
        ++count;
    }
    config.attrs = attributes;
    config.numAttrs = count;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

// Dynamic shared memory of a kernel beyond 48 KB, and clusters of more than 8 CTAs, allowed once per device: the calls cost as much
// as a small launch.
template <auto Kernel, bool LargeClusters = false>
cudaError_t allow_shared_memory(size_t bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    const uint64_t bit = uint64_t{1} << (device & 63);
    if (status != cudaSuccess || (done.load(std::memory_order_relaxed) & bit) != 0) {
        return status;
    }
    status = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (status == cudaSuccess && LargeClusters) {
        status = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    }
    if (status == cudaSuccess) {
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    return status;
}

}  // namespace lfm25
