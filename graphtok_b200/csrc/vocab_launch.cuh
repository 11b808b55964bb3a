// Kernel launches that overlap the end of the one before on the stream.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <utility>

namespace gtok {

// A kernel launched so may begin while the one before it on the stream still runs; what it reads of that one's it reads behind this.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches that may begin before the kernel in front of them on the stream has ended (see after_previous).
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), int64_t blocks, int threads, int smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}

}  // namespace gtok
