// Programmatic dependent launch: the blocks of a launch may come up while the launch ahead of it in the stream still runs.
//
// Such a kernel calls grid_wait() before it touches what the launch ahead wrote, and in every block before the block ends, so
// that its own end implies the end of everything ahead of it. A kernel whose successor is launched that way calls
// grid_release() when the successor's blocks may come up; they take no room from its own blocks that have not started.
#ifndef MCSPARSE_B200_LAUNCH_H_
#define MCSPARSE_B200_LAUNCH_H_

#include <cuda_runtime.h>

namespace mcsp_b200 {

// Waits until the launch ahead of this one is done and its writes are seen.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// early = false: an ordinary launch.
template <typename... P, typename... A>
cudaError_t launch_behind(cudaStream_t s, bool early, void (*kernel)(P...), unsigned blocks, int threads, int shared, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)shared;
    cfg.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace mcsp_b200

#endif  // MCSPARSE_B200_LAUNCH_H_
