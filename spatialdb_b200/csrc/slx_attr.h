// slx_attr.h -- per-device launch settings shared by the kernel launchers.
#pragma once
#include <cstddef>
#include <cuda_runtime.h>

namespace slx {

// Raises `func`'s dynamic shared memory limit to at least `bytes` on the current device.
// cudaFuncSetAttribute acts on one device only, so the setting is recorded per (kernel, device):
// a process that drives several GPUs (one context per device) sets it once on each. Thread-safe.
// Requests up to the 48 KiB default need no attribute and return at once.
cudaError_t ensure_smem(const void* func, size_t bytes);

// Streaming multiprocessors of the current device (cached per device).
int device_sm_count();

// Launches `fn` so that it may start while the kernel before it in the stream still runs (programmatic stream
// serialization): its prologue, and loads of what no kernel in the stream writes, overlap that kernel's last
// blocks. The kernel calls grid_wait() before it touches anything else, and grid_release() once it has started.
template <class... P, class... A>
cudaError_t launch_early(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = (unsigned)cluster;
        at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    cfg.attrs = at;
    return cudaLaunchKernelEx(&cfg, fn, P(args)...);
}
#ifdef __CUDACC__
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

}  // namespace slx
