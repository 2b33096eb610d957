// launch.cuh -- programmatic dependent launch for the small operator kernels: every kernel is launched so that it may
// start while the kernel ahead of it is still running; it waits for that kernel (griddepcontrol.wait: all prerequisite
// grids complete, their writes visible) before it reads anything, then lets the kernel after it launch at once (dep_enter;
// one kernel does it in parts of its own: kv4_prompt_kernel reads early what the kernel before the last one left, and one warp
// of each CTA waits for the last one). Without such a launch both are no-ops. And the encoder of tensor maps.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

__device__ __forceinline__ void dep_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// a kernel launch that lets the kernel start before the one ahead of it on the stream finishes (see dep_enter)
template <typename Kern, typename... Args>
cudaError_t launch_dep(Kern k, dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

// cuTensorMapEncodeTiled, or null
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)f;
  }
  return fn;
}
