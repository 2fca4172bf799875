// dense_launch.h — launching the dense-layer kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "eas_internal.h"

// EAS_PDL=0 turns programmatic dependent launch off, here as for generated kernels.
inline bool dense_pdl_on() {
  static const bool on = [] {
    const char* e = getenv("EAS_PDL");
    return !(e && (e[0] == '0' || e[0] == 0 || !strcmp(e, "off")));
  }();
  return on;
}

// The grid before this one in the stream may still be running: nothing of global memory is touched
// before it has finished.  The next grid may be set up meanwhile, and waits in the same place.  What comes
// behind it reads by plain loads: read-only ones (__ldg) promise that nobody writes while the kernel runs,
// which the grid before may do, and could be moved before the wait.
__device__ __forceinline__ void grid_order() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One launch with one parameter struct.  cluster: CTAs per cluster where the kernel does not say
// itself, else 0.  The kernel begins with grid_order(), so it may be scheduled while the
// grid before it in the stream is finishing.
inline int dense_launch(const void* kernel, dim3 blocks, int cluster, int threads, int smem, cudaStream_t s,
                        void* params, const char* who) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dense_pdl_on()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)n;
  void* args[] = {params};
  return eas_cuda_check(cudaLaunchKernelExC(&cfg, kernel, args), who, EAS_ERR_LAUNCH);
}

inline int dense_sms(int dev) {
  static int cached[64] = {0};
  if (dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev);
  return cached[dev];
}
