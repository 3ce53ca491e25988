// Launch with programmatic dependent launch: the grid may start while the
// kernel before it on the stream drains; it waits (grid_dependency_wait)
// before it touches memory.
#pragma once

#include "common.cuh"

namespace ic {

inline int launch_pdl(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t st, void** args,
                      const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelExC(&cfg, fn, args);
  return launch_status(what);
}

}  // namespace ic
