#pragma once
#include "common.cuh"

namespace hipattn {

// A launch that may be prepared while the kernel before it on the stream is still running, and a kernel so launched: in_turn() stands before all that it
// reads and writes, waits for all of that kernel (and so for everything before it), and lets the launch behind this one be prepared.
// One exception: paged_decode_merge_kernel reads rows and lengths before it.  The launch before is always the kernel whose parts it joins, which has
// waited itself before it let this one be prepared, so that all before it is over, and which writes neither.
// Such a kernel may have begun before what it reads was written, so it reads nothing by way of the read-only cache (no __ldg).
// Back to back on a stream: a few requests' pages freed and dealt out 10.2 us, 6.7 so.
struct InTurn {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  InTurn(int64_t grid, int threads, size_t smem, cudaStream_t stream, int cluster = 1) {
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
  }
};
__device__ __forceinline__ void in_turn() { asm volatile("griddepcontrol.wait;\ngriddepcontrol.launch_dependents;\n" ::: "memory"); }

}  // namespace hipattn
