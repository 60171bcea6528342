// launch.cuh -- launches that may start before the kernel ahead of them in the stream has ended.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace cvattn {

// fn calls griddep_wait() in every thread, or in some of each CTA's before a barrier of all, before it reads or writes global
// memory: only its launch and what it does with its own SM (barriers, TMEM, the first instructions) overlap the end of the
// kernel before it.  (Graph of 20 calls: commit of one utterance's path 2.8 -> 2.3 us, scores of one row over 500 positions
// 4.5 -> 4.2, eviction of 576 to 512 8.1 -> 7.9.)
template <class... P, class... A>
inline cudaError_t launch_overlapped(void (*fn)(P...), dim3 grid, int block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, std::forward<A>(args)...);
}

// The same with `cluster` CTAs of the grid's first dimension to a cluster.
template <class... P, class... A>
inline cudaError_t launch_overlapped_clusters(void (*fn)(P...), dim3 grid, int block, size_t smem, int cluster, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fn, std::forward<A>(args)...);
}

}  // namespace cvattn
