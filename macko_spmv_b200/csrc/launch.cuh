// Launches with programmatic stream serialization: the kernel may start while the previous one of the stream finishes and waits
// for it itself (griddepcontrol.wait).
#pragma once

#include "common.cuh"

namespace macko {

template <typename T> struct Same { using type = T; };

// `cluster` > 1: thread-block clusters of that many CTAs along x (the grid is a multiple of it). `smem`: dynamic shared memory.
template <typename... Args>
int launch_pdl(const char *what, void (*kernel)(Args...), dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t stream,
               typename Same<Args>::type... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return fail(MACKO_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
    return MACKO_OK;
}

}  // namespace macko
