/*
 * ops_launch.cuh -- a kernel's launch and its own error: what the runtime holds as the last error may be an earlier call's,
 * and what a launch that fails leaves there is not left for others to find.
 */
#pragma once
#include <cuda_runtime.h>

/* at: launch attributes */
template <typename... P, typename... A>
static int ops_launch(void (*k)(P...), dim3 grid, int threads, int smem, cudaStream_t st, cudaLaunchAttribute *at, int n_at, A... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    c.attrs = at;
    c.numAttrs = n_at;
    const cudaError_t rc = cudaLaunchKernelEx(&c, k, args...);
    if (rc != cudaSuccess) cudaGetLastError();
    return (int)rc;
}

template <typename... P, typename... A>
static int ops_launch(void (*k)(P...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
    return ops_launch(k, grid, threads, smem, st, (cudaLaunchAttribute *)nullptr, 0, args...);
}
