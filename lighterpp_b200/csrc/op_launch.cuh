// Launching stand-alone operator kernels: shared by the files that hold their entry points.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/lpp_b200.h"

namespace {

inline lpp_status chk() { return cudaGetLastError() == cudaSuccess ? LPP_OK : LPP_ERR_CUDA; }
inline cudaStream_t S(void* s) { return (cudaStream_t)s; }
inline int blocks(long long n, int t) { return (int)std::max<long long>(1, (n + t - 1) / t); }

// Launches an operator kernel.  It may start while the kernel before it in the stream ends (it waits for it in op_begin):
// 18 operators of a layer one after the other take about a microsecond less each.  A stream that is being captured gets a plain
// launch, because what comes before it in the graph need not be a kernel; behind: it is one, this operator's own.  cluster: CTAs of a cluster along x.
template <typename... KArgs, typename... Args>
lpp_status launch_op_cluster(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, bool behind, cudaStream_t s, Args... args) {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (!behind && cudaStreamIsCapturing(s, &capturing) != cudaSuccess) {
        (void)cudaGetLastError();
        capturing = cudaStreamCaptureStatusActive;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2] = {};
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    if (capturing == cudaStreamCaptureStatusNone) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
    return chk();
}
// Lets a kernel have `bytes` (the same at every call) of shared memory: once on every device, since asked at every launch it is 0.4 us of
// the host's time.
template <auto KERNEL>
bool allow_smem(int bytes) {
    static std::atomic<bool> allowed[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (allowed[dev].load(std::memory_order_relaxed)) return true;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        return false;
    }
    allowed[dev].store(true, std::memory_order_relaxed);
    return true;
}
template <typename... KArgs, typename... Args>
lpp_status launch_op(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s, Args... args) {
    return launch_op_cluster(kernel, grid, threads, smem, 1, false, s, args...);
}
template <typename... KArgs, typename... Args>
lpp_status launch_behind(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s, Args... args) {
    return launch_op_cluster(kernel, grid, threads, smem, 1, true, s, args...);
}

}  // namespace
