// What the entry points of the operators on device memory share: the bound device, the caller's stream, launches, set-up inside a caller's capture.
#pragma once
#include "../../include/fastllm_b200.h"
#include "bert_model.cuh"
#include "runtime.cuh"

namespace fl {

// The bound device for the length of a call; the caller's own is put back.
struct DeviceScope {
    int before = -1, now;
    DeviceScope() : now(bound_device()) {
        FL_CUDA(cudaGetDevice(&before));
        if (before != now) FL_CUDA(cudaSetDevice(now));
    }
    ~DeviceScope() { if (before >= 0 && before != now) cudaSetDevice(before); }
};

inline LaunchCtx op_ctx(void* stream) {
    LaunchCtx lc;
    lc.stream = static_cast<cudaStream_t>(stream);
    lc.pdl = false;
    if (g_prof.on) {                        // (no events inside a caller's capture)
        cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
        FL_CUDA(cudaStreamIsCapturing(lc.stream, &st));
        lc.capturing = st != cudaStreamCaptureStatusNone;
    }
    return lc;
}
inline size_t dtype_size(int dtype) { return dtype == FL_DTYPE_F32 ? 4 : dtype == FL_DTYPE_I8 ? 1 : 2; }
inline bool is_float(int dtype) { return dtype == FL_DTYPE_F32 || dtype == FL_DTYPE_BF16 || dtype == FL_DTYPE_F16; }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxRows = (int64_t)1 << 30;
// Launch of an operator's kernel in clusters of `cluster` blocks; pdl: it may start under the kernel before it, which this call launched too
// (never under a caller's).
template <typename... KArgs, typename... Args>
inline void launch_op(LaunchCtx& lc, const char* tag, uint64_t bytes, void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, bool pdl, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = lc.stream;
    cudaLaunchAttribute attr[2];
    const bool prof = g_prof.on && !lc.capturing;
    if (pdl && !prof) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    ProfEntry pe;
    if (prof) {
        pe.tag = tag;
        pe.bytes = bytes;
        FL_CUDA(cudaEventCreate(&pe.e0));
        FL_CUDA(cudaEventCreate(&pe.e1));
        FL_CUDA(cudaEventRecord(pe.e0, lc.stream));
    }
    FL_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
    if (prof) {
        FL_CUDA(cudaEventRecord(pe.e1, lc.stream));
        g_prof.entries.push_back(pe);
    }
    if (lc.capturing) lc.captured++;
    else g_launches.fetch_add(1, std::memory_order_relaxed);
}

// Unsafe calls for the length of a scope: set-up does not belong to a graph that the caller's thread may be capturing.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { FL_CUDA(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
template <typename... Kernels>
inline void load_kernels(Kernels... kernels) {
    cudaFuncAttributes at;
    for (cudaError_t e : {cudaFuncGetAttributes(&at, kernels)...}) FL_CUDA(e);
}

}  // namespace fl
