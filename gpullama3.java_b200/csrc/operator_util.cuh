// operator_util.cuh -- what the entry points of the operators on device memory share: messages, the caller's device, dispatch by head size and type, launches.
#pragma once
#include "../../include/b200llama.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

namespace {

int say(char *err, size_t len, int code, const char *fmt, ...) {
    if (err && len) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, len, fmt, ap);
        va_end(ap);
    }
    return code;
}
int cuda_code(cudaError_t e) { return e == cudaErrorMemoryAllocation ? B200_ERR_OOM : B200_ERR_CUDA; }

// The calling thread's device is what it was when an entry point returns.
struct OnDevice {
    int before = -1;
    cudaError_t error;
    explicit OnDevice(int device) {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

template <typename F> cudaError_t by_head_size(int hs, F &&f) { // f(integral_constant<head size>)
    switch (hs) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 96: return f(std::integral_constant<int, 96>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
    }
    return cudaErrorInvalidValue;
}
template <typename F> cudaError_t by_type(int type, F &&f) { // f(a value of the type)
    if (type == B200_GGML_F32) return f(0.0f);
    if (type == B200_GGML_F16) return f(__half());
    return f(__nv_bfloat16());
}
bool known_type(int type) { return type == B200_GGML_F32 || type == B200_GGML_F16 || type == B200_GGML_BF16; }
int type_bytes(int type) { return type == B200_GGML_F32 ? 4 : 2; }
bool aligned16(const void *p, long long stride, int bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0; }

template <typename... KA, typename... A>
cudaError_t launch(void (*kern)(KA...), dim3 grid, int block, size_t smem, int cluster, bool pdl, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KA>(args)...);
}
// Shared memory limit of a kernel, set in front of every launch that needs more than the usual 48 KB: an attribute of the function in the current device's context, so that nothing is kept
// here by device or by thread (0.2 us).
template <typename K> cudaError_t allow_smem(K kern, size_t smem) {
    return smem > 48 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
}
int sm_count(int device) {
    int n = 0;
    return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess && n > 0 ? n : 148;
}
int cluster_for(long long units, long long wanted, long long most) { // the largest power of two with units * cluster <= wanted, at most `most`
    int c = 1;
    while (2 * c <= most && units * 2 * c <= wanted) c *= 2;
    return c;
}

} // namespace
