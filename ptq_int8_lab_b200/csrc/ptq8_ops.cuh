// What the host sides of the token operators share: the handle, refusals, launches.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "ptq8.h"
#include "ptq8_ptx.cuh"

struct ptq8_ops {
    int device = 0;
    int sms = 0;
    int* error = nullptr;       // pinned host word that a kernel whose bounded wait ran out sets (error_word())
    int* error_dev = nullptr;   // its device address
    long long wait_limit = ptq8::kWaitLimitCycles;
    int stall = 0;
    int variant = -1, split = 1;   // test hook: the tile variant of every product
    PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    char err[512] = "";         // message of the last refusal: a fixed buffer, since refusing must not throw
};

namespace ptq8 {

inline int fail(ptq8_ops* o, int status, const char* f, ...) {
    va_list ap;
    va_start(ap, f);
    std::vsnprintf(o->err, sizeof o->err, f, ap);
    va_end(ap);
    return status;
}

// A message for a caller who has no handle yet.
inline void say(char* err, size_t n, const char* f, const char* more = "") {
    if (err && n) std::snprintf(err, n, f, more);
}

// The device becomes current for the call and is given back: a process may drive several.
struct OnDevice {
    int before = -1;
    cudaError_t rc;
    explicit OnDevice(int device) {
        rc = cudaGetDevice(&before);
        if (rc == cudaSuccess && before != device) rc = cudaSetDevice(device);
        if (before == device) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// One launch with programmatic stream serialization: the kernel may be scheduled while the kernel
// before it on the stream drains, and waits (griddepcontrol.wait) before it touches global memory.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline size_t type_size(int t) { return t == PTQ8_F32 ? 4 : 2; }

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// What every call checks first: a wait of an earlier call that ran out, until it is cleared.
inline int ready(ptq8_ops* o) {
    if (*static_cast<volatile int*>(o->error))
        return fail(o, PTQ8_ERR_TIMEOUT, "a device wait of an earlier call ran out (code %d); its outputs are invalid",
                    *o->error);
    return PTQ8_OK;
}

inline int cuda_fail(ptq8_ops* o, const char* what, cudaError_t e) {
    cudaGetLastError();   // reported here: the process's next check must not find it again
    return fail(o, PTQ8_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// What the kernels of the other sources need set once per device, at a handle's creation.
cudaError_t cache_attributes();
cudaError_t w4_attributes();

}  // namespace ptq8
