// capi.cuh — what the C entry points share: status errors and their message,
// the guard that keeps exceptions inside the library, launches, the device
// guard.
#pragma once
#include <cuda_runtime.h>

#include <new>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/forge_b200.h"
#include "forgemodel.hpp"

// ---------------------------------------------------------------------------
// errors
// ---------------------------------------------------------------------------
inline thread_local std::string g_last_error;

struct Fb2Error {
    int status;
    std::string msg;
};

[[noreturn]] inline void fail(int status, const std::string& msg) { throw Fb2Error{status, msg}; }

inline void ck(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return;
    cudaGetLastError();  // the status reports it; the caller's next check must not
    if (e == cudaErrorMemoryAllocation) {
        fail(FB2_OUT_OF_MEMORY, std::string(what) + ": " + cudaGetErrorString(e));
    }
    fail(FB2_CUDA_ERROR, std::string(what) + ": " + cudaGetErrorString(e));
}
#define CK(x) ck((x), #x)

// Launch with programmatic stream serialization (the kernel itself waits in
// pdl_wait before touching global memory), so consecutive kernels of a step
// overlap launch and prologue; inside a stream capture this becomes a
// programmatic edge of the graph.
template <class... KArgs, class... Args>
void launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ck(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), "cudaLaunchKernelEx");
}

template <class F>
int32_t guarded(F&& f) {
    try {
        f();
        return FB2_OK;
    } catch (const Fb2Error& e) {
        g_last_error = e.msg;
        return e.status;
    } catch (const fb2::fm::InvalidData& e) {
        g_last_error = e.what();
        return FB2_INVALID_DATA;
    } catch (const std::bad_alloc&) {
        g_last_error = "host out of memory";
        return FB2_OUT_OF_MEMORY;
    } catch (const std::exception& e) {
        g_last_error = e.what();
        return FB2_CUDA_ERROR;
    }
}

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        cudaGetDevice(&prev);
        CK(cudaSetDevice(dev));
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};
