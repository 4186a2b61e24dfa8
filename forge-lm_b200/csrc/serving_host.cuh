// serving_host.cuh — what the serving operators' C entries share: checks of
// arguments, the element type, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <mutex>
#include <set>

#include "capi.cuh"

inline void need(bool ok, const char* msg) {
    if (!ok) fail(FB2_INVALID_ARG, msg);
}
inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline bool pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }
inline int log2_of(int v) {
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}
inline size_t size_of(int dtype) { return dtype == FB2_F32 ? 4 : 2; }
inline void check_dtype(int dtype) { need(dtype == FB2_F32 || dtype == FB2_BF16 || dtype == FB2_F16, "dtype must be FB2_F32, FB2_BF16 or FB2_F16"); }

// f(T{}) for the element type of `dtype`
template <class F>
void with_type(int dtype, F&& f) {
    if (dtype == FB2_F32)
        f(float{});
    else if (dtype == FB2_BF16)
        f(__nv_bfloat16{});
    else
        f(__half{});
}

inline void launched() { CK(cudaGetLastError()); }

// Dynamic shared memory above 48 KB, once per kernel and device.
inline void opt_in_smem(const void* kernel, int bytes) {
    static std::mutex lock;
    static std::set<std::pair<const void*, int>> done;
    int device = 0;
    CK(cudaGetDevice(&device));
    std::lock_guard<std::mutex> hold(lock);
    if (done.count({kernel, device})) return;
    CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert({kernel, device});
}
