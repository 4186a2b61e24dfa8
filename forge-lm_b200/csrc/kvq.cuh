// kvq.cuh — the paged, quantised K/V cache: formats, write and read back.
//
// A row (one token's K or V of one head, head_dim values) is quantised by
// itself, so a write touches nothing but its own bytes and meta word:
//   int8: scale = max|x| / 127, code = rint(x * (127 / max|x|)), byte = code + 128;
//   int4: min = bf16(min x), scale = bf16((max x - min x) / 15),
//         code = clamp(rint((x - min) * (1 / scale)), 0, 15).
// All in fp32 with IEEE division and rounding to nearest even; the codes use
// the rounded scale and minimum, so the stored row is the best one for them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fb2 {

constexpr int KVQ_INT8 = 0, KVQ_INT4 = 1;
constexpr float kKvqTiny = 1e-35f;  // below: the row (or 4-bit group) is a constant, its 1 / scale would overflow

// The cache as the kernels see it.
struct KvqView {
    unsigned char* codes;
    uint32_t* meta;
    int n_slots;      // n_pages * page_size
    int page_shift;   // log2 page_size
    int heads, hd;
    int row_bytes;
    // index of (slot, head, kind)'s row: the rows of a page's head lie together
    FB2_DEV size_t row(int slot, int head, int kind) const {
        const size_t page = (uint32_t)slot >> page_shift;
        return ((((page * heads + head) * 2 + kind) << page_shift) | (slot & ((1 << page_shift) - 1)));
    }
};

FB2_DEV float bf16_bits_to_float(uint32_t b) { return __uint_as_float(b << 16); }
FB2_DEV uint32_t float_to_bf16_bits(float f) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// Element types of dense tensors: 8 consecutive values <-> fp32.
template <class T>
struct Dense;
template <>
struct Dense<float> {
    static FB2_DEV float get(float v) { return v; }
    static FB2_DEV float put(float v) { return v; }
};
template <>
struct Dense<__nv_bfloat16> {
    static FB2_DEV float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static FB2_DEV __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Dense<__half> {
    static FB2_DEV float get(__half v) { return __half2float(v); }
    static FB2_DEV __half put(float v) { return __float2half_rn(v); }
};

// 8 values from p (VEC: p is 16-byte aligned).
template <class T, bool VEC>
FB2_DEV void load8(const T* p, float (&x)[8]) {
    if constexpr (VEC) {
        constexpr int N = sizeof(T) / 2;  // 16-byte pieces of 8 values
        uint4 w[N];
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Dense<T>::get(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Dense<T>::get(p[i]);
    }
}
template <class T>
FB2_DEV void store8(T* p, const float (&x)[8]) {
    constexpr int N = sizeof(T) / 2;
    uint4 w[N];
    T* t = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = Dense<T>::put(x[i]);
#pragma unroll
    for (int i = 0; i < N; i++) reinterpret_cast<uint4*>(p)[i] = w[i];
}

// 8 codes (8 bytes of int8, 4 bytes of int4) and the row's meta word -> values.
FB2_DEV void kvq_decode8(uint2 c, float scale, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t byte = ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xffu;
        x[i] = (float)((int)byte - 128) * scale;
    }
}
FB2_DEV void kvq_decode8(uint32_t c, float scale, float least, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = fmaf((float)((c >> (4 * i)) & 15u), scale, least);
}

// A row's lanes are `width` (a power of two, >= head_dim / 8) neighbours of a
// warp, 8 values each; blockIdx.y: K or V.
constexpr int KVQ_THREADS = 256;

template <class T, int FMT, bool VEC>
__global__ void __launch_bounds__(KVQ_THREADS)
    k_kvq_write(KvqView c, int n_rows, const T* __restrict__ k, const T* __restrict__ v, long long k_row, long long k_head,
                long long v_row, long long v_head, const int* __restrict__ slots, int width) {
    const int kind = blockIdx.y;
    const long long item = ((long long)blockIdx.x * KVQ_THREADS + threadIdx.x) / width;
    const int part = threadIdx.x & (width - 1);
    const int row = (int)(item / c.heads), head = (int)(item - (long long)row * c.heads);
    // lanes of a row agree on `live`; the shuffles below run with the whole warp
    const int slot = row < n_rows ? __ldg(slots + row) : -1;
    const bool live = (uint32_t)slot < (uint32_t)c.n_slots;
    const bool mine = live && part * 8 < c.hd;
    float x[8];
    if (mine) {
        const T* p = kind ? v + row * v_row + head * v_head : k + row * k_row + head * k_head;
        load8<T, VEC>(p + part * 8, x);
    }
    if constexpr (FMT == KVQ_INT8) {
        // max|x| through the bits: NaN > inf > finite
        uint32_t top = 0;
        if (mine)
#pragma unroll
            for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        for (int o = width / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool finite = top < 0x7f800000u;
        const float amax = __uint_as_float(top);
        const bool some = finite && amax >= kKvqTiny;
        const float inv = some ? 127.0f / amax : 0.0f;
        if (!mine) return;
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int code = some ? (int)fminf(fmaxf(rintf(x[i] * inv), -127.0f), 127.0f) : 0;
            w[i >> 2] |= (uint32_t)(code + 128) << (8 * (i & 3));
        }
        const size_t at = c.row(slot, head, kind);
        *reinterpret_cast<uint2*>(c.codes + at * c.row_bytes + part * 8) = make_uint2(w[0], w[1]);
        if (part == 0)
            c.meta[at] = finite ? __float_as_uint(some ? amax / 127.0f : 0.0f) : 0x7fc00000u;
    } else {
        const float inf = __uint_as_float(0x7f800000u);
        float lo = inf, hi = -inf;
        if (mine)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool nan = x[i] != x[i];
                lo = fminf(lo, nan ? -inf : x[i]);
                hi = fmaxf(hi, nan ? inf : x[i]);
            }
        for (int o = width / 2; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        if (!mine) return;
        uint32_t scale_b = float_to_bf16_bits((hi - lo) / 15.0f);
        const uint32_t least_b = float_to_bf16_bits(lo);
        const float least = bf16_bits_to_float(least_b);
        float scale = bf16_bits_to_float(scale_b);
        const bool finite = scale < inf && fabsf(least) < inf;  // false for NaN
        const bool some = finite && scale >= kKvqTiny;
        const float inv = some ? 1.0f / scale : 0.0f;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int code = some ? (int)fminf(fmaxf(rintf((x[i] - least) * inv), 0.0f), 15.0f) : 0;
            w |= (uint32_t)code << (4 * i);
        }
        const size_t at = c.row(slot, head, kind);
        *reinterpret_cast<uint32_t*>(c.codes + at * c.row_bytes + part * 4) = w;
        if (part == 0) c.meta[at] = finite ? ((some ? scale_b : 0u) | (least_b << 16)) : 0x7fc07fc0u;
    }
}

template <class T, int FMT>
__global__ void __launch_bounds__(KVQ_THREADS)
    k_kvq_read(KvqView c, int n_rows, const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int width) {
    const int kind = blockIdx.y;
    const long long item = ((long long)blockIdx.x * KVQ_THREADS + threadIdx.x) / width;
    const int part = threadIdx.x & (width - 1);
    const int row = (int)(item / c.heads), head = (int)(item - (long long)row * c.heads);
    if (row >= n_rows || part * 8 >= c.hd) return;
    const int slot = __ldg(slots + row);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if ((uint32_t)slot < (uint32_t)c.n_slots) {
        const size_t at = c.row(slot, head, kind);
        const uint32_t m = c.meta[at];
        if constexpr (FMT == KVQ_INT8)
            kvq_decode8(*reinterpret_cast<const uint2*>(c.codes + at * c.row_bytes + part * 8), __uint_as_float(m), x);
        else
            kvq_decode8(*reinterpret_cast<const uint32_t*>(c.codes + at * c.row_bytes + part * 4),
                        bf16_bits_to_float(m & 0xffffu), __uint_as_float(m & 0xffff0000u), x);
    }
    store8((kind ? v : k) + (size_t)item * c.hd + part * 8, x);
}

}  // namespace fb2
