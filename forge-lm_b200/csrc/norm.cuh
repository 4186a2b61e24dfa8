// norm.cuh — a block's output onto the residual stream and the norm before the
// next block, in one pass, and rows as 8-bit codes (include/forge_b200.h,
// fb2_residual_norm and fb2_quantise_rows, has the formulas).
//
// A row is held in the registers of the threads that share it, as fp32, from the
// first load to the last store: h and x are read once, the stream and the normed
// row written once, and means and variances are taken of values at hand (the
// variance of differences from the mean, not of squares).  What bounds it is HBM
// where there are rows enough.
#pragma once
#include "kvq.cuh"

namespace fb2 {

constexpr int NORM_E = 8;         // consecutive values of a thread
constexpr int NORM_MOST = 32768;  // of a row: 1024 threads with 32 each

struct NormArgs {
    const void *h, *x, *gate;  // gate NULL: 1
    const float *w, *b, *post_w, *post_b;
    void *sum, *y;
    signed char* codes;
    float* scales;
    long long h_row, x_row, gate_row, sum_row, y_row, code_row;
    int rows, dim;
    float scale, eps;
    bool rms, post;
};

namespace nrm {

// Sum (or, of bits, largest) over the G threads that share a row.
template <int G>
FB2_DEV float sum(float v, float* s) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        __syncthreads();  // s may still be read from the last time
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < G / 32; i++) v += s[i];
    }
    return v;
}
template <int G>
FB2_DEV uint32_t largest(uint32_t v, float* s) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (G > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = __uint_as_float(v);
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < G / 32; i++) v = max(v, __float_as_uint(s[i]));
    }
    return v;
}

// 8 values of a row from `at` on; those past `n` are 0.
template <class T, bool VEC>
FB2_DEV void load(const T* row, int at, int n, float (&v)[NORM_E]) {
    if constexpr (VEC) {
        if (at < n) {
            load8(row + at, v);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < NORM_E; i++) v[i] = at + i < n ? Dense<T>::get(row[at + i]) : 0.f;
}
template <class T, bool VEC>
FB2_DEV void store(T* row, int at, int n, const float (&v)[NORM_E]) {
    if constexpr (VEC) {
        if (at >= n) return;
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < NORM_E; i += N) *reinterpret_cast<uint4*>(row + at + i) = pack16<T>(v + i);
    } else {
#pragma unroll
        for (int i = 0; i < NORM_E; i++)
            if (at + i < n) row[at + i] = Dense<T>::put(v[i]);
    }
}

// 127 / top and top / 127 of a row whose largest |value| has these bits: (0, 0)
// where it is too small to be divided by, a NaN scale where it is not finite.
FB2_DEV void code_scale(uint32_t top_bits, float& inv, float& scale) {
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) {
        inv = 0.f;
        scale = __uint_as_float(0x7fc00000u);
    } else if (top < kKvqTiny) {
        inv = scale = 0.f;
    } else {
        inv = 127.f / top;
        scale = top / 127.f;
    }
}
FB2_DEV uint32_t code(float x, float inv) {
    // no code is past 127: x * inv is at most 127 and two roundings
    return inv == 0.f ? 0u : (uint32_t)__float2int_rn(x * inv) & 0xffu;
}
template <bool VEC>
FB2_DEV void store_codes(signed char* row, int at, int n, const float (&v)[NORM_E], float inv) {
    if (VEC || at + NORM_E <= n) {  // rows of codes begin on 16 bytes
        if (at >= n) return;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < NORM_E; i++) w[i / 4] |= code(v[i], inv) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(row + at) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < NORM_E; i++)
            if (at + i < n) row[at + i] = (signed char)code(v[i], inv);
    }
}

}  // namespace nrm

// T: h, gate and y; X: x and the sum.  G threads share a row and hold 8 * NJ of
// its values each; blockDim: G, or rows / warp of 4 for G = 32.
template <class T, class X, int G, int NJ, bool VEC>
__global__ void __launch_bounds__(G == 32 ? 128 : G) k_residual_norm(NormArgs a) {
    __shared__ float s[32];
    const int tid = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int row = G == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    const int n = a.dim;
    const float count = (float)n;
    float v[NJ][NORM_E];
    // (v - mean) / sqrt(var + eps), or v / sqrt(mean square + eps)
    auto normed = [&](const float* w, const float* b) {
        float mean = 0.f, part = 0.f;
        if (!a.rms) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < NORM_E; i++) part += v[j][i];
            mean = nrm::sum<G>(part, s) / count;
        }
        part = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int i = 0; i < NORM_E; i++) {
                const float d = v[j][i] - mean;
                if ((tid + j * G) * NORM_E + i < n) part += d * d;
            }
        const float r = 1.f / sqrtf(nrm::sum<G>(part, s) / count + a.eps);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int at = (tid + j * G) * NORM_E;
            float wv[NORM_E], bv[NORM_E];
            nrm::load<float, VEC>(w, at, n, wv);
            if (b) nrm::load<float, VEC>(b, at, n, bv);
#pragma unroll
            for (int i = 0; i < NORM_E; i++) {
                v[j][i] = (v[j][i] - mean) * r * wv[i];
                if (b) v[j][i] += bv[i];
                if constexpr (!VEC) v[j][i] = at + i < n ? v[j][i] : 0.f;
            }
        }
    };
    const X* x = static_cast<const X*>(a.x) + row * a.x_row;
    if (a.h) {
        const T* h = static_cast<const T*>(a.h) + row * a.h_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) nrm::load<T, VEC>(h, (tid + j * G) * NORM_E, n, v[j]);
        if (a.post) normed(a.post_w, a.post_b);
        const T* gate = static_cast<const T*>(a.gate) + (a.gate ? row * a.gate_row : 0);
        X* sum = static_cast<X*>(a.sum) + row * a.sum_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int at = (tid + j * G) * NORM_E;
            float xv[NORM_E], gv[NORM_E];
            nrm::load<X, VEC>(x, at, n, xv);
            if (a.gate) nrm::load<T, VEC>(gate, at, n, gv);
#pragma unroll
            for (int i = 0; i < NORM_E; i++) {
                if (a.gate) v[j][i] *= gv[i];
                v[j][i] = xv[i] + a.scale * v[j][i];
            }
            nrm::store<X, VEC>(sum, at, n, v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NJ; j++) nrm::load<X, VEC>(x, (tid + j * G) * NORM_E, n, v[j]);
    }
    normed(a.w, a.b);
    if (!a.codes) {
        T* y = static_cast<T*>(a.y) + row * a.y_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) nrm::store<T, VEC>(y, (tid + j * G) * NORM_E, n, v[j]);
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int i = 0; i < NORM_E; i++) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
    float inv, scale;
    nrm::code_scale(nrm::largest<G>(top, s), inv, scale);
#pragma unroll
    for (int j = 0; j < NJ; j++) nrm::store_codes<VEC>(a.codes + row * a.code_row, (tid + j * G) * NORM_E, n, v[j], inv);
    if (tid == 0) a.scales[row] = scale;
}

// Rows x [rows][n] as codes: a CTA of 256 threads takes a row, of any length.
constexpr int QR_THREADS = 256;
template <class T, bool VEC>
__global__ void __launch_bounds__(QR_THREADS) k_quantise_rows(const T* x, long long x_row, int n, signed char* codes, long long code_row,
                                                              float* scales) {
    __shared__ float s[32];
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;
    x += row * x_row;
    codes += row * code_row;
    uint32_t top = 0;
    float v[NORM_E];
    for (int at = tid * NORM_E; at < n; at += QR_THREADS * NORM_E) {
        nrm::load<T, VEC>(x, at, n, v);
#pragma unroll
        for (int i = 0; i < NORM_E; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    float inv, scale;
    nrm::code_scale(nrm::largest<QR_THREADS>(top, s), inv, scale);
    for (int at = tid * NORM_E; at < n; at += QR_THREADS * NORM_E) {
        nrm::load<T, VEC>(x, at, n, v);
        nrm::store_codes<VEC>(codes, at, n, v, inv);
    }
    if (tid == 0) scales[row] = scale;
}

}  // namespace fb2
