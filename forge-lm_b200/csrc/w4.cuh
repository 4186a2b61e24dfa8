// w4.cuh — linear layers with 4-bit weights and a scale and minimum for each
// output and group of inputs: packing, and products with few rows.
//
// y[m][n] = sum_g (scale[g][n] * sum_{k in g} code[k][n] x[m][k]
//                  + min[g][n] * sum_{k in g} x[m][k]) + bias[n]
// Blocks of 16 outputs x 64 inputs, 32 lanes x 4 words: nibble p of word j of
// lane 4g + t is output 8 (p & 1) + g, input 16 t + 4 j + (p & 2) + (p >> 2).
#pragma once
#include "kvq.cuh"

namespace fb2 {

struct W4View {
    const uint4* codes;   // [n16][k64][32] uint4
    const uint32_t* meta; // [n16][groups][16]
    const float* bias;
    int K, N, group_shift;
    int k64, groups;
};

// One thread: outputs g and g + 8 of a block of 16, one group of inputs.
template <class T>
__global__ void __launch_bounds__(128)
    k_w4_pack(uint32_t* codes, uint32_t* meta, const T* __restrict__ w, long long w_row, int K, int N, int group_shift,
              int k64, int groups) {
    const int g = threadIdx.x & 7;
    const long long unit = ((long long)blockIdx.x * 128 + threadIdx.x) >> 3;
    const int block = (int)(unit / groups), grp = (int)(unit - (long long)block * groups);
    if (block >= (N + 15) / 16) return;
    const float inf = __uint_as_float(0x7f800000u);
    const int k0 = grp << group_shift, k1 = min(K, k0 + (1 << group_shift));
    float least[2], inv[2];
    for (int half = 0; half < 2; half++) {
        const int n = block * 16 + half * 8 + g;
        float lo = inf, hi = -inf;
        if (n < N)
            for (int k = k0; k < k1; k++) {
                const float x = Dense<T>::get(w[k * w_row + n]);
                const bool nan = x != x;
                lo = fminf(lo, nan ? -inf : x);
                hi = fmaxf(hi, nan ? inf : x);
            }
        else
            lo = hi = 0.f;
        const uint32_t scale_b = float_to_bf16_bits((hi - lo) / 15.0f), least_b = float_to_bf16_bits(lo);
        const float scale = bf16_bits_to_float(scale_b);
        least[half] = bf16_bits_to_float(least_b);
        const bool finite = scale < inf && fabsf(least[half]) < inf;
        const bool some = finite && scale >= kKvqTiny;
        inv[half] = some ? 1.0f / scale : 0.0f;
        meta[((size_t)block * groups + grp) * 16 + half * 8 + g] =
            finite ? ((some ? scale_b : 0u) | (least_b << 16)) : 0x7fc07fc0u;
    }
    for (int k = k0; k < k0 + (1 << group_shift); k += 4) {
        uint32_t word = 0;
#pragma unroll
        for (int p = 0; p < 8; p++) {
            const int half = p & 1, kk = k + (p & 2) + (p >> 2), n = block * 16 + half * 8 + g;
            if (kk < K && n < N && inv[half] != 0.f) {
                const float x = Dense<T>::get(w[kk * w_row + n]);
                word |= (uint32_t)fminf(fmaxf(rintf((x - least[half]) * inv[half]), 0.f), 15.f) << (4 * p);
            }
        }
        const int kb = k >> 6, t = (k & 63) >> 4, j = (k & 15) >> 2;
        if (kb < k64) codes[(((size_t)block * k64 + kb) * 32 + 4 * g + t) * 4 + j] = word;
    }
}

// One warp per output and row.
template <class T>
__global__ void __launch_bounds__(128)
    k_w4_matvec(W4View w, const T* __restrict__ x, long long x_row, T* __restrict__ y, long long y_row) {
    const int lane = threadIdx.x & 31, n = blockIdx.x * 4 + (threadIdx.x >> 5), m = blockIdx.y;
    if (n >= w.N) return;
    const int block = n >> 4, half = (n >> 3) & 1, g = n & 7;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(w.codes);
    float acc = 0.f;
    for (int k = lane; k < w.K; k += 32) {
        const uint32_t word = __ldg(codes + (((size_t)block * w.k64 + (k >> 6)) * 32 + 4 * g + ((k & 63) >> 4)) * 4 + ((k & 15) >> 2));
        const int p = half | (k & 2) | ((k & 1) << 2);
        const uint32_t meta = __ldg(w.meta + ((size_t)block * w.groups + (k >> w.group_shift)) * 16 + (n & 15));
        const float v = fmaf((float)((word >> (4 * p)) & 15u), bf16_bits_to_float(meta & 0xffffu),
                             __uint_as_float(meta & 0xffff0000u));
        acc = fmaf(v, Dense<T>::get(x[m * x_row + k]), acc);
    }
    acc = warp_sum(acc);
    if (lane == 0) y[m * y_row + n] = Dense<T>::put(acc + (w.bias ? __ldg(w.bias + n) : 0.f));
}

}  // namespace fb2
