// logit_controls.cuh — penalties for repeated tokens, biases and grammar masks
// on logit rows (include/forge_b200.h, fb2_logit_controls, has the formula).
#pragma once
#include "kvq.cuh"

namespace fb2 {

struct ControlArgs {
    const void* logits;
    void* out;
    const int* tokens;
    const int* token_starts;
    const float *repetition, *presence, *frequency;
    const int* bias_ids;
    const float* bias_values;
    const int* bias_starts;
    const uint32_t* allowed;
    const int* mask_rows;
    long long in_row, out_row, n_tokens, n_biases;
    int n_rows, vocab, n_masks, mask_words;
};

constexpr int CTL_CHUNK = 4096;  // vocabulary entries of a CTA
constexpr int CTL_THREADS = 256;

// A CTA takes one chunk of one row: it counts the row's tokens that fall in
// the chunk, finds each id's last bias, and passes over the chunk once.
template <class T>
__global__ void __launch_bounds__(CTL_THREADS) k_logit_controls(ControlArgs a) {
    __shared__ int count[CTL_CHUNK];
    __shared__ int bias[CTL_CHUNK];  // 1 + index in the row's list; 0: none
    const int row = blockIdx.y, v0 = blockIdx.x * CTL_CHUNK, n = min(CTL_CHUNK, a.vocab - v0);
    for (int i = threadIdx.x; i < CTL_CHUNK; i += CTL_THREADS) count[i] = bias[i] = 0;
    __syncthreads();
    if (a.tokens) {
        const long long lo = max(__ldg(a.token_starts + row), 0);
        const long long hi = min((long long)__ldg(a.token_starts + row + 1), a.n_tokens);
        for (long long i = lo + threadIdx.x; i < hi; i += CTL_THREADS) {
            const unsigned at = (unsigned)(__ldg(a.tokens + i) - v0);
            if (at < (unsigned)n) atomicAdd(count + at, 1);
        }
    }
    long long b0 = 0;
    if (a.bias_ids) {
        b0 = max(__ldg(a.bias_starts + row), 0);
        const long long hi = min((long long)__ldg(a.bias_starts + row + 1), a.n_biases);
        for (long long i = b0 + threadIdx.x; i < hi; i += CTL_THREADS) {
            const unsigned at = (unsigned)(__ldg(a.bias_ids + i) - v0);
            if (at < (unsigned)n) atomicMax(bias + at, (int)(i - b0) + 1);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? __ldg(a.repetition + row) : 1.f;
    const float pres = a.presence ? __ldg(a.presence + row) : 0.f;
    const float freq = a.frequency ? __ldg(a.frequency + row) : 0.f;
    const int mask = a.allowed ? (a.mask_rows ? __ldg(a.mask_rows + row) : row) : -1;
    const uint32_t* words = (unsigned)mask < (unsigned)a.n_masks ? a.allowed + (size_t)mask * a.mask_words : nullptr;
    const T* in = (const T*)a.logits + row * a.in_row;
    T* out = (T*)a.out + row * a.out_row;
    for (int i = threadIdx.x; i < n; i += CTL_THREADS) {
        const int v = v0 + i;
        float x = Dense<T>::get(in[v]);
        if (count[i]) {
            if (a.repetition) x = x < 0.f ? x * rep : x / rep;
            x = x - pres - freq * (float)count[i];
        }
        if (bias[i]) x += __ldg(a.bias_values + b0 + bias[i] - 1);
        if (words && !((__ldg(words + (v >> 5)) >> (v & 31)) & 1)) x = -INFINITY;
        out[v] = Dense<T>::put(x);
    }
}

}  // namespace fb2
