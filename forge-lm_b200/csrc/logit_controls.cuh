// logit_controls.cuh — penalties for repeated tokens, biases and grammar masks
// on logit rows (include/forge_b200.h, fb2_logit_controls, has the formula).
#pragma once
#include <cstring>
#include <type_traits>

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

constexpr int CTL_THREADS = 256;

// A CTA takes `chunk` vocabulary entries (a multiple of 32) of one row.  The
// ids that the row's window or bias list names are few: they get a bit each,
// and a word in a table that only they initialise (how often the window has
// the id, and which bias is its last).  Then one pass over the chunk: entries
// without a bit are copied or masked as they are, sixteen bytes at a time,
// the others computed in fp32.
// Table words: bias index + 1 in the high half, count in the low half; lists
// too long for 16 bits use two words, half as many entries at a time.
template <class T>
struct ControlRow {
    const ControlArgs& a;
    const uint32_t* allowed;  // null: everything
    float rep, pres, freq;
    const float* biases;      // of the row's list
    FB2_DEV float value(float x, uint32_t count, uint32_t bias) const {
        if (count) {
            if (a.repetition) x = x < 0.f ? x * rep : x / rep;
            x = x - pres - freq * (float)count;
        }
        if (bias) x += __ldg(biases + bias - 1);
        return x;
    }
};

// 32 bits of a bit string from bit `at` on; words past `last` are not read.
FB2_DEV uint32_t bits_from(const uint32_t* w, int at, int last) {
    const int i = at >> 5;
    return __funnelshift_r(w[i], i < last ? w[i + 1] : 0u, at & 31);
}

template <class T>
__global__ void __launch_bounds__(CTL_THREADS, 3) k_logit_controls(ControlArgs a, int chunk) {
    extern __shared__ uint32_t ctl_smem[];
    uint32_t* table = ctl_smem;          // [chunk]
    uint32_t* bits = ctl_smem + chunk;   // [chunk / 32]
    const int tid = threadIdx.x, row = blockIdx.y;
    const int c0 = blockIdx.x * chunk, c1 = min(c0 + chunk, a.vocab);

    long long t0 = 0, t1 = 0, b0 = 0, b1 = 0;
    if (a.tokens) {
        t0 = max(__ldg(a.token_starts + row), 0);
        t1 = min((long long)__ldg(a.token_starts + row + 1), a.n_tokens);
    }
    if (a.bias_ids) {
        b0 = max(__ldg(a.bias_starts + row), 0);
        b1 = min((long long)__ldg(a.bias_starts + row + 1), a.n_biases);
    }
    ControlRow<T> r{a, nullptr, 1.f, 0.f, 0.f, a.bias_values + b0};
    if (a.repetition) r.rep = __ldg(a.repetition + row);
    if (a.presence) r.pres = __ldg(a.presence + row);
    if (a.frequency) r.freq = __ldg(a.frequency + row);
    if (a.allowed) {
        const int mask = a.mask_rows ? __ldg(a.mask_rows + row) : row;
        if ((unsigned)mask < (unsigned)a.n_masks) r.allowed = a.allowed + (size_t)mask * a.mask_words;
    }
    const T* in = (const T*)a.logits + row * a.in_row;
    T* out = (T*)a.out + row * a.out_row;

    const bool shared_word = t1 - t0 <= 0xffff && b1 - b0 <= 0xfffe;
    const int cap = shared_word ? chunk : chunk / 2;  // chunk is a multiple of 64
    for (int v0 = c0; v0 < c1; v0 += cap) {
        const int n = min(cap, c1 - v0);
        uint32_t* bias_table = shared_word ? table : table + cap;
        for (int i = tid; i < cap / 32; i += CTL_THREADS) bits[i] = 0;
        __syncthreads();
        auto touch = [&](int id) {
            const uint32_t at = (uint32_t)id - (uint32_t)v0;
            if (at < (uint32_t)n) {
                atomicOr(bits + (at >> 5), 1u << (at & 31));
                table[at] = 0;
                if (!shared_word) bias_table[at] = 0;
            }
        };
#pragma unroll 4
        for (long long i = t0 + tid; i < t1; i += CTL_THREADS) touch(__ldg(a.tokens + i));
        for (long long i = b0 + tid; i < b1; i += CTL_THREADS) touch(__ldg(a.bias_ids + i));
        __syncthreads();
        for (long long i = b0 + tid; i < b1; i += CTL_THREADS) {
            const uint32_t at = (uint32_t)__ldg(a.bias_ids + i) - (uint32_t)v0;
            if (at < (uint32_t)n) atomicMax(bias_table + at, (uint32_t)(i - b0 + 1) << (shared_word ? 16 : 0));
        }
        __syncthreads();
#pragma unroll 4
        for (long long i = t0 + tid; i < t1; i += CTL_THREADS) {
            const uint32_t at = (uint32_t)__ldg(a.tokens + i) - (uint32_t)v0;
            if (at < (uint32_t)n) atomicAdd(table + at, 1u);
        }
        __syncthreads();

        auto touched = [&](float x, int at) {
            const uint32_t w = table[at];
            return shared_word ? r.value(x, w & 0xffffu, w >> 16) : r.value(x, w, bias_table[at]);
        };
        auto one = [&](int at) {
            const int v = v0 + at;
            if (r.allowed && !((__ldg(r.allowed + (v >> 5)) >> (v & 31)) & 1)) {
                out[v] = Dense<T>::put(-INFINITY);
            } else if ((bits[at >> 5] >> (at & 31)) & 1) {
                out[v] = Dense<T>::put(touched(Dense<T>::get(in[v]), at));
            } else {
                out[v] = in[v];
            }
        };
        constexpr int PER = 16 / sizeof(T);  // entries of 16 bytes
        const uint32_t in_at = (uint32_t)reinterpret_cast<uintptr_t>(in + v0) & 15, out_at = (uint32_t)reinterpret_cast<uintptr_t>(out + v0) & 15;
        if (in_at != out_at) {  // in and out of different alignment: one entry at a time
            for (int i = tid; i < n; i += CTL_THREADS) one(i);
        } else {
            const int head = min(n, (int)((16 - in_at) & 15) / (int)sizeof(T)), vecs = (n - head) / PER;
            if (tid < head) one(tid);
            if (head + vecs * PER + tid < n) one(head + vecs * PER + tid);
            const uint4* from = reinterpret_cast<const uint4*>(in + v0 + head);
            uint4* to = reinterpret_cast<uint4*>(out + v0 + head);
            constexpr int U = 4;  // loads in flight
            for (int i0 = tid; i0 < vecs; i0 += CTL_THREADS * U) {
                uint4 x[U];
                uint32_t ok[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int i = i0 + u * CTL_THREADS;
                    if (i < vecs) {
                        x[u] = __ldcs(from + i);
                        ok[u] = r.allowed ? bits_from(r.allowed, v0 + head + i * PER, a.mask_words - 1) : 0xffffffffu;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int i = i0 + u * CTL_THREADS, at = head + i * PER;
                    if (i >= vecs) break;
                    uint32_t hit = bits_from(bits, at, cap / 32 - 1) & ((1u << PER) - 1);
                    uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                    if (hit &= ok[u]) {
#pragma unroll
                        for (int e = 0; e < PER; e++)
                            if ((hit >> e) & 1) {
                                if constexpr (sizeof(T) == 4) {
                                    w[e] = __float_as_uint(touched(__uint_as_float(w[e]), at + e));
                                } else {
                                    const unsigned short h = (unsigned short)(w[e / 2] >> (16 * (e & 1)));
                                    T v;
                                    memcpy(&v, &h, 2);
                                    v = Dense<T>::put(touched(Dense<T>::get(v), at + e));
                                    unsigned short z;
                                    memcpy(&z, &v, 2);
                                    w[e / 2] = __byte_perm(w[e / 2], z, e & 1 ? 0x5410 : 0x3254);
                                }
                            }
                    }
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        constexpr uint32_t NEG = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
                        if constexpr (sizeof(T) == 4) {
                            if (!((ok[u] >> e) & 1)) w[e] = 0xff800000u;
                        } else {
                            if (!((ok[u] >> e) & 1)) w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | NEG << 16 : (w[e / 2] & 0xffff0000u) | NEG;
                        }
                    }
                    __stcs(to + i, make_uint4(w[0], w[1], w[2], w[3]));
                }
            }
        }
        __syncthreads();  // the table is written again
    }
}

}  // namespace fb2
