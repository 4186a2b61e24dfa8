// logit_controls.cuh — penalties for repeated tokens, biases and grammar masks
// on logit rows (include/forge_b200.h, fb2_logit_controls, has the formula).
#pragma once
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

// A CTA takes a row, or, of few rows, a slice of one.  It gathers what the
// row's window and bias list name in a hash table in shared memory (how often
// the window has the id, which bias is its last), copies the slice, or -inf
// where the mask does not allow an entry, sixteen bytes at a time, and then
// writes the entries that the lists name.  Few beside the vocabulary, these
// still cost more than the copies, as each is a load and a store of its own:
// 256 rows x 131071 in bf16 with windows of 4096 take 47 us, the copies alone
// 20 (6.7 TB/s); one row x 16384 in fp32 with a window of 576 takes 5.0, as
// long as its chain of dependent loads.
constexpr int CTL_THREADS = 512, CTL_VECS = 4;
// List entries a thread, and the table's slots at most: at most three quarters
// of them are taken.
constexpr int CTL_IDS = 12, CTL_SLOTS = CTL_THREADS * CTL_IDS / 3 * 4;

// blockIdx: slice of `slice` entries (a multiple of 32), row; `max_slots` (a
// power of two, at least 1024): what the shared memory has room for, two words
// each.
template <class T>
__global__ void __launch_bounds__(CTL_THREADS, 2) k_logit_controls(ControlArgs a, int slice, int max_slots, bool copies) {
    extern __shared__ uint32_t ctl_smem[];
    const int tid = threadIdx.x, row = blockIdx.y, v0 = blockIdx.x * slice, len = min(slice, a.vocab - v0);
    long long t0 = 0, b0 = 0, nt = 0, nb = 0;
    if (a.tokens) {
        t0 = max(__ldg(a.token_starts + row), 0);
        nt = max(0ll, min((long long)__ldg(a.token_starts + row + 1), a.n_tokens) - t0);
    }
    if (a.bias_ids) {
        b0 = max(__ldg(a.bias_starts + row), 0);
        nb = max(0ll, min((long long)__ldg(a.bias_starts + row + 1), a.n_biases) - b0);
    }
    const float rep = a.repetition ? __ldg(a.repetition + row) : 1.f;
    const float pres = a.presence ? __ldg(a.presence + row) : 0.f, freq = a.frequency ? __ldg(a.frequency + row) : 0.f;
    const uint32_t* words = nullptr;  // the row's mask; null: everything is allowed
    if (a.allowed) {
        const int mask = a.mask_rows ? __ldg(a.mask_rows + row) : row;
        if ((unsigned)mask < (unsigned)a.n_masks) words = a.allowed + (size_t)mask * a.mask_words + (v0 >> 5);
    }
    const T* in = (const T*)a.logits + row * a.in_row + v0;
    T* out = (T*)a.out + row * a.out_row + v0;
    auto allows = [&](int i) { return !words || ((__ldg(words + (i >> 5)) >> (i & 31)) & 1); };
    auto clear = [&](int n) {
        for (int i = tid; i < n / 4; i += CTL_THREADS) reinterpret_cast<uint4*>(ctl_smem)[i] = make_uint4(0, 0, 0, 0);
    };
    // the logit x of an id that the window has `count` times; `bias`: 1 + the
    // index of its last bias
    auto changed = [&](float x, uint32_t count, uint32_t bias) {
        if (count) {
            if (a.repetition) x = x < 0.f ? x * rep : x / rep;
            x = x - pres - freq * (float)count;
        }
        return bias ? x + __ldg(a.bias_values + b0 + bias - 1) : x;
    };
    auto copy = [&]() {
        constexpr int PER = 16 / sizeof(T);
        auto one = [&](int i) { out[i] = allows(i) ? in[i] : Dense<T>::put(-INFINITY); };
        const uint32_t in_at = (uint32_t)reinterpret_cast<uintptr_t>(in) & 15, out_at = (uint32_t)reinterpret_cast<uintptr_t>(out) & 15;
        if (in_at != out_at) {  // of different alignment: one entry at a time
            for (int i = tid; i < len; i += CTL_THREADS) one(i);
            return;
        }
        const int head = min(len, (int)((16 - in_at) & 15) / (int)sizeof(T)), vecs = (len - head) / PER;
        const int n_words = a.mask_words - (v0 >> 5);
        const uint4* from = reinterpret_cast<const uint4*>(in + head);
        uint4* to = reinterpret_cast<uint4*>(out + head);
        if (tid < head) one(tid);
        if (head + vecs * PER + tid < len) one(head + vecs * PER + tid);
        for (int i0 = tid; i0 < vecs; i0 += CTL_THREADS * CTL_VECS) {
            uint4 x[CTL_VECS];
            uint32_t ok[CTL_VECS];  // PER bits each
#pragma unroll
            for (int u = 0; u < CTL_VECS; u++)
                if (i0 + u * CTL_THREADS < vecs) x[u] = from[i0 + u * CTL_THREADS];
            if (words) {
#pragma unroll
                for (int u = 0; u < CTL_VECS; u++) {
                    const int e = min(head + (i0 + u * CTL_THREADS) * PER, len - 1), at = e >> 5;
                    ok[u] = __funnelshift_r(__ldg(words + at), at + 1 < n_words ? __ldg(words + at + 1) : 0u, e & 31);
                }
            }
#pragma unroll
            for (int u = 0; u < CTL_VECS; u++) {
                const int i = i0 + u * CTL_THREADS;
                if (i >= vecs) break;
                uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                if (words) {
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        constexpr uint32_t NEG = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
                        if constexpr (sizeof(T) == 4) {
                            if (!((ok[u] >> e) & 1)) w[e] = 0xff800000u;
                        } else {
                            if (!((ok[u] >> e) & 1)) w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | NEG << 16 : (w[e / 2] & 0xffff0000u) | NEG;
                        }
                    }
                }
                to[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    };

    if (nt + nb <= min(max_slots / 4 * 3, CTL_THREADS * CTL_IDS)) {
        // key: 1 + entry of the slice, 0 if free; value: bias << 16 | count.
        // The thread that takes a slot writes its entry.
        const int n = (int)(nt + nb), nbias = (int)nb;
        int slots = 1024;  // half of them free, where there is room
        while (slots < max_slots && slots / 2 < n) slots *= 2;
        const int shift = 32 - __popc(slots - 1);
        uint32_t *keys = ctl_smem, *values = ctl_smem + slots;
        int at[CTL_IDS];
        uint32_t mine = 0;
        if (n) {
#pragma unroll
            for (int u = 0; u < CTL_IDS; u++) {
                const int j = u * CTL_THREADS + tid;
                at[u] = -1;
                if (u * CTL_THREADS < n && j < n) at[u] = __ldg(j < nbias ? a.bias_ids + b0 + j : a.tokens + t0 + (j - nbias));
            }
            clear(2 * slots);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < CTL_IDS; u++) {
                if (u * CTL_THREADS >= n) break;
                const int e = (uint32_t)at[u] < (uint32_t)a.vocab ? at[u] - v0 : -1;
                at[u] = -1;
                if ((uint32_t)e >= (uint32_t)len) continue;
                uint32_t s = ((uint32_t)e * 0x9e3779b1u) >> shift;
                for (;;) {
                    const uint32_t was = atomicCAS(keys + s, 0u, (uint32_t)e + 1u);
                    if (was == 0u) mine |= 1u << u;
                    if (was == 0u || was == (uint32_t)e + 1u) break;
                    s = (s + 1) & (slots - 1);
                }
                at[u] = (int)s;
                if (u * CTL_THREADS + tid < nbias) atomicMax(values + s, (uint32_t)(u * CTL_THREADS + tid + 1) << 16);
            }
            if (nbias) __syncthreads();  // counts are added to finished indexes of biases
#pragma unroll
            for (int u = 0; u < CTL_IDS; u++)
                if (u * CTL_THREADS < n && at[u] >= 0 && u * CTL_THREADS + tid >= nbias) atomicAdd(values + at[u], 1u);
            __syncthreads();
            // the new values into the table: the registers are for the copies.  (The
            // loads of x before the counts, to hide their wait: 47 -> 83 us for 256
            // rows x 131071 in bf16 with windows of 4096.)
            T x[CTL_IDS];
#pragma unroll
            for (int u = 0; u < CTL_IDS; u++)
                if ((mine >> u) & 1) {
                    const int e = (int)keys[at[u]] - 1;
                    if (allows(e))
                        x[u] = in[e];
                    else
                        mine &= ~(1u << u);
                }
#pragma unroll
            for (int u = 0; u < CTL_IDS; u++)
                if ((mine >> u) & 1) {
                    const uint32_t value = values[at[u]];
                    values[at[u]] = __float_as_uint(changed(Dense<T>::get(x[u]), value & 0xffffu, value >> 16));
                }
        }
        if (copies) copy();
        __syncthreads();
#pragma unroll
        for (int u = 0; u < CTL_IDS; u++)
            if ((mine >> u) & 1) out[keys[at[u]] - 1] = Dense<T>::put(__uint_as_float(values[at[u]]));
        return;
    }
    // longer lists: ranges of ids, two words for each
    if (copies) copy();
    uint32_t *counts = ctl_smem, *biases = ctl_smem + max_slots;
    for (int e0 = 0; e0 < len; e0 += max_slots) {
        const int range = min(max_slots, len - e0), base = v0 + e0;
        __syncthreads();
        clear(2 * max_slots);
        __syncthreads();
        for (long long i = tid; i < nb; i += CTL_THREADS) {
            const int e = __ldg(a.bias_ids + b0 + i) - base;
            if ((uint32_t)e < (uint32_t)range) atomicMax(biases + e, (uint32_t)i + 1u);
        }
#pragma unroll 4
        for (long long i = tid; i < nt; i += CTL_THREADS) {
            const int e = __ldg(a.tokens + t0 + i) - base;
            if ((uint32_t)e < (uint32_t)range) atomicAdd(counts + e, 1u);
        }
        __syncthreads();
        for (int i = tid; i < range; i += CTL_THREADS)
            if ((counts[i] | biases[i]) && allows(e0 + i)) out[e0 + i] = Dense<T>::put(changed(Dense<T>::get(in[e0 + i]), counts[i], biases[i]));
    }
}

}  // namespace fb2
