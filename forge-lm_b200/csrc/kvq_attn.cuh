// kvq_attn.cuh — attention of new tokens (single ones or drafted trees) over
// the paged, quantised K/V cache.
//
// out = sum_p softmax_p(scale q.k_p) v_p over the positions a row sees, in one
// pass: the running maximum m, l = sum exp(s - m) and o = sum exp(s - m) v,
// rescaled when m grows; parts merge by the same rule.
#pragma once
#include "kvq.cuh"

namespace fb2 {

struct KvqAttnArgs {
    KvqView c;
    const void* q;
    void* out;
    float* lse;
    const int* table;
    const int* prefix;
    const int* starts;       // null: one row per sequence
    const uint32_t* mask;    // null: causal
    long long q_row, q_head, table_stride;
    int n_seqs, n_rows, n_heads, max_pages, max_nodes, max_len, mask_words;
    float scale;
    FB2_DEV void rows_of(int b, int& first, int& count) const {
        first = starts ? __ldg(starts + b) : b;
        const int last = starts ? __ldg(starts + b + 1) : b + 1;
        // a malformed list must not reach past the tensors
        first = max(first, 0);
        count = min(min(last, n_rows) - first, max_nodes);
    }
    FB2_DEV int slot(int b, int p) const {  // -1: not in the cache
        const int page = __ldg(table + b * table_stride + (p >> c.page_shift));
        if ((uint32_t)page >= (uint32_t)(c.n_slots >> c.page_shift)) return -1;
        return (page << c.page_shift) | (p & ((1 << c.page_shift) - 1));
    }
};

// One warp per (row, head).
template <class T, int FMT>
__global__ void __launch_bounds__(128) k_kvq_attend(KvqAttnArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z, i = blockIdx.y, h = blockIdx.x * 4 + warp;
    int first, count;
    a.rows_of(b, first, count);
    if (i >= count || h >= a.n_heads) return;
    const int row = first + i, g = h / (a.n_heads / a.c.heads);
    const int prefix = max(__ldg(a.prefix + b), 0);
    const int len = (int)min((long long)prefix + count, (long long)a.max_len);
    float q[8], o[8], x[8];
    const bool mine = lane * 8 < a.c.hd;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        q[j] = 0.f;
        o[j] = 0.f;
    }
    if (mine) load8<T, false>((const T*)a.q + row * a.q_row + h * a.q_head + lane * 8, q);
    float m = -INFINITY, l = 0.f;
    auto values = [&](size_t at) {
        const uint32_t w = a.c.meta[at];
        if constexpr (FMT == KVQ_INT8)
            kvq_decode8(*reinterpret_cast<const uint2*>(a.c.codes + at * a.c.row_bytes + lane * 8), __uint_as_float(w), x);
        else
            kvq_decode8(*reinterpret_cast<const uint32_t*>(a.c.codes + at * a.c.row_bytes + lane * 4),
                        bf16_bits_to_float(w & 0xffffu), __uint_as_float(w & 0xffff0000u), x);
    };
    for (int p = 0; p < len; p++) {
        const int j = p - prefix;
        if (j >= 0) {
            const bool see = a.mask ? (__ldg(a.mask + (size_t)row * a.mask_words + (j >> 5)) >> (j & 31)) & 1 : j <= i;
            if (!see) continue;
        }
        const int slot = a.slot(b, p);
        if (slot < 0) continue;
        float s = 0.f;
        if (mine) {
            values(a.c.row(slot, g, 0));
#pragma unroll
            for (int d = 0; d < 8; d++) s = fmaf(q[d], x[d], s);
        }
        s = warp_sum(s) * a.scale;
        const float n = fmaxf(m, s), f = __expf(m - n), e = expf(s - n);
        m = n;
        l = l * f + e;
        if (mine) {
            values(a.c.row(slot, g, 1));
#pragma unroll
            for (int d = 0; d < 8; d++) o[d] = fmaf(o[d], f, e * x[d]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (mine) {
#pragma unroll
        for (int d = 0; d < 8; d++) o[d] *= inv;
        store8((T*)a.out + ((size_t)row * a.n_heads + h) * a.c.hd + lane * 8, o);
    }
    if (a.lse && lane == 0) a.lse[(size_t)row * a.n_heads + h] = m + logf(l);
}

}  // namespace fb2
