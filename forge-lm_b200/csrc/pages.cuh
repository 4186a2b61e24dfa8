// pages.cuh — pages for the tokens of sequences: the page table that attention
// reads and the slots that the cache's write takes, made on the device from how
// many tokens each sequence adds, and the way back (include/forge_b200.h,
// fb2_pages_extend and fb2_pages_truncate, has the rules).
//
// Two sums over the sequences (tokens and pages that those before ask for) say
// which of them are served and where their rows and pages begin; then every row
// finds its sequence by a binary search of the starts and its page in the table
// or, for a page that it opens, in the list of free ones.  Nothing here moves
// more than some words a row: a call is one launch and a chain of loads, sums and
// stores.  One cluster does it, so that all CTAs have read lengths and list
// before the first of them writes; each sums for itself in its own shared memory,
// which costs less than handing sums over.  32 sequences of up to 8 tokens take 3.3 us, and
// 2.7 to give them back; 512 with 131 thousand rows 9 and 6.
#pragma once
#include "common.cuh"

namespace fb2 {

constexpr int PG_SEQS = 16384;  // sequences: three words each in shared memory

struct PagesView {
    int* table;  // [n_seqs], rows `stride` apart
    int* lens;
    int* free;
    int* n_free;
    long long stride;
    int n_seqs, max_pages, n_pages, shift;
    FB2_DEV long long cap() const { return (long long)max_pages << shift; }
    FB2_DEV int pages(long long n) const { return (int)((n + (1 << shift) - 1) >> shift); }
    FB2_DEV int list() const { return min(max(*n_free, 0), n_pages); }  // entries of the list of free pages
};

namespace pg {

struct Pair {
    long long a, b;
};
FB2_DEV Pair up(Pair v) {  // sums over the lanes up to this one
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
        if (lane >= o) v.a += a, v.b += b;
    }
    return v;
}
// Sums of a and b over the threads before this one; totals in `all`.  `s`: a place
// for each call.
template <int THREADS>
FB2_DEV Pair before(Pair v, Pair& all, Pair (&s)[THREADS / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Pair in = up(v);
    if (lane == 31) s[warp] = in;
    __syncthreads();
    const Pair w = up(lane < THREADS / 32 ? s[lane] : Pair{0, 0});
    all = {__shfl_sync(0xffffffffu, w.a, 31), __shfl_sync(0xffffffffu, w.b, 31)};
    const Pair base{__shfl_sync(0xffffffffu, w.a, warp - 1), __shfl_sync(0xffffffffu, w.b, warp - 1)};
    return {(warp ? base.a : 0) + in.a - v.a, (warp ? base.b : 0) + in.b - v.b};
}
// The last b in 0..n-1 with starts[b] <= i; starts[0] <= i, ascending.
FB2_DEV int owner(const int* starts, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}
FB2_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace pg

// gridDim.x: the CTAs of the one cluster; RUN: neighbouring rows of a thread, 1 or 4 (one
// search, one store where there are many rows; where there are few, a thread's rows would
// be of different sequences); `vec`: slots and positions begin on 16 bytes
template <int THREADS, int RUN>
__global__ void __launch_bounds__(THREADS, 1)
    k_pages_extend(PagesView p, const int* counts, int max_rows, int* starts, int* prefix, int* slots, int* positions, bool vec) {
    extern __shared__ int pg_smem[];
    __shared__ pg::Pair s_sum[2][THREADS / 32];
    int *s_start = pg_smem, *s_page = s_start + p.n_seqs, *s_len = s_page + p.n_seqs;
    const int tid = threadIdx.x, per = (p.n_seqs + THREADS - 1) / THREADS;
    const int b0 = min(tid * per, p.n_seqs), b1 = min(b0 + per, p.n_seqs);
    const int n_free = p.list();
    // what a sequence asks for; nothing where it cannot have it whoever else asks
    pg::Pair sum{0, 0}, all;
    for (int b = b0; b < b1; b++) {
        const int len = p.lens[b], count = counts[b];
        const bool fits = len >= 0 && count >= 0 && (long long)len + count <= p.cap();
        s_len[b] = len;
        s_start[b] = fits ? count : 0;
        s_page[b] = fits ? p.pages((long long)len + count) - p.pages(len) : 0;
        sum.a += s_start[b], sum.b += s_page[b];
    }
    pg::Pair at = pg::before<THREADS>(sum, all, s_sum[0]);
    if (all.a > max_rows || all.b > n_free) {  // not all can be served
        sum = {0, 0};
        for (int b = b0; b < b1; b++) {
            at.a += s_start[b], at.b += s_page[b];
            if (at.a > max_rows || (s_page[b] && at.b > n_free)) s_start[b] = s_page[b] = 0;
            sum.a += s_start[b], sum.b += s_page[b];
        }
        at = pg::before<THREADS>(sum, all, s_sum[1]);
    }
    for (int b = b0; b < b1; b++) {  // from counts to where they begin
        const int r = s_start[b], n = s_page[b];
        s_start[b] = (int)at.a, s_page[b] = (int)at.b;
        at.a += r, at.b += n;
    }
    const int total = (int)all.a;
    __syncthreads();
    if (gridDim.x > 1) pg::cluster_sync();
    const int rank = blockIdx.x, ranks = gridDim.x;
    if (rank == 0) {
        for (int b = tid; b < p.n_seqs; b += THREADS) {
            starts[b] = s_start[b];
            prefix[b] = s_len[b];
            const int next = b + 1 < p.n_seqs ? s_start[b + 1] : total;
            if (next > s_start[b]) p.lens[b] = s_len[b] + next - s_start[b];
        }
        if (tid == 0) {
            starts[p.n_seqs] = total;
            *p.n_free = n_free - (int)all.b;
        }
    }
    const int mask = (1 << p.shift) - 1;
    for (int r0 = (rank * THREADS + tid) * RUN; r0 < max_rows; r0 += ranks * THREADS * RUN) {
        int slot[RUN], pos[RUN];
        int b = -1, end = r0, last = -1, page = -1;  // the sequence of the row before, where it ends; its last page
#pragma unroll
        for (int i = 0; i < RUN; i++) {
            const int r = r0 + i;
            slot[i] = -1, pos[i] = 0;
            if (r >= total) continue;
            if (r >= end) {
                b = pg::owner(s_start, p.n_seqs, r);
                end = b + 1 < p.n_seqs ? s_start[b + 1] : total;
                last = -1;
            }
            pos[i] = s_len[b] + r - s_start[b];
            const int place = pos[i] >> p.shift, within = pos[i] & mask;
            if (place != last) {
                const int held = p.pages(s_len[b]);
                int* entry = p.table + b * p.stride + place;
                last = place;
                if (place < held) {
                    page = *entry;
                } else {  // the row that opens a page enters it
                    page = p.free[n_free - 1 - (s_page[b] + place - held)];
                    if (within == 0) *entry = page;
                }
            }
            if ((unsigned)page < (unsigned)p.n_pages) slot[i] = (page << p.shift) + within;
        }
        if constexpr (RUN == 4) {
            if (vec && r0 + 4 <= max_rows) {
                *reinterpret_cast<int4*>(slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                *reinterpret_cast<int4*>(positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < RUN; i++)
            if (r0 + i < max_rows) slots[r0 + i] = slot[i], positions[r0 + i] = pos[i];
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1) k_pages_truncate(PagesView p, const int* to) {
    extern __shared__ int pg_smem[];
    __shared__ pg::Pair s_sum[THREADS / 32];
    int *s_at = pg_smem, *s_keep = s_at + p.n_seqs;
    const int tid = threadIdx.x, per = (p.n_seqs + THREADS - 1) / THREADS;
    const int b0 = min(tid * per, p.n_seqs), b1 = min(b0 + per, p.n_seqs);
    const int n_free = p.list();
    pg::Pair sum{0, 0}, all;
    for (int b = b0; b < b1; b++) {
        const int len = p.lens[b], want = max(to[b], 0);
        const bool fewer = want < len && len <= p.cap();
        s_keep[b] = fewer ? p.pages(want) : 0;
        s_at[b] = fewer ? p.pages(len) - s_keep[b] : 0;
        sum.a += s_at[b];
        if (fewer) p.lens[b] = want;
    }
    pg::Pair at = pg::before<THREADS>(sum, all, s_sum);
    for (int b = b0; b < b1; b++) {
        const int n = s_at[b];
        s_at[b] = (int)at.a;
        at.a += n;
    }
    __syncthreads();
    const int total = (int)min(all.a, (long long)INT32_MAX);
    if (tid == 0) *p.n_free = (int)min((long long)n_free + total, (long long)p.n_pages);
    // the first page dropped ends up last on the list: the next to be taken
    for (int j = tid; j < total; j += THREADS) {
        const int b = pg::owner(s_at, p.n_seqs, j);
        int* entry = p.table + b * p.stride + s_keep[b] + (j - s_at[b]);
        const long long i = (long long)n_free + total - 1 - j;
        if (i < p.n_pages) p.free[i] = *entry;
        *entry = -1;
    }
}

}  // namespace fb2
