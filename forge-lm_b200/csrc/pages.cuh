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
// which costs less than handing sums over.
#pragma once
#include "common.cuh"

namespace fb2 {

constexpr int PG_THREADS = 1024, PG_SEQS = 16384;  // sequences: three words each in shared memory

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
// Sums of a and b over the threads before this one; totals in `all`.
FB2_DEV Pair before(Pair v, Pair& all) {
    __shared__ Pair s[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Pair in = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long a = __shfl_up_sync(0xffffffffu, in.a, o), b = __shfl_up_sync(0xffffffffu, in.b, o);
        if (lane >= o) in.a += a, in.b += b;
    }
    __syncthreads();  // s may still be read from the last time
    if (lane == 31) s[warp] = in;
    __syncthreads();
    Pair base{0, 0};
    all = {0, 0};
    for (int w = 0; w < PG_THREADS / 32; w++) {
        if (w == warp) base = all;
        all.a += s[w].a, all.b += s[w].b;
    }
    return {base.a + in.a - v.a, base.b + in.b - v.b};
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

// gridDim.x: the CTAs of the one cluster
__global__ void __launch_bounds__(PG_THREADS, 1)
    k_pages_extend(PagesView p, const int* counts, int max_rows, int* starts, int* prefix, int* slots, int* positions) {
    extern __shared__ int pg_smem[];
    int *s_start = pg_smem, *s_page = s_start + p.n_seqs, *s_len = s_page + p.n_seqs;
    const int tid = threadIdx.x, per = (p.n_seqs + PG_THREADS - 1) / PG_THREADS;
    const int b0 = min(tid * per, p.n_seqs), b1 = min(b0 + per, p.n_seqs);
    const int n_free = p.list();
    for (int b = tid; b < p.n_seqs; b += PG_THREADS) {
        s_start[b] = counts[b];
        s_len[b] = p.lens[b];
    }
    __syncthreads();
    // what a sequence asks for; nothing where it cannot have it whoever else asks
    auto asked = [&](int b, int& rows, int& pages) {
        const int len = s_len[b], count = s_start[b];
        const bool fits = len >= 0 && count >= 0 && (long long)len + count <= p.cap();
        rows = fits ? count : 0;
        pages = fits ? p.pages((long long)len + count) - p.pages(len) : 0;
    };
    pg::Pair sum{0, 0}, all;
    int rows, pages;
    for (int b = b0; b < b1; b++) {
        asked(b, rows, pages);
        sum.a += rows, sum.b += pages;
    }
    pg::Pair at = pg::before(sum, all);
    sum = {0, 0};
    for (int b = b0; b < b1; b++) {
        asked(b, rows, pages);
        at.a += rows, at.b += pages;
        const bool served = at.a <= max_rows && (pages == 0 || at.b <= n_free);
        s_start[b] = served ? rows : 0;  // counts from here on
        s_page[b] = served ? pages : 0;
        sum.a += s_start[b], sum.b += s_page[b];
    }
    at = pg::before(sum, all);
    for (int b = b0; b < b1; b++) {
        const int r = s_start[b], n = s_page[b];
        s_start[b] = (int)at.a, s_page[b] = (int)at.b;
        at.a += r, at.b += n;
    }
    const int total = (int)all.a;
    pg::cluster_sync();
    const int rank = blockIdx.x, ranks = gridDim.x;
    if (rank == 0) {
        for (int b = tid; b < p.n_seqs; b += PG_THREADS) {
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
    for (int r = rank * PG_THREADS + tid; r < max_rows; r += ranks * PG_THREADS) {
        int slot = -1, pos = 0;
        if (r < total) {
            const int b = pg::owner(s_start, p.n_seqs, r);
            pos = s_len[b] + r - s_start[b];
            const int place = pos >> p.shift, held = p.pages(s_len[b]), within = pos & ((1 << p.shift) - 1);
            int* entry = p.table + b * p.stride + place;
            int page;
            if (place < held) {
                page = *entry;
            } else {  // the row that opens a page enters it
                page = p.free[n_free - 1 - (s_page[b] + place - held)];
                if (within == 0) *entry = page;
            }
            if ((unsigned)page < (unsigned)p.n_pages) slot = (page << p.shift) + within;
        }
        slots[r] = slot;
        positions[r] = pos;
    }
}

__global__ void __launch_bounds__(PG_THREADS, 1) k_pages_truncate(PagesView p, const int* to) {
    extern __shared__ int pg_smem[];
    int *s_at = pg_smem, *s_keep = s_at + p.n_seqs;
    const int tid = threadIdx.x, per = (p.n_seqs + PG_THREADS - 1) / PG_THREADS;
    const int b0 = min(tid * per, p.n_seqs), b1 = min(b0 + per, p.n_seqs);
    const int n_free = p.list();
    const int rank = blockIdx.x, ranks = gridDim.x;
    for (int b = tid; b < p.n_seqs; b += PG_THREADS) {
        const int len = p.lens[b], want = max(to[b], 0);
        const bool fewer = want < len && len <= p.cap();
        s_keep[b] = fewer ? p.pages(want) : 0;
        s_at[b] = fewer ? p.pages(len) - p.pages(want) : 0;
    }
    __syncthreads();
    pg::Pair sum{0, 0}, all;
    for (int b = b0; b < b1; b++) sum.a += s_at[b];
    pg::Pair at = pg::before(sum, all);
    for (int b = b0; b < b1; b++) {
        const int n = s_at[b];
        s_at[b] = (int)at.a;
        at.a += n;
    }
    const int total = (int)min(all.a, (long long)INT32_MAX);
    pg::cluster_sync();
    if (rank == 0) {
        for (int b = tid; b < p.n_seqs; b += PG_THREADS) {
            const int len = p.lens[b], want = max(to[b], 0);
            if (want < len && len <= p.cap()) p.lens[b] = want;
        }
        if (tid == 0) *p.n_free = (int)min((long long)n_free + total, (long long)p.n_pages);
    }
    // the first page dropped ends up last on the list: the next to be taken
    for (int j = rank * PG_THREADS + tid; j < total; j += ranks * PG_THREADS) {
        const int b = pg::owner(s_at, p.n_seqs, j);
        int* entry = p.table + b * p.stride + s_keep[b] + (j - s_at[b]);
        const long long i = (long long)n_free + total - 1 - j;
        if (i < p.n_pages) p.free[i] = *entry;
        *entry = -1;
    }
}

}  // namespace fb2
