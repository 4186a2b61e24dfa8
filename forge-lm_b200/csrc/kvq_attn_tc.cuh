// kvq_attn_tc.cuh — attention over the quantised cache for many rows of a K/V
// head at once (drafted trees, shared heads), 16-bit types, head_dim <= 128:
// both products on the 5th-generation tensor cores.
//
// The same sums as kvq_attn.cuh, with 128 rows instead of 16 to each pass over
// the codes: the way from bytes to fp16 and the reading of K and V are paid
// once for 128 rows, and the tiles of tcgen05.mma take the products off the
// warps.  What is left for them (codes to fp16, scores, maxima, 16384 exponentials
// a tile, 0.5 us at 16 a clock) comes in the steps below, one after another: some
// 3.2 us a tile of 128 positions, in which neither the tensor pipe nor the issue
// slots are busy.  4 trees of 23 to 64 tokens over 9 to 33 K int8 positions, 32 heads on 8 of
// 128, bf16: 254 us, 198 TFLOP/s (450 on mma.sync tiles).
//
// 512 threads of a CTA take one chunk of a sequence's positions, one K/V head
// and 128 rows; row r is TMEM lane r; warps w, w + 4, w + 8, w + 12 read lane
// quarter w % 4, each the scores of 32 of a tile's 128 positions.  The bytes of
// K and V come to shared memory two tiles ahead (cp.async; every thread turns
// what it copied itself into fp16, so that this needs no barrier), and become
// operands of 128-byte rows, [64 dims][position], 128-byte swizzled: K-major
// for S = Q K^T and, with the positions as the contraction, MN-major for O = P V.
// q is scaled by a power of two to just below 2^13 (exact: the 16-bit types'
// values fit fp16 then); P carries the V scales and the row's power of two, with the
// references that lag of kvq_attn.cuh, so that O stays in TMEM and is rescaled
// only when one of them moves.  Iteration t:
//   1. wait for S(t); K(t+1) becomes an operand, S(t+1) goes to the other tile;
//   2. scores, their largest; wait for O(t-1); where a row's references have to
//      move, the largest weight, and rescale;
//   3. weights into P(t), V(t) becomes an operand, O(t).
// One more warp issues the MMAs (which takes as long as the tensor cores need)
// and looks up the pages of later tiles.
// Every mbarrier wait is bounded (2 s); on expiry the CTA stops, drains its MMAs
// (bounded as well), frees its TMEM and writes NaN for its rows.
#pragma once
#include "kvq_attn.cuh"
#include "tc.cuh"

namespace fb2 {

constexpr int KVT_THREADS = 512, KVT_ROWS = 128, KVT_KEYS = 128;
constexpr int KVT_LAUNCH = KVT_THREADS + 32;  // and a warp that issues the MMAs and looks up pages
constexpr int KVT_PARTS = KVT_THREADS / KVT_ROWS;  // threads of a row, each for a part of a tile's columns
constexpr int KVT_COLS = KVT_KEYS / KVT_PARTS;

template <int HD, int FMT>
struct KvtShape {
    static constexpr int BLOCKS = HD / 64;              // of 64 dims
    static constexpr int OPERAND = BLOCKS * 128 * 128;  // Q, K or V: [dims / 64][128 rows][128 bytes]
    static constexpr int P = 2 * 128 * 128;
    static constexpr int UNIT = FMT == KVQ_INT8 ? 16 : 8;               // bytes of 16 dims
    static constexpr int UNITS = KVT_KEYS * HD / 16 / KVT_THREADS;      // of a thread and tile
    static constexpr int RAW = UNITS * KVT_THREADS * UNIT;              // a tile's bytes
    static constexpr int SMEM = 3 * OPERAND + P + 4 * RAW + 1024;       // two tiles of K, of V
    static constexpr uint32_t O_COL = 256, TMEM_COLS = 512;  // S: columns 0..127 and 128..255, O from 256 on
};

namespace kvt {

// Byte offset of 16-byte chunk `chunk` (8 fp16) of row `row` in an operand.
FB2_DEV uint32_t place(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * (128 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}
// K-major descriptor of an operand, and what k-step kk (16 values) adds to it
// (the address field counts 16 bytes).
FB2_DEV uint64_t desc_k(uint32_t base) { return tc::sw128_desc(base, 16, 1024); }
constexpr uint64_t step_k(int kk) { return (uint64_t)(((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4); }
// MN-major: 64 values to a row, blocks of 64 16 KB apart, 8 rows 1 KB apart;
// k-step kk is 16 rows.
FB2_DEV uint64_t desc_mn(uint32_t base) { return tc::sw128_desc(base, 128 * 128, 1024); }
constexpr uint64_t step_mn(int kk) { return (uint64_t)((kk * 2048) >> 4); }
// A, B fp16, D fp32, M = 128.
constexpr uint32_t idesc(int N, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
}
FB2_DEV void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
// 32 or 16 columns of the warp's lanes; wait_ld() before v is used
FB2_DEV void ld(uint32_t at, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
FB2_DEV void ld(uint32_t at, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
FB2_DEV void st(uint32_t at, const float (&v)[32]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
        : "memory");
}
FB2_DEV void st(uint32_t at, const float (&v)[16]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
        : "memory");
}
FB2_DEV void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
FB2_DEV void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
FB2_DEV void st4(uint32_t at, uint4 v) {
    // no memory clobber: only the tensor cores read what it writes, after publish()
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}
// 8 codes of a row as fp16; int4: dims in the order 0, 4, 1, 5, 2, 6, 3, 7
template <int FMT>
FB2_DEV uint4 fp16_codes(const uint32_t* w) {
    if constexpr (FMT == KVQ_INT8)
        return make_uint4(kva::codes8<false>(w[0]), kva::codes8<true>(w[0]), kva::codes8<false>(w[1]), kva::codes8<true>(w[1]));
    return make_uint4(kva::codes4<0>(w[0]), kva::codes4<1>(w[0]), kva::codes4<2>(w[0]), kva::codes4<3>(w[0]));
}
// the dim at place p of 8
template <int FMT>
constexpr int dim_at(int p) {
    return FMT == KVQ_INT8 ? p : (p >> 1) + 4 * (p & 1);
}

}  // namespace kvt

template <int HD, int FMT>
__global__ void __launch_bounds__(KVT_LAUNCH, 1) k_kvq_attend_tc(KvqAttnArgs a) {
    using S = KvtShape<HD, FMT>;
    extern __shared__ unsigned char kvt_raw[];
    __shared__ __align__(8) uint64_t bar_s, bar_o, drain;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int s_abort;
    __shared__ uint32_t s_ids[4][KVT_KEYS / 8], s_live[4];  // groups of 8 positions of a tile; which have a page
    __shared__ __align__(16) float s_k[2][2][KVT_KEYS], s_v[2][2][KVT_KEYS];  // [tile parity][scale, centre]
    __shared__ uint32_t s_vtop[2][4];
    __shared__ float s_red[KVT_PARTS][KVT_ROWS], s_sum[2][KVT_PARTS][KVT_ROWS];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(kvt_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t Q = tc::smem_addr(sm), K = Q + S::OPERAND, V = K + S::OPERAND, P = V + S::OPERAND, RAW = P + S::P;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quarter = warp & 3, part = warp >> 2;
    const bool worker = warp < KVT_THREADS / 32;

    const int b = blockIdx.y;
    if (b >= a.n_seqs) return a.fill_rest();
    const int rb = blockIdx.x % a.row_blocks, rest = blockIdx.x / a.row_blocks;
    const int split = rest % a.splits, head = rest / a.splits;
    if (a.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge's launch
    int first, count;
    a.rows_of(b, first, count);
    const int row0 = rb * KVT_ROWS, n_rows = min(KVT_ROWS, count * a.share - row0);
    if (n_rows <= 0) return;
    const int prefix = max(__ldg(a.prefix + b), 0);
    const int len = (int)min((long long)prefix + count, (long long)a.max_len);
    const int c0 = split * a.chunk, c1 = len - c0 > a.chunk ? c0 + a.chunk : len;
    const int r = 32 * quarter + lane, node = (row0 + r) / a.share, h = head * a.share + (row0 + r) - node * a.share;
    const bool mine = worker && r < n_rows;
    const size_t item = (size_t)(first + node) * a.n_heads + h;
    const int hd = a.c.hd;
    if (c0 >= c1) {
        if (a.splits > 1) {  // the merge has to know
            if (mine && part == 0) a.part_ml[item * a.splits + split] = make_float2(-INFINITY, 0.f);
        } else if (mine) {
            for (int d = part; d < hd; d += KVT_PARTS) a.store_out(item * hd + d, 0.f);
            if (a.lse && part == 0) a.lse[item] = -INFINITY;
        }
        return;
    }

    if (tid == 0) {
        s_abort = 0;
        tc::bar_init(&bar_s, 1);
        tc::bar_init(&bar_o, 1);
        tc::bar_init(&drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // ---- loads ---------------------------------------------------------------------
    const int ps = 1 << a.c.page_shift, rbytes = a.c.row_bytes;
    const uint32_t n_pages = a.c.n_slots >> a.c.page_shift;
    const int* table = a.table + b * a.table_stride;
    const int ntiles = (c1 - c0 + KVT_KEYS - 1) / KVT_KEYS;
    // the issuing warp: lane i looks up group i of a tile
    auto page_of = [&](int tile) {
        const int pos = c0 + tile * KVT_KEYS + lane * 8;
        return lane < KVT_KEYS / 8 && pos < c1 ? (uint32_t)__ldg(table + (pos >> a.c.page_shift)) : n_pages;
    };
    auto put_ids = [&](int tile, uint32_t page) {
        const int pos = c0 + tile * KVT_KEYS + lane * 8;
        const uint32_t live = __ballot_sync(0xffffffffu, page < n_pages);
        if (lane < KVT_KEYS / 8)
            s_ids[tile & 3][lane] = page < n_pages ? (((page * a.c.heads + head) * 2) << (a.c.page_shift - 3)) + ((pos & (ps - 1)) >> 3) : 0;
        if (lane == 0) s_live[tile & 3] = live;
    };
    // 16 dims at a time: thread i, i + 512, .. over [position][dims / 16]; dims
    // past head_dim are left as they are (q is 0 there, and O is not read),
    // positions without a page are zeros
    constexpr int PER = HD / 16;
    auto fetch = [&](int tile, int kind) {
        const uint32_t live = s_live[tile & 3];
#pragma unroll
        for (int j = 0; j < S::UNITS; j++) {
            const int i = tid + KVT_THREADS * j, key = i / PER, unit = i % PER;
            const bool there = (live >> (key >> 3)) & 1;
            const unsigned char* from = a.c.codes + (uint64_t)s_ids[tile & 3][key >> 3] * (uint32_t)(8 * rbytes) +
                                        (kind * ps + (key & 7)) * rbytes + unit * S::UNIT;
            const uint32_t to = RAW + ((tile & 1) * 2 + kind) * S::RAW + i * S::UNIT;
            if (unit * 16 < hd) {
                if constexpr (S::UNIT == 16)
                    copy16(to, from, there);
                else
                    copy8(to, from, there);
            }
        }
    };
    auto convert = [&](int tile, int kind, uint32_t to) {
#pragma unroll
        for (int j = 0; j < S::UNITS; j++) {
            const int i = tid + KVT_THREADS * j, key = i / PER, unit = i % PER;
            const uint32_t from = RAW + ((tile & 1) * 2 + kind) * S::RAW + i * S::UNIT;
            uint32_t w[4];
            if constexpr (S::UNIT == 16) {
                const uint4 v = lds4(from);
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                kvt::st4(to + kvt::place(key, 2 * unit), kvt::fp16_codes<FMT>(w));
                kvt::st4(to + kvt::place(key, 2 * unit + 1), kvt::fp16_codes<FMT>(w + 2));
            } else {
                const float2 v = lds2(from);
                w[0] = __float_as_uint(v.x), w[1] = __float_as_uint(v.y);
                kvt::st4(to + kvt::place(key, 2 * unit), kvt::fp16_codes<FMT>(w));
                kvt::st4(to + kvt::place(key, 2 * unit + 1), kvt::fp16_codes<FMT>(w + 1));
            }
        }
    };
    uint32_t meta = 0;
    // threads 0..127: a position's K meta word, 128..255: its V meta word; 0 past the end
    const int key = tid & 127, kind = tid >> 7;
    auto load_meta = [&](int tile) {
        meta = 0;
        if (kind < 2 && ((s_live[tile & 3] >> (key >> 3)) & 1) && c0 + tile * KVT_KEYS + key < c1)
            asm volatile("ld.global.nc.u32 %0, [%1];"
                         : "=r"(meta)
                         : "l"(a.c.meta + (uint64_t)s_ids[tile & 3][key >> 3] * 8 + kind * ps + (key & 7)));
    };
    auto store_meta = [&](int tile) {
        if (kind > 1) return;
        float* to = (kind ? s_v : s_k)[tile & 1][0];
        to[key] = FMT == KVQ_INT8 ? __uint_as_float(meta) : bf16_bits_to_float(meta & 0xffffu);
        if constexpr (FMT == KVQ_INT4) to[KVT_KEYS + key] = kva::centre(meta);
        if (kind) {  // the largest finite V scale's bits
            uint32_t bits = (FMT == KVQ_INT8 ? meta : meta << 16) & 0x7fffffffu;
            bits = __reduce_max_sync(0xffffffffu, bits < 0x7f800000u ? bits : 0u);
            if (lane == 0) s_vtop[tile & 1][warp & 3] = bits;
        }
    };
    // shared-memory operands written by the threads -> one thread issues
    auto publish = [&]() {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc::fence_before();
        __syncthreads();
    };

    if (!worker) {
        const uint32_t page0 = page_of(0), page1 = page_of(1), page2 = page_of(2);
        put_ids(0, page0);
        put_ids(1, page1);
        put_ids(2, page2);
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(&tmem_base)), "r"(S::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;

    // ---- the warp that issues: the workers' barriers in the same order ------------------
    if (!worker) {
        const uint64_t q_desc = kvt::desc_k(Q), k_desc = kvt::desc_k(K), p_desc = kvt::desc_k(P), v_desc = kvt::desc_mn(V);
        auto issue_s = [&](int t) {
            if (lane == 0) {
                tc::fence_after();
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++)
                    kvt::mma(tmem + 128u * (t & 1), q_desc + kvt::step_k(kk), k_desc + kvt::step_k(kk), kvt::idesc(KVT_KEYS, false), kk != 0);
                tc::mma_commit(&bar_s);
            }
            __syncwarp();
        };
        __syncthreads();  // q's largest values
        if constexpr (FMT == KVQ_INT4) {
            __syncthreads();
            __syncthreads();
        }
        __syncthreads();  // Q and K(0)
        issue_s(0);
        int t = 0;
        for (; t < ntiles; t++) {
            if (!__syncthreads_and(1)) break;
            if (t + 1 < ntiles) {
                issue_s(t + 1);
                put_ids(t + 3, page_of(t + 3));  // of tiles up to t + 2 the others may still read
            }
            if (__syncthreads_or(0)) {
                if (s_abort) break;
                __syncthreads();  // the rows' largest scores are read
                __syncthreads();  // their largest weights
            }
            __syncthreads();  // P(t), V(t)
            if (lane == 0) {
                tc::fence_after();
#pragma unroll
                for (int kk = 0; kk < KVT_KEYS / 16; kk++)
                    kvt::mma(tmem + S::O_COL, p_desc + kvt::step_k(kk), v_desc + kvt::step_mn(kk), kvt::idesc(HD, true), t > 0 || kk != 0);
                if (t != a.withhold || (blockIdx.x | blockIdx.y)) tc::mma_commit(&bar_o);
            }
            __syncwarp();
        }
        if (t == ntiles) __syncthreads_and(1);
        __syncthreads();  // the rows' sums
        if (s_abort && lane == 0) {
            // every MMA issued completes before tensor memory is freed
            tc::mma_commit(&drain);
            const unsigned long long t0 = tc::now_ns();
            while (!tc::bar_try(&drain, 0) && tc::now_ns() - t0 < kTcTimeoutNs) {
            }
        }
        __syncwarp();
        __syncthreads();  // the workers have read TMEM
        tc::fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
        return;
    }

    // ---- the workers ---------------------------------------------------------------------
    // two copy groups to a tile, K's and V's, in this order throughout
    fetch(0, 0);
    copies_commit();
    fetch(0, 1);
    copies_commit();
    fetch(1, 0);
    copies_commit();
    fetch(1, 1);
    copies_commit();
    load_meta(0);

    // q: a row's threads take turns at its chunks of 8 dims
    float f, qsum = 0.f;  // score factor of the row (positive: the scale's sign is in q), sum of its q
    {
        constexpr int N = HD / 8 / KVT_PARTS;
        float x[N][8], top = 0.f;
        const unsigned short* q = static_cast<const unsigned short*>(a.q) + (first + node) * a.q_row + h * a.q_head;
        const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
        uint4 raw[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int d = (KVT_PARTS * j + part) * 8;
            raw[j] = make_uint4(0, 0, 0, 0);
            if (mine && d < hd) {
                if (vec) {
                    raw[j] = __ldg(reinterpret_cast<const uint4*>(q + d));
                } else {
                    raw[j] = make_uint4(q[d] | q[d + 1] << 16, q[d + 2] | q[d + 3] << 16, q[d + 4] | q[d + 5] << 16, q[d + 6] | q[d + 7] << 16);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                constexpr int order[8] = {kvt::dim_at<FMT>(0), kvt::dim_at<FMT>(1), kvt::dim_at<FMT>(2), kvt::dim_at<FMT>(3),
                                          kvt::dim_at<FMT>(4), kvt::dim_at<FMT>(5), kvt::dim_at<FMT>(6), kvt::dim_at<FMT>(7)};
                const uint32_t pair[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
                const uint32_t bits = (pair[order[i] / 2] >> (16 * (order[i] & 1))) & 0xffffu;
                x[j][i] = a.dtype == 1 ? bf16_bits_to_float(bits) : __half2float(__ushort_as_half((unsigned short)bits));
                top = max_nan(top, fabsf(x[j][i]));
            }
        s_red[part][r] = top;
        __syncthreads();
        top = max_nan(max_nan(s_red[0][r], s_red[1][r]), max_nan(s_red[2][r], s_red[3][r]));
        const bool finite = top < INFINITY;
        const int e = finite ? max((int)(__float_as_uint(top) >> 23) - 126, -95) : 0;  // max|q| < 2^e
        const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23) * (a.scale < 0.f ? -1.f : 1.f);
        f = finite ? fabsf(a.scale) * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - 13 + e) << 23) : NAN;
#pragma unroll
        for (int j = 0; j < N; j++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[j][i] = finite ? x[j][i] * up : 0.f;
                qsum += x[j][i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = kva::h2_pack(x[j][2 * i], x[j][2 * i + 1]);
            kvt::st4(Q + kvt::place(r, KVT_PARTS * j + part), make_uint4(w[0], w[1], w[2], w[3]));
        }
        if constexpr (FMT == KVQ_INT4) {
            __syncthreads();
            s_red[part][r] = qsum;
            __syncthreads();
            qsum = (s_red[0][r] + s_red[1][r]) + (s_red[2][r] + s_red[3][r]);
        }
    }
    copies_wait<3>();
    convert(0, 0, K);
    store_meta(0);
    publish();
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    load_meta(1);

    // ---- the tiles -----------------------------------------------------------------------
    constexpr int OD = HD / KVT_PARTS;  // dims of O that a thread rescales and writes
    constexpr float kLag = 9.f, kMost = 32768.f, kNone = -3.402823466e38f;  // as in k_kvq_attend
    constexpr uint32_t kUnit = 241;
    float base = kNone, l[4] = {0.f, 0.f, 0.f, 0.f}, z[4] = {0.f, 0.f, 0.f, 0.f};
    float unit = __uint_as_float(kUnit << 23);
    const bool busy = 32 * quarter < n_rows;  // warps whose rows are all past the end only keep step
    const uint32_t o_at = tmem + lanes + S::O_COL + part * OD;
    bool ok = true;
    int t = 0;
    for (; t < ntiles; t++) {
        const int p0 = c0 + t * KVT_KEYS;
        // copies: K(t), V(t) [K(t) done], K(t+1), V(t+1) outstanding at most
        if (t + 1 < ntiles) {
            copies_wait<1>();  // V(t) and K(t+1) are there
        } else {
            copies_wait<0>();
        }
        ok = tc::bar_wait(&bar_s, (uint32_t)(t & 1), &s_abort, a.wait_ns);
        tc::fence_after();
        const uint32_t live = s_live[t & 3];
        if (t + 1 < ntiles) {
            convert(t + 1, 0, K);
            store_meta(t + 1);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc::fence_before();
        if (!__syncthreads_and(ok)) break;
        if (t + 1 < ntiles) load_meta(t + 2);  // (positions past c1 give 0)
        const bool full = p0 + KVT_KEYS <= min(prefix, c1) && live == 0xffffu;
        const float vtop = __uint_as_float(max(max(s_vtop[t & 1][0], s_vtop[t & 1][1]), max(s_vtop[t & 1][2], s_vtop[t & 1][3])));
        bool over = false;
        // the row's scores of columns c .. c + 15 of its part (without f); they
        // are read twice, as registers are short
        auto scores = [&](int c, float (&s)[16]) {
            kvt::ld(tmem + lanes + 128u * (t & 1) + KVT_COLS * part + c, s);
            const float* ks = &s_k[t & 1][0][KVT_COLS * part + c];
            kvt::wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(ks + j);
                if constexpr (FMT == KVQ_INT8) {
                    s[j] *= k4.x, s[j + 1] *= k4.y, s[j + 2] *= k4.z, s[j + 3] *= k4.w;
                } else {
                    const float4 c4 = *reinterpret_cast<const float4*>(ks + KVT_KEYS + j);
                    s[j] = fmaf(s[j], k4.x, c4.x * qsum), s[j + 1] = fmaf(s[j + 1], k4.y, c4.y * qsum);
                    s[j + 2] = fmaf(s[j + 2], k4.z, c4.z * qsum), s[j + 3] = fmaf(s[j + 3], k4.w, c4.w * qsum);
                }
            }
        };
        uint32_t see = 0xffffffffu;
        if (busy) {
            if (!full) {
                // bit i: position at0 + i is there and seen by the row
                const int at0 = p0 + KVT_COLS * part, n0 = at0 - prefix;
                see = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) see |= ((live >> (4 * part + i)) & 1) * (0xffu << (8 * i));
                see &= at0 >= c1 ? 0u : c1 - at0 >= 32 ? 0xffffffffu : (1u << (c1 - at0)) - 1;
                if (n0 > -32 && mine) {  // some of them are drafted tokens
                    auto word = [&](int n) {  // the row's bits n .. n + 31, n a multiple of 32
                        if (a.mask) return n >= 0 && n / 32 < a.mask_words ? __ldg(a.mask + (size_t)(first + node) * a.mask_words + n / 32) : 0u;
                        return node >= n + 31 ? 0xffffffffu : node < n ? 0u : (2u << (node - n)) - 1;
                    };
                    const int low = n0 & ~31;
                    see &= n0 < 0 ? (word(0) << (-n0)) | ((1u << (-n0)) - 1) : __funnelshift_r(word(low), word(low + 32), n0 & 31);
                }
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains
            auto largest = [&](auto all) {
#pragma unroll
                for (int c = 0; c < KVT_COLS; c += 16) {
                    float s[16];
                    scores(c, s);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        if constexpr (!decltype(all)::value) s[j] = (see >> (c + j)) & 1 ? s[j] : -INFINITY;
                        top[j & 3] = fmaxf(top[j & 3], s[j]);
                    }
                }
            };
            if (full)
                largest(std::true_type{});
            else
                largest(std::false_type{});
            const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            s_red[part][r] = most;
            over = most * f > base || vtop * unit >= kMost;
        }
        if (t > 0) ok = tc::bar_wait(&bar_o, (uint32_t)((t - 1) & 1), &s_abort, a.wait_ns);  // P, V and O are free
        if (__syncthreads_or(over || !ok)) {
            if (s_abort) break;
            tc::fence_after();
            // f > 0: the largest product is the largest score
            const float top = fmaxf(fmaxf(s_red[0][r], s_red[1][r]), fmaxf(s_red[2][r], s_red[3][r])) * f;
            __syncthreads();
            const bool rise = top > base;
            const float to = rise ? top + kLag : base, by = rise ? to - base : 0.f;
            base = to;
            if (busy) {
                float most = 0.f;  // (NaN: not counted)
#pragma unroll
                for (int c = 0; c < KVT_COLS; c += 16) {
                    float s[16];
                    scores(c, s);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float w = fabsf(kva::exp2_fast(fmaf(s[j], f, -base)) * s_v[t & 1][0][KVT_COLS * part + c + j]);
                        most = fmaxf(most, (see >> (c + j)) & 1 ? w : 0.f);
                    }
                }
                s_red[part][r] = most;
            }
            __syncthreads();
            if (busy) {
                const float most = fmaxf(fmaxf(s_red[0][r], s_red[1][r]), fmaxf(s_red[2][r], s_red[3][r]));
                const uint32_t field = __float_as_uint(unit) >> 23, grow = min((uint32_t)fminf(by, 300.f), kUnit - field);
                const uint32_t next = by > 0.f || vtop * unit >= kMost ? min(field + grow, 256u - (__float_as_uint(most) >> 23)) : field;
                unit = __uint_as_float(next << 23);
#pragma unroll
                for (int i = 0; i < 4; i++) l[i] *= kva::exp2_fast(-by), z[i] *= kva::exp2_fast(-by);
                if (t > 0) {
                    const float beta = kva::exp2_fast((float)(int)(next - field) - by);
                    float v[OD];
                    kvt::ld(o_at, v);
                    kvt::wait_ld();
#pragma unroll
                    for (int i = 0; i < OD; i++) v[i] *= beta;
                    kvt::st(o_at, v);
                    kvt::wait_st();
                }
            }
        }
        tc::fence_after();
        if (busy) {
            // weights of 8 columns at a time; `all`: the row sees every one
            auto weights = [&](auto all) {
#pragma unroll
                for (int c = 0; c < KVT_COLS; c += 16) {
                    float s[16];
                    scores(c, s);
#pragma unroll
                    for (int j = 0; j < 16; j += 8) {
                        float w[8];
#pragma unroll
                        for (int i = 0; i < 8; i += 4) {
                            const float* to = &s_v[t & 1][0][KVT_COLS * part + c + j + i];
                            const float4 v4 = *reinterpret_cast<const float4*>(to);
                            const float vs[4] = {v4.x, v4.y, v4.z, v4.w};
                            float vc[4] = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (FMT == KVQ_INT4) {
                                const float4 c4 = *reinterpret_cast<const float4*>(to + KVT_KEYS);
                                vc[0] = c4.x, vc[1] = c4.y, vc[2] = c4.z, vc[3] = c4.w;
                            }
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                float p = kva::exp2_fast(fmaf(s[j + i + e], f, -base)), v = vs[e] * unit;
                                if constexpr (!decltype(all)::value) {  // nothing of what it does not see, NaN or not
                                    const bool seen = (see >> (c + j + i + e)) & 1;
                                    p = seen ? p : 0.f, v = seen ? v : 0.f, vc[e] = seen ? vc[e] : 0.f;
                                }
                                w[i + e] = p * v;
                                l[e] += p;
                                if constexpr (FMT == KVQ_INT4) z[e] = fmaf(p, vc[e], z[e]);
                            }
                        }
                        kvt::st4(P + kvt::place(r, (KVT_COLS * part + c + j) / 8),
                                 make_uint4(kva::h2_pack(w[0], w[1]), kva::h2_pack(w[2], w[3]), kva::h2_pack(w[4], w[5]), kva::h2_pack(w[6], w[7])));
                    }
                }
            };
            if (full)
                weights(std::true_type{});
            else
                weights(std::false_type{});
        }
        convert(t, 1, V);
        publish();
        // this tile's raw bytes are used up
        if (t + 2 < ntiles) {
            fetch(t + 2, 0);
            copies_commit();
            fetch(t + 2, 1);
            copies_commit();
        }
    }
    float o[OD];
    if (t == ntiles) {
        ok = tc::bar_wait(&bar_o, (uint32_t)((ntiles - 1) & 1), &s_abort, a.wait_ns);
        if (__syncthreads_and(ok)) {
            tc::fence_after();
            kvt::ld(o_at, o);
            kvt::wait_ld();
        }
    }
    copies_wait<0>();
    const float back = __uint_as_float((254u << 23) - __float_as_uint(unit));  // 1 / unit
    const bool gave_up = s_abort;
    s_sum[0][part][r] = (l[0] + l[1]) + (l[2] + l[3]);
    s_sum[1][part][r] = (z[0] + z[1]) + (z[2] + z[3]);
    __syncthreads();
    float ls = 0.f, zs = 0.f;
#pragma unroll
    for (int i = 0; i < KVT_PARTS; i++) ls += s_sum[0][i][r], zs += s_sum[1][i][r];
    if (gave_up) ls = NAN;
    if (mine && part == 0) {
        if (a.splits > 1)
            a.part_ml[item * a.splits + split] = make_float2(base == kNone ? -INFINITY : base, ls);
        else if (a.lse)
            a.lse[item] = 0.693147180559945309f * ((ls == 0.f ? -INFINITY : base) + log2f(ls));
    }
    // rows of O through shared memory (the operands are done with), so that
    // they are written as runs: [row][dim], 16-byte chunks moved by the row
    const float inv = a.splits > 1 ? 1.f : ls == 0.f ? 0.f : 1.0f / ls;
    float* so = reinterpret_cast<float*>(sm);
    auto so_at = [&](int row, int dim) { return row * HD + ((((dim >> 2) ^ row) & 7) | ((dim >> 2) & ~7)) * 4 + (dim & 3); };
#pragma unroll
    for (int d = 0; d < OD; d++) {
        const int col = part * OD + d, dim = (col & ~7) + kvt::dim_at<FMT>(d & 7);
        so[so_at(r, dim)] = gave_up ? NAN : fmaf(o[d], back, zs) * inv;
    }
    __syncwarp();
    // a warp wrote 32 rows x OD dims: it writes out those
    for (int i = lane; i < 32 * (OD / 4); i += 32) {
        const int row = 32 * quarter + i / (OD / 4), dim = part * OD + i % (OD / 4) * 4;
        const int token = (row0 + row) / a.share, qh = head * a.share + (row0 + row) - token * a.share;
        if (row >= n_rows || dim >= hd) continue;
        const float4 v = *reinterpret_cast<const float4*>(so + so_at(row, dim));
        const size_t at = (size_t)(first + token) * a.n_heads + qh;
        if (a.splits > 1) {
            *reinterpret_cast<float4*>(a.part_o + (at * a.splits + split) * hd + dim) = v;
        } else {
            const uint2 two = a.dtype == 1 ? make_uint2(float_to_bf16_bits(v.x) | float_to_bf16_bits(v.y) << 16,
                                                        float_to_bf16_bits(v.z) | float_to_bf16_bits(v.w) << 16)
                                           : make_uint2(kva::h2_pack(v.x, v.y), kva::h2_pack(v.z, v.w));
            *reinterpret_cast<uint2*>(static_cast<unsigned short*>(a.out) + at * hd + dim) = two;
        }
    }
    tc::fence_before();
    __syncthreads();
}

}  // namespace fb2
