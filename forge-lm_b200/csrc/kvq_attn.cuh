// kvq_attn.cuh — attention of new tokens (single ones or drafted trees) over
// the paged, quantised K/V cache.
//
// out = sum_p softmax_p(scale q.k_p) v_p over the positions a row sees, in one
// pass: the running maximum m, l = sum exp(s - m) and o = sum exp(s - m) v,
// rescaled when m grows; parts merge by the same rule.  With codes c and the
// row's scale a and (int4) minimum b, k = a c + b:
//   q.k = a (q.c) + b sum(q),    sum_p w_p v_p = sum_p (w_p a_p) c_p + sum_p w_p b_p,
// so both products run on the codes themselves, which fp16 holds exactly, and
// the scales are applied to scores and probabilities.
#pragma once
#include <type_traits>

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
    float* part_o;           // [n_rows][n_heads][splits][hd], and
    float2* part_ml;         // (m, l) of each, where splits > 1
    long long q_row, q_head, table_stride;
    int n_seqs, n_rows, n_heads, share, max_nodes, max_len, mask_words, dtype;
    int fill;                // 1: a row of blocks for fill_rest
    int splits, chunk, row_blocks, block_rows, warps;  // block_rows 8, 16: k_kvq_attend; 128: k_kvq_attend_tc
    float scale;
    int withhold;            // test hook: block 0 does not announce the end of this tile's O; -1: every block does
    unsigned long long wait_ns;  // limit of k_kvq_attend_tc's waits
    // a malformed list must not reach past the tensors: each start is cut to them
    FB2_DEV int start_of(int b) const { return starts ? min(max(__ldg(starts + b), 0), n_rows) : b; }
    FB2_DEV void rows_of(int b, int& first, int& count) const {
        first = start_of(b);
        count = min(max(start_of(b + 1) - first, 0), max_nodes);
    }
    // Zeros and -inf for the rows that lie past those that their sequence may have,
    // before the first sequence or after the last: the work of a row of blocks of its
    // own after the sequences' (as a part of theirs it cost the loops registers: 16
    // long sequences 257 -> 260 to 272 us).
    FB2_DEV void fill_rest() const {
        auto fill_rows = [&](int from, int to) {
            const size_t heads = (size_t)max(to - from, 0) * n_heads, at = (size_t)from * n_heads;
            const int vecs = c.hd * (dtype == 0 ? 4 : 2) / 16;  // of a head
            uint4* o = static_cast<uint4*>(out) + at * vecs;
            for (size_t i = threadIdx.x; i < heads * vecs; i += blockDim.x) o[i] = make_uint4(0, 0, 0, 0);
            if (lse)
                for (size_t i = threadIdx.x; i < heads; i += blockDim.x) lse[at + i] = -INFINITY;
        };
        for (int b = blockIdx.x; b < n_seqs; b += gridDim.x) {
            int first, count;
            rows_of(b, first, count);
            if (b == 0) fill_rows(0, first);
            fill_rows(first + count, b + 1 < n_seqs ? start_of(b + 1) : n_rows);
        }
    }
    FB2_DEV float load_q(long long row, int head, int d) const {
        const long long at = row * q_row + head * q_head + d;
        if (dtype == 0) return __ldg(static_cast<const float*>(q) + at);
        if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(q)[at]);
        return __half2float(static_cast<const __half*>(q)[at]);
    }
    FB2_DEV void store_out(size_t at, float v) const {
        if (dtype == 0)
            static_cast<float*>(out)[at] = v;
        else if (dtype == 1)
            static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
        else
            static_cast<__half*>(out)[at] = __float2half_rn(v);
    }
};

namespace kva {

FB2_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a fresh sum
FB2_DEV void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
FB2_DEV void mma_u8s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a sum that starts at z
FB2_DEV void mma_u8s8_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&z)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(z[0]), "r"(z[1]), "r"(z[2]), "r"(z[3]));
}
FB2_DEV uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
FB2_DEV uint32_t h2_sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
FB2_DEV uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
FB2_DEV uint32_t h2_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
FB2_DEV float2 h2_floats(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// fp16 pairs of codes.  0x6400 | b is 1024 + b (b < 1024), exactly.
// int8 bytes 0,1 (2,3 with `high`) of w as code = byte - 128.
template <bool HIGH>
FB2_DEV uint32_t codes8(uint32_t w) {
    return h2_sub(__byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140), 0x64806480u);
}
// Nibbles I and I + 4 of w as codes - 8 (a nibble at bits 4..7 of its half
// is 16 c in the sum: times 1/16, minus 72).  Around 8 they nearly cancel in
// the sums, so that the probabilities' roundings do too; the minimum that
// goes with them is b + 8 a.
template <int I>
FB2_DEV uint32_t codes4(uint32_t w) {
    const uint32_t v = I < 2 ? w : w >> 8;
    if constexpr (I % 2 == 0) return h2_sub((v & 0x000f000fu) | 0x64006400u, 0x64086408u);
    return h2_fma((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
}

// b + 8 a of an int4 row's meta word
FB2_DEV float centre(uint32_t w) { return fmaf(8.0f, bf16_bits_to_float(w & 0xffffu), __uint_as_float(w & 0xffff0000u)); }

FB2_DEV float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace kva

// A CTA takes one chunk of one sequence's positions for one K/V
// head and a block of 8 NT rows (the rows of its tokens and of the query
// heads that share the K/V head).  Each warp works on its own tiles of 16 MT
// positions through its own ring in shared memory (two tiles ahead by cp.async;
// straight to registers: 472 us for what the ring took to 268), with no barrier
// until the end:
//   S^T[position][row] = K codes (A, 16 positions) x q (B, 8 rows),
//   O^T[dim][row]     += V codes^T (A, 16 dims) x P^T (B, 16 positions x 8 rows),
// the same column = row layout for both accumulators, so maxima and rescaling
// need no exchange between the two; P's 8 x 8 blocks are transposed by
// movmatrix.  Dimensions and positions are assigned to fragments so that a
// lane's K and V codes are consecutive bytes (K: 16 dims of a position; V: HD/8
// dims of 2 positions); q's fragments are built in that order once.
//
// Scores take 8-bit integer tiles (16 positions x 32 dims, exact sums): the
// codes are bytes as they lie in memory (int4: one or two logical operations
// per four), and q is in fixed point, rint(q 2^(22 - e)) for max|q| < 2^e of
// its row, in three digits of 8 bits, which is exact to 2^-23 of max|q|.  The
// codes' offset (128, 8) is taken off where the sums start.
// Values take fp16 tiles: what a probability adds can be of any size, so P
// stays in floating point, scaled together with the V scales: one fp16 term for
// the 16-bit types, whose results have no more bits (a second one brings the error
// of fp16 against 64 bits from 2.8e-4 to 2.1e-4, its rounding alone, and takes 279
// us for 258 on the long sequences below, 15.3 for 14.4 on the short ones in fp16); two for
// fp32, whose sums over a tile start at zero and are added to the running ones.
//
// What bounds it: with many long sequences the instructions that make operands
// of the codes and probabilities of the scores (16 sequences of 40 to 65 K int4
// positions, 32 heads on 8 of 128, fp16: 259 us, 3.5 TB/s; 32 sequences of up to
// 1023 int8 positions, 12 heads of 64, fp32: 15.1 us, 1.9 TB/s); with few the
// chain from a launch over the page table to the merge (one of 576: 7.6 us).
template <int HD, int FMT, int NT, bool SPLIT, int WARPS>
struct KvaShape {
    static constexpr int MT = HD > 128 ? 1 : 2;       // 16-position groups of a tile
    static constexpr int TT = 16 * MT;                // positions of a tile
    static constexpr int RB = FMT == KVQ_INT8 ? HD : HD / 2;  // bytes of a row in shared memory
    static constexpr int KCH = HD / 64;               // 16-dim chunks of K per lane and position
    static constexpr int KW = FMT == KVQ_INT8 ? 4 : 2;  // words of a chunk
    static constexpr int VD = HD / 8;                 // dims of V per lane and position
    static constexpr int VW = FMT == KVQ_INT8 ? VD / 4 : VD / 8;
    static constexpr int STEPS = HD / 32;             // of 32 dims
    static constexpr int PARTS = SPLIT ? 2 : 1;       // terms of P
    static constexpr int ROWS = 8 * NT;
    // a warp's ring: two tiles of K rows, V rows (by groups of 8 positions) and
    // meta words
    static constexpr int GROUP = 16 * RB, META = TT / 8 * GROUP, SLOT = META + 2 * TT * 4, DEPTH = 2;
    static constexpr int RING = WARPS * DEPTH * SLOT;
    static constexpr int Q_BYTES = NT * 3 * STEPS * 32 * 8;
    static constexpr int O_STRIDE = HD + 8;
    static constexpr int O_BYTES = WARPS * ROWS * O_STRIDE * 4;
    static constexpr int BIG = RING > O_BYTES ? RING : O_BYTES;  // the merge takes the rings' place
    static constexpr int SMEM = BIG + Q_BYTES + ROWS * 8 + ROWS * 16 + WARPS * ROWS * 8;
    // CTAs per SM that the registers are kept to (shared memory allows them)
    static constexpr int RESIDENT = WARPS == 8 ? 1 : NT == 1 ? (HD == 64 || (HD == 128 && FMT == KVQ_INT4) ? 4 : HD == 128 ? 3 : 2) : 2;
    // Where 16-byte unit u of 8 rows lies: moved within its 128-byte line so
    // that the K reads (8 neighbouring rows, a run of each) and the V reads
    // (every second row, another run) both spread over the banks.
    static FB2_DEV uint32_t place(uint32_t u) {
        if constexpr (RB == 32) return u ^ (((u >> 3) & 1) << 1);
        if constexpr (RB == 64) return u ^ (((u >> 3) & 3) << 1);
        const uint32_t row = u / (RB / 16);
        return u ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2));
    }
};

template <int HD, int FMT, int NT, bool SPLIT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, KvaShape<HD, FMT, NT, SPLIT, WARPS>::RESIDENT) k_kvq_attend(KvqAttnArgs a) {
    using namespace kva;
    using S = KvaShape<HD, FMT, NT, SPLIT, WARPS>;
    extern __shared__ __align__(16) unsigned char smem[];
    float* so = reinterpret_cast<float*>(smem);
    unsigned char* sq = smem + S::BIG;                                  // [row tile][digit][two steps][lane] 16 bytes
    float4* szero = reinterpret_cast<float4*>(sq + S::Q_BYTES);         // what to take off each digit's sums
    float2* srow = reinterpret_cast<float2*>(sq + S::Q_BYTES + S::ROWS * 16);  // (score factor, factor * sum q)
    float2* sml = srow + S::ROWS;                                       // [warp][row] (m, l)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int b = blockIdx.y;
    if (b >= a.n_seqs) return a.fill_rest();
    const int rb = blockIdx.x % a.row_blocks, rest = blockIdx.x / a.row_blocks;
    const int split = rest % a.splits, head = rest / a.splits;
    int first, count;
    a.rows_of(b, first, count);
    const int row0 = rb * S::ROWS, n_rows = min(S::ROWS, count * a.share - row0);
    if (n_rows <= 0) return;
    const int prefix = max(__ldg(a.prefix + b), 0);
    const int len = (int)min((long long)prefix + count, (long long)a.max_len);
    const int c0 = split * a.chunk, c1 = len - c0 > a.chunk ? c0 + a.chunk : len;
    // row r of the block: token (row0 + r) / share of the sequence, query head
    // head * share + (row0 + r) % share
    if (c0 >= c1 && a.splits > 1) {  // nothing here: the merge has to know
        for (int r = tid; r < n_rows; r += WARPS * 32) {
            const int node = (row0 + r) / a.share, h = head * a.share + (row0 + r) - node * a.share;
            a.part_ml[((size_t)(first + node) * a.n_heads + h) * a.splits + split] = make_float2(-INFINITY, 0.f);
        }
        return;
    }

    // ---- the tile loop's addresses -------------------------------------------
    const int ps = 1 << a.c.page_shift, rbytes = a.c.row_bytes, hd = a.c.hd;
    const uint32_t n_pages = a.c.n_slots >> a.c.page_shift;
    const int tiles = (c1 - c0 + S::TT - 1) / S::TT;
    constexpr int GR = 2 * S::MT;        // 8-position groups of a tile, each in one page
    constexpr int AHEAD = 32 / GR;       // tiles whose groups a warp holds, one per lane
    const int* table = a.table + b * a.table_stride;
    // index of a group among all groups of 8 K or V rows (V's lie ps / 8 after K's)
    uint32_t ids = 0, valid = 0;         // one group per lane; which of them have a page
    auto load_ids = [&](int tile) {      // of tiles tile, tile + WARPS, ..
        const int pos = c0 + (tile + (lane / GR) * WARPS) * S::TT + (lane % GR) * 8;
        const uint32_t page = pos < c1 ? (uint32_t)__ldg(table + (pos >> a.c.page_shift)) : n_pages;
        valid = __ballot_sync(0xffffffffu, page < n_pages);
        ids = page < n_pages ? (((page * a.c.heads + head) * 2) << (a.c.page_shift - 3)) + ((pos & (ps - 1)) >> 3) : 0;
    };
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::DEPTH * S::SLOT;
    // 16-byte units of 8 rows; a lane's of a group: of K, then as many of V, or (16
    // units) the lower lanes of K and the others of V
    constexpr int UNITS = S::RB / 2, KINDS = UNITS >= 32 ? 2 : 1, COPIES = 2 * UNITS / 32 / KINDS;
    const unsigned char* copy_from[COPIES];
    uint32_t copy_to[COPIES];
    const uint32_t v_from = ps * S::RB;  // where V lies after K
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const uint32_t u = 32 * i + lane, kind = u / UNITS, at = u % UNITS;
        copy_from[i] = a.c.codes + kind * v_from + at * 16;
        copy_to[i] = kind * (8 * S::RB) + S::place(at) * 16;
    }
    const uint32_t* meta_from = a.c.meta + ((lane >> 1) & 1) * ps + (lane & 1) * 4;
    const uint32_t meta_to = S::META + ((lane >> 1) & 1) * (S::TT * 4) + (lane >> 2) * 32 + (lane & 1) * 16;
    // Starts the copies of a tile; returns which of its groups have a page (the
    // others are zeros).  Positions past c1 bring whatever the page holds there.
    auto fetch = [&](int held, uint32_t to) {
        const uint32_t live = (valid >> (held * GR)) & ((1u << GR) - 1);
        const uint32_t mine = __shfl_sync(0xffffffffu, ids, (held * GR + (lane >> 2)) & 31);
        const bool all = hd == HD && live == (1u << GR) - 1;
#pragma unroll
        for (int j = 0; j < GR; j++) {
            const uint64_t skip = (uint64_t)__shfl_sync(0xffffffffu, ids, held * GR + j) * (uint32_t)(8 * rbytes);
            const bool there = (live >> j) & 1;
            if (all) {
#pragma unroll
                for (int i = 0; i < COPIES * KINDS; i++)
                    copy16(to + copy_to[i % COPIES] + j * S::GROUP + i / COPIES * (8 * S::RB), copy_from[i % COPIES] + skip + i / COPIES * v_from);
            } else if (hd == HD) {
#pragma unroll
                for (int i = 0; i < COPIES * KINDS; i++)
                    copy16(to + copy_to[i % COPIES] + j * S::GROUP + i / COPIES * (8 * S::RB), copy_from[i % COPIES] + skip + i / COPIES * v_from,
                           there);
            } else {
                // rows shorter than in shared memory: two lanes to a row
                const int row = lane >> 1, kind = row >> 3, r = row & 7;
                const unsigned char* from = a.c.codes + skip + kind * (ps * rbytes) + r * rbytes;
                const uint32_t base = to + j * S::GROUP + kind * (8 * S::RB);
                if ((rbytes & 15) == 0) {
#pragma unroll 1
                    for (int u = lane & 1; u < rbytes / 16; u += 2) copy16(base + S::place(r * (S::RB / 16) + u) * 16, from + u * 16, there);
                } else {
#pragma unroll 1
                    for (int u = lane & 1; u < rbytes / 8; u += 2)
                        copy8(base + S::place(r * (S::RB / 16) + (u >> 1)) * 16 + (u & 1) * 8, from + u * 8, there);
                }
            }
        }
        if (lane < 4 * GR) {  // group lane / 4: K's and V's 8 words, 4 at a time
            copy16(to + meta_to, meta_from + (uint64_t)mine * 8, (live >> (lane >> 2)) & 1);
        }
        return live;
    };
    // a lane's reads in the first group: K chunks of position g, V of positions 2 t, 2 t + 1
    uint32_t k_at[S::KCH], v_at[2][S::VW > 4 ? 2 : 1];
#pragma unroll
    for (int cc = 0; cc < S::KCH; cc++) {
        const uint32_t byte = g * S::RB + (t + 4 * cc) * (S::KW * 4);
        k_at[cc] = S::place(byte >> 4) * 16 + (byte & 15);
    }
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int i = 0; i < (S::VW > 4 ? 2 : 1); i++) {
            const uint32_t byte = (2 * t + e) * S::RB + g * (S::VW * 4) + 16 * i;
            v_at[e][i] = 8 * S::RB + S::place(byte >> 4) * 16 + (byte & 15);
        }
    auto read_words = [&](uint32_t at, uint32_t* w, auto n) {
        constexpr int N = decltype(n)::value;
        if constexpr (N == 1) {
            w[0] = lds(at);
        } else if constexpr (N == 2) {
            const float2 v = lds2(at);
            w[0] = __float_as_uint(v.x), w[1] = __float_as_uint(v.y);
        } else {
            const uint4 v = lds4(at);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
    };
    int held = 0;  // tiles of `ids` used up
    uint32_t live_next = 0;
    if (warp < tiles) {
        load_ids(warp);
        live_next = fetch(0, ring);
    }
    copies_commit();

    // ---- q's fragments (while the first tile is on its way) --------------------
    // Integer sums start at the bits of 1.5 2^23: up to 2^22 in size, they are
    // then the bits of 1.5 2^23 + sum (over 256 dims and bytes they are larger
    // and converted).
    constexpr bool BITS = !(HD == 256 && FMT == KVQ_INT8);
    constexpr int START = BITS ? (int)kRintBits : 0;
    for (int r = warp; r < S::ROWS; r += WARPS) {
        float x[HD / 32], top = 0.f, sum = 0.f;
        int digits[3] = {0, 0, 0};
        const int node = (row0 + r) / a.share, h = head * a.share + (row0 + r) - node * a.share;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            const int d = lane + 32 * i;
            x[i] = r < n_rows && d < hd ? a.load_q(first + node, h, d) : 0.f;
            top = max_nan(top, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool finite = top < INFINITY;
        // max|q| < 2^e; below 2^-95 only what no score keeps is lost
        const int e = finite ? max((int)(__float_as_uint(top) >> 23) - 126, -95) : 0;
        const float up = __uint_as_float((uint32_t)(127 + 22 - e) << 23);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            const int d = lane + 32 * i, c = d >> 4, w = d & 15;
            x[i] = finite ? rintf(x[i] * up) : 0.f;
            sum += x[i];
            // digits of q + 128 (1 + 2^8 + 2^16), each less 128
            const uint32_t q = (uint32_t)(int)x[i] + 0x808080u;
            int step = 2 * (c >> 2) + (w >> 3), reg, byte;
            if constexpr (FMT == KVQ_INT8)
                reg = (w >> 2) & 1, byte = w & 3;
            else
                reg = w & 1, byte = (w >> 1) & 3;
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const int digit = (int)((q >> (8 * k)) & 0xffu) - 128;
                digits[k] += digit;
                sq[((((r >> 3) * 3 + k) * (S::STEPS / 2) + step / 2) * 32 + 4 * (r & 7) + (c & 3)) * 16 + 8 * (step & 1) + 4 * reg + byte] =
                    (unsigned char)digit;
            }
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int k = 0; k < 3; k++) digits[k] = __reduce_add_sync(0xffffffffu, digits[k]);
        if (lane == 0) {
            const float f = finite ? a.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - 22 + e) << 23) : NAN;
            constexpr int off = FMT == KVQ_INT8 ? 128 : 8;
            srow[r] = make_float2(f, sum * f);
            constexpr float start = BITS ? kRint : 0.f;
            szero[r] = make_float4(start + (float)(off * digits[0]), start + (float)(off * digits[1]), start + (float)(off * digits[2]), 0.f);
        }
    }
    __syncthreads();

    // ---- the pass over the positions --------------------------------------------
    // A row's probabilities are exp2(s - base), at most 1: base is kLag above the
    // largest score at the last time that one exceeded base.  Its weights are
    // probability * V scale, and unit, a power of two, brings the largest that the
    // row had so far to 2^2..2^3 at times.  Those times are when base moves and
    // when V scale * unit, the most that a weight can be, reaches kMost; so fp16
    // holds every weight, with at least 16 bits below the row's largest, whatever
    // other rows or masked positions have.  (One unit for all rows, by the tile's
    // largest V scale: 256 us for 259 on the long sequences, 14.4 for 15.1 on the short
    // ones; but a V row 2^20 times the others, seen or not, left the others' weights
    // 4 bits.)  o is in units of 1 / unit.
    constexpr float kLag = 9.f, kMost = 32768.f, kNone = -3.402823466e38f;  // kNone: nothing seen yet
    constexpr uint32_t kUnit = 241;  // exponent field of the largest unit
    float vlim = kMost * __uint_as_float((254u - kUnit) << 23);  // kMost / the lane's largest unit
    float o[S::VD / 2][NT][4], base[NT][2], unit[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int i = 0; i < 2; i++) base[n][i] = kNone, unit[n][i] = __uint_as_float(kUnit << 23), l[n][i] = 0.f, z[n][i] = 0.f;
#pragma unroll
        for (int i = 0; i < S::VD / 2; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][n][c] = 0.f;
    }
    float2 rowf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) rowf[n][i] = srow[8 * n + 2 * t + i];
    float zero[NT][2][3];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4 v = szero[8 * n + 2 * t + i];
            zero[n][i][0] = v.x, zero[n][i][1] = v.y, zero[n][i][2] = v.z;
        }
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(sq) + lane * 16;

    int slot = 0;
    for (int tile = warp; tile < tiles; tile += WARPS) {
        const int pos0 = c0 + tile * S::TT;
        const uint32_t live = live_next, at = ring + slot * S::SLOT;  // live: groups with a page
        slot ^= 1;
        __syncwarp();  // every lane is done with the slot that is filled now
        if (tile + WARPS < tiles) {
            if (++held == AHEAD) {
                held = 0;
                load_ids(tile + WARPS);
            }
            live_next = fetch(held, ring + slot * S::SLOT);
        }
        copies_commit();
        copies_wait<1>();
        __syncwarp();
        // every position seen by every row?
        const bool full = pos0 + S::TT <= min(prefix, c1) && live == (1u << GR) - 1;
        uint32_t km[GR], vm[GR];
#pragma unroll
        for (int j = 0; j < GR; j++) {
            km[j] = lds(at + S::META + (8 * j + g) * 4);
            vm[j] = lds(at + S::META + (S::TT + 8 * j + g) * 4);
            if (!full) vm[j] = pos0 + 8 * j + g < c1 ? vm[j] : 0;
        }

        const int start[4] = {START, START, START, START};
        float s[S::MT][NT][4];
#pragma unroll
        for (int i = 0; i < S::MT; i++) {
            int acc[NT][3][4];
            uint32_t kr[2][S::KCH][S::KW];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int cc = 0; cc < S::KCH; cc++)
                    read_words(at + (2 * i + j) * S::GROUP + k_at[cc], kr[j][cc], std::integral_constant<int, S::KW>{});
#pragma unroll
            for (int st = 0; st < S::STEPS; st += 2) {
                uint32_t f[2][4];  // positions g | g + 8, first | second four dims
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if constexpr (FMT == KVQ_INT8) {
                            f[e][j] = kr[j][st / 2][2 * e];
                            f[e][2 + j] = kr[j][st / 2][2 * e + 1];
                        } else {
                            const uint32_t w = kr[j][st / 2][e];
                            f[e][j] = w & 0x0f0f0f0fu;
                            f[e][2 + j] = (w >> 4) & 0x0f0f0f0fu;
                        }
                    }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int k = 0; k < 3; k++) {
                        const uint4 qf = lds4(q_at + ((n * 3 + k) * (S::STEPS / 2) + st / 2) * 512);
                        if (st == 0)
                            mma_u8s8_first(acc[n][k], f[0], qf.x, qf.y, start);
                        else
                            mma_u8s8(acc[n][k], f[0], qf.x, qf.y);
                        mma_u8s8(acc[n][k], f[1], qf.z, qf.w);
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float d[3];
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        d[k] = (BITS ? __int_as_float(acc[n][k][c]) : (float)acc[n][k][c]) - zero[n][c & 1][k];
                    s[i][n][c] = fmaf(fmaf(d[2], 256.f, d[1]), 256.f, d[0]);
                }
        }
        // scores in units of log2
#pragma unroll
        for (int i = 0; i < S::MT; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t w = km[2 * i + (c >> 1)];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float2 f = rowf[n][c & 1];
                    if constexpr (FMT == KVQ_INT8)
                        s[i][n][c] *= __uint_as_float(w) * f.x;
                    else
                        s[i][n][c] = fmaf(s[i][n][c], bf16_bits_to_float(w & 0xffffu) * f.x, centre(w) * f.y);
                }
            }
        if (!full) {
#pragma unroll
            for (int i = 0; i < S::MT; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int j = 2 * i + (c >> 1), pos = pos0 + 8 * j + g, node = pos - prefix;
                    const bool there = ((live >> j) & 1) && pos < c1;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const int r = 8 * n + 2 * t + (c & 1);
                        bool see = there && r < n_rows;
                        if (see && node >= 0) {
                            const int mine = (row0 + r) / a.share;
                            see = a.mask ? (__ldg(a.mask + (size_t)(first + mine) * a.mask_words + (node >> 5)) >> (node & 31)) & 1
                                         : node <= mine;
                        }
                        if (!see) s[i][n][c] = -INFINITY;
                    }
                }
        }
        float top[NT][2], vs[GR], vl[GR], vmax = 0.f;
        bool over = false;
#pragma unroll
        for (int j = 0; j < GR; j++) {
            vs[j] = FMT == KVQ_INT8 ? __uint_as_float(vm[j]) : bf16_bits_to_float(vm[j] & 0xffffu);
            vl[j] = FMT == KVQ_INT8 ? 0.f : centre(vm[j]);
            vmax = fmaxf(vmax, fabsf(vs[j]));
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                top[n][c] = fmaxf(s[0][n][c], s[0][n][c + 2]);
                if constexpr (S::MT == 2) top[n][c] = fmaxf(top[n][c], fmaxf(s[1][n][c], s[1][n][c + 2]));
                over |= top[n][c] > base[n][c];
            }
        over |= vmax >= vlim;
        if (__any_sync(0xffffffffu, over)) {
            // a row's own scores and the tile's V decide, not the rows beside it
            vmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vmax)));
            uint32_t high = 0;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float beta[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) top[n][c] = fmaxf(top[n][c], __shfl_xor_sync(0xffffffffu, top[n][c], x));
                    const bool rise = top[n][c] > base[n][c];
                    const float to = rise ? top[n][c] + kLag : base[n][c], by = rise ? to - base[n][c] : 0.f;
                    base[n][c] = to;
                    l[n][c] *= exp2_fast(-by);
                    z[n][c] *= exp2_fast(-by);
                    // unit grows as the old weights shrink, up to what the tile's largest weight allows
                    float most = 0.f;  // (NaN: not counted)
#pragma unroll
                    for (int i = 0; i < S::MT; i++)
#pragma unroll
                        for (int e = 0; e < 2; e++) most = fmaxf(most, fabsf(exp2_fast(s[i][n][c + 2 * e] - to) * vs[2 * i + e]));
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
                    const uint32_t field = __float_as_uint(unit[n][c]) >> 23, grow = min((uint32_t)fminf(by, 300.f), kUnit - field);
                    const uint32_t next = rise || vmax * unit[n][c] >= kMost ? min(field + grow, 256u - (__float_as_uint(most) >> 23)) : field;
                    unit[n][c] = __uint_as_float(next << 23);
                    high = max(high, next);
                    beta[c] = exp2_fast((float)(int)(next - field) - by);
                }
#pragma unroll
                for (int i = 0; i < S::VD / 2; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][n][c] *= beta[c & 1];
            }
            vlim = kMost * __uint_as_float((254u - high) << 23);
        }
        uint32_t pb[S::MT][NT][S::PARTS][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < S::MT; i++) {
                float w[4];
                auto weigh = [&](int c, bool none) {
                    const int j = 2 * i + (c >> 1);
                    const float p = exp2_fast(s[i][n][c] - base[n][c & 1]);
                    l[n][c & 1] += p;
                    if (FMT == KVQ_INT4 && !none) z[n][c & 1] = fmaf(p, vl[j], z[n][c & 1]);
                    w[c] = none ? 0.f : p * (vs[j] * unit[n][c & 1]);
                };
                if (full) {
#pragma unroll
                    for (int c = 0; c < 4; c++) weigh(c, false);
                } else {  // what a row does not see has weight 0 even where V is NaN
#pragma unroll
                    for (int c = 0; c < 4; c++) weigh(c, s[i][n][c] == -INFINITY);
                }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t hi = h2_pack(w[2 * j], w[2 * j + 1]);
                    pb[i][n][0][j] = transpose8x8(hi);
                    if constexpr (SPLIT) {
                        const float2 f = h2_floats(hi);
                        pb[i][n][1][j] = transpose8x8(h2_pack(w[2 * j] - f.x, w[2 * j + 1] - f.y));
                    }
                }
            }
        uint32_t vr[GR][2][S::VW];
#pragma unroll
        for (int j = 0; j < GR; j++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < S::VW; i += 4)
                    read_words(at + j * S::GROUP + v_at[e][i / 4], vr[j][e] + i, std::integral_constant<int, (S::VW > 4 ? 4 : S::VW)>{});
        // O^T += V^T P^T, two rows of 8 dims (dims 2 i, 2 i + 1 of each lane) at a time
#pragma unroll
        for (int i = 0; i < S::VD / 2; i++) {
            float acc[NT][4];
#pragma unroll
            for (int k = 0; k < S::MT; k++) {
                uint32_t f[2][2];  // [dim][positions 2t,2t+1 | +8]
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int gr = 2 * k + j;
                    if constexpr (FMT == KVQ_INT8) {
                        const uint32_t x = __byte_perm(vr[gr][0][i / 2], vr[gr][1][i / 2], i % 2 ? 0x7362 : 0x5140);
                        f[0][j] = codes8<false>(x);
                        f[1][j] = codes8<true>(x);
                    } else {
                        const uint32_t x = __byte_perm(vr[gr][0][i / 4], vr[gr][1][i / 4], (i % 4) / 2 ? 0x7632 : 0x5410);
                        f[0][j] = i % 2 ? codes4<2>(x) : codes4<0>(x);
                        f[1][j] = i % 2 ? codes4<3>(x) : codes4<1>(x);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int p = 0; p < S::PARTS; p++) {
                        if (!SPLIT)
                            mma_f16(o[i][n], f[0][0], f[1][0], f[0][1], f[1][1], pb[k][n][p][0], pb[k][n][p][1]);
                        else if (k == 0 && p == 0)
                            mma_f16_first(acc[n], f[0][0], f[1][0], f[0][1], f[1][1], pb[k][n][p][0], pb[k][n][p][1]);
                        else
                            mma_f16(acc[n], f[0][0], f[1][0], f[0][1], f[1][1], pb[k][n][p][0], pb[k][n][p][1]);
                    }
            }
            if constexpr (SPLIT)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][n][c] += acc[n][c];
        }
    }

    // ---- merge the warps ------------------------------------------------------------
    copies_wait<0>();
    __syncthreads();  // the rings are done with
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
                l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
                z[n][c] += __shfl_xor_sync(0xffffffffu, z[n][c], x);
            }
            const int r = 8 * n + 2 * t + c;
            if (g == 0) sml[warp * S::ROWS + r] = make_float2(base[n][c] == kNone ? -INFINITY : base[n][c], l[n][c]);
            const float back = __uint_as_float((254u << 23) - __float_as_uint(unit[n][c]));  // 1 / unit
            float* to = so + (warp * S::ROWS + r) * S::O_STRIDE + g * S::VD;
#pragma unroll
            for (int i = 0; i < S::VD / 2; i++)
                *reinterpret_cast<float2*>(to + 2 * i) =
                    make_float2(fmaf(o[i][n][c], back, z[n][c]), fmaf(o[i][n][c + 2], back, z[n][c]));
        }
    __syncthreads();
    for (int at = tid; at < n_rows * hd; at += WARPS * 32) {
        const int r = at / hd, d = at - r * hd;
        float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, sml[w * S::ROWS + r].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float2 ml = sml[w * S::ROWS + r];
            const float f = exp2_fast(ml.x - base);
            sum = fmaf(ml.y, f, sum);
            x = fmaf(so[(w * S::ROWS + r) * S::O_STRIDE + d], f, x);
        }
        const int node = (row0 + r) / a.share, h = head * a.share + (row0 + r) - node * a.share;
        const size_t item = (size_t)(first + node) * a.n_heads + h;
        if (a.splits == 1) {
            a.store_out(item * hd + d, sum == 0.f ? 0.f : x / sum);  // 0: nothing seen (NaN stays)
            if (d == 0 && a.lse) a.lse[item] = 0.693147180559945309f * (top + log2f(sum));
        } else {
            a.part_o[(item * a.splits + split) * hd + d] = x;
            if (d == 0) a.part_ml[item * a.splits + split] = make_float2(top, sum);
        }
    }
}

// One warp per (row, head): the chunks' parts by their maxima.
__global__ void __launch_bounds__(128) k_kvq_attend_merge(KvqAttnArgs a) {
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.y;
    int first, count;
    a.rows_of(b, first, count);
    const int at = blockIdx.x * 4 + warp;
    if (at >= count * a.n_heads) return;
    const size_t item = (size_t)first * a.n_heads + at;
    const float2* ml = a.part_ml + item * a.splits;
    const float* part = a.part_o + item * a.splits * a.c.hd;
    float top = -INFINITY;
    for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, __ldcg(ml + s).x);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    const int hd = a.c.hd, d0 = 4 * lane;  // a lane's dims: d0 .. d0 + 3, and 128 further
    float sum = 0.f, x[2][4] = {};
    for (int s0 = 0; s0 < a.splits; s0 += 32) {
        const float2 w = s0 + lane < a.splits ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
        const float scale = kva::exp2_fast(w.x - base);
        sum = fmaf(w.y, scale, sum);
        // parts in which nothing was seen may not have been written
        uint32_t there = __ballot_sync(0xffffffffu, w.y != 0.f);
        while (there) {
            float4 v[4][2];
            float f[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {  // four parts' loads before their sums
                const int s = there ? __ffs(there) - 1 : 0;
                f[u] = there ? __shfl_sync(0xffffffffu, scale, s) : 0.f;
                const float4* p = reinterpret_cast<const float4*>(part + (size_t)(s0 + s) * hd + d0);
                v[u][0] = there && d0 < hd ? __ldcg(p) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[u][1] = there && d0 + 128 < hd ? __ldcg(p + 32) : make_float4(0.f, 0.f, 0.f, 0.f);
                there &= there - 1;
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    x[i][0] = fmaf(v[u][i].x, f[u], x[i][0]);
                    x[i][1] = fmaf(v[u][i].y, f[u], x[i][1]);
                    x[i][2] = fmaf(v[u][i].z, f[u], x[i][2]);
                    x[i][3] = fmaf(v[u][i].w, f[u], x[i][3]);
                }
        }
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (d0 + 128 * i < hd)
#pragma unroll
            for (int e = 0; e < 4; e++) a.store_out(item * hd + d0 + 128 * i + e, sum == 0.f ? 0.f : x[i][e] / sum);
    if (a.lse && lane == 0) a.lse[item] = 0.693147180559945309f * (top + log2f(sum));
}

}  // namespace fb2
