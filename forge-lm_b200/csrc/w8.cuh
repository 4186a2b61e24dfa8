// w8.cuh — linear layers in 8-bit integers on tcgen05 tiles: weights with a scale
// for each output, rows of x with a scale each (include/forge_b200.h,
// fb2_w8_matmul, has the formula).
//
// y = (codes of x . codes of W) * scale of W * scale of x + bias: the products and
// their sums are exact in 32-bit integers, in tensor memory, whatever the order
// (127 * 127 * in_features < 2^31), so that splitting the inputs over CTAs changes
// no bit; only the epilogue rounds.  Both operands are K-major rows of bytes, TMA
// boxes of 128 bytes x rows, 128-byte swizzled.
//
// k_w8_rows: up to 4 rows of x, on the warps' dot products, quantised on the way.
// k_w8_few: up to 128 rows of x to a tile, as the N side of the tiles, the weights
// as the M side: each weight is read once.  A cluster shares a tile's inputs where
// there are fewer tiles than SMs.  64 x 8192 x 28672 46 us (5.1 TB/s of weights), 61 x 1024 x
// 4096 6.3 us, of which the products are a small part.
// k_w8_many: 256 rows of x by 256 outputs, a pair of CTAs to a tile.
// All of them may begin while the launch before still writes what they read, weights among it
// (quantise_rows makes them too): all of it comes by TMA or by w8::late and w8::stream, which
// stay behind pdl_wait; __ldg would say that it does not change while the kernel runs.
// Every wait is bounded: 2 s for a stage or an accumulator, 4 for a tile's sums (which come
// after those); on expiry a CTA stops, waits up to 2 s more for its copies and MMAs in
// flight, frees its tensor memory, and its rows of y are NaN.
#pragma once
#include <type_traits>

#include "norm.cuh"
#include "pages.cuh"
#include "tc.cuh"

namespace fb2 {

constexpr int W8_K = 128;  // bytes of a stage's rows
constexpr int W8_THREADS = 192, W8_TILE = 128 * W8_K;

struct W8Args {
    const float *x_scales, *w_scales, *bias;
    void* y;
    long long y_row;
    int rows, in, out;
    bool vec;       // rows of y begin on 16 bytes
    int withhold;   // test hook: the k block of block 0 whose copy is left out; -1: none
    unsigned long long wait_ns;
};

namespace w8 {

// A, B signed 8-bit, D 32-bit integers, both operands K-major.
constexpr uint32_t idesc(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
FB2_DEV void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5}, p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
FB2_DEV void ld16(uint32_t at, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
FB2_DEV void prefetch(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }
// Loads that no compiler moves over pdl_wait, as both are volatile: past L1; of what is read once.
FB2_DEV float late(const float* p) {
    float v;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
FB2_DEV int4 late(const int4* p) {
    int4 v;
    asm volatile("ld.global.cg.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
FB2_DEV int4 stream(const int4* p) {
    int4 v;
    asm volatile("ld.global.cs.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
FB2_DEV int peek(uint32_t at, int rank) {
    uint32_t r;
    int v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(r) : "memory");
    return v;
}
FB2_DEV int4 peek4(uint32_t at, int rank) {
    uint32_t r;
    int4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(r) : "memory");
    return v;
}
FB2_DEV float value(int sum, float w_scale, float x_scale, float bias) {
    return fmaf((float)sum * w_scale, x_scale, bias);
}

}  // namespace w8

template <int BN>
struct W8Few {
    static constexpr int STAGE = W8_TILE + BN * W8_K;
    static constexpr int STAGES = (108 * 1024) / STAGE;  // two CTAs to an SM
    static constexpr int PART = BN * 128 * 4;  // sums of a tile
    static constexpr int SMEM = (STAGES * STAGE > PART ? STAGES * STAGE : PART) + 1024;
    static constexpr uint32_t COLS = BN < 32 ? 32 : BN;
};

// blockIdx.x: tile of 128 outputs and, fastest, the CTA's rank in the cluster that
// shares its inputs; blockIdx.y: tile of BN rows of x.
template <class T, int BN>
__global__ void __launch_bounds__(W8_THREADS, 2)
    k_w8_few(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, W8Args a, int ranks) {
    using S = W8Few<BN>;
    extern __shared__ unsigned char w8_raw[];
    __shared__ __align__(8) uint64_t full[S::STAGES], empty[S::STAGES], done;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int s_abort;
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(w8_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % ranks, o0 = blockIdx.x / ranks * 128, r0 = blockIdx.y * BN;
    const int blocks = (a.in + W8_K - 1) / W8_K;
    const int k0 = (int)((long long)blocks * rank / ranks), nk = (int)((long long)blocks * (rank + 1) / ranks) - k0;
    if (tid == 0) {
        w8::prefetch(&map_w), w8::prefetch(&map_x);
        s_abort = 0;
        for (int i = 0; i < S::STAGES; i++) {
            tc::bar_init(&full[i], 1);
            tc::bar_init(&empty[i], 1);
        }
        tc::bar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(&tmem_base)), "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    pdl_wait();

    if (warp == 0 && lane == 0) {
        int i = 0;
        for (; i < nk; i++) {
            const int st = i % S::STAGES;
            if (i >= S::STAGES && !tc::bar_wait(&empty[st], (i / S::STAGES - 1) & 1, &s_abort, a.wait_ns)) break;
            unsigned char* at = sm + st * S::STAGE;
            const bool leave = i == a.withhold && blockIdx.x == 0 && blockIdx.y == 0;
            tc::bar_expect_tx(&full[st], S::STAGE);
            tc::tma_load_2d(at, &map_w, (k0 + i) * W8_K, o0, &full[st]);
            if (leave) break;  // the rest never comes
            tc::tma_load_2d(at + W8_TILE, &map_x, (k0 + i) * W8_K, r0, &full[st]);
        }
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < nk; i++) {
            const int st = i % S::STAGES;
            if (!tc::bar_wait(&full[st], (i / S::STAGES) & 1, &s_abort, a.wait_ns)) break;
            tc::fence_after();
            const uint32_t at = tc::smem_addr(sm + st * S::STAGE);
            const uint64_t w = tc::sw128_desc(at, 16, 1024), x = tc::sw128_desc(at + W8_TILE, 16, 1024);
#pragma unroll
            for (int k = 0; k < W8_K / 32; k++) w8::mma(tmem, w + 2 * k, x + 2 * k, w8::idesc(128, BN), (i | k) != 0);
            tc::mma_commit(&empty[st]);
        }
        tc::mma_commit(&done);
    }
    __syncwarp();
    // all MMAs have completed, with all copies that they read (warp 1 says so after its own
    // waits, whose limit is half of this one's); after an abort the copies in flight land
    // before the ring is used again
    bool ok = tc::bar_try(&done, 0);
    if (!ok) {
        const unsigned long long t0 = tc::now_ns();
        while (!(ok = tc::bar_try(&done, 0)) && tc::now_ns() - t0 < 2 * kTcTimeoutNs) {
        }
        if (!ok) s_abort = 1;
    }
    __syncthreads();
    tc::fence_after();
    const bool failed = s_abort != 0;
    const int quarter = warp & 3;
    const float nan = __uint_as_float(0x7fc00000u);
    T* y = static_cast<T*>(a.y);
    if (failed) {
        // a copy of a stage that never filled may still land: nothing is written there
        if (tid == 0) {
            const unsigned long long t0 = tc::now_ns();
            for (int st = 0; st < S::STAGES && st < nk; st++) {
                const int last = st + (nk - 1 - st) / S::STAGES * S::STAGES;
                while (!tc::bar_try(&full[st], (last / S::STAGES) & 1) && tc::now_ns() - t0 < a.wait_ns) {
                }
            }
        }
        __syncthreads();
    }
    if (ranks == 1) {
        if (warp < 4) {
            const int o = o0 + 32 * quarter + lane;
            const float ws = o < a.out ? w8::late(a.w_scales + o) : 0.f, bias = a.bias && o < a.out ? w8::late(a.bias + o) : 0.f;
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                if (r0 + c >= a.rows) break;
                int v[16];
                w8::ld16(tmem + ((uint32_t)(32 * quarter) << 16) + c, v);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = r0 + c + i;
                    if (r < a.rows && o < a.out)
                        y[r * a.y_row + o] = Dense<T>::put(failed ? nan : w8::value(v[i], ws, w8::late(a.x_scales + r), bias));
                }
            }
        }
    } else {
        int* part = reinterpret_cast<int*>(sm);  // [BN][128]
        __shared__ int s_failed;
        if (tid == 0) s_failed = failed;
        if (warp < 4) {
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                int v[16];
                w8::ld16(tmem + ((uint32_t)(32 * quarter) << 16) + c, v);
#pragma unroll
                for (int i = 0; i < 16; i++) part[(c + i) * 128 + 32 * quarter + lane] = v[i];
            }
        }
        pg::cluster_sync();
        // each CTA sums and writes some of the rows: a warp a row, a lane four outputs
        const bool bad = __any_sync(0xffffffffu, lane < ranks && w8::peek(tc::smem_addr(&s_failed), lane) != 0);
        const int o = o0 + 4 * lane;
        float ws[4], bias[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            ws[j] = o + j < a.out ? w8::late(a.w_scales + o + j) : 0.f;
            bias[j] = a.bias && o + j < a.out ? w8::late(a.bias + o + j) : 0.f;
        }
        const bool whole = a.vec && o + 4 <= a.out && a.out % 4 == 0;
        for (int c = rank + warp * ranks; c < BN && r0 + c < a.rows; c += ranks * (W8_THREADS / 32)) {
            const int r = r0 + c;
            const float xs = w8::late(a.x_scales + r);
            int4 sum = make_int4(0, 0, 0, 0);
            for (int k = 0; k < ranks; k++) {
                const int4 v = w8::peek4(tc::smem_addr(part + c * 128 + 4 * lane), k);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            const int s4[4] = {sum.x, sum.y, sum.z, sum.w};
            T* to = y + r * a.y_row + o;
            __align__(16) T out[4];
#pragma unroll
            for (int j = 0; j < 4; j++) out[j] = Dense<T>::put(bad ? nan : w8::value(s4[j], ws[j], xs, bias[j]));
            if (whole) {
                if constexpr (sizeof(T) == 4)
                    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(out);
                else
                    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(out);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (o + j < a.out) to[j] = out[j];
            }
        }
        pg::cluster_sync();  // the others' shared memory stays until it is read
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
}

// ---- up to four rows, on the integer dot products of the warps ---------------------------
// One launch from x to y.  Each CTA makes the codes of x for itself, in shared memory; a
// lane takes its inputs of them (16 bytes for each row and piece of 512 inputs of a warp)
// into registers and the weights of one output after another against them, W8R_AHEAD
// pieces in flight.  `per_k` warps share an output's inputs; the sums meet in shared
// memory as integers.  The weights' bytes bound it: 1 x 8192 x 28672, bf16, 41 us, 5.7 TB/s
// (on tcgen05 tiles after a launch for the codes 53); 1 x 768 x 2304, fp32, 4.1 us, a
// launch and a chain of loads (7.1).
constexpr int W8R_THREADS = 512, W8R_WARPS = W8R_THREADS / 32, W8R_AHEAD = 8;
constexpr int W8R_SUMS = 3200;       // sums of a CTA: outputs times rows (with the codes below 48 KB)
constexpr int W8R_CODES = 32 * 1024;  // bytes of x's codes: what a lane's registers take of them
template <class X, int ROWS, int PIECES>
constexpr int w8r_resident = sizeof(X) > 1 && ROWS * PIECES == 1 ? 2 : 1;  // CTAs of an SM, by registers

// T: type of y; X: of x, signed char for codes; PIECES: of a lane's inputs; `vec`: rows of
// values can be read 16 bytes at a time
template <class T, class X, int ROWS, int PIECES>
__global__ void __launch_bounds__(W8R_THREADS, w8r_resident<X, ROWS, PIECES>)
    k_w8_rows(W8Args a, const X* x, long long x_row, const signed char* w, long long w_row, int per_k, bool vec) {
    constexpr bool CODES = sizeof(X) == 1;
    constexpr int AHEAD = W8R_AHEAD / PIECES;  // outputs
    extern __shared__ __align__(16) signed char s_code[];  // [ROWS][in, rounded up to 16]
    __shared__ int s_sum[W8R_SUMS];
    __shared__ uint32_t s_top[ROWS][W8R_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slots = W8R_WARPS / per_k, slot = warp / per_k, part = warp % per_k;
    const int o0 = (int)((long long)a.out * blockIdx.x / gridDim.x), o1 = (int)((long long)a.out * (blockIdx.x + 1) / gridDim.x);
    // piece p of the lane: inputs at(p) .. at(p) + 15
    auto at = [&](int p) { return ((part + p * per_k) * 32 + lane) * 16; };
    const long long step = slots * w_row;
    // the weights of a piece; those behind the row's end may be anything, as x is 0 there.
    // What is behind the last row may not be memory: its last piece comes at the end.
    auto weights = [&](int o, const signed char* row, int p) {
        const bool there = at(p) < a.in && (o < a.out - 1 || at(p) + 16 <= a.in);
        return there ? w8::stream(reinterpret_cast<const int4*>(row + at(p))) : make_int4(0, 0, 0, 0);
    };
    for (int i = tid; i < (o1 - o0) * ROWS; i += W8R_THREADS) s_sum[i] = 0;
    pdl_wait();
    int4 held[AHEAD][PIECES];
    const signed char* from = w + (o0 + slot) * w_row;
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
#pragma unroll
        for (int p = 0; p < PIECES; p++)
            if (o0 + slot + u * slots < o1) held[u][p] = weights(o0 + slot + u * slots, from + u * step, p);
    int4 code[ROWS][PIECES];
    float x_scale[ROWS];
    if constexpr (CODES) {
        __syncthreads();  // the sums are 0
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            x_scale[r] = r < a.rows ? w8::late(a.x_scales + r) : 0.f;
#pragma unroll
            for (int p = 0; p < PIECES; p++) {
                code[r][p] = make_int4(0, 0, 0, 0);
                const signed char* xr = (const signed char*)x + r * x_row + at(p);
                if (r < a.rows && at(p) + 16 <= a.in) {
                    code[r][p] = w8::late(reinterpret_cast<const int4*>(xr));
                } else if (r < a.rows && at(p) < a.in) {  // the row ends inside the piece
                    int c[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 15; i++) c[i / 4] |= at(p) + i < a.in ? (xr[i] & 0xff) << (8 * (i & 3)) : 0;
                    code[r][p] = make_int4(c[0], c[1], c[2], c[3]);
                }
            }
        }
    } else {
        const int pad = (a.in + 15) & ~15;
        auto values = [&](int r, int i, float (&v)[NORM_E]) {
            const X* row = x + r * x_row;
            if (vec && i + NORM_E <= a.in) {
                load8(row + i, v);
            } else {
#pragma unroll
                for (int j = 0; j < NORM_E; j++) v[j] = i + j < a.in ? Dense<X>::get(row[i + j]) : 0.f;
            }
        };
        uint32_t top[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) top[r] = 0;
        for (int i = tid * NORM_E; i < a.in; i += W8R_THREADS * NORM_E)
#pragma unroll
            for (int r = 0; r < ROWS; r++)
                if (r < a.rows) {
                    float v[NORM_E];
                    values(r, i, v);
#pragma unroll
                    for (int j = 0; j < NORM_E; j++) top[r] = max(top[r], __float_as_uint(v[j]) & 0x7fffffffu);
                }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            top[r] = __reduce_max_sync(0xffffffffu, top[r]);
            if (lane == 0) s_top[r][warp] = top[r];
        }
        __syncthreads();
        float inv[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) nrm::code_scale(__reduce_max_sync(0xffffffffu, s_top[r][lane % W8R_WARPS]), inv[r], x_scale[r]);
        for (int i = tid * NORM_E; i < pad; i += W8R_THREADS * NORM_E)
#pragma unroll
            for (int r = 0; r < ROWS; r++)
                if (r < a.rows) {
                    float v[NORM_E];
                    values(r, i, v);
                    uint32_t c[2] = {0, 0};
#pragma unroll
                    for (int j = 0; j < NORM_E; j++) c[j / 4] |= nrm::code(v[j], inv[r]) << (8 * (j & 3));
                    *reinterpret_cast<uint2*>(s_code + r * pad + i) = make_uint2(c[0], c[1]);
                }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROWS; r++)
#pragma unroll
            for (int p = 0; p < PIECES; p++)
                code[r][p] = r < a.rows && at(p) < a.in ? *reinterpret_cast<const int4*>(s_code + r * pad + at(p)) : make_int4(0, 0, 0, 0);
    }
    for (int o = o0 + slot; o < o1; o += AHEAD * slots, from += AHEAD * step) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            if (o + u * slots >= o1) break;
            int4 now[PIECES];
#pragma unroll
            for (int p = 0; p < PIECES; p++) {
                now[p] = held[u][p];
                const int next = o + (u + AHEAD) * slots;
                if (next < o1) held[u][p] = weights(next, from + (u + AHEAD) * step, p);
            }
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                int sum = 0;
#pragma unroll
                for (int p = 0; p < PIECES; p++) {
                    sum = __dp4a(now[p].x, code[r][p].x, sum);
                    sum = __dp4a(now[p].y, code[r][p].y, sum);
                    sum = __dp4a(now[p].z, code[r][p].z, sum);
                    sum = __dp4a(now[p].w, code[r][p].w, sum);
                }
                sum = __reduce_add_sync(0xffffffffu, sum);
                if (lane == 0) atomicAdd(&s_sum[(o + u * slots - o0) * ROWS + r], sum);
            }
        }
    }
    if (o1 == a.out && warp < ROWS && warp < a.rows && lane < (a.in & 15)) {  // the last row's last piece
        const int i = (a.in & ~15) + lane;
        const int x_code = CODES ? ((const signed char*)x)[warp * x_row + i] : s_code[warp * ((a.in + 15) & ~15) + i];
        atomicAdd(&s_sum[(o1 - 1 - o0) * ROWS + warp], x_code * w[(o1 - 1) * w_row + i]);
    }
    __syncthreads();
    T* y = static_cast<T*>(a.y);
#pragma unroll
    for (int r = 0; r < ROWS; r++)
        for (int i = tid; r < a.rows && i < o1 - o0; i += W8R_THREADS)
            y[r * a.y_row + o0 + i] = Dense<T>::put(w8::value(s_sum[i * ROWS + r], w8::late(a.w_scales + o0 + i), x_scale[r], a.bias ? w8::late(a.bias + o0 + i) : 0.f));
}

// ---- many rows -------------------------------------------------------------------------
// A pair of CTAs (on the two SMs of a TPC) takes a tile of 256 rows of x by 256 outputs:
// one MMA of both, whose A and B tiles lie half in each one's shared memory, so that a
// stage brings 32 KB to an SM for the products that cost one SM by itself 48 KB.  8192 x
// 4096 x 14336 takes 336 us, 2.87 POP/s (354 with tiles of one CTA): the tensor pipe is
// active for 77 % of the cycles, at the 1.64 GHz that the power limit leaves; the
// operands, 64 bytes a cycle and SM at the pipe's full rate, are what it waits for.
constexpr int W8M_N = 256, W8M_STAGE = 2 * W8_TILE, W8M_STAGES = 6;
constexpr int W8M_SMEM = W8M_STAGES * W8M_STAGE + 1024;
constexpr int W8M_GROUP = 8;  // tiles of rows that are walked together: what runs at a time shares operands in L2

namespace w8 {
FB2_DEV uint32_t at_leader(const void* p) {  // the same place in the pair's first CTA
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_addr(p)));
    return r;
}
// A box into this CTA's memory, counted at the barrier `bar` of the pair's first CTA.
FB2_DEV void load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            tc::smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
FB2_DEV void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
// Arrives at the barrier at this place in both CTAs once the MMAs before are done.
FB2_DEV void commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tc::smem_addr(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
FB2_DEV void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
}  // namespace w8

// Pairs of CTAs walk the tiles.  Warp 0 of each copies its halves, warp 1 of the first
// issues the MMAs into one of two accumulators, warps 2..5 of each bring its rows of the
// other one out: lane r of quarter q is row 32 q + r, its columns are outputs.
template <class T>
__global__ void __launch_bounds__(W8_THREADS, 1)
    k_w8_many(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, W8Args a) {
    extern __shared__ unsigned char w8_raw[];
    // full and taken: the first CTA's count for both
    __shared__ __align__(8) uint64_t full[W8M_STAGES], empty[W8M_STAGES], ready[2], taken[2], drain;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int s_abort;
    __shared__ __align__(16) float s_scale[2][W8M_N], s_bias[2][W8M_N];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(w8_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles_r = (a.rows + 255) / 256, tiles_o = (a.out + W8M_N - 1) / W8M_N;
    const int tiles = tiles_r * tiles_o;
    const int nk = (a.in + W8_K - 1) / W8_K;
    // groups of W8M_GROUP tiles of rows, through all outputs; r0: this CTA's rows
    auto place = [&](int t, int& r0, int& o0) {
        const int group = t / (W8M_GROUP * tiles_o), within = t - group * W8M_GROUP * tiles_o;
        const int high = min(W8M_GROUP, tiles_r - group * W8M_GROUP);
        r0 = (group * W8M_GROUP + within % high) * 256 + 128 * rank;
        o0 = within / high * W8M_N;
    };
    if (tid == 0) {
        w8::prefetch(&map_w), w8::prefetch(&map_x);
        s_abort = 0;
        for (int i = 0; i < W8M_STAGES; i++) {
            tc::bar_init(&full[i], 1);
            tc::bar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            tc::bar_init(&ready[i], 1);
            tc::bar_init(&taken[i], 8);
        }
        tc::bar_init(&drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(&tmem_base)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    pg::cluster_sync();  // both have their barriers and tensor memory
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    pdl_wait();

    if (warp == 0 && lane == 0) {
        uint32_t it = 0;
        bool stop = false;
        for (int t = pair; t < tiles && !stop; t += pairs) {
            int r0, o0;
            place(t, r0, o0);
            for (int i = 0; i < nk; i++, it++) {
                const int st = it % W8M_STAGES;
                if (it >= W8M_STAGES && !tc::bar_wait(&empty[st], (it / W8M_STAGES - 1) & 1, &s_abort, a.wait_ns)) {
                    stop = true;
                    break;
                }
                unsigned char* at = sm + st * W8M_STAGE;
                const uint32_t bar = w8::at_leader(&full[st]);
                if (rank == 0) tc::bar_expect_tx(&full[st], 2 * W8M_STAGE);
                w8::load_pair(at, &map_x, i * W8_K, r0, bar);
                if (blockIdx.x == 0 && (int)it == a.withhold) {
                    stop = true;
                    break;
                }
                w8::load_pair(at + W8_TILE, &map_w, i * W8_K, o0 + 128 * rank, bar);
            }
        }
        // after an abort, copies of both may still be landing, which the first CTA sees
        if (rank == 0 && (s_abort || stop)) {
            const unsigned long long t0 = tc::now_ns();
            for (uint32_t j = it > W8M_STAGES ? it - W8M_STAGES : 0; j <= it; j++)
                while (!tc::bar_try(&full[j % W8M_STAGES], (j / W8M_STAGES) & 1) && tc::now_ns() - t0 < a.wait_ns) {
                }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        uint32_t it = 0, local = 0;
        bool stop = false;
        for (int t = pair; t < tiles && !stop; t += pairs, local++) {
            const uint32_t acc = local & 1;
            if (local >= 2 && !tc::bar_wait(&taken[acc], (local / 2 - 1) & 1, &s_abort, a.wait_ns)) break;
            tc::fence_after();
            for (int i = 0; i < nk; i++, it++) {
                const int st = it % W8M_STAGES;
                if (!tc::bar_wait(&full[st], (it / W8M_STAGES) & 1, &s_abort, a.wait_ns)) {
                    stop = true;
                    break;
                }
                tc::fence_after();
                const uint32_t at = tc::smem_addr(sm + st * W8M_STAGE);
                const uint64_t x = tc::sw128_desc(at, 16, 1024), w = tc::sw128_desc(at + W8_TILE, 16, 1024);
#pragma unroll
                for (int k = 0; k < W8_K / 32; k++)
                    w8::mma_pair(tmem + acc * W8M_N, x + 2 * k, w + 2 * k, w8::idesc(256, W8M_N), (i | k) != 0);
                w8::commit_pair(&empty[st]);
            }
            if (!stop) w8::commit_pair(&ready[acc]);
        }
        // every MMA issued completes before the accumulators are freed
        w8::commit_pair(&drain);
        const unsigned long long t0 = tc::now_ns();
        while (!tc::bar_try(&drain, 0) && tc::now_ns() - t0 < kTcTimeoutNs) {
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, thread = tid - 64;
        const float nan = __uint_as_float(0x7fc00000u);
        T* y = static_cast<T*>(a.y);
        uint32_t local = 0;
        bool failed = false;  // from the first tile that never came on: the rest is NaN
        for (int t = pair; t < tiles; t += pairs, local++) {
            const uint32_t acc = local & 1;
            int r0, o0;
            place(t, r0, o0);
            // the four warps fill the tile's scales; the one before last may still be read
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int i = thread; i < W8M_N; i += 128) {
                const int o = o0 + i;
                s_scale[acc][i] = o < a.out ? w8::late(a.w_scales + o) : 0.f;
                s_bias[acc][i] = a.bias && o < a.out ? w8::late(a.bias + o) : 0.f;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const bool ok = !failed && tc::bar_wait(&ready[acc], (local / 2) & 1, &s_abort, 2 * a.wait_ns);
            failed = !__all_sync(0xffffffffu, ok);
            tc::fence_after();
            const int r = r0 + 32 * quarter + lane;
            const float xs = r < a.rows ? w8::late(a.x_scales + r) : 0.f;
            T* to = y + r * a.y_row + o0;
#pragma unroll 1
            for (int c = 0; c < W8M_N; c += 16) {
                int v[16];
                w8::ld16(tmem + acc * W8M_N + ((uint32_t)(32 * quarter) << 16) + c, v);
                if (r >= a.rows || o0 + c >= a.out) continue;
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 s4 = *reinterpret_cast<const float4*>(&s_scale[acc][c + i]);
                    const float4 b4 = *reinterpret_cast<const float4*>(&s_bias[acc][c + i]);
                    f[i] = w8::value(v[i], s4.x, xs, b4.x), f[i + 1] = w8::value(v[i + 1], s4.y, xs, b4.y);
                    f[i + 2] = w8::value(v[i + 2], s4.z, xs, b4.z), f[i + 3] = w8::value(v[i + 3], s4.w, xs, b4.w);
                }
                if (failed) {
#pragma unroll
                    for (int i = 0; i < 16; i++) f[i] = nan;
                }
                if (a.vec && o0 + c + 16 <= a.out) {
                    constexpr int N = 16 / sizeof(T);
#pragma unroll
                    for (int i = 0; i < 16; i += N) *reinterpret_cast<uint4*>(to + c + i) = pack16<T>(f + i);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (o0 + c + i < a.out) to[c + i] = Dense<T>::put(f[i]);
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) w8::arrive_at(w8::at_leader(&taken[acc]));
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    pg::cluster_sync();  // neither ends or frees while the other's MMAs or copies go on
    if (warp == 0) {
        tc::fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// W [in][out] as codes [out][in] with a scale for each output: a warp's lanes take 32
// neighbouring outputs, 8 warps the inputs in turns; codes go through shared memory,
// so that both sides are read and written in runs.  Once for a model's weights, and far from
// the bytes' time, as few CTAs read W twice with a load at a time: 4096 x 14336 fp32 306 us
// (bytes 45), bf16 355, 8192 x 28672 714 and 788.
constexpr int W8P_THREADS = 256;
template <class T>
__global__ void __launch_bounds__(W8P_THREADS) k_w8_pack(const T* w, long long w_row, int in, int out, signed char* codes, long long code_row,
                                                         float* scales) {
    __shared__ uint32_t s_top[8][32];
    __shared__ signed char s_code[32][128 + 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, o0 = blockIdx.x * 32, o = o0 + lane;
    uint32_t top = 0;
    if (o < out)
        for (int i = warp; i < in; i += 8) top = max(top, __float_as_uint(Dense<T>::get(w[i * w_row + o])) & 0x7fffffffu);
    s_top[warp][lane] = top;
    __syncthreads();
    for (int k = 0; k < 8; k++) top = max(top, s_top[k][lane]);
    float inv, scale;
    nrm::code_scale(top, inv, scale);
    if (warp == 0 && o < out) scales[o] = scale;
    for (int i0 = 0; i0 < in; i0 += 128) {
        __syncthreads();
        for (int i = warp; i < 128; i += 8)
            s_code[lane][i] = o < out && i0 + i < in ? (signed char)nrm::code(Dense<T>::get(w[(i0 + i) * w_row + o]), inv) : 0;
        __syncthreads();
        for (int k = threadIdx.x; k < 32 * 128; k += W8P_THREADS) {
            const int to = o0 + k / 128, i = i0 + k % 128;
            if (to < out && i < in) codes[to * code_row + i] = s_code[k / 128][k % 128];
        }
    }
}

}  // namespace fb2
