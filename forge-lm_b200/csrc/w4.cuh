// w4.cuh — linear layers with 4-bit weights and a scale and minimum for each
// output and group of inputs: packing, and products with few rows.
//
// y[m][n] = sum_g (scale[g][n] * sum_{k in g} code[k][n] x[m][k]
//                  + min[g][n] * sum_{k in g} x[m][k]) + bias[n]
// Blocks of 16 outputs x 64 inputs, 32 lanes x 4 words: nibble p of word j of
// lane 4g + t is output 8 (p & 1) + g, input 16 t + 4 j + (p & 2) + (p >> 2).
#pragma once
#include <cstring>

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

// ---- products ------------------------------------------------------------------
//
// The weights are the 16-row side of mma.sync tiles (16 outputs x 16 inputs),
// the rows of x its columns, so a block's 512 bytes (one 16-byte load per
// lane) go through the tensor cores once for 8 columns.  The codes enter as
// fp16 or bf16 values that one shift and one logical operation make of four
// bits; a group's sum and the sum of its x (k_w4_columns adds it up) then
// give scale * sum(code x) + minimum * sum(x) in fp32:
//   bf16 x: 128 + code (bit pattern 0x4300 | code);
//   fp16 x: 1 + code / 16 (0x3c00 | code << 6);
//   fp32 x: three bf16 terms that add up to x exactly, in three columns, and
//           code - 8, as no offset may cost fp32 sums their last bits.
// For the 16-bit types the offset costs 8 bits at most of fp32 sums that are
// rounded to 8 or 11 bits: of 61 bf16 rows x 1024 x 16384, one value in a thousand
// is not the rounding of the exact one (one in ten thousand with code - 8, which
// takes 18.5 us for 17.8), and values 100 times below the rest are as exact.
namespace w4 {

FB2_DEV void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
FB2_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

FB2_DEV void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// c = a b + z for the first product of a sum
template <bool BF16>
FB2_DEV void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// What a type of x needs: columns per row, the four fragment words of a word
// of codes, ones, and the scale and minimum that go with the codes' values.
template <class T>
struct Form;
template <>
struct Form<__nv_bfloat16> {
    static constexpr bool BF16 = true;
    static constexpr int PARTS = 1;
    static FB2_DEV void codes(uint32_t w, uint32_t (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    }
    static FB2_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
    static FB2_DEV float2 affine(uint32_t m) {
        const float s = bf16_bits_to_float(m & 0xffffu);
        return make_float2(s, fmaf(-128.0f, s, __uint_as_float(m & 0xffff0000u)));
    }
    static FB2_DEV float sum_of(uint32_t v) { return __uint_as_float(v << 16) + __uint_as_float(v & 0xffff0000u); }
    static FB2_DEV uint32_t pair(const __nv_bfloat16* x, int) { return (uint32_t)__bfloat16_as_ushort(x[0]) | (uint32_t)__bfloat16_as_ushort(x[1]) << 16; }
};
template <>
struct Form<__half> {
    static constexpr bool BF16 = false;
    static constexpr int PARTS = 1;
    static FB2_DEV void codes(uint32_t w, uint32_t (&f)[4]) {
        f[0] = ((w << 6) & 0x03c003c0u) | 0x3c003c00u;
        f[1] = ((w << 2) & 0x03c003c0u) | 0x3c003c00u;
        f[2] = ((w >> 2) & 0x03c003c0u) | 0x3c003c00u;
        f[3] = ((w >> 6) & 0x03c003c0u) | 0x3c003c00u;
    }
    static FB2_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_f16(c, a, b0, b1); }
    static FB2_DEV float2 affine(uint32_t m) {
        const float s = 16.0f * bf16_bits_to_float(m & 0xffffu);
        return make_float2(s, __uint_as_float(m & 0xffff0000u) - s);
    }
    static FB2_DEV float sum_of(uint32_t v) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
        return f.x + f.y;
    }
    static FB2_DEV uint32_t pair(const __half* x, int) { return (uint32_t)__half_as_ushort(x[0]) | (uint32_t)__half_as_ushort(x[1]) << 16; }
};
template <>
struct Form<float> {
    static constexpr bool BF16 = true;
    static constexpr int PARTS = 3;
    static FB2_DEV void codes(uint32_t w, uint32_t (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(f[i]) : "r"(v), "r"(0x43084308u));  // - 136
        }
    }
    static FB2_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
    static FB2_DEV float2 affine(uint32_t m) {
        const float s = bf16_bits_to_float(m & 0xffffu);
        return make_float2(s, fmaf(8.0f, s, __uint_as_float(m & 0xffff0000u)));
    }
    static FB2_DEV float sum_of(uint32_t v) { return __uint_as_float(v << 16) + __uint_as_float(v & 0xffff0000u); }
    // term `part` of the exact split x = t0 + t1 + t2 into bf16 values
    static FB2_DEV float term(float x, int part) {
        const float t0 = __bfloat162float(__float2bfloat16_rn(x));
        if (part == 0) return t0;
        const float r = x - t0, t1 = __bfloat162float(__float2bfloat16_rn(r));
        return part == 1 ? t1 : r - t1;
    }
    static FB2_DEV uint32_t pair(const float* x, int part) {
        return float_to_bf16_bits(term(x[0], part)) | float_to_bf16_bits(term(x[1], part)) << 16;
    }
};

// A group of 32 inputs is half of a block: the lanes t < 2 hold the first, the
// others the second.  Two steps' words are exchanged between lanes t and t ^ 2
// so that step 0 has the first group's inputs in all lanes and step 1 the
// second's (for codes and for x alike).
FB2_DEV void by_group(uint32_t& w0, uint32_t& w1) {
    const bool low = (threadIdx.x & 2) == 0;
    const uint32_t v = __shfl_xor_sync(0xffffffffu, low ? w1 : w0, 2);
    if (low)
        w1 = v;
    else
        w0 = v;
}

// Lane (g, t)'s 16 values of one column for a block of 64 inputs: inputs
// k0 .. k0 + 15, k0 = 16 t in it, as the B fragments of its four steps.
template <class T>
FB2_DEV void column(const T* __restrict__ x, long long x_row, int row, int part, bool live, int k0, int K, bool vec,
                    uint32_t (&f)[8]) {
    const T* p = x + row * x_row + k0;
    if (sizeof(T) == 2 && live && vec && k0 + 16 <= K) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p)), v = __ldg(reinterpret_cast<const uint4*>(p) + 1);
        f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = v.x, f[5] = v.y, f[6] = v.z, f[7] = v.w;
        return;
    }
    T v[16];
    if (sizeof(T) == 4 && live && vec && k0 + 16 <= K) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
            memcpy(reinterpret_cast<char*>(v) + 16 * i, &u, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = live && k0 + i < K ? p[i] : Dense<T>::put(0.f);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = Form<T>::pair(v + 2 * i, part);
}

FB2_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
FB2_DEV uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
FB2_DEV uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
FB2_DEV float cluster_ld(uint32_t at, uint32_t rank) {
    uint32_t there;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there));
    return v;
}

// A unit of the loops: 128 inputs (two blocks) of one block of 16 outputs,
// 1024 bytes of codes and up to 256 of meta words, as it lies in shared memory.
constexpr int UNIT = 1280;

// Starts the copy of unit `u` of output block `block`; blocks and groups past
// the end are filled with zeros.
FB2_DEV void fetch_unit(const W4View& w, int block, int u, uint32_t to, int lane) {
    const uint4* from = w.codes + ((size_t)block * w.k64 + 2 * u) * 32 + lane;
    copy16(to + lane * 16, from, true);
    const bool second = 2 * u + 1 < w.k64;
    copy16(to + 512 + lane * 16, second ? from + 32 : from, second);
    const int per = 128 >> w.group_shift;  // groups of a unit
    if (lane < per * 4) {
        const int grp = u * per + (lane >> 2);
        const bool there = grp < w.groups;
        copy16(to + 1024 + lane * 16, w.meta + ((size_t)block * w.groups + (there ? grp : 0)) * 16 + (lane & 3) * 4, there);
    }
}

// The group sums of a unit: acc, xs -> sum, with the group's scale and minimum.
template <class T, int NT>
FB2_DEV void close_group(uint32_t meta, int grp, int g, const float (&acc)[NT][4], const float (&xs)[NT][4], float (&sum)[NT][4]) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const float2 sm = Form<T>::affine(lds(meta + grp * 64 + (half * 8 + g) * 4));
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float& s = sum[n][2 * half + c];
                s = fmaf(sm.x, acc[n][2 * half + c], fmaf(sm.y, xs[n][c], s));
            }
    }
}

// Adds the cluster's CTAs' sums own[out][COLS + 1] (OUT outputs from n0 on, P
// columns to a row) for every row and writes y; each CTA of the cluster takes its share.
template <class T, int OUT, int COLS, int P, int THREADS>
FB2_DEV void finish(const W4View& w, const float* own, int n0, int rows, T* __restrict__ y, long long y_row) {
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    if (ranks > 1)
        cluster_sync();
    else
        __syncthreads();
    constexpr int LD = COLS + 1;  // rows apart by an odd number: no bank conflicts down a column
    const uint32_t at0 = (uint32_t)__cvta_generic_to_shared(own);
    for (int i = threadIdx.x + (int)rank * THREADS; i < rows * OUT; i += THREADS * (int)ranks) {
        const int row = i / OUT, out = i - row * OUT, n = n0 + out, at = out * LD + row * P;
        float s = 0.f;
        if (ranks == 1) {
#pragma unroll
            for (int p = 0; p < P; p++) s += own[at + p];
        } else {
            float v[8][P];  // all loads before the first sum
#pragma unroll
            for (int q = 0; q < 8; q++)
#pragma unroll
                for (int p = 0; p < P; p++) v[q][p] = q < ranks ? cluster_ld(at0 + (at + p) * 4u, q) : 0.f;
#pragma unroll
            for (int q = 0; q < 8; q++)
#pragma unroll
                for (int p = 0; p < P; p++) s += v[q][p];
        }
        if (n < w.N) y[row * y_row + n] = Dense<T>::put(s + (w.bias ? __ldg(w.bias + n) : 0.f));
    }
    if (ranks > 1) cluster_sync();  // nobody leaves while its sums are still read
}

}  // namespace w4

// x for the 16-bit tiles, in fragment order: [chunk of `per` rows][unit of 128
// inputs][2 blocks of 64][tile of 8 columns][2 steps' half][lane] 4 words; and the sums
// of x over the groups, [chunk][unit][group][column].
template <class T>
__global__ void __launch_bounds__(128)
    k_w4_columns(const T* __restrict__ x, long long x_row, int rows, int per, int K, int units, int tiles, int chunks,
                 int group_shift, uint4* __restrict__ to, float* __restrict__ sums, int vec) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the product fetches its first codes meanwhile
    const long long at = ((long long)blockIdx.x * 128 + threadIdx.x) >> 5;  // (chunk, unit, tile)
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (at >= (long long)chunks * units * tiles) return;
    const long long cu = at / tiles;
    const int tile = (int)(at - cu * tiles), chunk = (int)(cu / units), u = (int)(cu - (long long)chunk * units);
    constexpr int P = w4::Form<T>::PARTS;
    const int col = tile * 8 + g, in = col / P, row = chunk * per + in;
    const bool live = in < per && row < rows;
    float part[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
        uint32_t f[8];
        w4::column<T>(x, x_row, row, col - in * P, live, u * 128 + b * 64 + 16 * t, K, vec, f);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) s += w4::Form<T>::sum_of(f[i]);
        part[b] = s;
        const bool by32 = group_shift == 5;
        if (by32) {
            w4::by_group(f[0], f[2]);
            w4::by_group(f[1], f[3]);
            w4::by_group(f[4], f[6]);
            w4::by_group(f[5], f[7]);
        }
        uint4* out = to + ((cu * 2 + b) * tiles + tile) * 64 + lane;  // a group's two steps together
        out[0] = by32 ? make_uint4(f[0], f[1], f[4], f[5]) : make_uint4(f[0], f[1], f[2], f[3]);
        out[32] = by32 ? make_uint4(f[2], f[3], f[6], f[7]) : make_uint4(f[4], f[5], f[6], f[7]);
    }
    // over the lanes of a group: 2 of a block, all 4, or both blocks
    part[0] += __shfl_xor_sync(0xffffffffu, part[0], 1);
    part[1] += __shfl_xor_sync(0xffffffffu, part[1], 1);
    if (group_shift > 5) {
        part[0] += __shfl_xor_sync(0xffffffffu, part[0], 2);
        part[1] += __shfl_xor_sync(0xffffffffu, part[1], 2);
    }
    float* out = sums + cu * (128 >> group_shift) * tiles * 8 + col;
    if (group_shift == 7) {
        if (t == 0) out[0] = part[0] + part[1];
    } else if (group_shift == 6) {
        if (t < 2) out[t * tiles * 8] = t ? part[1] : part[0];
    } else {
        // lanes 0, 2: the first block's groups; 1, 3: the second's
        out[(2 * (t & 1) + (t >> 1)) * tiles * 8] = t & 1 ? part[1] : part[0];
    }
}

// ---- few rows: 8-bit integer tiles ------------------------------------------------
//
// With few columns the weights' way through the registers bounds the product,
// and the cheapest operand that codes can be made into is bytes: four of them
// per logical operation, for mma.sync tiles of 16 outputs x 32 inputs with
// exact 32-bit integer sums (measured here: the same rate as the 16-input fp16
// tiles).  x is written in fixed point for that: over each unit of 128 inputs,
// q = rint(x 2^(22 - e)) with |x| <= 2^e (16-bit types: 3 digits of 8 bits;
// fp32: 2^(30 - e), 4 digits), one column for each digit in -128..127.  What q
// drops is below 2^-23 (2^-31) of the unit's largest |x|.
//
// One row x 16384 x 16384, groups of 128, bf16: 29.3 us, 4.9 TB/s of codes and
// meta words (on the fp32 cores: 354); 8192 x 57344: 46.3 us, 5.4 TB/s; below
// some 4096 x 4096 (5.8 us) the two launches and their chains are most of it,
// 768 x 2304 in fp32 takes 3.2 with one.

// One column of a unit in lane (g, t): digit `digit` of the 32 inputs
// 64 b + 16 t + i of row `row`, as the B words f[4 b + j] of inputs
// 16 t + 4 j + (0, 2, 1, 3); the digit's weight; and the sums of x over the
// groups of the unit (sum[0..3]; one value for 128, two for 64).
template <class T>
FB2_DEV void w4_digits(const T* __restrict__ x, long long x_row, int row, int digit, bool live, int k0, int K, bool vec,
                       int group_shift, uint32_t (&f)[8], float& weight, float (&sum)[4]) {
    constexpr int D = sizeof(T) == 4 ? 4 : 3, TOP = sizeof(T) == 4 ? 30 : 22;
    const int t = threadIdx.x & 3;
    float v[32], part[2];
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int k = k0 + 64 * b + 16 * t;
        const T* p = x + row * x_row + k;
        if (live && vec && k + 16 <= K) {
            float a[8];
            load8<T>(p, a);
#pragma unroll
            for (int i = 0; i < 8; i++) v[16 * b + i] = a[i];
            load8<T>(p + 8, a);
#pragma unroll
            for (int i = 0; i < 8; i++) v[16 * b + 8 + i] = a[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[16 * b + i] = live && k + i < K ? Dense<T>::get(p[i]) : 0.f;
        }
        part[b] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            part[b] += v[16 * b + i];
            top = fmaxf(top, fabsf(v[16 * b + i]));
        }
    }
    // 2^e > the row's largest |x| in the unit; a NaN or inf makes the sums,
    // and with them the row's results, non-finite
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max((int)(__float_as_uint(top) >> 23) - 126, -95);  // the scale must be finite
    const bool finite = top < INFINITY;
    const float scale = __uint_as_float((uint32_t)(127 + TOP - e) << 23);
    weight = finite ? __uint_as_float((uint32_t)(127 - TOP + e + 8 * digit) << 23) : 0.f;
    constexpr uint32_t BIAS = D == 4 ? 0x80808080u : 0x00808080u;
    const uint32_t pick = 0x0040u + 0x0011u * digit;  // byte `digit` of each of two words
#pragma unroll
    for (int i = 0; i < 8; i++) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) q[j] = finite ? (uint32_t)__float2int_rn(v[4 * i + j] * scale) + BIAS : BIAS;
        const uint32_t a = __byte_perm(q[0], q[2], pick), c = __byte_perm(q[1], q[3], pick);
        f[i] = __byte_perm(a, c, 0x5410) ^ 0x80808080u;
    }
    part[0] += __shfl_xor_sync(0xffffffffu, part[0], 1);
    part[1] += __shfl_xor_sync(0xffffffffu, part[1], 1);
    const float o0 = __shfl_xor_sync(0xffffffffu, part[0], 2), o1 = __shfl_xor_sync(0xffffffffu, part[1], 2);
    const bool low = t < 2;
    sum[0] = low ? part[0] : o0, sum[1] = low ? o0 : part[0];
    sum[2] = low ? part[1] : o1, sum[3] = low ? o1 : part[1];
    if (group_shift > 5) sum[0] += sum[1], sum[1] = sum[2] + sum[3];
    if (group_shift > 6) sum[0] += sum[1];
    if (digit != 0)  // once per row
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] = 0.f;
    if (group_shift == 5) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            w4::by_group(f[i], f[i + 1]);
            w4::by_group(f[i + 2], f[i + 3]);
            const uint32_t m = f[i + 1];  // a group's two words together
            f[i + 1] = f[i + 2];
            f[i + 2] = m;
        }
    }
}

// The columns of a unit in the products' order: [unit][tile of 8 columns]
// 1024 bytes of B words ([block of 64][lane] 4 words), 8 weights, 4 x 8 group sums.
constexpr int W4_COL = 1024 + 32 + 128;

template <class T>
__global__ void __launch_bounds__(128)
    k_w4_digits(const T* __restrict__ x, long long x_row, int rows, int K, int units, int tiles, int group_shift,
                unsigned char* __restrict__ to, int vec) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the product fetches its first codes meanwhile
    const long long at = ((long long)blockIdx.x * 128 + threadIdx.x) >> 5;
    if (at >= (long long)units * tiles) return;
    constexpr int D = sizeof(T) == 4 ? 4 : 3;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int u = (int)(at / tiles), tile = (int)(at - (long long)u * tiles), col = tile * 8 + g, row = col / D;
    uint32_t f[8];
    float weight, sum[4];
    w4_digits<T>(x, x_row, row, col - row * D, row < rows, u * 128, K, vec, group_shift, f, weight, sum);
    unsigned char* out = to + at * W4_COL;
    reinterpret_cast<uint4*>(out)[lane] = make_uint4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<uint4*>(out)[lane + 32] = make_uint4(f[4], f[5], f[6], f[7]);
    float* tail = reinterpret_cast<float*>(out + 1024);
    if (t == 0) tail[g] = weight;
    tail[8 + t * 8 + g] = t == 0 ? sum[0] : t == 1 ? sum[1] : t == 2 ? sum[2] : sum[3];
}

// A CTA: RT blocks of 16 outputs; its 8 warps (and the CTAs of its cluster)
// take every 8th (8 * cluster) unit of 128 inputs.  Each warp keeps DEPTH
// units in flight in a ring of its own in shared memory (cp.async: no
// registers, no barrier), and all add up at the end, in a fixed order.
// DIRECT: the warp makes the digits itself (NT = 1); else k_w4_digits has.
constexpr int W4_WARPS = 8;

template <int RT, int NT, bool DIRECT>
struct W4Narrow {
    static constexpr int DEPTH = RT == 1 && NT == 1 ? 4 : 2;
    static constexpr int SLOT = RT * w4::UNIT + (DIRECT ? 0 : NT * W4_COL);
    static constexpr int RING = W4_WARPS * DEPTH * SLOT;
    static constexpr int RED = (W4_WARPS * 8 * NT + 8 * NT + 1) * RT * 16 * 4;
    static constexpr int SMEM = RING > RED ? RING : RED;
};

template <class T, int RT, int NT, bool DIRECT>
__global__ void __launch_bounds__(W4_WARPS * 32, 2)
    k_w4_narrow(W4View w, const T* __restrict__ x, long long x_row, const unsigned char* __restrict__ columns, int rows,
                T* __restrict__ y, long long y_row, int vec) {
    using S = W4Narrow<RT, NT, DIRECT>;
    constexpr int D = sizeof(T) == 4 ? 4 : 3;
    extern __shared__ __align__(16) unsigned char w4_smem[];
    constexpr int COLS = 8 * NT, OUT = RT * 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)w4::cluster_rank(), ranks = (int)w4::cluster_size();
    const int block0 = (int)blockIdx.x / ranks * RT, blocks = (w.N + 15) >> 4;
    const int units = (w.k64 + 1) >> 1, stride = W4_WARPS * ranks;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(w4_smem) + warp * S::DEPTH * S::SLOT;

    float sum[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) sum[r][n][c] = 0.f;
    int u = rank * W4_WARPS + warp, ahead = u, slot = 0, fill = 0;
    auto fetch_codes = [&](int unit, int to) {
        if (unit < units)
#pragma unroll
            for (int r = 0; r < RT; r++)
                w4::fetch_unit(w, min(block0 + r, blocks - 1), unit, ring + to * S::SLOT + r * w4::UNIT, lane);
    };
    auto fetch_x = [&](int unit, int to) {
        if (DIRECT || unit >= units) return;
        const unsigned char* from = columns + (size_t)unit * (NT * W4_COL);
#pragma unroll
        for (int i = 0; i < NT * W4_COL / 16; i += 32)
            if (i + lane < NT * W4_COL / 16)
                copy16(ring + to * S::SLOT + RT * w4::UNIT + (i + lane) * 16, from + (i + lane) * 16, true);
    };
    // the first units' codes before the columns are there
#pragma unroll
    for (int i = 0; i < S::DEPTH - 1; i++) fetch_codes(u + i * stride, i);
    if constexpr (!DIRECT) pdl_wait();
#pragma unroll
    for (int i = 0; i < S::DEPTH - 1; i++) {
        fetch_x(u + i * stride, i);
        copies_commit();
    }
    ahead = u + (S::DEPTH - 1) * stride, fill = S::DEPTH - 1;
    for (; u < units; u += stride) {
        __syncwarp();  // every lane is done with the slot that is filled next
        fetch_codes(ahead, fill);
        fetch_x(ahead, fill);
        copies_commit();
        ahead += stride;
        fill = fill + 1 == S::DEPTH ? 0 : fill + 1;
        uint32_t xf[NT][8];
        float2 weight[NT];
        float own_weight, own_sum[4];
        if constexpr (DIRECT) {
            const int row = g / D;
            w4_digits<T>(x, x_row, row, g - row * D, row < rows, u * 128, w.K, vec, w.group_shift, xf[0], own_weight, own_sum);
            weight[0] = make_float2(__shfl_sync(0xffffffffu, own_weight, 8 * t), __shfl_sync(0xffffffffu, own_weight, 8 * t + 4));
        }
        copies_wait<S::DEPTH - 1>();
        __syncwarp();
        const uint32_t at = ring + slot * S::SLOT, xat = at + RT * w4::UNIT;
        slot = slot + 1 == S::DEPTH ? 0 : slot + 1;
        if constexpr (!DIRECT)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 a = lds4(xat + n * W4_COL + lane * 16), b = lds4(xat + n * W4_COL + 512 + lane * 16);
                xf[n][0] = a.x, xf[n][1] = a.y, xf[n][2] = a.z, xf[n][3] = a.w;
                xf[n][4] = b.x, xf[n][5] = b.y, xf[n][6] = b.z, xf[n][7] = b.w;
                weight[n] = lds2(xat + n * W4_COL + 1024 + 8 * t);
            }
        // integer sums start at the bits of 1.5 2^23: below 2^22 in size, they
        // are then the bits of 1.5 2^23 + sum
        constexpr int ZERO = 0x4b400000;
        constexpr float ZERO_F = 12582912.0f;
        int acc[RT][NT][4];
        auto clear = [&]() {
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[r][n][c] = ZERO;
        };
        auto step = [&](int r, uint32_t w0, uint32_t w1, int i) {
            const uint32_t a0 = w0 & 0x0f0f0f0fu, a1 = (w0 >> 4) & 0x0f0f0f0fu, a2 = w1 & 0x0f0f0f0fu, a3 = (w1 >> 4) & 0x0f0f0f0fu;
#pragma unroll
            for (int n = 0; n < NT; n++) w4::mma_u8s8(acc[r][n], a0, a1, a2, a3, xf[n][2 * i], xf[n][2 * i + 1]);
        };
        auto close = [&](int grp) {
            float2 xs[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if constexpr (DIRECT) {
                    xs[n].x = __shfl_sync(0xffffffffu, own_sum[grp], 8 * t);
                    xs[n].y = __shfl_sync(0xffffffffu, own_sum[grp], 8 * t + 4);
                } else {
                    xs[n] = lds2(xat + n * W4_COL + 1056 + grp * 32 + 8 * t);
                }
            }
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint32_t m = lds(at + r * w4::UNIT + 1024 + grp * 64 + (half * 8 + g) * 4);
                    const float s = bf16_bits_to_float(m & 0xffffu), low = __uint_as_float(m & 0xffff0000u);
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float& to = sum[r][n][2 * half + c];
                            const float a = __int_as_float(acc[r][n][2 * half + c]) - ZERO_F;
                            to = fmaf(s * (c ? weight[n].y : weight[n].x), a, fmaf(low, c ? xs[n].y : xs[n].x, to));
                        }
                }
        };
        clear();
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint4 word[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) word[r] = lds4(at + r * w4::UNIT + b * 512 + lane * 16);
            if (w.group_shift == 5) {
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    w4::by_group(word[r].x, word[r].y);
                    w4::by_group(word[r].z, word[r].w);
                    step(r, word[r].x, word[r].z, 2 * b);
                }
                close(2 * b);
                clear();
#pragma unroll
                for (int r = 0; r < RT; r++) step(r, word[r].y, word[r].w, 2 * b + 1);
                close(2 * b + 1);
                clear();
            } else {
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    step(r, word[r].x, word[r].y, 2 * b);
                    step(r, word[r].z, word[r].w, 2 * b + 1);
                }
                if (w.group_shift == 6) {
                    close(b);
                    clear();
                } else if (b == 1) {
                    close(0);
                }
            }
        }
    }
    copies_wait<0>();
    __syncthreads();  // the rings are done with
    float* red = reinterpret_cast<float*>(w4_smem);  // [warp][OUT][COLS], then the CTA's sums
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int half = 0; half < 2; half++)
                *reinterpret_cast<float2*>(red + ((warp * OUT + r * 16 + half * 8 + g) * COLS + 8 * n + 2 * t)) =
                    make_float2(sum[r][n][2 * half], sum[r][n][2 * half + 1]);
    __syncthreads();
    float* own = red + W4_WARPS * OUT * COLS;
    for (int i = threadIdx.x; i < OUT * COLS; i += W4_WARPS * 32) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < W4_WARPS; v++) s += red[v * OUT * COLS + i];
        own[i / COLS * (COLS + 1) + i % COLS] = s;
    }
    w4::finish<T, OUT, COLS, D, W4_WARPS * 32>(w, own, block0 * 16, rows, y, y_row);
}

// ---- more rows: 16-bit tiles --------------------------------------------------------
//
// A CTA: each of its 8 warps one block of 16 outputs, for one chunk of 8 NT
// columns (blockIdx.y); the units of 128 inputs go round the CTAs of
// the cluster.  A unit's x (in fragment order, with its group sums) is staged
// once for the CTA, next to the warps' codes, DEPTH units deep.  Instructions
// bound it: 16 for each tile product with groups of 32, of which 4 apply the
// groups' scales and minimums and 2 make fp16 of codes.  61 rows x 1024 x
// 16384, groups of 32, fp16: 18.2 us, of them 3 before it starts; 113 TFLOP/s.
template <int NT>
struct W4Wide {
    static constexpr int DEPTH = 3;
    static constexpr int X = 2 * NT * 1024, SUMS = 4 * NT * 32;
    static constexpr int STAGE = X + SUMS + W4_WARPS * w4::UNIT;
    static constexpr int OUT = W4_WARPS * 16;
    static constexpr int RED = OUT * (8 * NT + 1) * 4;
    static constexpr int SMEM = DEPTH * STAGE > RED ? DEPTH * STAGE : RED;
};

template <class T, int NT, int GS>
__global__ void __launch_bounds__(W4_WARPS * 32, 2)
    k_w4_wide(W4View w, const uint4* __restrict__ columns, const float* __restrict__ sums, int rows, int per, T* __restrict__ y,
              long long y_row) {
    using F = w4::Form<T>;
    using S = W4Wide<NT>;
    extern __shared__ __align__(16) unsigned char w4_smem[];
    constexpr int GROUPS = 128 >> GS;  // of a unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)w4::cluster_rank(), ranks = (int)w4::cluster_size();
    const int cta0 = (int)blockIdx.x / ranks * W4_WARPS, block = min(cta0 + warp, ((w.N + 15) >> 4) - 1);
    const int units = (w.k64 + 1) >> 1, row0 = blockIdx.y * per;
    const uint32_t smem = (uint32_t)__cvta_generic_to_shared(w4_smem);

    auto fetch_codes = [&](int u, int st) {
        if (u < units) w4::fetch_unit(w, block, u, smem + st * S::STAGE + S::X + S::SUMS + warp * w4::UNIT, lane);
    };
    auto fetch_x = [&](int u, int st) {
        if (u >= units) return;
        const size_t cu = (size_t)blockIdx.y * units + u;
        const uint32_t to = smem + st * S::STAGE;
        const uint4* from = columns + cu * (S::X / 16);
#pragma unroll
        for (int i = 0; i < S::X / 16; i += W4_WARPS * 32) copy16(to + (i + threadIdx.x) * 16, from + i + threadIdx.x, true);
        if (threadIdx.x < GROUPS * NT * 2)
            copy16(to + S::X + threadIdx.x * 16, sums + cu * (GROUPS * NT * 8) + threadIdx.x * 4, true);
    };

    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) sum[n][c] = 0.f;
    // codes of the first stages before the columns are there
#pragma unroll
    for (int i = 0; i < S::DEPTH - 1; i++) fetch_codes(rank + i * ranks, i);
    pdl_wait();
#pragma unroll
    for (int i = 0; i < S::DEPTH - 1; i++) {
        fetch_x(rank + i * ranks, i);
        copies_commit();
    }
    int slot = 0;
    for (int u = rank; u < units; u += ranks) {
        copies_wait<S::DEPTH - 2>();
        __syncthreads();  // the unit is there for all, and all are done with the stage that is filled next
        {
            const int ahead = u + (S::DEPTH - 1) * ranks, st = slot == 0 ? S::DEPTH - 1 : slot - 1;
            fetch_codes(ahead, st);
            fetch_x(ahead, st);
            copies_commit();
        }
        const uint32_t xat = smem + slot * S::STAGE, sat = xat + S::X, cat = sat + S::SUMS + warp * w4::UNIT;
        slot = slot + 1 == S::DEPTH ? 0 : slot + 1;
        float acc[NT][4];
        auto close = [&](int grp) {
            float xs[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float2 v = lds2(sat + (grp * NT * 8 + n * 8 + 2 * t) * 4);
                xs[n][0] = v.x, xs[n][1] = v.y;
            }
            w4::close_group<T, NT>(cat + 1024, grp, g, acc, xs, sum);
        };
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint4 words = lds4(cat + b * 512 + lane * 16);
            uint32_t word[4] = {words.x, words.y, words.z, words.w};
            if constexpr (GS == 5) {
                w4::by_group(word[0], word[1]);
                w4::by_group(word[2], word[3]);
            }
            // two steps at a time, those of one group: 0, 2 and 1, 3 for groups of 32
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t f[2][4];
                F::codes(word[GS == 5 ? h : 2 * h], f[0]);
                F::codes(word[GS == 5 ? 2 + h : 2 * h + 1], f[1]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 v = lds4(xat + ((b * NT + n) * 2 + h) * 512 + lane * 16);
                    if (GS == 5 || (h == 0 && (b == 0 || GS == 6)))
                        w4::mma_first<F::BF16>(acc[n], f[0], v.x, v.y);
                    else
                        F::mma(acc[n], f[0], v.x, v.y);
                    F::mma(acc[n], f[1], v.z, v.w);
                }
                if constexpr (GS == 5) close(2 * b + h);
            }
            if constexpr (GS == 6) close(b);
        }
        if constexpr (GS == 7) close(0);
    }
    copies_wait<0>();
    __syncthreads();
    float* own = reinterpret_cast<float*>(w4_smem);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++)
            own[(warp * 16 + (c >> 1) * 8 + g) * (8 * NT + 1) + 8 * n + 2 * t + (c & 1)] = sum[n][c];
    w4::finish<T, S::OUT, 8 * NT, F::PARTS, W4_WARPS * 32>(w, own, cta0 * 16, min(per, rows - row0), y + row0 * y_row, y_row);
}

}  // namespace fb2
