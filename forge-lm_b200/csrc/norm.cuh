// norm.cuh — a block's output onto the residual stream and the norm before the
// next block, in one pass, and rows as 8-bit codes (include/forge_b200.h,
// fb2_residual_norm and fb2_quantise_rows, has the formulas).
//
// A row is held by the threads that share it, as fp32, from the first load to the last
// store, in registers up to 16384 values (beyond, 1024 threads have 64 registers each for 64
// values, and some are spilled: 2000 x 32768 bf16 172 us, fp32 228, with both norms 231 and 340,
// where x 16384 takes 75, 100, 96 and 132): h and x are read once, the stream and the normed
// row written once, and means and variances are taken of values at hand (the
// variance of differences from the mean, not of squares).  All of a row's loads go out
// before the first sum (with x behind the norm of h: 226 us instead of 137 for 16383 x
// 4096, h bf16, x fp32, both norms).  What bounds it is HBM where there are rows enough:
// that case moves 805 MB at 5.9 TB/s, 30000 x 1999 in fp32 6.6 TB/s; rows of 16-bit values
// that do not begin on 16 bytes go by accesses of two bytes a lane (30000 x 1999 bf16 174
// us, x 2000 87).  Rows of up to 256 have a warp each, whatever their length, and are
// bound by its instructions: 100 thousand x 256 bf16 50 us where the bytes take 31, 200 thousand x
// 128 85, 400 thousand x 64 162, x 70 180 (their codes 27, 53, 105 and 105; bytes 12).  One row
// takes as long as a launch, its loads and its sums: 2.3 us (768),
// 4.2 (8192).
#pragma once
#include "kvq.cuh"

namespace fb2 {

constexpr int NORM_E = 8;         // consecutive values of a thread
constexpr int NORM_MOST = 32768;  // of a row: 1024 threads with 32 each

struct NormArgs {
    const void *h, *x, *gate;  // gate NULL: 1
    const float *w, *b, *post_w, *post_b;
    void *sum, *y;
    signed char* codes;
    float* scales;
    long long h_row, x_row, gate_row, sum_row, y_row, code_row;
    int rows, dim;
    float scale, eps;
    bool rms, post;
};

namespace nrm {

// Sum (or, of bits, largest) over the G threads that share a row; `turn` counts the
// calls: the place of the one before may still be read.
template <int G>
FB2_DEV float sum(float v, float (*s)[32], int& turn) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        float* to = s[turn++ & 1];
        if ((threadIdx.x & 31) == 0) to[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < G / 32; i++) v += to[i];
    }
    return v;
}
template <int G>
FB2_DEV uint32_t largest(uint32_t v, float (*s)[32], int& turn) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (G > 32) {
        float* to = s[turn++ & 1];
        if ((threadIdx.x & 31) == 0) to[threadIdx.x >> 5] = __uint_as_float(v);
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < G / 32; i++) v = max(v, __float_as_uint(to[i]));
    }
    return v;
}

// How a row's n values lie with its G threads.  VEC (rows that begin on 16 bytes and are
// a multiple of 8 values): piece j of a thread is 8 neighbours, read 16 bytes at a time.
// Else neighbouring threads have neighbouring values, so that a warp's accesses are runs;
// pieces that are inside the row for all threads are not checked value by value.  (Rows
// that begin anywhere read 16 bytes at a time, with the weights moved in registers to fit,
// took 240 us where this takes 174: 30000 x 1999, bf16.)
template <int G, bool VEC>
struct Lie {
    int tid, n;
    FB2_DEV bool whole(int j) const { return VEC ? (tid + j * G) * NORM_E < n : (j + 1) * NORM_E * G <= n; }
    FB2_DEV bool inside(int j, int i) const { return VEC ? whole(j) : whole(j) || tid + (j * NORM_E + i) * G < n; }
    // values outside the row are 0
    template <class T>
    FB2_DEV void load(const T* row, int j, float (&v)[NORM_E]) const {
        if constexpr (VEC) {
            if (whole(j)) {
                load8(row + (tid + j * G) * NORM_E, v);
            } else {
#pragma unroll
                for (int i = 0; i < NORM_E; i++) v[i] = 0.f;
            }
        } else {
            const T* p = row + tid;
            if (whole(j)) {
#pragma unroll
                for (int i = 0; i < NORM_E; i++) v[i] = Dense<T>::get(p[(j * NORM_E + i) * G]);
            } else {
#pragma unroll
                for (int i = 0; i < NORM_E; i++) v[i] = inside(j, i) ? Dense<T>::get(p[(j * NORM_E + i) * G]) : 0.f;
            }
        }
    }
    template <class T>
    FB2_DEV void store(T* row, int j, const float (&v)[NORM_E]) const {
        if constexpr (VEC) {
            if (!whole(j)) return;
            T* to = row + (tid + j * G) * NORM_E;
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < NORM_E; i += N) *reinterpret_cast<uint4*>(to + i) = pack16<T>(v + i);
        } else {
#pragma unroll
            for (int i = 0; i < NORM_E; i++)
                if (inside(j, i)) (row + tid)[(j * NORM_E + i) * G] = Dense<T>::put(v[i]);
        }
    }
};

// 127 / top and top / 127 of a row whose largest |value| has these bits: (0, 0)
// where it is too small to be divided by, a NaN scale where it is not finite.
FB2_DEV void code_scale(uint32_t top_bits, float& inv, float& scale) {
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) {
        inv = 0.f;
        scale = __uint_as_float(0x7fc00000u);
    } else if (top < kKvqTiny) {
        inv = scale = 0.f;
    } else {
        inv = 127.f / top;
        scale = top / 127.f;
    }
}
FB2_DEV uint32_t code(float x, float inv) {
    // no code is past 127: x * inv is at most 127 and two roundings
    return inv == 0.f ? 0u : (uint32_t)__float2int_rn(x * inv) & 0xffu;
}
template <int G, bool VEC>
FB2_DEV void store_codes(signed char* row, const Lie<G, VEC>& lie, int j, const float (&v)[NORM_E], float inv) {
    if constexpr (VEC) {  // rows of codes begin on 16 bytes
        if (!lie.whole(j)) return;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < NORM_E; i++) w[i / 4] |= code(v[i], inv) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(row + (lie.tid + j * G) * NORM_E) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < NORM_E; i++)
            if (lie.inside(j, i)) (row + lie.tid)[(j * NORM_E + i) * G] = (signed char)code(v[i], inv);
    }
}

}  // namespace nrm

// T: h, gate and y; X: x and the sum.  G threads share a row and hold 8 * NJ of
// its values each; blockDim: G, or four rows of a warp each for G = 32.
template <class T, class X, int G, int NJ, bool VEC>
__global__ void __launch_bounds__(G == 32 ? 128 : G, G == 32 ? 5 : G < 640 ? 640 / G : 1) k_residual_norm(NormArgs a) {
    __shared__ float s[2][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product's launch; it waits for this grid's end
    const int row = G == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    const nrm::Lie<G, VEC> lie{G == 32 ? (int)threadIdx.x & 31 : (int)threadIdx.x, a.dim};
    const float count = (float)a.dim;
    int turn = 0;
    float v[NJ][NORM_E], xv[NJ][NORM_E];
    // (v - mean) / sqrt(var + eps), or v / sqrt(mean square + eps)
    auto normed = [&](const float* w, const float* b) {
        float mean = 0.f, part = 0.f;
        if (!a.rms) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < NORM_E; i++) part += v[j][i];
            mean = nrm::sum<G>(part, s, turn) / count;
        }
        part = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int i = 0; i < NORM_E; i++) {
                const float d = v[j][i] - mean;
                if (lie.inside(j, i)) part += d * d;
            }
        const float r = 1.f / sqrtf(nrm::sum<G>(part, s, turn) / count + a.eps);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            float wv[NORM_E], bv[NORM_E];
            lie.load(w, j, wv);
            if (b) lie.load(b, j, bv);
#pragma unroll
            for (int i = 0; i < NORM_E; i++) {
                v[j][i] = (v[j][i] - mean) * r * wv[i];
                if (b) v[j][i] += bv[i];
            }
        }
    };
    // all of the row's loads at once
    const X* x = static_cast<const X*>(a.x) + row * a.x_row;
#pragma unroll
    for (int j = 0; j < NJ; j++) lie.load(x, j, xv[j]);
    if (a.h) {
        const T* h = static_cast<const T*>(a.h) + row * a.h_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) lie.load(h, j, v[j]);
        if (a.post) normed(a.post_w, a.post_b);
        if (a.gate) {
            const T* gate = static_cast<const T*>(a.gate) + row * a.gate_row;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                float gv[NORM_E];
                lie.load(gate, j, gv);
#pragma unroll
                for (int i = 0; i < NORM_E; i++) v[j][i] *= gv[i];
            }
        }
        X* sum = static_cast<X*>(a.sum) + row * a.sum_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
#pragma unroll
            for (int i = 0; i < NORM_E; i++) v[j][i] = xv[j][i] + a.scale * v[j][i];
            lie.store(sum, j, v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int i = 0; i < NORM_E; i++) v[j][i] = xv[j][i];
    }
    normed(a.w, a.b);
    if (!a.codes) {
        T* y = static_cast<T*>(a.y) + row * a.y_row;
#pragma unroll
        for (int j = 0; j < NJ; j++) lie.store(y, j, v[j]);
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int i = 0; i < NORM_E; i++)
            if (lie.inside(j, i)) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
    float inv, scale;
    nrm::code_scale(nrm::largest<G>(top, s, turn), inv, scale);
#pragma unroll
    for (int j = 0; j < NJ; j++) nrm::store_codes(a.codes + row * a.code_row, lie, j, v[j], inv);
    if (lie.tid == 0) a.scales[row] = scale;
}

// Rows x [rows][n] as codes, 8 * NJ values to a thread; NJ = 0: of any length, read
// twice.
template <class T, int G, int NJ, bool VEC>
__global__ void __launch_bounds__(G == 32 ? 128 : G) k_quantise_rows(const T* x, long long x_row, int rows, int n, signed char* codes,
                                                                     long long code_row, float* scales) {
    __shared__ float s[2][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const long long row = G == 32 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= rows) return;
    const nrm::Lie<G, VEC> lie{G == 32 ? (int)threadIdx.x & 31 : (int)threadIdx.x, n};
    x += row * x_row;
    codes += row * code_row;
    uint32_t top = 0;
    float v[NJ ? NJ : 1][NORM_E];
    auto most = [&](const float (&p)[NORM_E]) {
#pragma unroll
        for (int i = 0; i < NORM_E; i++) top = max(top, __float_as_uint(p[i]) & 0x7fffffffu);
    };
    const int pieces = (n + G * NORM_E - 1) / (G * NORM_E);
    if constexpr (NJ > 0) {
#pragma unroll
        for (int j = 0; j < NJ; j++) lie.load(x, j, v[j]);
#pragma unroll
        for (int j = 0; j < NJ; j++) most(v[j]);
    } else {
        for (int j = 0; j < pieces; j++) {
            lie.load(x, j, v[0]);
            most(v[0]);
        }
    }
    float inv, scale;
    int turn = 0;
    nrm::code_scale(nrm::largest<G>(top, s, turn), inv, scale);
    if constexpr (NJ > 0) {
#pragma unroll
        for (int j = 0; j < NJ; j++) nrm::store_codes(codes, lie, j, v[j], inv);
    } else {
        for (int j = 0; j < pieces; j++) {
            lie.load(x, j, v[0]);
            nrm::store_codes(codes, lie, j, v[0], inv);
        }
    }
    if (lie.tid == 0) scales[row] = scale;
}

}  // namespace fb2
