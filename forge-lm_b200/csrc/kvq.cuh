// kvq.cuh — the paged, quantised K/V cache: formats, write and read back.
//
// A row (one token's K or V of one head, head_dim values) is quantised by
// itself, so a write touches nothing but its own bytes and meta word:
//   int8: scale = max|x| / 127, code = rint(x * (127 / max|x|)), byte = code + 128;
//   int4: min = bf16(min x), scale = bf16((max x - min x) / 15),
//         code = clamp(rint((x - min) * (1 / scale)), 0, 15).
// All in fp32 with IEEE division and rounding to nearest even; the codes use
// the rounded scale and minimum, so the stored row is the best one for them.
#pragma once
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

#include "common.cuh"

namespace fb2 {

constexpr int KVQ_INT8 = 0, KVQ_INT4 = 1;
constexpr float kKvqTiny = 1e-35f;  // below: the row (or 4-bit group) is a constant, its 1 / scale would overflow

// The cache as the kernels see it.
struct KvqView {
    unsigned char* codes;
    uint32_t* meta;
    int n_slots;      // n_pages * page_size
    int page_shift;   // log2 page_size
    int heads, hd;
    int row_bytes;
    // index of (slot, head, kind)'s row: the rows of a page's head lie together
    FB2_DEV size_t row(int slot, int head, int kind) const {
        const size_t page = (uint32_t)slot >> page_shift;
        return ((((page * heads + head) * 2 + kind) << page_shift) | (slot & ((1 << page_shift) - 1)));
    }
};

FB2_DEV float bf16_bits_to_float(uint32_t b) { return __uint_as_float(b << 16); }
FB2_DEV uint32_t float_to_bf16_bits(float f) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// Copies from global to shared memory that wait nowhere (cp.async), and reads
// of shared memory by its 32-bit addresses.  `live` false: zeros are written.
FB2_DEV void copy16(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
FB2_DEV void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
FB2_DEV void copy8(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(live ? 8 : 0) : "memory");
}
FB2_DEV void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
FB2_DEV void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
FB2_DEV uint4 lds4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
FB2_DEV float2 lds2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}
FB2_DEV uint32_t lds(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

// Element types of dense tensors: 8 consecutive values <-> fp32.
template <class T>
struct Dense;
template <>
struct Dense<float> {
    static FB2_DEV float get(float v) { return v; }
    static FB2_DEV float put(float v) { return v; }
};
template <>
struct Dense<__nv_bfloat16> {
    static FB2_DEV float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static FB2_DEV __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Dense<__half> {
    static FB2_DEV float get(__half v) { return __half2float(v); }
    static FB2_DEV __half put(float v) { return __float2half_rn(v); }
};

// 16 bytes <-> their values, two at a time for the 16-bit types.
template <class T>
FB2_DEV void unpack16(const uint4& w, float* x) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(v[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
template <class T>
FB2_DEV uint4 pack16(const float* x) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __float_as_uint(x[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            memcpy(&v[i], &h, 4);
        } else {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            memcpy(&v[i], &h, 4);
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// 8 values from p, 16-byte aligned.
template <class T>
FB2_DEV void load8(const T* p, float (&x)[8]) {
    constexpr int N = sizeof(T) / 2;  // 16-byte pieces of 8 values
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = Dense<T>::get(t[i]);
}
// A row is shared by `width` = 1 << `shift` neighbouring lanes of a warp; a
// lane holds NP pieces of 16 bytes, piece j at index part + width * j, so that
// every load and store of a row is one run of bytes.  32 values per lane: the
// reductions over the row, the divisions and the addresses are paid once for
// them.  Memory bounds both kernels where there are rows enough.  32785 rows x 8
// heads x 128 in bf16 written as int4 and read back (304 MB): 67.9 us, 4.5 TB/s
// (16 values a lane: 75.1), the instructions of the write still showing; 131072
// rows of int8 read back as bf16 (814 MB): 138 us, 5.9 TB/s.  Few rows take as
// long as a launch and a chain of loads, 4.2 us with the read back (16 values: 3.9).
constexpr int KVQ_THREADS = 128;

template <class T>
struct KvqPiece {
    static constexpr int N = 16 / sizeof(T);  // values
    static constexpr int NP = 32 / N;         // per lane
};

// The code bytes of a piece: N bytes (int8) or N / 2 (int4).
template <int FMT, int N>
FB2_DEV void kvq_store_codes(unsigned char* row, int piece, const uint32_t* w) {
    if constexpr (FMT == KVQ_INT8) {
        if constexpr (N == 8)
            *reinterpret_cast<uint2*>(row + piece * 8) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(row + piece * 4) = w[0];
    } else {
        if constexpr (N == 8)
            *reinterpret_cast<uint32_t*>(row + piece * 4) = w[0];
        else
            *reinterpret_cast<unsigned short*>(row + piece * 2) = (unsigned short)w[0];
    }
}
template <int FMT, int N>
FB2_DEV void kvq_load_codes(const unsigned char* row, int piece, uint32_t* w) {
    if constexpr (FMT == KVQ_INT8) {
        if constexpr (N == 8) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(row + piece * 8));
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = __ldcs(reinterpret_cast<const uint32_t*>(row + piece * 4));
        }
    } else {
        if constexpr (N == 8)
            w[0] = __ldcs(reinterpret_cast<const uint32_t*>(row + piece * 4));
        else
            w[0] = __ldcs(reinterpret_cast<const unsigned short*>(row + piece * 2));
    }
}

FB2_DEV float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
FB2_DEV float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

FB2_DEV float min3_nan(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
FB2_DEV float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// rint(x) for |x| < 2^22 as the low bits of 1.5 2^23 + x
constexpr float kRint = 12582912.0f;
constexpr uint32_t kRintBits = 0x4b400000u;

// blockIdx: rows, K/V head, K or V.
template <class T, int FMT, bool VEC>
__global__ void __launch_bounds__(KVQ_THREADS)
    k_kvq_write(KvqView c, int n_rows, const T* __restrict__ k, const T* __restrict__ v, long long k_row, long long k_head,
                long long v_row, long long v_head, const int* __restrict__ slots, int shift) {
    constexpr int N = KvqPiece<T>::N, NP = KvqPiece<T>::NP;
    const int kind = blockIdx.z, head = blockIdx.y;
    const int width = 1 << shift;
    const int row = blockIdx.x * (KVQ_THREADS >> shift) + (threadIdx.x >> shift), part = threadIdx.x & (width - 1);
    // lanes of a row agree on `live`; the shuffles below run with the whole warp
    const int slot = row < n_rows ? __ldg(slots + row) : -1;
    const bool live = (uint32_t)slot < (uint32_t)c.n_slots;
    const T* p = kind ? v + row * v_row + head * v_head : k + row * k_row + head * k_head;
    float x[NP][N];
    bool mine[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        const int piece = part + width * j;
        mine[j] = live && piece * N < c.hd;
        if constexpr (VEC) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (mine[j]) w = __ldcs(reinterpret_cast<const uint4*>(p) + piece);
            unpack16<T>(w, x[j]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) x[j][i] = mine[j] ? Dense<T>::get(p[piece * N + i]) : 0.f;
        }
    }
    const size_t at = live ? c.row(slot, head, kind) : 0;
    unsigned char* to = c.codes + at * c.row_bytes;
    if constexpr (FMT == KVQ_INT8) {
        float amax = 0.f;  // NaN stays
#pragma unroll
        for (int j = 0; j < NP; j++)
#pragma unroll
            for (int i = 0; i < N; i += 2) amax = max3_nan(amax, fabsf(x[j][i]), fabsf(x[j][i + 1]));
        for (int o = width / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const bool finite = amax < INFINITY;  // false for NaN
        const bool some = finite && amax >= kKvqTiny;
        const float inv = some ? 127.0f / amax : 0.0f;
#pragma unroll
        for (int j = 0; j < NP; j++) {
            if (!mine[j]) continue;
            // |x inv| <= 127 (1 + 2^-23): it rounds to 127 at most; NaN rows hold code 0.
            // The product is rounded by itself, as the formula says.
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                uint32_t q[4];
#pragma unroll
                for (int l = 0; l < 4; l++) q[l] = __float_as_uint(__fmul_rn(x[j][i + l], inv) + (kRint + 128.0f));
                const uint32_t four = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                w[i / 4] = finite ? four : 0x80808080u;
            }
            kvq_store_codes<FMT, N>(to, part + width * j, w);
        }
        if (part == 0 && live) c.meta[at] = finite ? __float_as_uint(some ? amax / 127.0f : 0.0f) : 0x7fc00000u;
    } else {
        const float inf = __uint_as_float(0x7f800000u);
        float lo = inf, hi = -inf;  // NaN stays
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (mine[j])
#pragma unroll
                for (int i = 0; i < N; i += 2) lo = min3_nan(lo, x[j][i], x[j][i + 1]), hi = max3_nan(hi, x[j][i], x[j][i + 1]);
        for (int o = width / 2; o > 0; o >>= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t scale_b = float_to_bf16_bits((hi - lo) / 15.0f), least_b = float_to_bf16_bits(lo);
        const float least = bf16_bits_to_float(least_b), scale = bf16_bits_to_float(scale_b);
        const bool finite = scale < inf && fabsf(least) < inf;  // false for NaN
        const bool some = finite && scale >= kKvqTiny;
        const float inv = some ? 1.0f / scale : 0.0f;
        // The minimum and scale are rounded, so that a code may lie outside 0..15,
        // but hardly ever does: the row's ends show it (rounding is monotonic).
        const bool inside = finite && (lo - least) * inv >= -0.5f && (hi - least) * inv < 15.5f;
        const bool all_inside = __all_sync(0xffffffffu, inside);
#pragma unroll
        for (int j = 0; j < NP; j++) {
            if (!mine[j]) continue;
            uint32_t w = 0;  // the sum of the shifted bits less that of kRint's
#pragma unroll
            for (int i = 0; i < N; i++) {
                float f = __fmul_rn(x[j][i] - least, inv);  // rounded as the formula says: not one step with the sum
                if (!all_inside) f = fminf(fmaxf(f, 0.0f), 15.0f);  // NaN (inf 0): 0
                w += __float_as_uint(f + kRint) << (4 * i);
            }
            w -= N == 8 ? kRintBits * 0x11111111u : kRintBits * 0x1111u;
            kvq_store_codes<FMT, N>(to, part + width * j, &w);
        }
        if (part == 0 && live) c.meta[at] = finite ? ((some ? scale_b : 0u) | (least_b << 16)) : 0x7fc07fc0u;
    }
}

template <class T, int FMT>
__global__ void __launch_bounds__(KVQ_THREADS)
    k_kvq_read(KvqView c, int n_rows, const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int shift) {
    constexpr int N = KvqPiece<T>::N, NP = KvqPiece<T>::NP;
    const int kind = blockIdx.z, head = blockIdx.y;
    const int width = 1 << shift;
    const int row = blockIdx.x * (KVQ_THREADS >> shift) + (threadIdx.x >> shift), part = threadIdx.x & (width - 1);
    if (row >= n_rows) return;
    const int slot = __ldg(slots + row);
    const bool live = (uint32_t)slot < (uint32_t)c.n_slots;
    uint32_t w[NP][2], m = 0;
#pragma unroll
    for (int j = 0; j < NP; j++) w[j][0] = w[j][1] = 0;
    if (live) {
        const size_t at = c.row(slot, head, kind);
        m = __ldg(c.meta + at);
#pragma unroll
        for (int j = 0; j < NP; j++)
            if ((part + width * j) * N < c.hd) kvq_load_codes<FMT, N>(c.codes + at * c.row_bytes, part + width * j, w[j]);
    }
    const float scale = bf16_bits_to_float(m & 0xffffu), scale16 = scale * 0.0625f, least = __uint_as_float(m & 0xffff0000u);
    uint4* to = reinterpret_cast<uint4*>((kind ? v : k) + ((size_t)row * c.heads + head) * c.hd);
#pragma unroll
    for (int j = 0; j < NP; j++) {
        if ((part + width * j) * N >= c.hd) continue;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (FMT == KVQ_INT8) {
                const float code = __uint_as_float(__byte_perm(w[j][i / 4], kRintBits, 0x7650 + i % 4)) - (kRint + 128.0f);
                x[i] = code * __uint_as_float(m);
            } else {
                // a byte's high nibble stays in place: 16 code, with scale / 16 (a power of two: exact)
                const uint32_t byte = w[j][0] >> (8 * (i / 2)), nibble = i & 1 ? 0xf0u : 0xfu;
                const float code = __uint_as_float((byte & nibble) | kRintBits) - kRint;
                x[i] = fmaf(code, i & 1 ? scale16 : scale, least);
            }
        }
        const uint4 o = live ? pack16<T>(x) : make_uint4(0, 0, 0, 0);
        __stcs(to + part + width * j, o);
    }
}

}  // namespace fb2
