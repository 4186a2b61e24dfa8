// step_ops.cu — C ABI of the serving operators around attention and 4-bit layers:
// pages of sequences, residual stream and norms, 8-bit linear layers, verification
// of drafts.  Checks of arguments and launches; the kernels are in pages.cuh,
// norm.cuh, w8.cuh and verify.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include <cudaTypedefs.h>

#include "../../include/forge_b200_testing.h"
#include "norm.cuh"
#include "pages.cuh"
#include "serving_host.cuh"
#include "verify.cuh"
#include "w8.cuh"

using namespace fb2;

namespace {

// A launch of clusters of `cluster` CTAs along x (`smem`: the same for every launch of a
// kernel, or opted in for its most before); `early`: it may begin before
// the launch before it has ended (the kernel waits in pdl_wait).
template <class... P, class... A>
void launch_cluster(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, bool early, void* stream, A... args) {
    if (smem > 48 * 1024) opt_in_smem((const void*)kernel, smem);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (cluster > 1) {
        cudaLaunchAttribute& a = attr[cfg.numAttrs++];
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim.x = cluster;
        a.val.clusterDim.y = a.val.clusterDim.z = 1;
    }
    if (early) {
        cudaLaunchAttribute& a = attr[cfg.numAttrs++];
        a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        a.val.programmaticStreamSerializationAllowed = 1;
    }
    CK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

}  // namespace

// ---- pages of sequences ------------------------------------------------------------
namespace {
PagesView pages_view(const fb2_pages* p) {
    need(p, "pages are NULL");
    need(p->n_seqs >= 0 && p->n_seqs <= PG_SEQS, "n_seqs must be in 0..16384");
    need(p->max_pages >= 0 && p->n_pages >= 0, "max_pages and n_pages must not be negative");
    need(pow2(p->page_size) && p->page_size >= 8 && p->page_size <= 1024, "page_size must be a power of two in 8..1024");
    need((int64_t)p->max_pages * p->page_size <= INT32_MAX, "max_pages * page_size must be at most 2^31 - 1");
    need((int64_t)p->n_pages * p->page_size <= INT32_MAX, "there must be at most 2^31 - 1 slots");
    need(p->table_stride >= p->max_pages, "table_stride must be at least max_pages");
    need(p->n_seqs == 0 || p->device_lens, "NULL argument");
    need(p->n_seqs == 0 || p->max_pages == 0 || p->device_table, "NULL argument");
    need((p->n_pages == 0 || p->device_free) && p->device_n_free, "NULL argument");
    need(aligned(p->device_table, 4) && aligned(p->device_lens, 4) && aligned(p->device_free, 4) && aligned(p->device_n_free, 4),
         "a tensor is not aligned to its element size");
    return {p->device_table, p->device_lens, p->device_free, p->device_n_free, p->table_stride,
            p->n_seqs,       p->max_pages,   p->n_pages,     log2_of(p->page_size)};
}
}  // namespace

int32_t fb2_pages_check(const fb2_pages* p) {
    return guarded([&] { pages_view(p); });
}

int32_t fb2_pages_extend(const fb2_pages* p, const int32_t* counts, int32_t max_rows, int32_t* starts, int32_t* prefix_lens,
                         int32_t* slots, int32_t* positions, void* stream) {
    return guarded([&] {
        const PagesView v = pages_view(p);
        need(max_rows >= 0 && max_rows <= INT32_MAX - 65536, "max_rows must be in 0..2^31 - 65537");
        need(starts && (v.n_seqs == 0 || (counts && prefix_lens)) && (max_rows == 0 || (slots && positions)), "NULL argument");
        need(aligned(counts, 4) && aligned(starts, 4) && aligned(prefix_lens, 4) && aligned(slots, 4) && aligned(positions, 4),
             "a tensor is not aligned to its element size");
        const bool vec = aligned(slots, 16) && aligned(positions, 16);
        auto launch = [&](auto kernel, int threads, int ranks) {
            opt_in_smem((const void*)kernel, 12 * PG_SEQS);
            if (ranks > 8) CK(cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            launch_cluster(kernel, dim3(ranks), threads, 12 * v.n_seqs, ranks, false, stream, v, counts, max_rows, starts, prefix_lens, slots,
                           positions, vec);
        };
        // CTAs of the cluster: where each has 4 rows to a thread (131 thousand rows: 14.6 us with
        // 8, 10.5 with 16, which is more than every device promises: this one has it)
        int ranks = 1;
        while (ranks < 16 && max_rows > 1024 * 4 * ranks) ranks *= 2;
        if (v.n_seqs <= 256 && max_rows <= 1024)
            launch(k_pages_extend<256, 1>, 256, 1);
        else
            launch(k_pages_extend<1024, 4>, 1024, ranks);
    });
}

int32_t fb2_pages_truncate(const fb2_pages* p, const int32_t* lens, void* stream) {
    return guarded([&] {
        const PagesView v = pages_view(p);
        if (v.n_seqs == 0) return;
        need(lens, "NULL argument");
        need(aligned(lens, 4), "a tensor is not aligned to its element size");
        auto launch = [&](auto kernel, int threads) {
            opt_in_smem((const void*)kernel, 8 * PG_SEQS);
            launch_cluster(kernel, dim3(1), threads, 8 * v.n_seqs, 1, false, stream, v, lens);
        };
        if (v.n_seqs <= 256)
            launch(k_pages_truncate<256>, 256);
        else
            launch(k_pages_truncate<1024>, 1024);
    });
}

// ---- residual stream and norms -------------------------------------------------------
namespace {
template <class T, class X, int G, int NJ>
void launch_norm(const NormArgs& a, bool vec, cudaStream_t stream) {
    constexpr int rows = G == 32 ? 4 : 1;
    const unsigned grid = (unsigned)(((int64_t)a.rows + rows - 1) / rows);
    (vec ? k_residual_norm<T, X, G, NJ, true> : k_residual_norm<T, X, G, NJ, false>)<<<grid, G == 32 ? 128 : G, 0, stream>>>(a);
}
template <class T, class X>
void launch_norm(const NormArgs& a, bool vec, cudaStream_t stream) {
    // threads of a row: few values each where rows are few (one of 768: 3.6 us with a warp,
    // 2.3 with 128 threads), else up to 32 (6000 x 8192 bf16: 88 us with 256 threads, 139
    // with 512)
    const bool few = a.rows <= 4 * 148;
    const int dim = a.dim;
    if (dim <= 256)
        launch_norm<T, X, 32, 1>(a, vec, stream);
    else if (dim <= 1024 && few)
        launch_norm<T, X, 128, 1>(a, vec, stream);
    else if (dim <= 1024)
        launch_norm<T, X, 32, 4>(a, vec, stream);
    else if (dim <= 4096 && few)
        launch_norm<T, X, 512, 1>(a, vec, stream);
    else if (dim <= 2048)
        launch_norm<T, X, 64, 4>(a, vec, stream);
    else if (dim <= 4096)
        launch_norm<T, X, 128, 4>(a, vec, stream);
    else if (dim <= 8192)
        launch_norm<T, X, 256, 4>(a, vec, stream);
    else if (dim <= 16384)
        launch_norm<T, X, 512, 4>(a, vec, stream);
    else
        launch_norm<T, X, 1024, 4>(a, vec, stream);
}
}  // namespace

int32_t fb2_residual_norm(const fb2_norm* n, void* stream) {
    return guarded([&] {
        need(n, "norm is NULL");
        check_dtype(n->dtype);
        need(n->stream_dtype == n->dtype || n->stream_dtype == FB2_F32, "stream_dtype must be dtype or FB2_F32");
        need(n->kind == FB2_NORM_LAYER || n->kind == FB2_NORM_RMS, "kind must be FB2_NORM_LAYER or FB2_NORM_RMS");
        need(n->n_rows >= 0 && n->n_rows <= INT32_MAX - 3, "n_rows must be in 0..2^31 - 4");
        need(n->dim >= 1 && n->dim <= NORM_MOST, "dim must be in 1..32768");
        need(std::isfinite(n->scale) && n->eps >= 0.f && std::isfinite(n->eps), "scale must be finite, eps finite and not negative");
        if (n->n_rows == 0) return;
        need(n->device_x && n->device_weight, "NULL argument");
        need(n->device_h ? n->device_sum != nullptr : !n->device_gate && !n->device_post_weight,
             "h needs a sum; without h there is no gate and no norm of it");
        need(n->device_post_weight || !n->device_post_bias, "post_bias needs post_weight");
        need(!n->device_codes == !n->device_scales && !n->device_codes != !n->device_y, "the result is y, or codes and scales");
        const size_t es = size_of(n->dtype), xs = size_of(n->stream_dtype);
        need(aligned(n->device_h, es) && aligned(n->device_gate, es) && aligned(n->device_y, es) && aligned(n->device_x, xs) &&
                 aligned(n->device_sum, xs) && aligned(n->device_weight, 4) && aligned(n->device_bias, 4) &&
                 aligned(n->device_post_weight, 4) && aligned(n->device_post_bias, 4) && aligned(n->device_scales, 4),
             "a tensor is not aligned to its element size");
        const bool many = n->n_rows > 1;
        need(!many || ((!n->device_sum || n->sum_row_stride >= n->dim) && (!n->device_y || n->y_row_stride >= n->dim)),
             "sum_row_stride and y_row_stride must be at least dim");
        need(!n->device_codes || (aligned(n->device_codes, 16) && (!many || (n->code_row_stride >= n->dim && n->code_row_stride % 16 == 0))),
             "rows of codes must begin on 16 bytes and not overlap");
        bool vec = n->dim % NORM_E == 0;  // rows that begin on 16 bytes throughout
        auto runs = [&](const void* p, int64_t row, size_t size) {
            if (p && (!aligned(p, 16) || (many && row * (int64_t)size % 16))) vec = false;
        };
        runs(n->device_h, n->h_row_stride, es), runs(n->device_gate, n->gate_row_stride, es), runs(n->device_y, n->y_row_stride, es);
        runs(n->device_x, n->x_row_stride, xs), runs(n->device_sum, n->sum_row_stride, xs);
        for (const float* p : {n->device_weight, n->device_bias, n->device_post_weight, n->device_post_bias}) runs(p, 0, 4);
        const NormArgs a{n->device_h,      n->device_x,       n->device_gate,      n->device_weight,    n->device_bias,    n->device_post_weight,
                         n->device_post_bias, n->device_sum,  n->device_y,         (signed char*)n->device_codes, n->device_scales,
                         n->h_row_stride,  n->x_row_stride,   n->gate_row_stride,  n->sum_row_stride,   n->y_row_stride,   n->code_row_stride,
                         n->n_rows,        n->dim,            n->scale,            n->eps,              n->kind == FB2_NORM_RMS,
                         n->device_post_weight != nullptr};
        with_type(n->dtype, [&](auto t) {
            using T = decltype(t);
            if (n->stream_dtype == n->dtype)
                launch_norm<T, T>(a, vec, (cudaStream_t)stream);
            else
                launch_norm<T, float>(a, vec, (cudaStream_t)stream);
        });
        launched();
    });
}

// ---- 8-bit linear layers ----------------------------------------------------------------
int32_t fb2_quantise_rows(int32_t n_rows, int32_t dim, const void* x, int32_t dtype, int64_t x_row, void* codes, int64_t code_row, float* scales,
                          void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        need(n_rows >= 0 && dim >= 1 && dim <= INT32_MAX - 4096, "n_rows must not be negative, dim in 1..2^31 - 4097");
        if (n_rows == 0) return;
        need(x && codes && scales, "NULL argument");
        const size_t es = size_of(dtype);
        need(aligned(x, es) && aligned(scales, 4), "a tensor is not aligned to its element size");
        need(aligned(codes, 16) && (n_rows == 1 || (code_row >= dim && code_row % 16 == 0)),
             "rows of codes must begin on 16 bytes and not overlap");
        const bool vec = aligned(x, 16) && dim % NORM_E == 0 && (n_rows == 1 || x_row * es % 16 == 0);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto launch = [&](auto threads, auto pieces) {
                constexpr int G = decltype(threads)::value, NJ = decltype(pieces)::value, rows = G == 32 ? 4 : 1;
                auto kernel = vec ? k_quantise_rows<T, G, NJ, true> : k_quantise_rows<T, G, NJ, false>;
                kernel<<<(unsigned)(((int64_t)n_rows + rows - 1) / rows), G == 32 ? 128 : G, 0, (cudaStream_t)stream>>>(
                    (const T*)x, x_row, n_rows, dim, (signed char*)codes, code_row, scales);
            };
            const bool few = n_rows <= 4 * 148;
            if (dim <= 256)
                launch(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
            else if (dim <= 1024 && !few)
                launch(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
            else if (dim <= 1024)
                launch(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
            else if (dim <= 2048)
                launch(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
            else if (dim <= 4096)
                launch(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{});
            else if (dim <= 8192)
                launch(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
            else if (dim <= 16384)
                launch(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
            else
                launch(std::integral_constant<int, 512>{}, std::integral_constant<int, 0>{});
        });
        launched();
    });
}

namespace {
void check_w8(const fb2_w8_linear* w) {
    need(w, "linear is NULL");
    need(w->in_features >= 1 && w->in_features <= 131072, "in_features must be in 1..131072");  // 127^2 a product, 2^31 the sum
    need(w->out_features >= 1 && w->out_features <= INT32_MAX - 255, "out_features must be in 1..2^31 - 256");
    need(w->out_features == 1 || (w->code_row_stride >= w->in_features && w->code_row_stride % 16 == 0),
         "code_row_stride must be a multiple of 16 and at least in_features");
    need(w->device_codes && w->device_scales, "a weight buffer is NULL");
    need(aligned(w->device_codes, 16) && aligned(w->device_scales, 4) && aligned(w->device_bias, 4),
         "codes must be 16-byte aligned, scales and bias to their element size");
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
        else
            cudaGetLastError();
    });
    return fn;
}
// Rows of `inner` bytes, `stride` bytes apart, in 128-byte swizzled boxes of 128
// bytes x `box` rows; what lies past the rows' ends or the last row reads as 0.
CUtensorMap byte_map(const void* base, int64_t inner, int64_t rows, int64_t stride, int box) {
    auto fn = encode_fn();
    if (!fn) fail(FB2_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t boxes[2] = {W8_K, (cuuint32_t)box}, steps[2] = {1, 1};
    if (fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(FB2_CUDA_ERROR, "cuTensorMapEncodeTiled failed");
    return map;
}
// A single row may have any stride; the map wants one that it can hold.
int64_t row_stride(int64_t rows, int64_t stride, int64_t inner) { return rows > 1 ? stride : (inner + 15) / 16 * 16; }

template <class T, int BN>
void launch_few(const CUtensorMap& mw, const CUtensorMap& mx, const W8Args& a, void* stream) {
    const int tiles = (a.out + 127) / 128, across = (a.rows + BN - 1) / BN, blocks = (a.in + W8_K - 1) / W8_K;
    // CTAs to a tile: of two blocks of inputs at least, up to one on each SM, two where
    // they have 16 blocks each (us with up to 148 and up to 296 CTAs of any length: 61 x
    // 1024 x 4096 6.3 and 8.8, 61 x 4096 x 4096 8.2 and 10.1, 16 x 8192 x 8192 17.0 and 16.0)
    int ranks = 1;
    while (ranks < 8 && ranks * 4 <= blocks && (int64_t)tiles * across * ranks * 2 <= (blocks >= ranks * 32 ? 2 : 1) * 148) ranks *= 2;
    launch_cluster(k_w8_few<T, BN>, dim3(tiles * ranks, across), W8_THREADS, W8Few<BN>::SMEM, ranks, true, stream, mw, mx, a, ranks);
}

// Few rows: pieces of a lane's inputs, warps that share an output's
struct W8Rows {
    int pieces, per_k;
};
// Up to 4 rows take the warps' dot products as far as a lane's registers hold their inputs
// (1 x 768 x 2304 4.1 us, 9.4 on tcgen05 tiles behind a launch for the codes; 1 x 8192 x 28672
// 41 and 53); more rows, at 4 instructions for 16 products each, would take longer than
// the weights' bytes.
constexpr int W8R_MOST = 4;
bool w8_by_rows(int rows, int in) {
    return rows <= W8R_MOST && in <= W8R_CODES && (rows > 2 ? 4 : rows) * ((in + 15) / 16 * 16) <= W8R_CODES;
}
W8Rows w8_rows_plan(int in) {
    W8Rows p{1, 1};
    while (p.per_k < W8R_WARPS && p.per_k * 512 < in) p.per_k *= 2;
    while (p.pieces * p.per_k * 512 < in) p.pieces *= 2;
    return p;
}
template <class T, class X, int ROWS, int PIECES>
void launch_rows(const fb2_w8_linear* w, const W8Args& a, const X* x, int64_t x_row, bool vec, bool early, int per_k, void* stream) {
    const int slots = W8R_WARPS / per_k, codes = sizeof(X) == 1 ? 0 : a.rows * (int)row_stride(1, 0, a.in);
    // every SM full, an output at least for each slot, and what the sums have room for
    int64_t grid = std::min<int64_t>(w8r_resident<X, ROWS, PIECES> * 148, (a.out + slots - 1) / slots);
    grid = std::max<int64_t>(grid, ((int64_t)a.out * ROWS + W8R_SUMS - ROWS - 1) / (W8R_SUMS - ROWS));
    launch_cluster(k_w8_rows<T, X, ROWS, PIECES>, dim3((unsigned)grid), W8R_THREADS, codes, 1, early, stream, a, x, x_row,
                   (const signed char*)w->device_codes, row_stride(a.out, w->code_row_stride, a.in), per_k, vec);
}
template <class T, class X>
void launch_rows(const fb2_w8_linear* w, const W8Args& a, const X* x, int64_t x_row, bool vec, bool early, void* stream) {
    const W8Rows p = w8_rows_plan(a.in);  // rows (3 count as 4) times pieces: at most 4
    auto go = [&](auto rows, auto pieces) {
        launch_rows<T, X, decltype(rows)::value, decltype(pieces)::value>(w, a, x, x_row, vec, early, p.per_k, stream);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    if (a.rows > 2)
        go(four, one);
    else if (a.rows == 2)
        p.pieces == 1 ? go(two, one) : go(two, two);
    else
        p.pieces == 1 ? go(one, one) : p.pieces == 2 ? go(one, two) : go(one, four);
}

// More than 128 rows: whether tiles of 128 x 128 whose inputs a cluster shares take less
// than 256 x 256 by pairs of CTAs that leave most SMs without one.  us, shared and not, of
// rows x inputs x outputs with so many of the larger tiles:
//   below 1024 inputs   256 x 512 x 1024, 4, 8.9 and 8.0; x 4096, 16, 9.3 and 8.3 (x 4608, 18, 9.3
//                       and 9.8)
//   1024 to 4095        256 x 1024 x 1024, 4, 7.6 and 9.5; x 4096, 16, 9.9 and 9.7; x 4608, 18, 9.9 and
//                       11.3; 256 x 2048 x 4096, 16, 11.2 and 12.2; x 6144, 24, 32 and 13.3 (2048 to
//                       4096 rows x 1024, 16: up to 10 % the other way)
//   4096 on             256 x 4096 x 4096, 16, 13.8 and 17.4; x 9472, 37, 19.7 and 20.2; x 11008, 43, 42 and
//                       21; 256 x 16384 x 8192, 32, 41 and 50 (256 x 5000 x 8192, 32, 29 and 22; 2048 x 4096 x
//                       1152, 40, 17.5 and 19.2)
bool w8_splits(int64_t tiles, int in) { return in >= 32 * W8_K ? tiles <= 37 : in >= 8 * W8_K && tiles <= 18; }

std::atomic<int> g_withhold_block{-1};
std::atomic<int64_t> g_withhold_wait_ns{0};
}  // namespace

// test hook: what the next product withholds
int32_t fb2_test_w8_withhold(int32_t block, int64_t wait_ns) {
    return guarded([&] {
        need(block >= 0 && wait_ns > 0 && wait_ns <= (int64_t)kTcTimeoutNs, "bad hook arguments");
        g_withhold_wait_ns = wait_ns;
        g_withhold_block = block;
    });
}

int32_t fb2_w8_check(const fb2_w8_linear* w) {
    return guarded([&] { check_w8(w); });
}

int32_t fb2_w8_pack(const fb2_w8_linear* w, const void* dense, int32_t dtype, int64_t w_row, void* stream) {
    return guarded([&] {
        check_w8(w);
        check_dtype(dtype);
        need(dense, "w is NULL");
        need(aligned(dense, size_of(dtype)), "w is not aligned to its element size");
        need(w_row == 0 || w_row >= w->out_features, "w_row_stride must be 0 or at least out_features");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            k_w8_pack<T><<<(unsigned)((w->out_features + 31) / 32), W8P_THREADS, 0, (cudaStream_t)stream>>>(
                (const T*)dense, w_row, w->in_features, w->out_features, (signed char*)const_cast<void*>(w->device_codes), w->code_row_stride,
                const_cast<float*>(w->device_scales));
        });
        launched();
    });
}

int32_t fb2_w8_matmul(const fb2_w8_linear* w, int32_t n_rows, const void* codes, int64_t code_row, const float* scales, void* y, int64_t y_row,
                      int32_t dtype, void* stream) {
    return guarded([&] {
        check_w8(w);
        check_dtype(dtype);
        need(n_rows >= 0 && n_rows <= INT32_MAX - 255, "n_rows must be in 0..2^31 - 256");
        if (n_rows == 0) return;
        need(codes && scales && y, "NULL argument");
        const size_t es = size_of(dtype);
        need(aligned(codes, 16) && (n_rows == 1 || (code_row >= w->in_features && code_row % 16 == 0)),
             "rows of codes must begin on 16 bytes and not overlap");
        need(aligned(scales, 4) && aligned(y, es), "a tensor is not aligned to its element size");
        need(n_rows == 1 || y_row >= w->out_features, "y_row_stride must be at least out_features");
        W8Args a{scales, w->device_scales, w->device_bias, y, y_row, n_rows, w->in_features, w->out_features,
                 aligned(y, 16) && (n_rows == 1 || y_row * es % 16 == 0), g_withhold_block.exchange(-1), kTcTimeoutNs};
        if (a.withhold >= 0) a.wait_ns = (unsigned long long)g_withhold_wait_ns.load();
        const int64_t tiles = (int64_t)((a.rows + 255) / 256) * ((a.out + W8M_N - 1) / W8M_N);  // of the largest kind
        auto x_map = [&](int box) { return byte_map(codes, a.in, a.rows, row_stride(a.rows, code_row, a.in), box); };
        auto w_map = [&](int box) { return byte_map(w->device_codes, a.in, a.out, row_stride(a.out, w->code_row_stride, a.in), box); };
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            if (w8_by_rows(n_rows, a.in))
                launch_rows<T>(w, a, (const signed char*)codes, code_row, true, true, stream);
            else if (n_rows <= 16)
                launch_few<T, 16>(w_map(128), x_map(16), a, stream);
            else if (n_rows <= 32)
                launch_few<T, 32>(w_map(128), x_map(32), a, stream);
            else if (n_rows <= 64)
                launch_few<T, 64>(w_map(128), x_map(64), a, stream);
            else if (n_rows <= 128 || w8_splits(tiles, a.in))
                launch_few<T, 128>(w_map(128), x_map(128), a, stream);
            else {
                need(tiles <= INT32_MAX - 65536, "too many rows for one call");
                launch_cluster(k_w8_many<T>, dim3((unsigned)std::min<int64_t>(2 * tiles, 148)), W8_THREADS, W8M_SMEM, 2, true, stream,
                               w_map(128), x_map(128), a);
            }
        });
        launched();
    });
}

int32_t fb2_w8_forward_workspace(const fb2_w8_linear* w, int32_t n_rows, int64_t* bytes) {
    return guarded([&] {
        check_w8(w);
        need(n_rows >= 0, "n_rows must not be negative");
        need(bytes, "bytes is NULL");
        // codes on 16 bytes, and scales
        *bytes = n_rows == 0 || w8_by_rows(n_rows, w->in_features) ? 0 : (int64_t)n_rows * (row_stride(1, 0, w->in_features) + 4);
    });
}

int32_t fb2_w8_forward(const fb2_w8_linear* w, int32_t n_rows, const void* x, int64_t x_row, void* y, int64_t y_row, int32_t dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_w8(w);
        check_dtype(dtype);
        need(n_rows >= 0 && n_rows <= INT32_MAX - 255, "n_rows must be in 0..2^31 - 256");
        if (n_rows == 0) return;
        need(x && y, "NULL argument");
        const size_t es = size_of(dtype);
        need(aligned(x, es) && aligned(y, es), "a tensor is not aligned to its element size");
        need(n_rows == 1 || y_row >= w->out_features, "y_row_stride must be at least out_features");
        if (w8_by_rows(n_rows, w->in_features)) {
            const W8Args a{nullptr, w->device_scales, w->device_bias, y, y_row, n_rows, w->in_features, w->out_features, false, -1, 0};
            const bool vec = aligned(x, 16) && (n_rows == 1 || x_row * es % 16 == 0);
            with_type(dtype, [&](auto t) {
                using T = decltype(t);
                launch_rows<T>(w, a, (const T*)x, x_row, vec, false, stream);
            });
            return;
        }
        const int64_t row = row_stride(1, 0, w->in_features), bytes = n_rows * (row + 4);
        need(workspace && workspace_bytes >= bytes, "the workspace is too small");
        need(aligned(workspace, 16), "the workspace must be 16-byte aligned");
        float* scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + n_rows * row);
        int32_t s = fb2_quantise_rows(n_rows, w->in_features, x, dtype, x_row, workspace, row, scales, stream);
        if (s == FB2_OK) s = fb2_w8_matmul(w, n_rows, workspace, row, scales, y, y_row, dtype, stream);
        if (s != FB2_OK) fail(s, std::string(fb2_last_error()));
    });
}

// ---- verification of drafts -----------------------------------------------------------
namespace {
// CTAs to a row: of at least 2048 ids each where rows leave SMs free, else of 32768
// and up to 8 on each SM (all of a call, us: 161 rows x 131071 bf16 53 with 4 CTAs, 57 with 2,
// 64 with 1; 289 x 50257 fp16 35 with 2, 37 with 4, 41 with 8).
int verify_ranks(int vocab, int rows) {
    int ranks = 1;
    while (ranks < VF_RANKS && vocab > 2048 * ranks &&
           ((int64_t)rows * ranks * 2 <= 2 * 148 || (vocab > 32768 * ranks && (int64_t)rows * ranks * 2 <= 8 * 148)))
        ranks *= 2;
    return ranks;
}
VerifyArgs verify_args(const fb2_verify* v) {
    need(v, "verify arguments are NULL");
    check_dtype(v->dtype);
    need(v->n_seqs >= 0 && v->n_rows >= 0 && v->vocab >= 1, "n_seqs and n_rows must not be negative, vocab positive");
    need(v->max_nodes >= 1 && v->max_nodes <= VF_NODES, "max_nodes must be in 1..1024");
    need(v->vocab <= INT32_MAX - 65536, "vocab is too large");
    need(v->n_seqs <= INT32_MAX / VF_RANKS && v->n_rows <= INT32_MAX / VF_RANKS, "too many rows for one call");
    need(v->device_row_starts || v->n_rows == v->n_seqs, "without row_starts there is one row per sequence");
    need(!(v->device_draft_probs && v->device_parents), "draft_probs go with chains: one draft to a node, parents NULL");
    VerifyArgs a{};
    a.logits = v->device_logits;
    a.probs = v->device_draft_probs;
    a.drafts = v->device_drafts;
    a.starts = v->device_row_starts;
    a.parents = v->device_parents;
    a.uniforms = v->device_uniforms;
    a.temperature = v->device_temperature;
    a.tokens = v->device_tokens;
    a.nodes = v->device_nodes;
    a.counts = v->device_counts;
    a.logits_row = v->logits_row_stride;
    a.probs_row = v->probs_row_stride;
    a.n_seqs = v->n_seqs;
    a.n_rows = v->n_rows;
    a.vocab = v->vocab;
    a.max_nodes = v->max_nodes;
    a.parts = verify_ranks(a.vocab, a.n_rows);
    a.ranks = verify_ranks(a.vocab, a.n_seqs);
    return a;
}
}  // namespace

int32_t fb2_verify_workspace(const fb2_verify* v, int64_t* bytes) {
    return guarded([&] {
        need(bytes, "bytes is NULL");
        const VerifyArgs a = verify_args(v);
        *bytes = (int64_t)a.n_rows * a.parts * (int64_t)sizeof(VerifyRow);
    });
}

int32_t fb2_verify_drafts(const fb2_verify* v, void* stream) {
    return guarded([&] {
        VerifyArgs a = verify_args(v);
        if (a.n_seqs == 0) return;
        need(a.tokens && a.nodes && a.counts, "NULL argument");
        need(a.n_rows == 0 || (a.logits && a.drafts && a.uniforms), "NULL argument");
        need(aligned(a.logits, size_of(v->dtype)) && aligned(a.probs, 4) && aligned(a.drafts, 4) && aligned(a.starts, 4) &&
                 aligned(a.parents, 4) && aligned(a.uniforms, 8) && aligned(a.temperature, 4) && aligned(a.tokens, 4) &&
                 aligned(a.nodes, 4) && aligned(a.counts, 4),
             "a tensor is not aligned to its element size");
        need(a.n_rows == 0 || (v->device_workspace && v->workspace_bytes >= (int64_t)a.n_rows * a.parts * (int64_t)sizeof(VerifyRow)),
             "the workspace is too small");
        need(aligned(v->device_workspace, 16), "the workspace must be 16-byte aligned");
        a.rows = static_cast<VerifyRow*>(v->device_workspace);
        with_type(v->dtype, [&](auto t) {
            using T = decltype(t);
            if (a.n_rows) k_verify_rows<T><<<a.n_rows * a.parts, VF_THREADS, 0, (cudaStream_t)stream>>>(a);
            launched();
            opt_in_smem((const void*)k_verify_walk<T>, VF_NODES * VW_NODE);
            launch_cluster(k_verify_walk<T>, dim3(a.n_seqs * a.ranks), VW_THREADS, a.max_nodes * VW_NODE, a.ranks, a.n_rows > 0, stream, a);
        });
    });
}
