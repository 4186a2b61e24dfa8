// serving_ops.cu — C ABI of the serving operators: the quantised paged K/V
// cache, attention over it, 4-bit linear layers, logit controls.  Checks of
// arguments and launches; the kernels are in kvq.cuh, kvq_attn.cuh, w4.cuh
// and logit_controls.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <set>

#include "../../include/forge_b200_testing.h"
#include "capi.cuh"
#include "kvq.cuh"
#include "kvq_attn.cuh"
#include "kvq_attn_tc.cuh"
#include "logit_controls.cuh"
#include "w4.cuh"

using namespace fb2;

namespace {

void need(bool ok, const char* msg) {
    if (!ok) fail(FB2_INVALID_ARG, msg);
}
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }
int log2_of(int v) {
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}
size_t size_of(int dtype) { return dtype == FB2_F32 ? 4 : 2; }
void check_dtype(int dtype) { need(dtype == FB2_F32 || dtype == FB2_BF16 || dtype == FB2_F16, "dtype must be FB2_F32, FB2_BF16 or FB2_F16"); }

// f(T{}) for the element type of `dtype`
template <class F>
void with_type(int dtype, F&& f) {
    if (dtype == FB2_F32)
        f(float{});
    else if (dtype == FB2_BF16)
        f(__nv_bfloat16{});
    else
        f(__half{});
}

void launched() { CK(cudaGetLastError()); }

// Dynamic shared memory above 48 KB, once per kernel and device.
void opt_in_smem(const void* kernel, int bytes) {
    static std::mutex lock;
    static std::set<std::pair<const void*, int>> done;
    int device = 0;
    CK(cudaGetDevice(&device));
    std::lock_guard<std::mutex> hold(lock);
    if (done.count({kernel, device})) return;
    CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert({kernel, device});
}

void check_cache_sizes(const fb2_kvq_cache* c) {
    need(c, "cache is NULL");
    need(c->format == FB2_KVQ_INT8 || c->format == FB2_KVQ_INT4, "format must be FB2_KVQ_INT8 or FB2_KVQ_INT4");
    need(c->n_pages >= 0, "n_pages must not be negative");
    need(pow2(c->page_size) && c->page_size >= 8 && c->page_size <= 1024, "page_size must be a power of two in 8..1024");
    need(c->n_kv_heads >= 1 && c->n_kv_heads <= 65535, "n_kv_heads must be in 1..65535");
    need(c->head_dim >= 16 && c->head_dim <= 256 && c->head_dim % 16 == 0, "head_dim must be a multiple of 16 in 16..256");
    need((int64_t)c->n_pages * c->page_size <= INT32_MAX, "the cache must have at most 2^31 - 1 slots");
}

KvqView view_of(const fb2_kvq_cache* c) {
    check_cache_sizes(c);
    need(c->n_pages == 0 || (c->device_codes && c->device_meta), "a cache buffer is NULL");
    need(aligned(c->device_codes, 16) && aligned(c->device_meta, 16), "the cache buffers must be 16-byte aligned");
    KvqView v;
    v.codes = static_cast<unsigned char*>(c->device_codes);
    v.meta = static_cast<uint32_t*>(c->device_meta);
    v.n_slots = c->n_pages * c->page_size;
    v.page_shift = log2_of(c->page_size);
    v.heads = c->n_kv_heads;
    v.hd = c->head_dim;
    v.row_bytes = c->format == FB2_KVQ_INT8 ? c->head_dim : c->head_dim / 2;
    return v;
}

// log2 of the lanes of a row at 32 values each
int row_shift(int hd) {
    int s = 0;
    while ((32 << s) < hd) s++;
    return s;
}
dim3 row_grid(int n_rows, int heads, int shift) {
    need(n_rows <= INT32_MAX - KVQ_THREADS, "n_rows must be at most 2^31 - 129");  // rows are counted in 32 bits
    const int per = KVQ_THREADS >> shift;
    return dim3((unsigned)(((int64_t)n_rows + per - 1) / per), heads, 2);
}

}  // namespace

int32_t fb2_kvq_sizes(const fb2_kvq_cache* c, int64_t* code_bytes, int64_t* meta_bytes) {
    return guarded([&] {
        check_cache_sizes(c);
        need(code_bytes && meta_bytes, "NULL argument");
        const int64_t rows = (int64_t)c->n_pages * c->page_size * c->n_kv_heads * 2;
        *code_bytes = rows * (c->format == FB2_KVQ_INT8 ? c->head_dim : c->head_dim / 2);
        *meta_bytes = rows * 4;
    });
}

int32_t fb2_kvq_write(const fb2_kvq_cache* c, int32_t n_rows, const void* k, const void* v, int32_t dtype, int64_t k_row,
                      int64_t k_head, int64_t v_row, int64_t v_head, const int32_t* slots, void* stream) {
    return guarded([&] {
        const KvqView view = view_of(c);
        check_dtype(dtype);
        need(n_rows >= 0, "n_rows must not be negative");
        if (n_rows == 0 || c->n_pages == 0) return;
        need(k && v && slots, "NULL argument");
        const size_t es = size_of(dtype);
        need(aligned(k, es) && aligned(v, es) && aligned(slots, 4), "a tensor is not aligned to its element size");
        const int shift = row_shift(view.hd);
        const dim3 grid = row_grid(n_rows, view.heads, shift);
        const bool vec = aligned(k, 16) && aligned(v, 16) && k_row * es % 16 == 0 && k_head * es % 16 == 0 &&
                         v_row * es % 16 == 0 && v_head * es % 16 == 0;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto kernel = view.row_bytes == view.hd ? (vec ? k_kvq_write<T, KVQ_INT8, true> : k_kvq_write<T, KVQ_INT8, false>)
                                                    : (vec ? k_kvq_write<T, KVQ_INT4, true> : k_kvq_write<T, KVQ_INT4, false>);
            kernel<<<grid, KVQ_THREADS, 0, (cudaStream_t)stream>>>(view, n_rows, (const T*)k, (const T*)v, k_row, k_head,
                                                                  v_row, v_head, slots, shift);
        });
        launched();
    });
}

int32_t fb2_kvq_read(const fb2_kvq_cache* c, int32_t n_rows, const int32_t* slots, void* k, void* v, int32_t dtype,
                     void* stream) {
    return guarded([&] {
        const KvqView view = view_of(c);
        check_dtype(dtype);
        need(n_rows >= 0, "n_rows must not be negative");
        if (n_rows == 0) return;
        need(k && v && slots, "NULL argument");
        need(aligned(k, 16) && aligned(v, 16), "k and v must be 16-byte aligned");
        need(aligned(slots, 4), "slots is not aligned to its element size");
        const int shift = row_shift(view.hd);
        const dim3 grid = row_grid(n_rows, view.heads, shift);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto kernel = view.row_bytes == view.hd ? k_kvq_read<T, KVQ_INT8> : k_kvq_read<T, KVQ_INT4>;
            kernel<<<grid, KVQ_THREADS, 0, (cudaStream_t)stream>>>(view, n_rows, slots, (T*)k, (T*)v, shift);
        });
        launched();
    });
}

// ---- attention ---------------------------------------------------------------
namespace {
// Rows to a block, chunks of positions, warps.  Measured (us):
// - Blocks of 128 rows on tcgen05 tiles where a K/V head has more than 32 rows,
//   else blocks of 8 or 16 on mma.sync tiles.  4 sequences of 8192 int8
//   positions, 8 K/V heads, bf16, head_dim 64 and 128: 32 rows 44 and 65 in
//   blocks of 16, 53 and 70 on tcgen05 tiles; 64 rows 73 and 111, 60 and 80.
// - Chunks of a size that gives some 888 CTAs (512 of the larger kind): 16
//   sequences of 40 to 65 K positions take 292 with chunks of 1024, 254 with
//   4096, 275 with 8192; 4 trees over 9 to 33 K, 263 with 2048, 257 with 4096,
//   450 with 16384.  Each chunk costs its start and its part of the merge: at
//   least 512 positions, and at most 64 chunks (one row over 60000 positions:
//   51, 29, 23, 23 with 256, 512, 1024, 2048).
// - A cache of up to 1024 positions is one chunk for blocks of 8 rows (12 heads
//   over 576: 7.4; 8.5 with 512, 8.0 with 256), and cut finer for a few blocks
//   of 16, which take longer per position (4 blocks over 1000: 19.5 with 256,
//   25.4 with 512; 128 blocks: 34 and 25).
// - 8 warps to a block of 8 rows where no SM gets two CTAs (60000 positions:
//   22.8, 26.5 with 4; 12 heads over 576: 7.4 and 8.7), else 4 (384 CTAs of up
//   to 1023 positions: 14.6, 22.1 with 8).
void plan_attention(KvqAttnArgs& k) {
    const int64_t rows = (int64_t)k.max_nodes * k.share;
    const bool tc = k.dtype != FB2_F32 && k.c.hd <= 128 && rows > 32;
    k.block_rows = tc ? KVT_ROWS : rows > 8 ? 16 : 8;
    k.row_blocks = (int)((rows + k.block_rows - 1) / k.block_rows);
    const int64_t units = (int64_t)k.n_seqs * k.c.heads * k.row_blocks;
    // counted as if all sequences were of max_len
    int64_t chunk = k.max_len * units / (tc ? 512 : 888), least = 512;
    if (!tc) {
        if (k.block_rows == 8 && k.max_len <= 1024) least = 1024;
        if (k.block_rows == 16 && k.max_len <= 1024 && units <= 16) least = 256;
        least = std::max<int64_t>(least, k.max_len / 64);
    }
    chunk = std::min<int64_t>(std::max(chunk, least), std::max<int64_t>(tc ? 8192 : 4096, k.max_len / 64));
    chunk = (chunk + 127) / 128 * 128;
    k.chunk = (int)chunk;
    k.splits = std::max(1, (int)((k.max_len + chunk - 1) / chunk));
    k.warps = k.block_rows == 8 && units * k.splits <= 148 ? 8 : 4;
}

KvqAttnArgs attn_args(const fb2_kvq_cache* c, const fb2_kvq_attention* a) {
    need(a, "attention arguments are NULL");
    KvqAttnArgs k{};
    k.c = view_of(c);
    check_dtype(a->dtype);
    need(a->n_seqs >= 0 && a->n_rows >= 0, "n_seqs and n_rows must not be negative");
    need(a->n_seqs <= (a->fill_rest ? 65534 : 65535), "n_seqs must be at most 65535, 65534 with fill_rest");
    need(a->n_heads >= 1 && a->n_heads % c->n_kv_heads == 0, "n_heads must be a positive multiple of n_kv_heads");
    need(a->n_heads <= 65535, "n_heads must be at most 65535");
    need(a->max_pages >= 0 && a->max_len >= 0, "max_pages and max_len must not be negative");
    need(a->max_nodes >= 1 && (int64_t)a->max_nodes * a->n_heads <= INT32_MAX - 1024, "max_nodes must be in 1..2^31 / n_heads");
    need(a->device_row_starts || (a->n_rows == a->n_seqs && a->max_nodes == 1),
         "without row_starts there is one row per sequence and max_nodes is 1");
    need(std::isfinite(a->scale), "scale must be finite");
    need(!a->device_mask || (int64_t)a->mask_words * 32 >= a->max_nodes, "mask_words must cover max_nodes");
    need(a->table_stride == 0 || a->table_stride >= a->max_pages, "table_stride must be 0 or at least max_pages");
    const int64_t cap = (int64_t)a->max_pages * c->page_size;
    need(cap <= INT32_MAX, "max_pages * page_size must be at most 2^31 - 1");
    // groups of 8 rows are counted in 32 bits (a cache of that size has over 270 GB)
    need((int64_t)c->n_pages * c->page_size / 8 * 2 * c->n_kv_heads < UINT32_MAX, "the cache is too large");
    k.q = a->device_q;
    k.out = a->device_out;
    k.lse = a->device_lse;
    k.table = a->device_page_table;
    k.prefix = a->device_prefix_lens;
    k.starts = a->device_row_starts;
    k.mask = a->device_mask;
    k.q_row = a->q_row_stride;
    k.q_head = a->q_head_stride;
    k.table_stride = a->table_stride;
    k.n_seqs = a->n_seqs;
    k.n_rows = a->n_rows;
    k.n_heads = a->n_heads;
    k.share = a->n_heads / c->n_kv_heads;
    k.dtype = a->dtype;
    k.max_nodes = a->max_nodes;
    k.max_len = c->n_pages == 0 ? 0 : a->max_len && a->max_len < cap ? a->max_len : (int)cap;  // no pages: no buffers to address
    // positions are counted in 32 bits, some thousands past the last one
    need(k.max_len <= INT32_MAX - 65535, "max_len (0: max_pages * page_size) must be at most 2^31 - 65536");
    k.mask_words = a->mask_words;
    k.scale = a->scale;
    k.fill = a->fill_rest != 0 && a->device_row_starts;
    plan_attention(k);
    return k;
}

int64_t attn_workspace(const KvqAttnArgs& k) {
    if (k.splits == 1) return 0;
    const int64_t parts = (int64_t)k.n_rows * k.n_heads * k.splits;
    return (parts * 8 + 15) / 16 * 16 + parts * k.c.hd * 4;
}

template <int HD, int FMT, int NT, bool SPLIT, int WARPS>
void launch_attend(const KvqAttnArgs& k, cudaStream_t stream) {
    using S = KvaShape<HD, FMT, NT, SPLIT, WARPS>;
    auto kernel = k_kvq_attend<HD, FMT, NT, SPLIT, WARPS>;
    if (S::SMEM > 48 * 1024) opt_in_smem((const void*)kernel, S::SMEM);
    const int64_t blocks = (int64_t)k.row_blocks * k.splits * k.c.heads;
    need(blocks <= INT32_MAX, "too many rows for one call");
    kernel<<<dim3((unsigned)blocks, k.n_seqs + k.fill), WARPS * 32, S::SMEM, stream>>>(k);
}
template <int HD, int FMT>
void launch_attend(const KvqAttnArgs& k, cudaStream_t stream) {
    const bool split = k.dtype == FB2_F32;
    if (k.block_rows == 16)
        split ? launch_attend<HD, FMT, 2, true, 4>(k, stream) : launch_attend<HD, FMT, 2, false, 4>(k, stream);
    else if (k.warps == 8)
        split ? launch_attend<HD, FMT, 1, true, 8>(k, stream) : launch_attend<HD, FMT, 1, false, 8>(k, stream);
    else
        split ? launch_attend<HD, FMT, 1, true, 4>(k, stream) : launch_attend<HD, FMT, 1, false, 4>(k, stream);
}
template <int HD, int FMT>
void launch_attend_tc(const KvqAttnArgs& k, cudaStream_t stream) {
    auto kernel = k_kvq_attend_tc<HD, FMT>;
    constexpr int smem = KvtShape<HD, FMT>::SMEM;
    opt_in_smem((const void*)kernel, smem);
    const int64_t blocks = (int64_t)k.row_blocks * k.splits * k.c.heads;
    need(blocks <= INT32_MAX, "too many rows for one call");
    kernel<<<dim3((unsigned)blocks, k.n_seqs + k.fill), KVT_LAUNCH, smem, stream>>>(k);
}
template <int FMT>
void launch_attend(const KvqAttnArgs& k, cudaStream_t stream) {
    if (k.block_rows == KVT_ROWS) {
        if (k.c.hd <= 64)
            launch_attend_tc<64, FMT>(k, stream);
        else
            launch_attend_tc<128, FMT>(k, stream);
        return;
    }
    if (k.c.hd <= 64)
        launch_attend<64, FMT>(k, stream);
    else if (k.c.hd <= 128)
        launch_attend<128, FMT>(k, stream);
    else
        launch_attend<256, FMT>(k, stream);
}
}  // namespace

int32_t fb2_kvq_attend_workspace(const fb2_kvq_cache* c, const fb2_kvq_attention* a, int64_t* bytes) {
    return guarded([&] {
        need(bytes, "bytes is NULL");
        *bytes = attn_workspace(attn_args(c, a));
    });
}

// test hook: what the next launch on tcgen05 tiles withholds
namespace {
std::atomic<int> g_withhold_tile{-1};
std::atomic<int64_t> g_withhold_wait_ns{0};
}  // namespace
int32_t fb2_test_kvq_withhold(int32_t tile, int64_t wait_ns) {
    return guarded([&] {
        need(tile >= 0 && wait_ns > 0 && wait_ns <= (int64_t)kTcTimeoutNs, "bad hook arguments");
        g_withhold_wait_ns = wait_ns;
        g_withhold_tile = tile;
    });
}

int32_t fb2_kvq_attend(const fb2_kvq_cache* c, const fb2_kvq_attention* a, void* stream) {
    return guarded([&] {
        const KvqAttnArgs k = attn_args(c, a);
        if (a->n_seqs == 0 || a->n_rows == 0) return;
        need(k.q && k.out && k.prefix && (k.table || a->max_pages == 0), "NULL argument");
        const size_t es = size_of(a->dtype);
        need(aligned(k.q, es) && aligned(k.lse, 4) && aligned(k.table, 4) && aligned(k.prefix, 4) && aligned(k.starts, 4) &&
                 aligned(k.mask, 4),
             "a tensor is not aligned to its element size");
        need(aligned(k.out, 16), "out must be 16-byte aligned");
        KvqAttnArgs args = k;
        const int64_t bytes = attn_workspace(k);
        if (bytes) {
            need(a->device_workspace && a->workspace_bytes >= bytes, "the workspace is too small");
            need(aligned(a->device_workspace, 16), "the workspace must be 16-byte aligned");
            const int64_t parts = (int64_t)k.n_rows * k.n_heads * k.splits;
            args.part_ml = static_cast<float2*>(a->device_workspace);
            args.part_o = reinterpret_cast<float*>(static_cast<char*>(a->device_workspace) + (parts * 8 + 15) / 16 * 16);
        }
        args.withhold = k.block_rows == KVT_ROWS ? g_withhold_tile.exchange(-1) : -1;
        args.wait_ns = args.withhold < 0 ? kTcTimeoutNs : (unsigned long long)g_withhold_wait_ns.load();
        if (c->format == FB2_KVQ_INT8)
            launch_attend<KVQ_INT8>(args, (cudaStream_t)stream);
        else
            launch_attend<KVQ_INT4>(args, (cudaStream_t)stream);
        launched();
        if (bytes) {
            const int64_t blocks = ((int64_t)k.max_nodes * k.n_heads + 3) / 4;
            launch_pdl(k_kvq_attend_merge, dim3((unsigned)blocks, k.n_seqs), dim3(128), 0, (cudaStream_t)stream, args);
        }
        launched();
    });
}

// ---- 4-bit linear layers --------------------------------------------------------
namespace {
W4View w4_view(const fb2_w4_linear* w) {
    need(w, "linear is NULL");
    need(w->in_features >= 1 && w->out_features >= 1, "in_features and out_features must be positive");
    need(w->in_features <= INT32_MAX - 127 && w->out_features <= INT32_MAX - 15, "in_features or out_features is too large");
    need(w->group == 32 || w->group == 64 || w->group == 128, "group must be 32, 64 or 128");
    W4View v;
    v.codes = static_cast<const uint4*>(w->device_codes);
    v.meta = static_cast<const uint32_t*>(w->device_meta);
    v.bias = w->device_bias;
    v.K = w->in_features;
    v.N = w->out_features;
    v.group_shift = log2_of(w->group);
    v.k64 = (v.K + 63) / 64;
    v.groups = (v.K + w->group - 1) / w->group;
    return v;
}
void check_w4_buffers(const fb2_w4_linear* w) {
    need(w->device_codes && w->device_meta, "a weight buffer is NULL");
    need(aligned(w->device_codes, 16) && aligned(w->device_meta, 16), "the weight buffers must be 16-byte aligned");
}
}  // namespace

int32_t fb2_w4_sizes(const fb2_w4_linear* w, int64_t* code_bytes, int64_t* meta_bytes) {
    return guarded([&] {
        const W4View v = w4_view(w);
        need(code_bytes && meta_bytes, "NULL argument");
        const int64_t blocks = (v.N + 15) / 16;
        *code_bytes = blocks * v.k64 * 512;
        *meta_bytes = blocks * v.groups * 64;
    });
}

int32_t fb2_w4_pack(const fb2_w4_linear* w, const void* dense, int32_t dtype, int64_t w_row, void* stream) {
    return guarded([&] {
        const W4View v = w4_view(w);
        check_w4_buffers(w);
        check_dtype(dtype);
        need(dense, "w is NULL");
        need(aligned(dense, size_of(dtype)), "w is not aligned to its element size");
        need(w_row == 0 || w_row >= v.N, "w_row_stride must be 0 or at least out_features");
        const int64_t units = (int64_t)((v.N + 15) / 16) * v.groups * 8;
        need((units + 127) / 128 <= INT32_MAX, "the layer is too large for one call");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            k_w4_pack<T><<<(unsigned)((units + 127) / 128), 128, 0, (cudaStream_t)stream>>>(
                (uint32_t*)w->device_codes, (uint32_t*)w->device_meta, (const T*)dense, w_row, v.K, v.N, v.group_shift,
                v.k64, v.groups);
        });
        launched();
    });
}

namespace {
// Few rows take the 8-bit tiles (up to 4 tiles of 8 columns, one column for a
// digit), more the 16-bit ones (one column, three for fp32).
int w4_digits_of(int dtype) { return dtype == FB2_F32 ? 4 : 3; }
int w4_parts(int dtype) { return dtype == FB2_F32 ? 3 : 1; }
struct W4Shape {
    bool narrow;
    int tiles;   // of 8 columns: all (narrow), of a chunk (wide)
    int per;     // rows of a chunk
    int chunks;
};
W4Shape w4_shape(int rows, int dtype) {
    const int64_t digits = (int64_t)rows * w4_digits_of(dtype), cols = (int64_t)rows * w4_parts(dtype);
    if (digits <= 32) return {true, (int)((digits + 7) / 8), rows, 1};
    const int tiles = cols <= 16 ? 2 : 4, per = tiles * 8 / w4_parts(dtype);
    return {false, tiles, per, (int)(((int64_t)rows + per - 1) / per)};
}

// Blocks of 16 outputs per warp, and CTAs per cluster (which share the inputs).
// More blocks per warp spread the columns' cost (16384 x 16384, one bf16 row:
// 37.7 us with 1, 34.3 with 2, 31.9 with 4) where enough CTAs are left (4096 x
// 4096: 7.6, 7.4, 8.7 us).  A cluster's sums cost 1 to 3 us, which pays only
// where less than half of the SMs have a CTA (16384 x 64: 10.5 us alone, 6.6
// by 4; 4096 x 4096: 7.4 alone, 7.7 by 2; 32 rows, 8192 x 2048: 62 alone, 25
// by 4, 33 by 8).
struct W4Plan {
    int rt, ranks;
};
W4Plan w4_plan(const W4View& v, const W4Shape& shape) {
    const int blocks = (v.N + 15) / 16, units = (v.k64 + 1) / 2;
    W4Plan p{1, 1};
    if (shape.narrow) {
        p.rt = blocks >= 512 ? 4 : blocks >= 128 ? 2 : 1;
        if (shape.tiles > 1) p.rt = std::min(p.rt, shape.tiles > 2 ? 1 : 2);  // registers
        const int ctas = (blocks + p.rt - 1) / p.rt;
        while (p.ranks < 8 && ctas * p.ranks * 2 <= 148 && p.ranks * 4 * W4_WARPS <= units) p.ranks *= 2;
    } else {
        const int ctas = (blocks + W4_WARPS - 1) / W4_WARPS;
        while (p.ranks < 4 && (int64_t)ctas * shape.chunks * p.ranks * 2 <= 148 && p.ranks * 4 <= units) p.ranks *= 2;
    }
    return p;
}
struct W4Workspace {
    int64_t columns, sums;
};
W4Workspace w4_workspace(const W4View& v, const W4Shape& s) {
    const int64_t units = (int64_t)(v.k64 + 1) / 2 * s.chunks;
    if (s.narrow) return {units * s.tiles * W4_COL, 0};
    return {units * s.tiles * 2048, units * (128 >> v.group_shift) * s.tiles * 32};
}
// x in fixed point is made by the product itself where each warp has one or
// two units of inputs, else by a launch before it (768 x 2304 fp32: 3.3 and 4.1
// us; 1024 x 4096 bf16: 3.7 and 5.0; 4096 x 4096 fp16: 9.3 and 5.8; 16384 x
// 16384 bf16: 44 and 29)
bool w4_direct(const W4View& v, int64_t rows, int dtype) { return rows * w4_digits_of(dtype) <= 8 && v.k64 <= 32; }

template <class K, class... A>
void launch_cluster(K kernel, dim3 grid, int threads, int smem, int ranks, bool early, cudaStream_t stream, A... args) {
    if (smem > 48 * 1024) opt_in_smem((const void*)kernel, smem);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 2 : 1;
    CK(cudaLaunchKernelEx(&cfg, kernel, args...));
}
template <class T, int RT, int NT, bool DIRECT>
void launch_narrow(const W4View& v, int ranks, const T* x, int64_t x_row, const unsigned char* columns, int rows, T* y,
                   int64_t y_row, int vec, cudaStream_t stream) {
    const unsigned grid = ((v.N + 15) / 16 + RT - 1) / RT * ranks;
    launch_cluster(k_w4_narrow<T, RT, NT, DIRECT>, dim3(grid), W4_WARPS * 32, W4Narrow<RT, NT, DIRECT>::SMEM, ranks, !DIRECT, stream,
                   v, x, (long long)x_row, columns, rows, y, (long long)y_row, vec);
}
template <class T, int NT, bool DIRECT, class... A>
void launch_narrow(const W4View& v, const W4Plan& p, A... args) {
    if constexpr (NT == 1)
        if (p.rt == 4) return launch_narrow<T, 4, NT, DIRECT>(v, p.ranks, args...);
    if constexpr (NT <= 2)
        if (p.rt == 2) return launch_narrow<T, 2, NT, DIRECT>(v, p.ranks, args...);
    launch_narrow<T, 1, NT, DIRECT>(v, p.ranks, args...);
}
template <class T, int NT, int GS>
void launch_wide(const W4View& v, const W4Shape& s, int ranks, const uint4* columns, const float* sums, int rows, T* y,
                 int64_t y_row, cudaStream_t stream) {
    launch_cluster(k_w4_wide<T, NT, GS>, dim3((unsigned)(((v.N + 15) / 16 + W4_WARPS - 1) / W4_WARPS * ranks), s.chunks),
                   W4_WARPS * 32, W4Wide<NT>::SMEM, ranks, true, stream, v, columns, sums, rows, s.per, y, (long long)y_row);
}
template <class T, int NT, class... A>
void launch_wide(const W4View& v, const W4Shape& s, A... args) {
    if (v.group_shift == 5)
        launch_wide<T, NT, 5>(v, s, args...);
    else if (v.group_shift == 6)
        launch_wide<T, NT, 6>(v, s, args...);
    else
        launch_wide<T, NT, 7>(v, s, args...);
}
template <class T, class... A>
void launch_wide(const W4View& v, const W4Shape& s, const W4Plan& p, A... args) {
    if (s.tiles == 2)
        launch_wide<T, 2>(v, s, p.ranks, args...);
    else
        launch_wide<T, 4>(v, s, p.ranks, args...);
}
}  // namespace

int32_t fb2_w4_matvec_workspace(const fb2_w4_linear* w, int32_t n_rows, int32_t dtype, int64_t* bytes) {
    return guarded([&] {
        const W4View v = w4_view(w);
        check_dtype(dtype);
        need(n_rows >= 0, "n_rows must not be negative");
        need(bytes, "bytes is NULL");
        *bytes = 0;
        if (n_rows == 0 || w4_direct(v, n_rows, dtype)) return;
        const W4Workspace ws = w4_workspace(v, w4_shape(n_rows, dtype));
        *bytes = ws.columns + ws.sums;
    });
}

int32_t fb2_w4_matvec(const fb2_w4_linear* w, int32_t n_rows, const void* x, int64_t x_row, void* y, int64_t y_row,
                      int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const W4View v = w4_view(w);
        check_dtype(dtype);
        need(n_rows >= 0, "n_rows must not be negative");
        if (n_rows == 0) return;
        check_w4_buffers(w);
        need(x && y, "NULL argument");
        const size_t es = size_of(dtype);
        need(aligned(x, es) && aligned(y, es) && aligned(v.bias, 4), "a tensor is not aligned to its element size");
        need(n_rows == 1 || y_row >= v.N, "y_row_stride must be at least out_features");
        int64_t bytes = 0;
        fb2_w4_matvec_workspace(w, n_rows, dtype, &bytes);
        need(bytes == 0 || (workspace && workspace_bytes >= bytes), "the workspace is too small");
        need(aligned(workspace, 16), "the workspace must be 16-byte aligned");
        const int vec = aligned(x, 16) && (n_rows == 1 || x_row * es % 16 == 0);
        const cudaStream_t st = (cudaStream_t)stream;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            const W4Shape shape = w4_shape(n_rows, dtype);
            const W4Plan plan = w4_plan(v, shape);
            const T* xt = (const T*)x;
            T* yt = (T*)y;
            if (bytes == 0) {
                launch_narrow<T, 1, true>(v, plan, xt, x_row, (const unsigned char*)nullptr, n_rows, yt, y_row, vec, st);
                return;
            }
            const W4Workspace ws = w4_workspace(v, shape);
            unsigned char* columns = static_cast<unsigned char*>(workspace);
            float* sums = reinterpret_cast<float*>(columns + ws.columns);
            const int units = (v.k64 + 1) / 2;
            const int64_t blocks = ((int64_t)units * shape.tiles * shape.chunks + 3) / 4;
            need(blocks <= INT32_MAX && shape.chunks <= 65535, "too many rows for one call");
            if (!shape.narrow) {
                k_w4_columns<T><<<(unsigned)blocks, 128, 0, st>>>(xt, x_row, n_rows, shape.per, v.K, units, shape.tiles, shape.chunks,
                                                                 v.group_shift, (uint4*)columns, sums, vec);
                launched();
                launch_wide<T>(v, shape, plan, (const uint4*)columns, (const float*)sums, n_rows, yt, y_row, st);
                return;
            }
            k_w4_digits<T><<<(unsigned)blocks, 128, 0, st>>>(xt, x_row, n_rows, v.K, units, shape.tiles, v.group_shift, columns, vec);
            launched();
            const unsigned char* cols = columns;
            if (shape.tiles == 1)
                launch_narrow<T, 1, false>(v, plan, xt, x_row, cols, n_rows, yt, y_row, vec, st);
            else if (shape.tiles == 2)
                launch_narrow<T, 2, false>(v, plan, xt, x_row, cols, n_rows, yt, y_row, vec, st);
            else if (shape.tiles == 3)
                launch_narrow<T, 3, false>(v, plan, xt, x_row, cols, n_rows, yt, y_row, vec, st);
            else
                launch_narrow<T, 4, false>(v, plan, xt, x_row, cols, n_rows, yt, y_row, vec, st);
        });
    });
}

// ---- logit controls --------------------------------------------------------------
namespace {
// Whether a row of logits shares entries with a row of out that is not its own in place.
bool rows_collide(const fb2_logit_control* c, int64_t size) {
    const int64_t from = (int64_t)(intptr_t)c->device_logits, to = (int64_t)(intptr_t)c->device_out, row = c->vocab * size;
    const int64_t si = c->n_rows > 1 ? c->logits_row_stride * size : 0, so = c->n_rows > 1 ? c->out_row_stride * size : row;
    const int64_t last = c->n_rows - 1;
    if (from + last * si + row <= to || to + last * so + row <= from || (from == to && (si == so || last == 0))) return false;
    for (int64_t r = 0; r <= last; r++) {
        const int64_t at = from + r * si - to;  // out's rows lie at q * so, so >= row
        for (int64_t q = std::max<int64_t>(0, at / so - 1); q <= std::min(last, at / so + 1); q++)
            if (at < q * so + row && q * so < at + row) return true;
    }
    return false;
}
}  // namespace

int32_t fb2_logit_controls(const fb2_logit_control* c, void* stream) {
    return guarded([&] {
        need(c, "controls are NULL");
        check_dtype(c->dtype);
        need(c->n_rows >= 0 && c->vocab >= 0, "n_rows and vocab must not be negative");
        need(c->n_rows <= 65535, "n_rows must be at most 65535");
        need(c->vocab <= INT32_MAX - 65536, "vocab is too large");
        if (c->n_rows == 0 || c->vocab == 0) return;
        need(c->device_logits && c->device_out, "NULL argument");
        const size_t es = size_of(c->dtype);
        need(aligned(c->device_logits, es) && aligned(c->device_out, es), "a tensor is not aligned to its element size");
        need(c->n_rows == 1 || (c->out_row_stride >= c->vocab && c->logits_row_stride >= 0),
             "out_row_stride must be at least vocab");
        need(!rows_collide(c, (int64_t)es), "out must be the logits, row for row, or not overlap them");
        need(!c->device_tokens || (c->device_token_starts && c->n_tokens >= 0), "tokens need token_starts and n_tokens");
        need(!c->device_bias_ids || (c->device_bias_values && c->device_bias_starts && c->n_biases >= 0),
             "bias_ids need bias_values, bias_starts and n_biases");
        need(!c->device_allowed || (c->n_masks >= 0 && (int64_t)c->mask_words * 32 >= c->vocab), "mask_words must cover vocab");
        for (const void* p : {(const void*)c->device_tokens, (const void*)c->device_token_starts,
                              (const void*)c->device_repetition, (const void*)c->device_presence,
                              (const void*)c->device_frequency, (const void*)c->device_bias_ids,
                              (const void*)c->device_bias_values, (const void*)c->device_bias_starts,
                              (const void*)c->device_allowed, (const void*)c->device_mask_rows})
            need(aligned(p, 4), "a tensor is not aligned to its element size");
        ControlArgs a{c->device_logits, c->device_out, c->device_tokens, c->device_token_starts, c->device_repetition,
                      c->device_presence, c->device_frequency, c->device_bias_ids, c->device_bias_values,
                      c->device_bias_starts, c->device_allowed, c->device_mask_rows, c->logits_row_stride,
                      c->out_row_stride, c->n_tokens, c->n_biases, c->n_rows, c->vocab, c->n_masks, c->mask_words};
        const bool copies = c->device_allowed || c->device_out != c->device_logits || c->out_row_stride != c->logits_row_stride;
        // a table with half of its slots free for a row that has all of the lists
        int slots = 1024;
        while (slots < CTL_SLOTS && slots / 2 < c->n_tokens + c->n_biases) slots *= 2;
        // two CTAs on each SM, of at least 2048 entries each
        const int slices = std::max(1, std::min(2 * 148 / std::max(c->n_rows, 1), c->vocab / 2048));
        const int slice = ((c->vocab + slices - 1) / slices + 31) / 32 * 32;
        with_type(c->dtype, [&](auto t) {
            using T = decltype(t);
            if (slots * 8 > 48 * 1024) opt_in_smem((const void*)k_logit_controls<T>, slots * 8);
            k_logit_controls<T><<<dim3((c->vocab + slice - 1) / slice, c->n_rows), CTL_THREADS, slots * 8, (cudaStream_t)stream>>>(
                a, slice, slots, copies);
        });
        launched();
    });
}
