// serving_ops.cu — C ABI of the serving operators: the quantised paged K/V
// cache, attention over it, 4-bit linear layers, logit controls.  Checks of
// arguments and launches; the kernels are in kvq.cuh, kvq_attn.cuh, w4.cuh
// and logit_controls.cuh.
#include <climits>
#include <cmath>
#include <cstdint>

#include "capi.cuh"
#include "kvq.cuh"
#include "kvq_attn.cuh"
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

// lanes of a row at 8 values each, a power of two
int row_lanes(int hd) {
    int w = 2;
    while (w * 8 < hd) w *= 2;
    return w;
}
unsigned row_blocks(int64_t n_rows, int heads, int width) {
    const int64_t blocks = (n_rows * heads * width + KVQ_THREADS - 1) / KVQ_THREADS;
    need(blocks <= INT32_MAX, "too many rows for one call");
    return (unsigned)blocks;
}

}  // namespace

extern "C" {

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
        const int width = row_lanes(view.hd);
        const dim3 grid(row_blocks(n_rows, view.heads, width), 2);
        const bool vec = aligned(k, 16) && aligned(v, 16) && k_row * es % 16 == 0 && k_head * es % 16 == 0 &&
                         v_row * es % 16 == 0 && v_head * es % 16 == 0;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto kernel = view.row_bytes == view.hd ? (vec ? k_kvq_write<T, KVQ_INT8, true> : k_kvq_write<T, KVQ_INT8, false>)
                                                    : (vec ? k_kvq_write<T, KVQ_INT4, true> : k_kvq_write<T, KVQ_INT4, false>);
            kernel<<<grid, KVQ_THREADS, 0, (cudaStream_t)stream>>>(view, n_rows, (const T*)k, (const T*)v, k_row, k_head,
                                                                  v_row, v_head, slots, width);
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
        const int width = row_lanes(view.hd);
        const dim3 grid(row_blocks(n_rows, view.heads, width), 2);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto kernel = view.row_bytes == view.hd ? k_kvq_read<T, KVQ_INT8> : k_kvq_read<T, KVQ_INT4>;
            kernel<<<grid, KVQ_THREADS, 0, (cudaStream_t)stream>>>(view, n_rows, slots, (T*)k, (T*)v, width);
        });
        launched();
    });
}

// ---- attention ---------------------------------------------------------------
namespace {
KvqAttnArgs attn_args(const fb2_kvq_cache* c, const fb2_kvq_attention* a) {
    need(a, "attention arguments are NULL");
    KvqAttnArgs k{};
    k.c = view_of(c);
    check_dtype(a->dtype);
    need(a->n_seqs >= 0 && a->n_rows >= 0, "n_seqs and n_rows must not be negative");
    need(a->n_seqs <= 65535, "n_seqs must be at most 65535");
    need(a->n_heads >= 1 && a->n_heads % c->n_kv_heads == 0, "n_heads must be a positive multiple of n_kv_heads");
    need(a->n_heads <= 65535, "n_heads must be at most 65535");
    need(a->max_pages >= 0 && a->max_len >= 0, "max_pages and max_len must not be negative");
    need(a->max_nodes >= 1 && a->max_nodes <= 65535, "max_nodes must be in 1..65535");
    need(a->device_row_starts || (a->n_rows == a->n_seqs && a->max_nodes == 1),
         "without row_starts there is one row per sequence and max_nodes is 1");
    need(std::isfinite(a->scale), "scale must be finite");
    need(!a->device_mask || (int64_t)a->mask_words * 32 >= a->max_nodes, "mask_words must cover max_nodes");
    need(a->table_stride >= a->max_pages, "table_stride must be at least max_pages");
    const int64_t cap = (int64_t)a->max_pages * c->page_size;
    need(cap <= INT32_MAX, "max_pages * page_size must be at most 2^31 - 1");
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
    k.max_pages = a->max_pages;
    k.max_nodes = a->max_nodes;
    k.max_len = a->max_len && a->max_len < cap ? a->max_len : (int)cap;
    k.mask_words = a->mask_words;
    k.scale = a->scale;
    return k;
}
}  // namespace

int32_t fb2_kvq_attend_workspace(const fb2_kvq_cache* c, const fb2_kvq_attention* a, int64_t* bytes) {
    return guarded([&] {
        need(bytes, "bytes is NULL");
        attn_args(c, a);
        *bytes = 0;
    });
}

int32_t fb2_kvq_attend(const fb2_kvq_cache* c, const fb2_kvq_attention* a, void* stream) {
    return guarded([&] {
        const KvqAttnArgs k = attn_args(c, a);
        if (a->n_seqs == 0 || a->n_rows == 0) return;
        need(k.q && k.out && k.prefix && (k.table || k.max_pages == 0), "NULL argument");
        const size_t es = size_of(a->dtype);
        need(aligned(k.q, es) && aligned(k.lse, 4) && aligned(k.table, 4) && aligned(k.prefix, 4) && aligned(k.starts, 4) &&
                 aligned(k.mask, 4),
             "a tensor is not aligned to its element size");
        need(aligned(k.out, 16), "out must be 16-byte aligned");
        const dim3 grid((k.n_heads + 3) / 4, k.max_nodes, k.n_seqs);
        with_type(a->dtype, [&](auto t) {
            using T = decltype(t);
            auto kernel = k.c.row_bytes == k.c.hd ? k_kvq_attend<T, KVQ_INT8> : k_kvq_attend<T, KVQ_INT4>;
            kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(k);
        });
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
        need(w_row >= v.N, "w_row_stride must be at least out_features");
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

int32_t fb2_w4_matvec_workspace(const fb2_w4_linear* w, int32_t n_rows, int32_t dtype, int64_t* bytes) {
    return guarded([&] {
        w4_view(w);
        check_dtype(dtype);
        need(n_rows >= 0, "n_rows must not be negative");
        need(bytes, "bytes is NULL");
        *bytes = 0;
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
        need(n_rows <= 65535, "n_rows must be at most 65535");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            k_w4_matvec<T><<<dim3((v.N + 3) / 4, n_rows), 128, 0, (cudaStream_t)stream>>>(v, (const T*)x, x_row, (T*)y, y_row);
        });
        launched();
    });
}

// ---- logit controls --------------------------------------------------------------
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
        const dim3 grid((c->vocab + CTL_CHUNK - 1) / CTL_CHUNK, c->n_rows);
        with_type(c->dtype, [&](auto t) {
            using T = decltype(t);
            k_logit_controls<T><<<grid, CTL_THREADS, 0, (cudaStream_t)stream>>>(a);
        });
        launched();
    });
}

}  // extern "C"
