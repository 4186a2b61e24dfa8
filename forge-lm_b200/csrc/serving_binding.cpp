// serving_binding.cpp — the serving operators on torch tensors, as a Python
// extension module (_serving) over the C entry points of forge_b200.h.
//
// A decode step calls these once per layer, and the smallest calls take a few
// microseconds on the GPU; checks, allocations and the call itself are done
// here because the same work in Python took 11 to 17 us a call.  Tensors come
// from and results go to torch's caching allocator, on the current stream of
// the tensors' device; workspaces live for the call (the allocator orders
// their reuse on the stream, and captured calls get theirs from the graph's
// pool).  serving.py holds the documented classes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <memory>
#include <string>

#include "../../include/forge_b200.h"

namespace {

PyObject* g_argument_error = nullptr;  // (status, message)
PyObject* g_check = nullptr;           // raises for a status of the library

struct Refusal {
    std::string message;
};
[[noreturn]] void refuse(std::string message) { throw Refusal{std::move(message)}; }
void need(bool ok, const char* message) {
    if (!ok) refuse(message);
}
struct Raised {};  // a Python exception is set
void status(int32_t s) {
    if (s == FB2_OK) return;
    PyObject* r = PyObject_CallFunction(g_check, "i", (int)s);
    Py_XDECREF(r);
    throw Raised{};
}

// Tells autograd and whoever else counts versions that a call changed t.
void changed(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool needs_gradient(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
// A result of `from`: no gradient is computed, and a backward pass that comes
// to it says so instead of stopping there.
PyObject* result(at::Tensor t, const at::Tensor& from, const char* call) {
    if (needs_gradient(from)) {
        const auto node = std::make_shared<torch::autograd::Error>(std::string(call) + " computes no gradient",
                                                                   torch::autograd::collect_next_edges(from));
        torch::autograd::set_history(t, node);
    }
    return THPVariable_Wrap(std::move(t));
}

// Python errors for what `f` throws
template <class F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refusal& r) {
        if (PyObject* args = Py_BuildValue("(is)", (int)FB2_INVALID_ARG, r.message.c_str())) {
            PyErr_SetObject(g_argument_error, args);
            Py_DECREF(args);
        }
        return nullptr;
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    // its memory holds the values with the other sign
    if (t.is_neg()) refuse(std::string(name) + " must not be a negated view (resolve_neg() makes a tensor of it)");
    return t;
}
int32_t code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return FB2_F32;
        case at::kBFloat16: return FB2_BF16;
        case at::kHalf: return FB2_F16;
        default: refuse("dtype must be float32, bfloat16 or float16");
    }
}
// A contiguous tensor of `type` on CUDA device `index`; null for None.
const at::Tensor* plain(PyObject* o, const char* name, at::ScalarType type, int index) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != index || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor on cuda:" + std::to_string(index));
    return &t;
}
template <class T>
T* data(const at::Tensor* t) {
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
int64_t integer(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(name) + " must be a whole number");
    }
    return v;
}
int32_t small(int64_t v, const char* name) {
    if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(name) + " is out of range");
    return (int32_t)v;
}

// The tensors' device, made current for the call, and its current stream.
struct OnDevice {
    int before, index;
    explicit OnDevice(int i) : before(c10::cuda::current_device()), index(i) {
        if (before != index) c10::cuda::set_device(index);
    }
    ~OnDevice() {
        if (before != index) c10::cuda::set_device(before);
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(index).stream(); }
};
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int index) {
    return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, index), std::nullopt);
}

template <class H>
void destroy(PyObject* capsule) {
    delete static_cast<H*>(PyCapsule_GetPointer(capsule, H::kName));
}
template <class H>
PyObject* capsule(std::unique_ptr<H> h) {
    PyObject* c = PyCapsule_New(h.get(), H::kName, destroy<H>);
    if (c) h.release();
    return c;
}
template <class H>
H& handle(PyObject* o) {
    void* p = PyCapsule_GetPointer(o, H::kName);
    if (!p) throw Raised{};
    return *static_cast<H*>(p);
}

#define ARGS(n)                                                              \
    if (count != (n)) {                                                      \
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", (n), count); \
        return nullptr;                                                      \
    }

// ---- the cache -------------------------------------------------------------------

// A buffer that a handle holds: still of the size and kind that it was made with?
// (resize_, set_ or .data may have changed the tensor since.)
void check_held(const at::Tensor& t, at::ScalarType type, int64_t bytes, int index, const char* name) {
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != index || !t.is_contiguous() ||
        t.numel() * (int64_t)t.element_size() != bytes)
        refuse(std::string(name) + " was given another size, type, layout or device since the object was made");
}

struct Cache {
    static constexpr const char* kName = "forge_b200.cache";
    at::Tensor codes, meta;
    fb2_kvq_cache c{};
    int64_t code_bytes = 0, meta_bytes = 0;
    int index = 0;
    // the cache with the buffers where they are now
    fb2_kvq_cache now() const {
        check_held(codes, at::kByte, code_bytes, index, "codes");
        check_held(meta, at::kInt, meta_bytes, index, "meta");
        fb2_kvq_cache n = c;
        n.device_codes = codes.data_ptr();
        n.device_meta = meta.data_ptr();
        return n;
    }
};

PyObject* cache_new(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(4)  // codes, meta, head_dim, format
    return guarded([&] {
        auto h = std::make_unique<Cache>();
        h->codes = tensor(args[0], "codes");
        h->meta = tensor(args[1], "meta");
        need(h->codes.dim() == 5 && h->codes.size(2) == 2 && h->codes.scalar_type() == at::kByte && h->codes.is_cuda(),
             "codes must be a CUDA uint8 tensor [pages, kv heads, 2, page size, row bytes]");
        h->index = h->codes.get_device();
        plain(args[0], "codes", at::kByte, h->index);
        plain(args[1], "meta", at::kInt, h->index);
        need(h->meta.sizes() == h->codes.sizes().slice(0, 4), "meta must be [pages, kv heads, 2, page size]");
        const int64_t dim = integer(args[2], "head_dim");
        h->c.format = (int32_t)integer(args[3], "format");
        need(dim == h->codes.size(4) * (h->c.format == FB2_KVQ_INT8 ? 1 : 2), "row bytes do not fit head_dim");
        h->c.n_pages = small(h->codes.size(0), "pages");
        h->c.n_kv_heads = small(h->codes.size(1), "kv heads");
        h->c.page_size = small(h->codes.size(3), "page size");
        h->c.head_dim = small(dim, "head_dim");
        status(fb2_kvq_sizes(&h->c, &h->code_bytes, &h->meta_bytes));
        return capsule(std::move(h));
    });
}

// k, v or q: [rows, heads, head_dim] on the cache's device, last dimension contiguous
const at::Tensor& rows_of(const Cache& h, PyObject* o, const char* name, int64_t rows, int64_t heads) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 3 || t.size(0) != rows || t.size(1) != heads || t.size(2) != h.c.head_dim)
        refuse(std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(heads) + ", " +
               std::to_string(h.c.head_dim) + "]");
    if (!t.is_cuda() || t.get_device() != h.index || t.stride(2) != 1)
        refuse(std::string(name) + " must be on cuda:" + std::to_string(h.index) + " with a contiguous last dimension");
    return t;
}

PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(4)  // handle, k, v, slots
    return guarded([&]() -> PyObject* {
        const Cache& h = handle<Cache>(args[0]);
        const at::Tensor* slots = plain(args[3], "slots", at::kInt, h.index);
        need(slots, "slots must be a tensor");
        const int64_t rows = slots->numel();
        const at::Tensor &k = rows_of(h, args[1], "k", rows, h.c.n_kv_heads), &v = rows_of(h, args[2], "v", rows, h.c.n_kv_heads);
        need(k.scalar_type() == v.scalar_type(), "k and v must have the same dtype");
        const int32_t code = code_of(k.scalar_type());
        const fb2_kvq_cache c = h.now();
        OnDevice on(h.index);
        status(fb2_kvq_write(&c, small(rows, "rows"), k.data_ptr(), v.data_ptr(), code, k.stride(0), k.stride(1), v.stride(0),
                             v.stride(1), data<int32_t>(slots), on.stream()));
        changed(h.codes), changed(h.meta);
        Py_RETURN_NONE;
    });
}

PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(3)  // handle, slots, dtype
    return guarded([&]() -> PyObject* {
        const Cache& h = handle<Cache>(args[0]);
        const at::Tensor* slots = plain(args[1], "slots", at::kInt, h.index);
        need(slots, "slots must be a tensor");
        need(args[2] == Py_None || THPDtype_Check(args[2]), "dtype must be a torch dtype");
        const at::ScalarType type = args[2] == Py_None ? at::kFloat : reinterpret_cast<THPDtype*>(args[2])->scalar_type;
        const int32_t code = code_of(type);
        const fb2_kvq_cache c = h.now();
        OnDevice on(h.index);
        const int64_t shape[3] = {slots->numel(), h.c.n_kv_heads, h.c.head_dim};
        at::Tensor k = empty(shape, type, h.index), v = empty(shape, type, h.index);
        status(fb2_kvq_read(&c, small(shape[0], "rows"), data<int32_t>(slots), k.data_ptr(), v.data_ptr(), code, on.stream()));
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
    });
}

PyObject* cache_attend(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(9)  // handle, q, page_table, prefix_lens, starts, mask, scale, max_nodes, max_len
    return guarded([&]() -> PyObject* {
        const Cache& h = handle<Cache>(args[0]);
        const at::Tensor& any = tensor(args[1], "q");
        need(any.dim() == 3, "q must be [rows, heads, head_dim]");
        const int64_t rows = any.size(0), heads = any.size(1);
        const at::Tensor& q = rows_of(h, args[1], "q", rows, heads);
        fb2_kvq_attention a{};
        a.dtype = code_of(q.scalar_type());
        const at::Tensor& table = tensor(args[2], "page_table");
        need(table.dim() == 2 && table.scalar_type() == at::kInt && table.is_cuda() && table.get_device() == h.index &&
                 (table.stride(1) == 1 || table.size(1) <= 1),
             "page_table must be an int32 tensor [sequences, pages] on the cache's device with contiguous rows");
        const int64_t seqs = table.size(0), pages = table.size(1);
        const at::Tensor* prefix = plain(args[3], "prefix_lens", at::kInt, h.index);
        need(prefix && prefix->numel() == seqs, "prefix_lens must have one entry per sequence");
        const at::Tensor* starts = plain(args[4], "starts", at::kInt, h.index);
        const at::Tensor* mask = plain(args[5], "mask", at::kInt, h.index);
        if (mask) {
            need(mask->dim() == 2 && mask->size(0) == rows && mask->size(1) > 0, "mask must be [rows, words]");
            a.mask_words = small(mask->size(1), "mask words");
        }
        int64_t nodes = args[7] == Py_None ? -1 : integer(args[7], "max_nodes");
        if (starts) {
            need(starts->numel() == seqs + 1, "starts must have one entry more than there are sequences");
            // a sequence has no more rows than the call, nor than its mask has bits
            if (args[7] == Py_None) nodes = std::max<int64_t>(mask ? std::min(rows, 32 * mask->size(1)) : rows, 1);
        } else {
            need(args[7] == Py_None || nodes == 1, "starts is needed for more than one row per sequence");
            nodes = 1;
        }
        a.scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)h.c.head_dim)) : (float)PyFloat_AsDouble(args[6]);
        if (args[6] != Py_None && PyErr_Occurred()) throw Raised{};
        a.max_len = args[8] == Py_None ? 0 : small(integer(args[8], "max_len"), "max_len");
        a.max_nodes = small(nodes, "max_nodes");
        a.n_seqs = small(seqs, "sequences");
        a.n_rows = small(rows, "rows");
        a.n_heads = small(heads, "heads");
        a.max_pages = small(pages, "pages");
        a.q_row_stride = q.stride(0);
        a.q_head_stride = q.stride(1);
        a.table_stride = seqs > 1 ? table.stride(0) : pages;  // one row may have any stride
        a.device_q = q.data_ptr();
        a.device_page_table = data<int32_t>(&table);
        a.device_prefix_lens = data<int32_t>(prefix);
        a.device_row_starts = data<int32_t>(starts);
        a.device_mask = data<uint32_t>(mask);
        const fb2_kvq_cache c = h.now();
        OnDevice on(h.index);
        int64_t size = 0;
        status(fb2_kvq_attend_workspace(&c, &a, &size));
        at::Tensor out = empty({rows, heads, h.c.head_dim}, q.scalar_type(), h.index), lse = empty({rows, heads}, at::kFloat, h.index), work;
        if (size) work = empty({size}, at::kByte, h.index);
        a.device_out = out.data_ptr();
        a.device_lse = static_cast<float*>(lse.data_ptr());
        a.device_workspace = size ? work.data_ptr() : nullptr;
        a.workspace_bytes = size;
        // fresh memory: rows of no sequence are filled by the call, or here where it has no room for that
        a.fill_rest = starts && seqs > 0 && seqs <= 65534;
        if (starts && !a.fill_rest) out.zero_(), lse.fill_(-INFINITY);
        status(fb2_kvq_attend(&c, &a, on.stream()));
        return Py_BuildValue("(NN)", result(std::move(out), q, "QuantKvCache.attend"), result(std::move(lse), q, "QuantKvCache.attend"));
    });
}

// ---- 4-bit linear layers ------------------------------------------------------------

struct Linear {
    static constexpr const char* kName = "forge_b200.linear";
    at::Tensor codes, meta, bias;
    fb2_w4_linear w{};
    int64_t code_bytes = 0, meta_bytes = 0;
    int index = 0;
    fb2_w4_linear now() const {
        check_held(codes, at::kInt, code_bytes, index, "codes");
        check_held(meta, at::kInt, meta_bytes, index, "meta");
        fb2_w4_linear n = w;
        n.device_codes = codes.data_ptr();
        n.device_meta = meta.data_ptr();
        if (bias.defined()) {
            check_held(bias, at::kFloat, (int64_t)w.out_features * 4, index, "bias");
            n.device_bias = static_cast<const float*>(bias.data_ptr());
        }
        return n;
    }
};

PyObject* linear_new(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(6)  // codes, meta, bias, in_features, out_features, group
    return guarded([&] {
        auto h = std::make_unique<Linear>();
        h->codes = tensor(args[0], "codes");
        h->meta = tensor(args[1], "meta");
        need(h->codes.is_cuda(), "codes must be a CUDA tensor");
        h->index = h->codes.get_device();
        plain(args[0], "codes", at::kInt, h->index);
        plain(args[1], "meta", at::kInt, h->index);
        if (const at::Tensor* b = plain(args[2], "bias", at::kFloat, h->index)) h->bias = *b;
        h->w.in_features = small(integer(args[3], "in_features"), "in_features");
        h->w.out_features = small(integer(args[4], "out_features"), "out_features");
        h->w.group = small(integer(args[5], "group"), "group");
        need(!h->bias.defined() || h->bias.numel() == h->w.out_features, "bias must have out_features entries");
        status(fb2_w4_sizes(&h->w, &h->code_bytes, &h->meta_bytes));
        if (h->codes.numel() * 4 != h->code_bytes || h->meta.numel() * 4 != h->meta_bytes)
            refuse("codes and meta must have " + std::to_string(h->code_bytes) + " and " + std::to_string(h->meta_bytes) + " bytes");
        return capsule(std::move(h));
    });
}

PyObject* linear_pack(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(2)  // handle, w
    return guarded([&]() -> PyObject* {
        const Linear& h = handle<Linear>(args[0]);
        const at::Tensor& w = tensor(args[1], "w");
        need(w.dim() == 2 && w.is_cuda() && w.get_device() == h.index && w.size(0) == h.w.in_features && w.size(1) == h.w.out_features &&
                 (w.stride(1) == 1 || w.size(1) == 1),
             "w must be a CUDA tensor [in, out] with contiguous rows");
        const int32_t code = code_of(w.scalar_type());
        const fb2_w4_linear l = h.now();
        OnDevice on(h.index);
        const int64_t row = w.size(0) > 1 ? w.stride(0) : w.size(1);  // one row may have any stride
        status(fb2_w4_pack(&l, w.data_ptr(), code, row, on.stream()));
        changed(h.codes), changed(h.meta);
        Py_RETURN_NONE;
    });
}

PyObject* linear_call(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(2)  // handle, x
    return guarded([&]() -> PyObject* {
        const Linear& h = handle<Linear>(args[0]);
        const at::Tensor& x = tensor(args[1], "x");
        const int64_t k = h.w.in_features, n = h.w.out_features;
        if (x.dim() == 0 || x.size(-1) != k || !x.is_cuda() || x.get_device() != h.index)
            refuse("x must be [..., " + std::to_string(k) + "] on cuda:" + std::to_string(h.index));
        const int32_t code = code_of(x.scalar_type());
        at::Tensor other;
        if (x.dim() != 2) other = x.reshape({-1, k});
        const at::Tensor& flat = x.dim() == 2 ? x : other;
        need(flat.stride(1) == 1 || k == 1, "x must have a contiguous last dimension");
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = n;
        const fb2_w4_linear l = h.now();
        OnDevice on(h.index);
        at::Tensor y = empty(shape, x.scalar_type(), h.index), work;
        const int32_t rows = small(flat.size(0), "rows");
        int64_t size = 0;
        status(fb2_w4_matvec_workspace(&l, rows, code, &size));
        if (size) work = empty({size}, at::kByte, h.index);
        status(fb2_w4_matvec(&l, rows, flat.data_ptr(), flat.stride(0), y.data_ptr(), n, code, size ? work.data_ptr() : nullptr,
                             size, on.stream()));
        return result(std::move(y), x, "W4Linear");
    });
}

// ---- logit controls --------------------------------------------------------------------

PyObject* controls(PyObject*, PyObject* const* args, Py_ssize_t count) {
    // logits, tokens, token_starts, repetition, presence, frequency, bias_ids,
    // bias_values, bias_starts, allowed, mask_rows, out
    ARGS(12)
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(args[0], "logits");
        need(logits.dim() == 2 && logits.is_cuda() && (logits.stride(1) == 1 || logits.size(1) <= 1),
             "logits must be a CUDA tensor [rows, vocab] with contiguous rows");
        const int64_t rows = logits.size(0), vocab = logits.size(1);
        const int index = logits.get_device();
        fb2_logit_control c{};
        c.dtype = code_of(logits.scalar_type());
        const at::Tensor* tokens = plain(args[1], "tokens", at::kInt, index);
        const at::Tensor* token_starts = plain(args[2], "token_starts", at::kInt, index);
        const at::Tensor* repetition = plain(args[3], "repetition", at::kFloat, index);
        const at::Tensor* presence = plain(args[4], "presence", at::kFloat, index);
        const at::Tensor* frequency = plain(args[5], "frequency", at::kFloat, index);
        const at::Tensor* ids = plain(args[6], "bias_ids", at::kInt, index);
        const at::Tensor* values = plain(args[7], "bias_values", at::kFloat, index);
        const at::Tensor* bias_starts = plain(args[8], "bias_starts", at::kInt, index);
        const at::Tensor* allowed = plain(args[9], "allowed", at::kInt, index);
        const at::Tensor* mask_rows = plain(args[10], "mask_rows", at::kInt, index);
        need(!tokens == !token_starts, "tokens and token_starts go together");
        need(tokens || (!repetition && !presence && !frequency), "penalties need tokens");
        need(!token_starts || token_starts->numel() == rows + 1, "token_starts must have rows + 1 entries");
        need(!ids == !values && !ids == !bias_starts, "bias_ids, bias_values and bias_starts go together");
        need(!ids || (values->numel() == ids->numel() && bias_starts->numel() == rows + 1),
             "bias_values must have one entry per id and bias_starts rows + 1");
        for (const at::Tensor* t : {repetition, presence, frequency, mask_rows})
            need(!t || t->numel() == rows, "repetition, presence, frequency and mask_rows must have one entry per row");
        if (allowed) {
            need(allowed->dim() == 2 && (mask_rows || allowed->size(0) == rows),
                 "allowed must be [masks, words], one mask per row without mask_rows");
            c.n_masks = small(allowed->size(0), "masks");
            c.mask_words = small(allowed->size(1), "mask words");
        } else {
            need(!mask_rows, "mask_rows needs allowed");
        }
        OnDevice on(index);
        at::Tensor fresh;
        const at::Tensor* out = args[11] == Py_None ? nullptr : &tensor(args[11], "out");
        need(!out || !(needs_gradient(logits) || needs_gradient(*out)), "out= goes without gradients: detach() or no_grad()");
        if (out)
            need(out->sizes() == logits.sizes() && out->scalar_type() == logits.scalar_type() && out->is_cuda() &&
                     out->get_device() == index && (out->stride(1) == 1 || vocab <= 1),
                 "out must have the logits' shape, dtype, device and contiguous rows");
        else
            out = &(fresh = empty({rows, vocab}, logits.scalar_type(), index));
        c.device_logits = logits.data_ptr();
        c.device_out = out->data_ptr();
        c.device_tokens = data<int32_t>(tokens);
        c.device_token_starts = data<int32_t>(token_starts);
        c.device_repetition = data<float>(repetition);
        c.device_presence = data<float>(presence);
        c.device_frequency = data<float>(frequency);
        c.device_bias_ids = data<int32_t>(ids);
        c.device_bias_values = data<float>(values);
        c.device_bias_starts = data<int32_t>(bias_starts);
        c.device_allowed = data<uint32_t>(allowed);
        c.device_mask_rows = data<int32_t>(mask_rows);
        c.logits_row_stride = logits.stride(0);
        c.out_row_stride = out->stride(0);
        c.n_tokens = tokens ? tokens->numel() : 0;
        c.n_biases = ids ? ids->numel() : 0;
        c.n_rows = small(rows, "rows");
        c.vocab = small(vocab, "vocab");
        if (rows && vocab) status(fb2_logit_controls(&c, on.stream()));
        if (fresh.defined()) return result(std::move(fresh), logits, "logit_controls");
        changed(*out);
        return Py_NewRef(args[11]);
    });
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t count) {
    ARGS(2)  // ArgumentError, check
    Py_XSETREF(g_argument_error, Py_NewRef(args[0]));
    Py_XSETREF(g_check, Py_NewRef(args[1]));
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(setup),      METHOD(cache_new),   METHOD(cache_write), METHOD(cache_read), METHOD(cache_attend),
                          METHOD(linear_new), METHOD(linear_pack), METHOD(linear_call), METHOD(controls),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_serving", "The serving operators on torch tensors (see serving.py).", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&kModule); }
