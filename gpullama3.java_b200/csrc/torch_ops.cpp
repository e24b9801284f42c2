// torch_ops.cpp -- the operators of operators.cu on torch tensors (operators.py has their documentation): checks of the tensors, the current stream, results from torch's allocator.
// A call through Python's ctypes costs 15 to 20 us of host time, more than most of these kernels run; here it is about 5.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>

#include "../../include/b200llama.h"

namespace py = pybind11;
using at::Tensor;
typedef std::optional<Tensor> Maybe;

#define NEED(ok, ...)                                                  \
    do {                                                               \
        if (C10_UNLIKELY(!(ok))) throw py::value_error(c10::str(__VA_ARGS__)); \
    } while (0)

namespace {

py::object *raise_error = nullptr; // native._raise(code, message); lives as long as the interpreter

[[noreturn]] void refused(int code, const char *message) {
    (*raise_error)(code, message);
    throw py::value_error(message); // (raise_error has raised)
}

std::string shape(const Tensor &t) { return t.defined() ? c10::str(t.sizes(), " of ", t.scalar_type(), " on ", t.device()) : "None"; }

int type_of(at::ScalarType t, const char *what) {
    switch (t) {
    case at::kFloat: return B200_GGML_F32;
    case at::kHalf: return B200_GGML_F16;
    case at::kBFloat16: return B200_GGML_BF16;
    default: NEED(false, what, ": FP32, FP16 or BF16 is wanted, got ", t);
    }
    return -1;
}

// There are no derivatives: a graph that led through a call, or a tangent carried into it, would end there without a word.
void outside_graph(const Tensor &t, const char *name) {
    NEED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name, " carries a forward-mode tangent, and the operators have none: detach it");
    NEED(!t.requires_grad() || !at::GradMode::is_enabled(), name, " requires a gradient, and the operators have none: detach it, or call under torch.no_grad()");
}

// A new tensor on a device, without the dispatcher (1 us of at::empty's 2).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, int device) {
    return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

struct Cache {
    b200_kv4 *kv;
    int64_t slots, context, kv_heads, head_size;
    int device;
    Cache(b200_kv4 *kv, int64_t slots, int64_t context, int64_t kv_heads, int64_t head_size, int device)
        : kv(kv), slots(slots), context(context), kv_heads(kv_heads), head_size(head_size), device(device) {}
    Cache(const Cache &) = delete;
    Cache &operator=(const Cache &) = delete;
    ~Cache() { free(); }
    void alive() const {
        if (!kv) refused(B200_ERR_STATE, "the cache has been freed");
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
    void check(int rc) const {
        if (rc != B200_OK) refused(rc, b200_kv4_last_error(kv));
    }

    // rows [n, heads, head_size] whose heads lie one behind the other: entries between rows
    int64_t rows(const Tensor &t, const char *name, int64_t n, int64_t heads) const {
        NEED(t.defined() && t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == head_size, name, ": [", n, ", ", heads, ", ", head_size, "] is wanted, got ", shape(t));
        NEED(t.is_cuda() && t.get_device() == device, name, " is on ", t.device(), ", the cache on cuda:", device);
        outside_graph(t, name);
        NEED(n == 0 || (t.stride(2) == 1 && (t.stride(1) == head_size || heads == 1)), name, ": the heads of a row have to lie one behind the other");
        return n > 1 ? t.stride(0) : heads * head_size;
    }
    const int32_t *indices(const Maybe &t, const char *name, int64_t n) const {
        if (!t) return nullptr;
        NEED(t->defined(), name, " are wanted");
        NEED(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n, name, ": ", n, " entries of int32 are wanted, got ", t->sizes(), " of ", t->scalar_type());
        NEED(t->is_cuda() && t->get_device() == device, name, " is on ", t->device(), ", the cache on cuda:", device);
        NEED(n <= 1 || t->stride(0) == 1, name, " has to be contiguous");
        return t->data_ptr<int32_t>();
    }
    const float *vector(const Maybe &t, const char *name, int64_t least, int64_t width) const {
        if (!t) return nullptr;
        outside_graph(*t, name);
        NEED(t->scalar_type() == at::kFloat && t->is_cuda() && t->get_device() == device && t->is_contiguous(), name, ": a contiguous FP32 tensor on cuda:", device, " is wanted");
        NEED(least ? t->dim() == 2 && t->size(0) >= least && t->size(1) == width : t->dim() == 1 && t->size(0) == width, name, ": has the shape ", t->sizes());
        return t->data_ptr<float>();
    }
    static int32_t rows_of(int64_t n) {
        NEED(n <= INT32_MAX, n, " rows in one call");
        return (int32_t)n;
    }

    Maybe append(const Tensor &k, const Tensor &v, const Tensor &positions, const Maybe &q, const Maybe &slot, const Maybe &q_norm, const Maybe &k_norm, double eps, const Maybe &cos,
                 const Maybe &sin, const std::string &layout, const Maybe &q_out) const {
        alive();
        NEED(k.defined() && v.defined() && k.dim() == 3, "k: [n, ", kv_heads, ", ", head_size, "] is wanted, got ", shape(k));
        const int64_t n = k.size(0);
        b200_kv4_append_args a = {};
        a.n = rows_of(n);
        a.type = type_of(k.scalar_type(), "k");
        NEED(v.scalar_type() == k.scalar_type(), "k and v have the same type: got ", k.scalar_type(), " and ", v.scalar_type());
        NEED(layout == "half" || layout == "interleaved", "layout ", layout);
        a.rope_layout = layout == "half" ? B200_ROPE_HALF : B200_ROPE_INTERLEAVED;
        a.eps = (float)eps;
        a.k_stride = rows(k, "k", n, kv_heads);
        a.v_stride = rows(v, "v", n, kv_heads);
        a.k = k.data_ptr();
        a.v = v.data_ptr();
        a.positions = indices(positions, "positions", n);
        a.slots = indices(slot, "slots", n);
        Maybe out = q_out;
        if (q) {
            NEED(q->scalar_type() == k.scalar_type() && q->dim() == 3, "q: rows of k's type are wanted");
            a.heads = rows_of(q->size(1));
            a.q_stride = rows(*q, "q", n, a.heads);
            a.q = q->data_ptr();
            if (!out) out = fresh({n, a.heads, head_size}, at::kFloat, device);
            NEED(out->scalar_type() == at::kFloat, "q_out is FP32");
            a.q_out_stride = rows(*out, "q_out", n, a.heads);
            a.q_out = out->data_ptr<float>();
        } else NEED(!q_out && !q_norm, "q_out and q_norm belong to q");
        a.q_norm = vector(q_norm, "q_norm", 0, head_size);
        a.k_norm = vector(k_norm, "k_norm", 0, head_size);
        NEED(cos.has_value() == sin.has_value(), "a rotation needs cos and sin");
        a.cos = vector(cos, "cos", context, head_size / 2);
        a.sin = vector(sin, "sin", context, head_size / 2);
        if (n) check(b200_kv4_append(kv, &a, stream()));
        return out;
    }

    Tensor attention(const Tensor &q, const Tensor &positions, const Maybe &slot, std::optional<double> scale, int64_t window, int64_t max_len, int64_t chunk, at::ScalarType dtype,
                     const Maybe &given) const {
        alive();
        NEED(q.defined() && q.dim() == 3 && q.scalar_type() == at::kFloat, "q: FP32 rows [n, heads, head_size] are wanted, got ", shape(q));
        NEED(q.size(1) > 0 && q.size(1) % kv_heads == 0, q.size(1), " query heads over ", kv_heads, " key/value heads");
        NEED(window >= 0 && max_len >= 0 && chunk >= 0, "a negative window, length or chunk");
        const int64_t n = q.size(0);
        b200_kv4_attention_args a = {};
        a.out_type = type_of(given ? given->scalar_type() : dtype, "results");
        a.n = rows_of(n);
        a.heads = rows_of(q.size(1));
        a.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
        a.max_len = (int32_t)std::min<int64_t>(max_len, INT32_MAX);
        a.chunk = (int32_t)std::min<int64_t>(chunk, INT32_MAX);
        a.q_stride = rows(q, "q", n, a.heads);
        a.positions = indices(positions, "positions", n);
        a.slots = indices(slot, "slots", n);
        const Tensor out = given ? *given : fresh({n, a.heads, head_size}, dtype, device);
        a.out_stride = rows(out, "out", n, a.heads);
        a.q = q.data_ptr<float>();
        a.out = out.data_ptr();
        a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)head_size));
        if (n == 0) return out;
        Tensor work; // from the stream's own pool: calls on other streams, and captured graphs, have theirs
        if ((a.workspace_bytes = b200_kv4_attention_workspace(kv, &a)) > 0) {
            work = fresh({(int64_t)(a.workspace_bytes / 4)}, at::kFloat, device);
            a.workspace = work.data_ptr<float>();
        }
        check(b200_kv4_attention(kv, &a, stream()));
        return out;
    }

    std::pair<Tensor, Tensor> read(const Tensor &positions, const Maybe &slot, at::ScalarType dtype) const {
        alive();
        b200_kv4_read_args a = {};
        a.type = type_of(dtype, "results");
        NEED(positions.defined() && positions.dim() == 1, "positions: one an entry");
        const int64_t n = positions.size(0);
        a.n = rows_of(n);
        a.positions = indices(positions, "positions", n);
        a.slots = indices(slot, "slots", n);
        Tensor k = fresh({n, kv_heads, head_size}, dtype, device), v = fresh({n, kv_heads, head_size}, dtype, device);
        a.k = k.data_ptr();
        a.v = v.data_ptr();
        if (n) check(b200_kv4_read(kv, &a, stream()));
        return {k, v};
    }

    void reset() const {
        alive();
        check(b200_kv4_reset(kv, stream()));
    }
    int64_t bytes() const { return b200_kv4_device_bytes(kv); }
    void free() { // waits for the device: not with the interpreter's lock, and not with a pointer that another thread could still use
        b200_kv4 *gone = kv;
        kv = nullptr;
        if (!gone) return;
        py::gil_scoped_release others;
        b200_kv4_free(gone);
    }
};

Cache *create(int64_t slots, int64_t context, int64_t kv_heads, int64_t head_size, int64_t device) {
    NEED(std::max({slots, context, kv_heads, head_size}) <= INT32_MAX && std::min({slots, context, kv_heads, head_size}) >= INT32_MIN, "sizes outside 32 bits");
    b200_kv4 *kv = nullptr;
    char err[256] = "";
    int rc;
    {
        py::gil_scoped_release others; // (it waits for the device)
        rc = b200_kv4_create((int32_t)slots, (int32_t)context, (int32_t)kv_heads, (int32_t)head_size, (int32_t)device, &kv, err, sizeof err);
    }
    if (rc != B200_OK) refused(rc, err);
    return new Cache(kv, slots, context, kv_heads, head_size, (int)device);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> log_probs(const Tensor &logits, const Maybe &targets, int64_t top) {
    NEED(logits.defined() && logits.dim() == 2 && logits.is_cuda(), "logits: rows [rows, vocab] on a GPU are wanted, got ", shape(logits));
    outside_graph(logits, "logits");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    b200_log_probs_args a = {};
    a.type = type_of(logits.scalar_type(), "logits");
    NEED(rows <= INT32_MAX && vocab <= INT32_MAX, "too many rows or logits");
    NEED(vocab > 0 && top >= 0 && top <= 32 && top <= vocab, top, " alternatives of ", vocab, " logits (at most 32)");
    NEED(rows == 0 || vocab == 1 || logits.stride(1) == 1, "the logits of a row have to lie one behind the other");
    a.device = logits.get_device();
    if (targets) {
        NEED(targets->scalar_type() == at::kInt && targets->dim() == 1 && targets->size(0) == rows, "targets: ", rows, " entries of int32 are wanted, got ", targets->sizes(), " of ",
                          targets->scalar_type());
        NEED(targets->is_cuda() && targets->get_device() == a.device && (rows <= 1 || targets->stride(0) == 1), "targets are contiguous and on ", logits.device());
        a.targets = targets->data_ptr<int32_t>();
    }
    Tensor lp = fresh({rows}, at::kFloat, a.device), entropy = fresh({rows}, at::kFloat, a.device), ids = fresh({rows, top}, at::kInt, a.device), values = fresh({rows, top}, at::kFloat, a.device);
    if (rows) {
        a.logits = logits.data_ptr();
        a.row_stride = rows > 1 ? logits.stride(0) : vocab;
        a.rows = (int32_t)rows;
        a.vocab = (int32_t)vocab;
        a.top = (int32_t)top;
        a.logprobs = lp.data_ptr<float>();
        a.entropy = entropy.data_ptr<float>();
        if (top) {
            a.top_ids = ids.data_ptr<int32_t>();
            a.top_logprobs = values.data_ptr<float>();
        }
        char err[256] = "";
        const int rc = b200_log_probs(&a, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream(), err, sizeof err);
        if (rc != B200_OK) refused(rc, err);
    }
    return {lp, entropy, ids, values};
}

// Checks of the calls on a pool of pages and of the verification (the 4-bit cache has its own, with its messages).
const int32_t *int_tensor(const Tensor &t, const char *name, int device, at::IntArrayRef sizes) {
    NEED(t.defined() && t.scalar_type() == at::kInt && t.sizes() == sizes, name, ": ", sizes, " of int32 is wanted, got ", shape(t));
    NEED(t.is_cuda() && t.get_device() == device, name, " is on ", t.device(), ", the call on cuda:", device);
    NEED(t.is_contiguous(), name, " has to be contiguous");
    return t.data_ptr<int32_t>();
}

struct Paged {
    Tensor keys, values;
    int64_t pages, page_size, kv_heads, head_size;
    int device;
    b200_paged_cache cache;
    Paged(const Tensor &k, const Tensor &v) : keys(k), values(v) {
        NEED(k.defined() && v.defined() && k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "keys and values: two of [pages, kv_heads, page_size, head_size] of one type are wanted, got ",
             shape(k), " and ", shape(v));
        NEED(k.is_cuda() && v.is_cuda() && k.get_device() == v.get_device(), "keys and values lie on one GPU: got ", k.device(), " and ", v.device());
        NEED(k.is_contiguous() && v.is_contiguous(), "keys and values have to be contiguous");
        outside_graph(k, "keys");
        outside_graph(v, "values");
        for (int i = 0; i < 4; i++) NEED(k.size(i) <= INT32_MAX, "sizes outside 32 bits");
        pages = k.size(0); kv_heads = k.size(1); page_size = k.size(2); head_size = k.size(3);
        device = k.get_device();
        cache = {k.data_ptr(), v.data_ptr(), (int32_t)pages, (int32_t)page_size, (int32_t)kv_heads, (int32_t)head_size, type_of(k.scalar_type(), "keys and values"), device};
        // what the library refuses of a cache it refuses here
        b200_paged_append_args none = {};
        none.rope_layout = B200_ROPE_HALF;
        char err[256] = "";
        const int rc = b200_paged_append(&cache, &none, nullptr, err, sizeof err);
        if (rc != B200_OK) refused(rc, err);
    }
    at::ScalarType dtype() const { return keys.scalar_type(); }
    // The memory as it is now: the tensors are the caller's too, who may free or move what they lie in (storage().resize_) between calls.
    const void *place(const Tensor &t, const char *name) const {
        outside_graph(t, name);
        NEED(t.sizes() == at::IntArrayRef({pages, kv_heads, page_size, head_size}) && t.is_contiguous() && t.scalar_type() == (cache.type == B200_GGML_F16 ? at::kHalf : at::kBFloat16) && t.get_device() == device, name,
             " are no longer the tensor of the cache's shape, type and device: ", shape(t));
        NEED(t.storage().nbytes() >= (size_t)(t.storage_offset() + t.numel()) * 2, name, ": their memory has been taken away");
        return t.data_ptr();
    }
    b200_paged_cache now() const {
        b200_paged_cache c = cache;
        c.keys = const_cast<void *>(place(keys, "keys"));
        c.values = const_cast<void *>(place(values, "values"));
        return c;
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

    // rows [n, heads, head_size] whose heads lie one behind the other: entries between rows
    int64_t rows(const Tensor &t, const char *name, int64_t n, int64_t heads) const {
        NEED(t.defined() && t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == head_size, name, ": [", n, ", ", heads, ", ", head_size, "] is wanted, got ", shape(t));
        NEED(t.is_cuda() && t.get_device() == device, name, " is on ", t.device(), ", the cache on cuda:", device);
        outside_graph(t, name);
        NEED(n == 0 || (t.stride(2) == 1 && (t.stride(1) == head_size || heads == 1)), name, ": the heads of a row have to lie one behind the other");
        return n > 1 ? t.stride(0) : heads * head_size;
    }
    const float *floats(const Maybe &t, const char *name) const {
        if (!t) return nullptr;
        outside_graph(*t, name);
        NEED(t->scalar_type() == at::kFloat && t->is_cuda() && t->get_device() == device && t->is_contiguous(), name, ": a contiguous FP32 tensor on cuda:", device, " is wanted");
        return t->data_ptr<float>();
    }
    const float *norm(const Maybe &t, const char *name) const {
        if (t) NEED(t->dim() == 1 && t->size(0) == head_size, name, ": has the shape ", t->sizes());
        return floats(t, name);
    }
    template <typename A> void places(A &a, int64_t n, const Tensor &positions, const Tensor &tables, const Maybe &sequences) const {
        NEED(n <= INT32_MAX, n, " rows in one call");
        a.n = (int32_t)n;
        a.positions = int_tensor(positions, "positions", device, {n});
        a.sequences = sequences ? int_tensor(*sequences, "sequences", device, {n}) : nullptr;
        NEED(tables.defined() && tables.scalar_type() == at::kInt && tables.dim() == 2, "tables: [sequences, pages] of int32 is wanted, got ", shape(tables));
        NEED(tables.is_cuda() && tables.get_device() == device, "tables are on ", tables.device(), ", the cache on cuda:", device);
        NEED(tables.size(0) <= INT32_MAX && tables.size(1) <= INT32_MAX, "sizes outside 32 bits");
        NEED(tables.size(1) <= 1 || tables.size(0) == 0 || tables.stride(1) == 1, "the pages of a table have to lie one behind the other");
        a.tables = tables.data_ptr<int32_t>();
        a.n_sequences = (int32_t)tables.size(0);
        a.table_width = (int32_t)tables.size(1);
        a.table_stride = tables.size(0) > 1 ? tables.stride(0) : tables.size(1);
    }

    Maybe append(const Tensor &k, const Tensor &v, const Tensor &positions, const Tensor &tables, const Maybe &sequences, const Maybe &q, const Maybe &q_norm, const Maybe &k_norm, double eps,
                 const Maybe &cos, const Maybe &sin, const std::string &layout, const Maybe &q_out) const {
        NEED(k.defined() && v.defined() && k.dim() == 3, "k: [n, ", kv_heads, ", ", head_size, "] is wanted, got ", shape(k));
        const int64_t n = k.size(0);
        b200_paged_append_args a = {};
        places(a, n, positions, tables, sequences);
        a.type = type_of(k.scalar_type(), "k");
        NEED(v.scalar_type() == k.scalar_type(), "k and v have the same type: got ", k.scalar_type(), " and ", v.scalar_type());
        NEED(layout == "half" || layout == "interleaved", "layout ", layout);
        a.rope_layout = layout == "half" ? B200_ROPE_HALF : B200_ROPE_INTERLEAVED;
        a.eps = (float)eps;
        a.k_stride = rows(k, "k", n, kv_heads);
        a.v_stride = rows(v, "v", n, kv_heads);
        a.k = k.data_ptr();
        a.v = v.data_ptr();
        Maybe out = q_out;
        if (q) {
            NEED(q->defined() && q->scalar_type() == k.scalar_type() && q->dim() == 3, "q: rows of k's type are wanted");
            NEED(q->size(1) <= INT32_MAX, "sizes outside 32 bits");
            a.heads = (int32_t)q->size(1);
            a.q_stride = rows(*q, "q", n, a.heads);
            a.q = q->data_ptr();
            if (!out) out = fresh({n, a.heads, head_size}, dtype(), device);
            NEED(out->defined() && out->scalar_type() == dtype(), "q_out is of the cache's type, ", dtype());
            NEED(n == 0 || out->data_ptr() != q->data_ptr(), "q_out may not overlap q");
            a.q_out_stride = rows(*out, "q_out", n, a.heads);
            a.q_out = out->data_ptr();
        } else NEED(!q_out && !q_norm, "q_out and q_norm belong to q");
        a.q_norm = norm(q_norm, "q_norm");
        a.k_norm = norm(k_norm, "k_norm");
        NEED(cos.has_value() == sin.has_value(), "a rotation needs cos and sin");
        if (cos) {
            NEED(cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->size(1) > 0 && 2 * cos->size(1) <= head_size, "cos and sin: [positions, up to ", head_size / 2, "] are wanted, got ", shape(*cos), " and ",
                 shape(*sin));
            a.cos = floats(cos, "cos");
            a.sin = floats(sin, "sin");
            a.rope_dims = (int32_t)(2 * cos->size(1));
            a.rope_rows = (int32_t)std::min<int64_t>(cos->size(0), INT32_MAX);
            if (a.rope_rows == 0) return out; // every row is padding
        }
        if (n) {
            char err[256] = "";
            const b200_paged_cache here = now();
            const int rc = b200_paged_append(&here, &a, stream(), err, sizeof err);
            if (rc != B200_OK) refused(rc, err);
        }
        return out;
    }

    Tensor attention(const Tensor &q, const Tensor &positions, const Tensor &tables, const Maybe &sequences, std::optional<double> scale, int64_t window, int64_t max_len, int64_t chunk,
                     std::optional<at::ScalarType> dtype_, const Maybe &given) const {
        NEED(q.defined() && q.dim() == 3 && q.scalar_type() == dtype(), "q: rows [n, heads, head_size] of the cache's type, ", dtype(), ", are wanted, got ", shape(q));
        NEED(q.size(1) > 0 && q.size(1) % kv_heads == 0, q.size(1), " query heads over ", kv_heads, " key/value heads");
        NEED(window >= 0 && max_len >= 0 && chunk >= 0, "a negative window, length or chunk");
        const int64_t n = q.size(0);
        b200_paged_attention_args a = {};
        places(a, n, positions, tables, sequences);
        if (given) NEED(given->defined(), "out is wanted");
        const at::ScalarType type = given ? given->scalar_type() : dtype_ ? *dtype_ : dtype();
        a.out_type = type_of(type, "results");
        NEED(q.size(1) <= INT32_MAX, "sizes outside 32 bits");
        a.heads = (int32_t)q.size(1);
        a.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
        a.max_len = (int32_t)std::min<int64_t>(max_len, INT32_MAX);
        a.chunk = (int32_t)std::min<int64_t>(chunk, INT32_MAX);
        a.q_stride = rows(q, "q", n, a.heads);
        const Tensor out = given ? *given : fresh({n, a.heads, head_size}, type, device);
        a.out_stride = rows(out, "out", n, a.heads);
        a.q = q.data_ptr();
        a.out = out.data_ptr();
        a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)head_size));
        if (n == 0) return out;
        Tensor work; // from the stream's own pool: calls on other streams, and captured graphs, have theirs
        const b200_paged_cache here = now();
        if ((a.workspace_bytes = b200_paged_attention_workspace(&here, &a)) > 0) {
            work = fresh({(int64_t)(a.workspace_bytes / 4)}, at::kFloat, device);
            a.workspace = work.data_ptr();
        }
        char err[256] = "";
        const int rc = b200_paged_attention(&here, &a, stream(), err, sizeof err);
        if (rc != B200_OK) refused(rc, err);
        return out;
    }
};

std::pair<Tensor, Tensor> verify_drafts(const Tensor &logits, const Tensor &drafts, const Maybe &uniforms, const Maybe &draft_logits, double temperature) {
    NEED(logits.defined() && logits.dim() == 3 && logits.is_cuda(), "logits: [sequences, drafts + 1, vocab] on a GPU is wanted, got ", shape(logits));
    outside_graph(logits, "logits");
    const int64_t S = logits.size(0), K = logits.size(1) - 1, V = logits.size(2);
    NEED(K >= 0 && V > 0 && S <= INT32_MAX && K <= INT32_MAX && V <= INT32_MAX, "logits: [sequences, drafts + 1, vocab] is wanted, got ", shape(logits));
    NEED(V == 1 || logits.stride(2) == 1, "the logits of a row have to lie one behind the other");
    b200_verify_drafts_args a = {};
    a.device = logits.get_device();
    a.type = type_of(logits.scalar_type(), "logits");
    a.sequences = (int32_t)S;
    a.drafts = (int32_t)K;
    a.vocab = (int32_t)V;
    a.temperature = (float)temperature;
    if (a.temperature == 0.0f && temperature != 0.0) refused(B200_ERR_BAD_ARG, c10::str("a temperature of ", temperature, " (0, or 1e-4 to 1e4)").c_str()); // (FP32 would make it 0)
    a.logits = logits.data_ptr();
    a.row_stride = K > 0 ? logits.stride(1) : V;
    a.sequence_stride = S > 1 ? logits.stride(0) : 0;
    a.tokens = int_tensor(drafts, "drafts", a.device, {S, K});
    if (uniforms) {
        NEED(uniforms->defined() && uniforms->scalar_type() == at::kFloat && uniforms->sizes() == at::IntArrayRef({S, K + 1}), "uniforms: [", S, ", ", K + 1, "] of FP32 is wanted, got ", shape(*uniforms));
        NEED(uniforms->is_cuda() && uniforms->get_device() == a.device && uniforms->is_contiguous(), "uniforms are contiguous and on ", logits.device());
        outside_graph(*uniforms, "uniforms");
        a.uniforms = uniforms->data_ptr<float>();
    } else NEED(temperature == 0.0, "uniforms are wanted unless the temperature is 0");
    if (draft_logits) {
        const Tensor &y = *draft_logits;
        NEED(y.defined() && y.dim() == 3 && y.size(0) == S && y.size(1) == K && y.size(2) == V && y.scalar_type() == logits.scalar_type(), "draft_logits: [", S, ", ", K, ", ", V, "] of ", logits.scalar_type(),
             " is wanted, got ", shape(y));
        NEED(y.is_cuda() && y.get_device() == a.device, "draft_logits are on ", y.device(), ", the logits on ", logits.device());
        outside_graph(y, "draft_logits");
        NEED(V == 1 || y.numel() == 0 || y.stride(2) == 1, "the logits of a row have to lie one behind the other");
        if (K > 0) {
            a.draft_logits = y.data_ptr();
            a.draft_row_stride = K > 1 ? y.stride(1) : V;
            a.draft_sequence_stride = S > 1 ? y.stride(0) : 0;
        }
    }
    Tensor tokens = fresh({S, K + 1}, at::kInt, a.device), accepted = fresh({S}, at::kInt, a.device);
    a.out_tokens = tokens.data_ptr<int32_t>();
    a.accepted = accepted.data_ptr<int32_t>();
    Tensor work; // from the stream's own pool
    if ((a.workspace_bytes = b200_verify_drafts_workspace(&a)) > 0) {
        work = fresh({(int64_t)(a.workspace_bytes / 4)}, at::kFloat, a.device);
        a.workspace = work.data_ptr();
    }
    char err[256] = "";
    const int rc = b200_verify_drafts(&a, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream(), err, sizeof err);
    if (rc != B200_OK) refused(rc, err);
    return {tokens, accepted};
}

} // namespace

PYBIND11_MODULE(_b200ops, m) {
    using py::arg;
    m.def("on_error", [](py::object f) { raise_error = new py::object(std::move(f)); });
    py::class_<Cache>(m, "Cache")
        .def(py::init(&create), arg("slots"), arg("context"), arg("kv_heads"), arg("head_size"), arg("device"))
        .def_readonly("slots", &Cache::slots)
        .def_readonly("context", &Cache::context)
        .def_readonly("kv_heads", &Cache::kv_heads)
        .def_readonly("head_size", &Cache::head_size)
        .def_readonly("device_index", &Cache::device)
        .def_property_readonly("device_bytes", &Cache::bytes)
        .def("append", &Cache::append, arg("k"), arg("v"), arg("positions").none(false), arg("q") = py::none(), arg("slots") = py::none(), arg("q_norm") = py::none(), arg("k_norm") = py::none(),
             arg("eps") = 1e-6, arg("cos") = py::none(), arg("sin") = py::none(), arg("layout") = "half", arg("q_out") = py::none())
        .def("attention", &Cache::attention, arg("q"), arg("positions").none(false), arg("slots") = py::none(), arg("scale") = py::none(), arg("window") = 0, arg("max_len") = 0, arg("chunk") = 1,
             arg("dtype") = at::kFloat, arg("out") = py::none())
        .def("read", &Cache::read, arg("positions").none(false), arg("slots") = py::none(), arg("dtype") = at::kFloat)
        .def("reset", &Cache::reset)
        .def("free", &Cache::free);
    py::class_<Paged>(m, "Paged")
        .def(py::init<const Tensor &, const Tensor &>(), arg("keys").none(false), arg("values").none(false))
        .def_readonly("keys", &Paged::keys)
        .def_readonly("values", &Paged::values)
        .def_readonly("pages", &Paged::pages)
        .def_readonly("page_size", &Paged::page_size)
        .def_readonly("kv_heads", &Paged::kv_heads)
        .def_readonly("head_size", &Paged::head_size)
        .def_readonly("device_index", &Paged::device)
        .def("append", &Paged::append, arg("k"), arg("v"), arg("positions").none(false), arg("tables").none(false), arg("sequences") = py::none(), arg("q") = py::none(), arg("q_norm") = py::none(),
             arg("k_norm") = py::none(), arg("eps") = 1e-6, arg("cos") = py::none(), arg("sin") = py::none(), arg("layout") = "half", arg("q_out") = py::none())
        .def("attention", &Paged::attention, arg("q"), arg("positions").none(false), arg("tables").none(false), arg("sequences") = py::none(), arg("scale") = py::none(), arg("window") = 0,
             arg("max_len") = 0, arg("chunk") = 1, arg("dtype") = py::none(), arg("out") = py::none());
    m.def("verify_drafts", &verify_drafts, arg("logits"), arg("drafts").none(false), arg("uniforms").none(true), arg("draft_logits") = py::none(), arg("temperature") = 1.0);
    m.def("log_probs", &log_probs, arg("logits"), arg("targets").none(true), arg("top") = 0);
}
