// torch_ops.cpp -- the operators of operators.cu on torch tensors (operators.py has their documentation): checks of the tensors, the current stream, results from torch's allocator.
// A call through Python's ctypes costs 15 to 20 us of host time, more than most of these kernels run; here it is about 5.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
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

// There are no backward passes: a graph that led through a call would end there without a word.
void outside_graph(const Tensor &t, const char *name) {
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
    m.def("log_probs", &log_probs, arg("logits"), arg("targets").none(true), arg("top") = 0);
}
