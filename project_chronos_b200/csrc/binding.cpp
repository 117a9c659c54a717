// binding.cpp — the Python module project_chronos_b200._binding: argument checks and calls of
// include/chronos_paged4.h for torch tensors.  What ops.py does in Python for the calls of
// chronos_paged.h (a dozen microseconds per call, more than a step's kernels take) is done
// here in native code: the same checks, the same errors, the current stream of the tensors'
// device, workspaces from torch's allocator.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstdarg>
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "chronos_paged4.h"

namespace {

PyObject* g_status = nullptr;   // device index -> address of its status word
PyObject* g_check = nullptr;    // return code -> raises the package's error
std::array<int32_t*, 64> g_words{};

// A Python error that is already set, on its way out.
struct Raised {};

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Raised{};
}

const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kByte: return "torch.uint8";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return c10::toString(t);
    }
}
std::string shape_text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}
int dtype_code(at::ScalarType t) {
    return t == at::kBFloat16 ? CHRONOS_DTYPE_BF16 : t == at::kHalf ? CHRONOS_DTYPE_FP16 : t == at::kFloat ? CHRONOS_DTYPE_FP32 : -1;
}
int known_dtype(at::ScalarType t) {
    const int code = dtype_code(t);
    if (code < 0) refuse(PyExc_TypeError, "unsupported dtype %s", type_name(t));
    return code;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor expected, got %s", name, Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw Raised{};
        PyErr_Clear();
        refuse(PyExc_ValueError, "%s %S does not fit 32 bits", name, o);
    }
    return v;
}
int32_t int32(PyObject* o, const char* name) {
    const int64_t v = integer(o, name);
    if (v != static_cast<int32_t>(v)) refuse(PyExc_ValueError, "%s %lld does not fit 32 bits", name, static_cast<long long>(v));
    return static_cast<int32_t>(v);
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return static_cast<float>(v);
}

// The device of a call and whether gradients are recorded.
struct Call {
    c10::Device device;
    bool grad;
    explicit Call(const at::Tensor& t) : device(t.device()), grad(at::GradMode::is_enabled()) {
        if (!t.is_cuda())
            refuse(PyExc_RuntimeError, "chronos paged kernels need CUDA tensors (no CPU path exists); got a tensor on %s",
                   device.str().c_str());
    }
    void like(const char* name, const at::Tensor& t, at::IntArrayRef shape, at::ScalarType dt) const {
        if (t.scalar_type() != dt || t.device() != device)
            refuse(PyExc_TypeError, "%s: %s on %s expected, got %s on %s", name, type_name(dt), device.str().c_str(),
                   type_name(t.scalar_type()), t.device().str().c_str());
        if (t.sizes() != shape)
            refuse(PyExc_ValueError, "%s must be %s, got %s", name, shape_text(shape).c_str(), shape_text(t.sizes()).c_str());
        if (grad && t.requires_grad())
            refuse(PyExc_RuntimeError, "forward-only kernels: call under torch.no_grad() or detach the inputs");
    }
    // A tensor of vectors: the last dimension contiguous, the others by their strides.
    void rows(const char* name, const at::Tensor& t, at::IntArrayRef shape, at::ScalarType dt) const {
        like(name, t, shape, dt);
        if (t.stride(-1) != 1 && t.size(-1) != 1) refuse(PyExc_ValueError, "%s's last dimension must be contiguous", name);
    }
    void written(const char* name, const at::Tensor& t) const {
        for (int64_t i = 0; i < t.dim(); ++i)
            if (t.size(i) > 1 && t.stride(i) == 0) refuse(PyExc_ValueError, "%s is written: it must not be expanded", name);
    }
    template <typename N>
    N* dense(const char* name, const at::Tensor& t, at::IntArrayRef shape, at::ScalarType dt) const {
        like(name, t, shape, dt);
        if (!t.is_contiguous()) refuse(PyExc_ValueError, "%s must be contiguous", name);
        return static_cast<N*>(t.data_ptr());
    }
    int32_t* ints(PyObject* o, const char* name, at::IntArrayRef shape) const {
        const at::Tensor* t = maybe(o, name);
        return t == nullptr ? nullptr : dense<int32_t>(name, *t, shape, at::kInt);
    }
    float* floats(PyObject* o, const char* name, at::IntArrayRef shape) const {
        const at::Tensor* t = maybe(o, name);
        return t == nullptr ? nullptr : dense<float>(name, *t, shape, at::kFloat);
    }
    int32_t* status() const {
        const size_t i = static_cast<size_t>(device.index());
        if (i < g_words.size() && g_words[i] != nullptr) return g_words[i];
        PyObject* r = PyObject_CallFunction(g_status, "i", static_cast<int>(device.index()));
        if (r == nullptr) throw Raised{};
        int32_t* p = static_cast<int32_t*>(PyLong_AsVoidPtr(r));
        Py_DECREF(r);
        if (p == nullptr && PyErr_Occurred()) throw Raised{};
        if (i < g_words.size()) g_words[i] = p;
        return p;
    }
    void raise(int rc) const {
        PyObject* r = PyObject_CallFunction(g_check, "i", rc);
        Py_XDECREF(r);
        if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "call failed with code %d", rc);
        throw Raised{};
    }
    // On the current stream of the tensors' device, whatever the current device is.
    template <typename A>
    void launch(int (*fn)(const A*, void*), const A& args) const {
        const c10::cuda::OptionalCUDAGuard guard(device);
        void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = fn(&args, stream);
        Py_END_ALLOW_THREADS;
        if (rc != CHRONOS_OK) raise(rc);
    }
    // The call's workspace, from torch's allocator: a captured graph keeps its own.
    template <typename A>
    at::Tensor workspace(size_t (*fn)(const A*), A& args) const {
        const c10::cuda::OptionalCUDAGuard guard(device);
        const size_t bytes = fn(&args);
        if (bytes == 0) {
            const char* error = chronos_moe_last_error();
            if (error != nullptr && error[0] != 0) raise(CHRONOS_ERR_INVALID_ARG);
            return at::Tensor();
        }
        at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device));
        args.workspace = ws.data_ptr();
        args.workspace_bytes = bytes;
        return ws;
    }
    at::Tensor fresh(at::IntArrayRef shape, at::ScalarType dt) const { return at::empty(shape, at::TensorOptions().dtype(dt).device(device)); }
};

int64_t columns_of(int64_t head_dim) {
    if (head_dim < 1 || head_dim > CHRONOS_PAGED_MAX_HEAD_DIM)
        refuse(PyExc_ValueError, "head_dim %lld must be 1..%d", static_cast<long long>(head_dim), CHRONOS_PAGED_MAX_HEAD_DIM);
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
}

// Page table and lengths into the cache part of a call's arguments.
void set_table(const Call& call, ChronosPagedCache& c, PyObject* table_o, PyObject* lens_o) {
    const at::Tensor& table = tensor(table_o, "page_table");
    if (table.scalar_type() != at::kInt || table.device() != call.device || table.dim() != 2 || (table.stride(1) != 1 && table.size(1) > 1))
        refuse(PyExc_ValueError, "page_table must be an int32 tensor [B, pages] on %s with contiguous rows", call.device.str().c_str());
    if (table.size(0) > INT32_MAX || table.size(1) > INT32_MAX) refuse(PyExc_ValueError, "page_table is too large");
    c.batch = static_cast<int32_t>(table.size(0));
    c.table_width = static_cast<int32_t>(table.size(1));
    c.page_table = static_cast<const int32_t*>(table.data_ptr());
    c.page_table_stride = table.stride(0);
    c.lens = call.dense<int32_t>("lens", tensor(lens_o, "lens"), {c.batch}, at::kInt);
}

// The cache part: pages of the layer type `dt` [pages, size, G, D] or, as uint8 [pages, G, bytes],
// of 4-bit values.  Returns whether they are packed.
int set_cache(const Call& call, ChronosPagedCache& c, PyObject* k_o, PyObject* v_o, PyObject* table_o, PyObject* lens_o, at::ScalarType dt,
              int64_t d, bool written) {
    const at::Tensor &k = tensor(k_o, "k_pages"), &v = tensor(v_o, "v_pages");
    c.dtype = known_dtype(dt);
    set_table(call, c, table_o, lens_o);
    const bool packed = k.scalar_type() == at::kByte;
    if (packed) {
        if (k.dim() != 3) refuse(PyExc_ValueError, "4-bit k_pages must be [pages, kv heads, bytes], got %s", shape_text(k.sizes()).c_str());
        const int64_t record = 9 * columns_of(d), bytes = k.size(2);
        if (bytes == 0 || bytes % record)
            refuse(PyExc_ValueError, "4-bit pages of heads of %lld have a multiple of %lld bytes, got %lld", static_cast<long long>(d),
                   static_cast<long long>(record), static_cast<long long>(bytes));
        call.rows("k_pages", k, k.sizes(), at::kByte);
        call.rows("v_pages", v, k.sizes(), at::kByte);
        c.kv_heads = static_cast<int32_t>(k.size(1));
        c.page_size = static_cast<int32_t>(bytes / record * 16);
        c.k_page_stride = k.stride(0);
        c.k_head_stride = k.stride(1);
        c.v_page_stride = v.stride(0);
        c.v_head_stride = v.stride(1);
    } else {
        if (k.dim() != 4) refuse(PyExc_ValueError, "k_pages must be [pages, page size, kv heads, head dim], got %s", shape_text(k.sizes()).c_str());
        if (k.scalar_type() != dt || k.size(3) != d)
            refuse(PyExc_TypeError, "pages: %s (or uint8) with heads of %lld expected, got %s with heads of %lld", type_name(dt),
                   static_cast<long long>(d), type_name(k.scalar_type()), static_cast<long long>(k.size(3)));
        call.rows("k_pages", k, k.sizes(), dt);
        call.rows("v_pages", v, k.sizes(), dt);
        if (k.size(1) > INT32_MAX || k.size(2) > INT32_MAX) refuse(PyExc_ValueError, "k_pages is too large");
        c.page_size = static_cast<int32_t>(k.size(1));
        c.kv_heads = static_cast<int32_t>(k.size(2));
        c.k_page_stride = k.stride(0);
        c.k_slot_stride = k.stride(1);
        c.k_head_stride = k.stride(2);
        c.v_page_stride = v.stride(0);
        c.v_slot_stride = v.stride(1);
        c.v_head_stride = v.stride(2);
    }
    if (k.size(0) > INT32_MAX || d > INT32_MAX) refuse(PyExc_ValueError, "k_pages is too large");
    c.num_pages = static_cast<int32_t>(k.size(0));
    c.head_dim = static_cast<int32_t>(d);
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    if (written) {
        call.written("k_pages", k);
        call.written("v_pages", v);
    }
    return packed ? 1 : 0;
}

// The rows that an attention call writes: given ones, or new ones.
at::Tensor rows_out(const Call& call, const char* name, PyObject* o, at::IntArrayRef shape, at::ScalarType dt) {
    const at::Tensor* t = maybe(o, name);
    if (t == nullptr) return call.fresh(shape, dt);
    call.rows(name, *t, shape, dt);
    call.written(name, *t);
    return *t;
}
PyObject* wrapped(PyObject* given, at::Tensor&& t) {
    if (given != Py_None) return Py_NewRef(given);
    return THPVariable_Wrap(std::move(t));
}
void three(const at::Tensor& t, const char* text) {
    if (t.dim() != 3) refuse(PyExc_ValueError, "%s, got %s", text, shape_text(t.sizes()).c_str());
}
float scale_or(PyObject* o, int64_t d) { return o == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(d))) : real(o); }

// k, v, k_pages, v_pages, page_table, lens, seen, cos, sin, q, q_out, k_out, cu_seqlens, rope_start, weights, positions,
// lens_out, seen_out, k_scale, v_scale
PyObject* append_rope(PyObject* const* a) {
    const at::Tensor& k = tensor(a[0], "k");
    const Call call(k);
    three(k, "k must be [tokens, kv heads, head dim]");
    const at::ScalarType dt = k.scalar_type();
    const int64_t t = k.size(0), g = k.size(1), d = k.size(2);
    ChronosPagedRopeArgs x{};
    x.packed = set_cache(call, x.cache, a[2], a[3], a[4], a[5], dt, d, true);
    const int64_t b = x.cache.batch;
    if (x.cache.kv_heads != g)
        refuse(PyExc_ValueError, "k has %lld kv heads, the pages %d", static_cast<long long>(g), x.cache.kv_heads);
    const at::Tensor& v = tensor(a[1], "v");
    call.rows("k", k, k.sizes(), dt);
    call.rows("v", v, k.sizes(), dt);
    x.num_tokens = t;
    x.k = k.data_ptr();
    x.v = v.data_ptr();
    x.k_row_stride = k.stride(0);
    x.k_head_stride = k.stride(1);
    x.v_row_stride = v.stride(0);
    x.v_head_stride = v.stride(1);
    at::Tensor q_out;
    const at::Tensor* q = maybe(a[9], "q");
    if (q != nullptr) {
        if (q->dim() != 3 || q->size(1) < 1 || q->size(1) > INT32_MAX)
            refuse(PyExc_ValueError, "q must be [tokens, heads, head dim], got %s", shape_text(q->sizes()).c_str());
        const std::array<int64_t, 3> shape{t, q->size(1), d};
        call.rows("q", *q, shape, dt);
        q_out = rows_out(call, "q_out", a[10], shape, dt);
        x.heads = static_cast<int32_t>(q->size(1));
        x.q = q->data_ptr();
        x.q_row_stride = q->stride(0);
        x.q_head_stride = q->stride(1);
        x.q_out = q_out.data_ptr();
        x.q_out_row_stride = q_out.stride(0);
        x.q_out_head_stride = q_out.stride(1);
    } else if (a[10] != Py_None) {
        refuse(PyExc_ValueError, "q_out needs q");
    }
    if (a[11] != Py_None) {
        const at::Tensor k_out = rows_out(call, "k_out", a[11], k.sizes(), dt);
        x.k_out = k_out.data_ptr();
        x.k_out_row_stride = k_out.stride(0);
        x.k_out_head_stride = k_out.stride(1);
    }
    const at::Tensor *cos = maybe(a[7], "cos"), *sin = maybe(a[8], "sin");
    if ((cos == nullptr) != (sin == nullptr)) refuse(PyExc_ValueError, "cos and sin go together");
    if (cos != nullptr) {
        if (cos->dim() != 2) refuse(PyExc_ValueError, "cos must be [positions, columns], got %s", shape_text(cos->sizes()).c_str());
        const at::ScalarType tt = cos->scalar_type();
        if (tt != at::kFloat && tt != dt) refuse(PyExc_TypeError, "cos and sin must be fp32 or %s, got %s", type_name(dt), type_name(tt));
        if (cos->size(0) > INT32_MAX || cos->size(1) > INT32_MAX) refuse(PyExc_ValueError, "cos is too large");
        call.rows("cos", *cos, cos->sizes(), tt);
        call.rows("sin", *sin, cos->sizes(), tt);
        if (a[6] == Py_None) refuse(PyExc_ValueError, "the rotation needs seen, the positions of the sequences' next tokens");
        x.table_len = static_cast<int32_t>(cos->size(0));
        x.rope_dim = static_cast<int32_t>(cos->size(1));
        x.table_dtype = dtype_code(tt);
        x.cos = cos->data_ptr();
        x.sin = sin->data_ptr();
        x.cos_row_stride = cos->stride(0);
        x.sin_row_stride = sin->stride(0);
    }
    x.rope_start = int32(a[13], "rope_start");
    const at::Tensor *weights = maybe(a[14], "weights"), *positions = maybe(a[15], "positions");
    for (const at::Tensor* s : {weights, positions})
        if (s != nullptr) {
            if (s->dim() != 3) refuse(PyExc_ValueError, "weights and positions must be [sequences, kv heads, slots]");
            if (weights != nullptr && s->size(2) != weights->size(2))
                refuse(PyExc_ValueError, "weights and positions must have the same number of slots");
            x.slot_cap = s->size(2);
        }
    x.weights = call.floats(a[14], "weights", {b, g, x.slot_cap});
    x.positions = call.ints(a[15], "positions", {b, g, x.slot_cap});
    x.cu_seqlens = call.ints(a[12], "cu_seqlens", {b + 1});
    x.seen = call.ints(a[6], "seen", {b});
    x.lens_out = call.ints(a[16], "lens_out", {b});
    x.seen_out = call.ints(a[17], "seen_out", {b});
    x.k_scale = real(a[18]);
    x.v_scale = real(a[19]);
    x.status = call.status();
    call.launch(chronos_paged_append_rope, x);
    if (q == nullptr) Py_RETURN_NONE;
    return wrapped(a[10], std::move(q_out));
}

// k_pages, v_pages, page_table, lens, cu_seqlens, k_out, v_out, first, k_scale, v_scale
PyObject* gather(PyObject* const* a) {
    const at::Tensor &k = tensor(a[5], "k_out"), &v = tensor(a[6], "v_out");
    const Call call(tensor(a[0], "k_pages"));
    three(k, "k_out must be [rows, kv heads, head dim]");
    const at::ScalarType dt = k.scalar_type();
    ChronosPagedGatherArgs x{};
    x.packed = set_cache(call, x.cache, a[0], a[1], a[2], a[3], dt, k.size(2), false);
    if (x.cache.kv_heads != k.size(1))
        refuse(PyExc_ValueError, "k_out has %lld kv heads, the pages %d", static_cast<long long>(k.size(1)), x.cache.kv_heads);
    call.rows("k_out", k, k.sizes(), dt);
    call.rows("v_out", v, k.sizes(), dt);
    call.written("k_out", k);
    call.written("v_out", v);
    x.k_scale = real(a[8]);
    x.v_scale = real(a[9]);
    x.num_tokens = k.size(0);
    x.k_out = k.data_ptr();
    x.v_out = v.data_ptr();
    x.k_row_stride = k.stride(0);
    x.k_head_stride = k.stride(1);
    x.v_row_stride = v.stride(0);
    x.v_head_stride = v.stride(1);
    x.cu_seqlens = call.dense<int32_t>("cu_seqlens", tensor(a[4], "cu_seqlens"), {x.cache.batch + int64_t{1}}, at::kInt);
    x.first = call.ints(a[7], "first", {x.cache.batch});
    x.status = call.status();
    call.launch(chronos_paged_gather, x);
    return PyTuple_Pack(2, a[5], a[6]);
}

// q, k_pages, v_pages, page_table, lens, scale, window, sinks, k_scale, v_scale, out, lse
PyObject* decode4(PyObject* const* a) {
    const at::Tensor& q = tensor(a[0], "q");
    const Call call(q);
    three(q, "q must be [sequences, heads, head dim]");
    const at::Tensor& pages = tensor(a[1], "k_pages");
    if (pages.scalar_type() != at::kByte)
        refuse(PyExc_TypeError, "k_pages: uint8 pages of 4-bit values expected, got %s", type_name(pages.scalar_type()));
    const at::ScalarType dt = q.scalar_type();
    const int64_t h = q.size(1), d = q.size(2);
    ChronosPagedDecode4Args x{};
    set_cache(call, x.cache, a[1], a[2], a[3], a[4], dt, d, false);
    const std::array<int64_t, 3> shape{x.cache.batch, h, d};
    if (h > INT32_MAX) refuse(PyExc_ValueError, "q has too many heads");
    call.rows("q", q, shape, dt);
    at::Tensor out = rows_out(call, "out", a[10], shape, dt);
    x.heads = static_cast<int32_t>(h);
    x.window = int32(a[6], "window");
    x.sinks = int32(a[7], "sinks");
    x.scale = scale_or(a[5], d);
    x.k_scale = real(a[8]);
    x.v_scale = real(a[9]);
    x.q = q.data_ptr();
    x.q_row_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.out = out.data_ptr();
    x.out_row_stride = out.stride(0);
    x.out_head_stride = out.stride(1);
    x.lse = call.floats(a[11], "lse", {x.cache.batch, h});
    x.status = call.status();
    const at::Tensor ws = call.workspace(chronos_paged_decode4_workspace, x);
    call.launch(chronos_paged_decode4, x);
    return wrapped(a[10], std::move(out));
}

void* bounds_of(const Call& call, const at::Tensor& bounds, const ChronosPagedCache& c) {
    known_dtype(bounds.scalar_type());
    return call.dense<void>("bounds", bounds, {c.num_pages, 2, c.kv_heads, c.head_dim}, bounds.scalar_type());
}

// k_pages, bounds, page_table, lens, cu_seqlens, num_tokens, full, k_scale
PyObject* bounds(PyObject* const* a) {
    const Call call(tensor(a[0], "k_pages"));
    const at::Tensor& b = tensor(a[1], "bounds");
    if (b.dim() != 4) refuse(PyExc_ValueError, "bounds must be [pages, 2, kv heads, head dim], got %s", shape_text(b.sizes()).c_str());
    ChronosPagedBoundsArgs x{};
    x.packed = set_cache(call, x.cache, a[0], a[0], a[2], a[3], b.scalar_type(), b.size(3), false);
    x.bounds = bounds_of(call, b, x.cache);
    x.cu_seqlens = call.ints(a[4], "cu_seqlens", {x.cache.batch + int64_t{1}});
    const int64_t slots = static_cast<int64_t>(x.cache.table_width) * x.cache.page_size;
    x.num_tokens = a[5] != Py_None ? integer(a[5], "num_tokens")
                   : x.cu_seqlens == nullptr ? x.cache.batch
                                             : std::min<int64_t>(INT32_MAX, slots > 0 && x.cache.batch > INT32_MAX / slots ? INT32_MAX : x.cache.batch * slots);
    const int full = PyObject_IsTrue(a[6]);
    if (full < 0) throw Raised{};
    x.full = full;
    x.k_scale = real(a[7]);
    x.status = call.status();
    call.launch(chronos_paged_bounds, x);
    return Py_NewRef(a[1]);
}

// q, bounds, page_table, lens, page_size, topk, first, last, cu_seqlens, out
PyObject* select(PyObject* const* a) {
    const at::Tensor &q = tensor(a[0], "q"), &b = tensor(a[1], "bounds");
    const Call call(q);
    if (q.dim() != 3 || b.dim() != 4)
        refuse(PyExc_ValueError, "q and bounds must be [tokens, heads, head dim] and [pages, 2, kv heads, head dim], got %s and %s",
               shape_text(q.sizes()).c_str(), shape_text(b.sizes()).c_str());
    const at::ScalarType dt = q.scalar_type();
    const int64_t t = q.size(0), h = q.size(1), d = q.size(2), g = b.size(2);
    if (h > INT32_MAX || d > INT32_MAX || g > INT32_MAX || b.size(0) > INT32_MAX) refuse(PyExc_ValueError, "q or bounds are too large");
    ChronosPagedSelectArgs x{};
    x.cache.dtype = known_dtype(dt);
    x.cache.kv_heads = static_cast<int32_t>(g);
    x.cache.head_dim = static_cast<int32_t>(d);
    x.cache.num_pages = static_cast<int32_t>(b.size(0));
    x.cache.page_size = int32(a[4], "page_size");
    x.topk = int32(a[5], "topk");
    x.first = int32(a[6], "first");
    x.last = int32(a[7], "last");
    set_table(call, x.cache, a[2], a[3]);
    if (b.scalar_type() != dt) refuse(PyExc_TypeError, "bounds: %s expected, got %s", type_name(dt), type_name(b.scalar_type()));
    x.bounds = bounds_of(call, b, x.cache);
    call.rows("q", q, q.sizes(), dt);
    if (x.topk < 1) refuse(PyExc_ValueError, "topk %d must be at least 1", x.topk);
    const std::array<int64_t, 3> shape{t, g, x.topk};
    const at::Tensor* given = maybe(a[9], "out");
    at::Tensor out = given == nullptr ? call.fresh(shape, at::kInt) : *given;
    if (given != nullptr) call.dense<int32_t>("out", out, shape, at::kInt);
    x.heads = static_cast<int32_t>(h);
    x.num_tokens = t;
    x.q = q.data_ptr();
    x.q_row_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.cu_seqlens = call.ints(a[8], "cu_seqlens", {x.cache.batch + int64_t{1}});
    x.pages = static_cast<int32_t*>(out.data_ptr());
    x.status = call.status();
    const at::Tensor ws = call.workspace(chronos_paged_select_workspace, x);
    call.launch(chronos_paged_select, x);
    return wrapped(a[9], std::move(out));
}

// q, k_pages, v_pages, page_table, lens, pages, cu_seqlens, scale, k_scale, v_scale, out, lse
PyObject* sparse(PyObject* const* a) {
    const at::Tensor &q = tensor(a[0], "q"), &pages = tensor(a[5], "pages");
    const Call call(q);
    if (q.dim() != 3 || pages.dim() != 3)
        refuse(PyExc_ValueError, "q and pages must be [tokens, heads, head dim] and [tokens, kv heads, n], got %s and %s",
               shape_text(q.sizes()).c_str(), shape_text(pages.sizes()).c_str());
    const at::ScalarType dt = q.scalar_type();
    const int64_t t = q.size(0), h = q.size(1), d = q.size(2), n = pages.size(2);
    if (h > INT32_MAX || n > INT32_MAX) refuse(PyExc_ValueError, "q or pages are too large");
    ChronosPagedSparseArgs x{};
    x.packed = set_cache(call, x.cache, a[1], a[2], a[3], a[4], dt, d, false);
    call.rows("q", q, q.sizes(), dt);
    at::Tensor out = rows_out(call, "out", a[10], q.sizes(), dt);
    x.heads = static_cast<int32_t>(h);
    x.topk = static_cast<int32_t>(n);
    x.scale = scale_or(a[7], d);
    x.k_scale = real(a[8]);
    x.v_scale = real(a[9]);
    x.num_tokens = t;
    x.q = q.data_ptr();
    x.q_row_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.out = out.data_ptr();
    x.out_row_stride = out.stride(0);
    x.out_head_stride = out.stride(1);
    x.lse = call.floats(a[11], "lse", {t, h});
    x.pages = call.dense<int32_t>("pages", pages, {t, x.cache.kv_heads, n}, at::kInt);
    x.cu_seqlens = call.ints(a[6], "cu_seqlens", {x.cache.batch + int64_t{1}});
    x.status = call.status();
    call.launch(chronos_paged_sparse, x);
    return wrapped(a[10], std::move(out));
}

// No C++ exception leaves the module.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Raised&) {
    } catch (...) {   // as torch's own calls raise it: torch.OutOfMemoryError among them
        if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

PyObject* init(PyObject*, PyObject* args) {
    PyObject *status, *check;
    if (!PyArg_ParseTuple(args, "OO", &status, &check)) return nullptr;
    Py_XSETREF(g_status, Py_NewRef(status));
    Py_XSETREF(g_check, Py_NewRef(check));
    Py_RETURN_NONE;
}

#define CHRONOS_ENTRY(name, n) \
    { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<name, n>)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {
    CHRONOS_ENTRY(append_rope, 20), CHRONOS_ENTRY(gather, 10), CHRONOS_ENTRY(decode4, 12), CHRONOS_ENTRY(bounds, 8),
    CHRONOS_ENTRY(select, 10), CHRONOS_ENTRY(sparse, 12), {"init", init, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&g_module); }
