// Python functions over the paged cache's C entry points, for tensors of torch: argument checks, outputs, scratch from
// torch's caching allocator, the current stream. A decoding step makes two of these calls per layer, and each is a few
// microseconds of device time, so what the host spends on one counts: attention of one token took 17.6 us through ctypes
// and checks in Python and takes 5 through this (one launch; 7 with two).
#include <Python.h>

#include <cmath>
#include <cstdlib>

#include <ATen/Context.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/smlm_b200.h"

namespace {

struct Refused {};  // a Python error is set

template <typename... A>
[[noreturn]] void refuse(const char* fmt, A... a) {
    PyErr_Format(PyExc_ValueError, fmt, a...);
    throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: %s has to be a tensor, got %s", what, name, Py_TYPE(o)->tp_name);
        throw Refused();
    }
    return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}

// All on the first tensor's CUDA device.
void same_device(const char* what, std::initializer_list<const at::Tensor*> ts) {
    const auto dev = (*ts.begin())->device();
    for (const at::Tensor* t : ts) {
        if (!t->is_cuda())
            refuse("%s: smlm_b200 kernels run on CUDA tensors only (there is no CPU fallback); got a tensor on %s", what,
                   t->device().str().c_str());
        if (t->device() != dev)
            refuse("%s: tensors on different devices: %s and %s", what, dev.str().c_str(), t->device().str().c_str());
    }
}

// The device's status word, asked from Python once per device (it is a tensor kept there). No word before a capture
// began: none for the calls captured.
PyObject* status_of_device = nullptr;
int* status_word[64] = {};

int* status(int dev) {
    if (dev < 64 && status_word[dev]) return status_word[dev];
    if (!status_of_device) return nullptr;
    PyObject* r = PyObject_CallFunction(status_of_device, "i", dev);
    if (!r) throw Refused();
    int* p = r == Py_None ? nullptr : static_cast<int*>(PyLong_AsVoidPtr(r));
    Py_DECREF(r);
    if (PyErr_Occurred()) throw Refused();
    if (dev < 64) status_word[dev] = p;
    return p;
}

// Device guard, stream, status and scratch of one call.
struct Call {
    c10::cuda::OptionalCUDAGuard guard;
    int* st;
    void* stream;
    c10::DataPtr scratch;
    explicit Call(const at::Tensor& t) {
        if (c10::cuda::current_device() != t.device().index()) guard.set_device(t.device());
        st = status(t.device().index());
        stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
    }
    void* workspace(size_t bytes) {
        if (!bytes) return nullptr;
        scratch = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
        return scratch.get();
    }
};

// An uninitialised tensor beside `like`.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// These calls have no gradient. Where one would be recorded, the output gets a node that says so in a backward pass (a
// forward pass outside no_grad is fine by itself).
void no_gradient(const char* what, std::initializer_list<const at::Tensor*> ins, std::initializer_list<at::Tensor*> outs) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list next;
    for (const at::Tensor* t : ins)
        if (t->requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(*t));
    if (next.empty()) return;
    auto node = std::make_shared<torch::autograd::Error>(std::string(what) + " has no gradient (decoding only)",
                                                         std::move(next));
    for (at::Tensor* t : outs)
        if (t->defined()) torch::autograd::set_history(*t, node);
}

void checked(const char* what, int rc) {
    if (rc == SMLM_OK) return;
    PyErr_Format(rc == SMLM_ERR_INVALID ? PyExc_ValueError : PyExc_RuntimeError, "%s: %s", what, smlm_last_error());
    throw Refused();
}

struct Layer {
    int code;
    int64_t pages, hkv, page, d;
    int64_t strides[6];
};

Layer layer(const char* what, const at::Tensor& x, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
            const at::Tensor& lengths, int64_t batch) {
    Layer l;
    if (k.dim() != 4 || k.sizes() != v.sizes())
        refuse("%s: k_pages and v_pages have to be (pages, key heads, page_size, head dimension)", what);
    if (x.scalar_type() != k.scalar_type() || x.scalar_type() != v.scalar_type())
        refuse("%s: activations and pages have to be of one type, got %s, %s, %s", what, toString(x.scalar_type()),
               toString(k.scalar_type()), toString(v.scalar_type()));
    switch (x.scalar_type()) {
        case at::kFloat: l.code = SMLM_F32; break;
        case at::kBFloat16: l.code = SMLM_BF16; break;
        case at::kHalf: l.code = SMLM_F16; break;
        default: refuse("%s: unsupported type %s (fp32, bf16 or fp16)", what, toString(x.scalar_type()));
    }
    if (k.stride(3) != 1 || v.stride(3) != 1) refuse("%s: the pages' head dimension has to be contiguous", what);
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != batch ||
        (batch && table.size(1) > 1 && table.stride(1) != 1))
        refuse("%s: the table has to be int32, (%lld sequences, blocks) with contiguous rows", what, (long long)batch);
    if (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != batch || !lengths.is_contiguous())
        refuse("%s: lengths has to be a contiguous int32 tensor of %lld lengths", what, (long long)batch);
    same_device(what, {&x, &k, &v, &table, &lengths});
    l.pages = k.size(0);
    l.hkv = k.size(1);
    l.page = k.size(2);
    l.d = k.size(3);
    for (int i = 0; i < 3; i++) {  // a dimension of one element may have any stride: it is not used
        l.strides[i] = k.size(i) > 1 ? k.stride(i) : 0;
        l.strides[3 + i] = v.size(i) > 1 ? v.stride(i) : 0;
    }
    return l;
}

// One row per sequence: torch reports any stride for a table of one row, and the C entry wants one no less than its
// columns.
int64_t row_stride(const at::Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

// A contiguous int32 tensor of n numbers on like's device, or None.
int32_t* optional_ints(const char* what, const char* name, PyObject* o, int64_t n, const at::Tensor& like) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, what, name);
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        refuse("%s: %s has to be a contiguous int32 tensor of %lld numbers", what, name, (long long)n);
    same_device(what, {&like, &t});
    return static_cast<int32_t*>(t.data_ptr());
}

template <typename F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

bool arity(const char* what, Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", what, want, n);
    return false;
}

// (q, k_pages, v_pages, table, lengths, window, sinks): the kernels that the call launches, one where it needs no scratch
PyObject* attention_launches(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "paged_attention";
    if (!arity(what, n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& q = tensor(a[0], what, "q");
        if (q.dim() != 3) refuse("%s: q has to be (sequences, heads, head dimension)", what);
        const at::Tensor& table = tensor(a[3], what, "table");
        const Layer l = layer(what, q, tensor(a[1], what, "k_pages"), tensor(a[2], what, "v_pages"), table,
                              tensor(a[4], what, "lengths"), q.size(0));
        const c10::cuda::OptionalCUDAGuard guard(q.device());
        const size_t bytes = smlm_paged_attention_workspace(q.size(0), q.size(1), l.hkv, l.d, l.code, l.page,
                                                            table.size(1), integer(a[5]), integer(a[6]));
        return PyLong_FromLong(q.size(0) ? 1 + (bytes > 0) : 0);
    });
}

// (q, k_pages, v_pages, table, lengths, scale, window, sinks, return_lse)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "paged_attention";
    if (!arity(what, n, 9)) return nullptr;
    return guarded([&]() -> PyObject* {
        at::Tensor q = tensor(a[0], what, "q");
        const at::Tensor &k = tensor(a[1], what, "k_pages"), &v = tensor(a[2], what, "v_pages");
        const at::Tensor &table = tensor(a[3], what, "table"), &lengths = tensor(a[4], what, "lengths");
        if (q.dim() != 3) refuse("%s: q has to be (sequences, heads, head dimension)", what);
        const int64_t batch = q.size(0), hq = q.size(1);
        const Layer l = layer(what, q, k, v, table, lengths, batch);
        if (q.size(2) != l.d || !l.hkv || hq % l.hkv)
            refuse("%s: %lld query heads of %lld over %lld key heads of %lld", what, (long long)hq, (long long)q.size(2),
                   (long long)l.hkv, (long long)l.d);
        const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)l.d) : PyFloat_AsDouble(a[5]);
        if (PyErr_Occurred()) throw Refused();
        const int64_t window = integer(a[6]), sinks = integer(a[7]);
        if (window < 0 || sinks < 0) refuse("%s: window %lld, sinks %lld", what, (long long)window, (long long)sinks);
        if (!q.is_contiguous()) q = q.contiguous();
        const bool with_lse = PyObject_IsTrue(a[8]) == 1;
        Call c(q);
        at::Tensor out = fresh(q.sizes(), q.scalar_type(), q);
        at::Tensor lse = with_lse ? fresh({batch, hq}, at::kFloat, q) : at::Tensor();
        const size_t bytes = smlm_paged_attention_workspace(batch, hq, l.hkv, l.d, l.code, l.page, table.size(1), window,
                                                            sinks);
        checked(what, smlm_paged_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), l.code, l.strides,
                                           static_cast<const int32_t*>(table.data_ptr()), row_stride(table),
                                           static_cast<const int32_t*>(lengths.data_ptr()), batch, hq, l.hkv, l.d,
                                           l.pages, l.page, table.size(1), (float)scale, window, sinks, out.data_ptr(),
                                           with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, c.workspace(bytes),
                                           bytes, c.st, c.stream));
        no_gradient(what, {&q, &k, &v}, {&out, &lse});
        PyObject* o = THPVariable_Wrap(std::move(out));
        return with_lse ? Py_BuildValue("(NN)", o, THPVariable_Wrap(std::move(lse))) : o;
    });
}

// (qkv, k_pages, v_pages, table, lengths, cos, sin, grown)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "paged_append";
    if (!arity(what, n, 8)) return nullptr;
    return guarded([&]() -> PyObject* {
        at::Tensor x = tensor(a[0], what, "qkv");
        const at::Tensor &k = tensor(a[1], what, "k_pages"), &v = tensor(a[2], what, "v_pages");
        const at::Tensor &table = tensor(a[3], what, "table"), &lengths = tensor(a[4], what, "lengths");
        if (x.dim() != 3) refuse("%s: qkv has to be (sequences, tokens, width)", what);
        const int64_t batch = x.size(0), tokens = x.size(1), width = x.size(2);
        const Layer l = layer(what, x, k, v, table, lengths, batch);
        const int64_t hq = l.d ? width / l.d - 2 * l.hkv : 0;
        if (!l.d || !l.hkv || width % l.d || hq < 1 || hq % l.hkv)
            refuse("%s: a projection of %lld values with %lld key heads of %lld", what, (long long)width,
                   (long long)l.hkv, (long long)l.d);
        const float *cos = nullptr, *sin = nullptr;
        int64_t positions = 0;
        if ((a[5] == Py_None) != (a[6] == Py_None)) refuse("%s: cos and sin come together", what);
        if (a[5] != Py_None) {
            const at::Tensor &c = tensor(a[5], what, "cos"), &s = tensor(a[6], what, "sin");
            if (c.scalar_type() != at::kFloat || s.scalar_type() != at::kFloat || c.dim() != 2 || c.sizes() != s.sizes() ||
                2 * c.size(1) != l.d || !c.is_contiguous() || !s.is_contiguous())
                refuse("%s: cos and sin have to be contiguous fp32 (positions, %lld)", what, (long long)(l.d / 2));
            same_device(what, {&x, &c, &s});
            cos = static_cast<const float*>(c.data_ptr());
            sin = static_cast<const float*>(s.data_ptr());
            positions = c.size(0);
        }
        const int32_t* grown = optional_ints(what, "grown", a[7], batch, x);
        if (!x.is_contiguous()) x = x.contiguous();
        Call c(x);
        at::Tensor q = fresh({batch, tokens, hq, l.d}, x.scalar_type(), x);
        checked(what, smlm_paged_append_grown(x.data_ptr(), k.data_ptr(), v.data_ptr(), l.code, l.strides,
                                              static_cast<const int32_t*>(table.data_ptr()), row_stride(table),
                                              static_cast<const int32_t*>(lengths.data_ptr()), batch, tokens, hq, l.hkv,
                                              l.d, l.pages, l.page, table.size(1), cos, sin, positions, grown,
                                              q.data_ptr(), c.st, c.stream));
        no_gradient(what, {&x}, {&q});
        return THPVariable_Wrap(std::move(q));
    });
}

// ------------------------------------------------------------------------------------------------- the pages
int32_t* ints(const char* what, const char* name, const at::Tensor& t, int64_t dim) {
    if (t.scalar_type() != at::kInt || t.dim() != dim || (t.numel() && t.size(dim - 1) > 1 && t.stride(dim - 1) != 1))
        refuse("%s: %s has to be an int32 tensor of %lld dimension(s) with contiguous rows", what, name, (long long)dim);
    return static_cast<int32_t*>(t.data_ptr());
}

struct Tables {
    const at::Tensor &table, &lengths, &refcount;
    int32_t *t, *l, *r;
    int64_t stride, rows, blocks, pages;
    Tables(const char* what, PyObject* const* a)
        : table(tensor(a[0], what, "table")), lengths(tensor(a[1], what, "lengths")),
          refcount(tensor(a[2], what, "refcount")) {
        t = ints(what, "table", table, 2);
        l = ints(what, "lengths", lengths, 1);
        r = ints(what, "refcount", refcount, 1);
        stride = row_stride(table);
        rows = table.size(0);
        blocks = table.size(1);
        pages = refcount.size(0);
        if (lengths.size(0) != rows)
            refuse("%s: %lld table rows, %lld lengths", what, (long long)rows, (long long)lengths.size(0));
    }
};

struct Pool {
    void* p;
    int64_t planes, heads, token_bytes, page;
    Pool(const char* what, const at::Tensor& t, const at::Tensor& refcount) {
        if (t.dim() != 6 || t.size(1) != 2 || !t.is_contiguous())
            refuse("%s: the pool has to be a contiguous (layers, 2, pages, key heads, page_size, head dimension) tensor",
                   what);
        if (t.size(2) != refcount.size(0))
            refuse("%s: %lld pages, %lld reference counts", what, (long long)t.size(2), (long long)refcount.size(0));
        same_device(what, {&refcount, &t});
        p = t.data_ptr();
        planes = 2 * t.size(0);
        heads = t.size(3);
        page = t.size(4);
        token_bytes = t.size(5) * t.element_size();
    }
};

// (table, lengths, refcount, rows)
PyObject* pages_free(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "pages_free";
    if (!arity(what, n, 4)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tables t(what, a);
        const at::Tensor& rows = tensor(a[3], what, "rows");
        const int32_t* r = ints(what, "row numbers", rows, 1);
        same_device(what, {&t.table, &t.lengths, &t.refcount, &rows});
        Call c(t.table);
        checked(what, smlm_pages_free(t.t, t.stride, t.rows, t.blocks, t.l, t.r, t.pages, r, rows.size(0), c.st, c.stream));
        Py_RETURN_NONE;
    });
}

// (table, lengths, refcount, rows, page_size, window, sinks)
PyObject* pages_trim(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "pages_trim";
    if (!arity(what, n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tables t(what, a);
        const at::Tensor& rows = tensor(a[3], what, "rows");
        const int32_t* r = ints(what, "row numbers", rows, 1);
        const int64_t page = integer(a[4]), window = integer(a[5]), sinks = integer(a[6]);
        same_device(what, {&t.table, &t.lengths, &t.refcount, &rows});
        Call c(t.table);
        checked(what, smlm_pages_trim(t.t, t.stride, t.rows, t.blocks, t.l, t.r, t.pages, page, r, rows.size(0), window,
                                      sinks, c.st, c.stream));
        Py_RETURN_NONE;
    });
}

// (table, lengths, refcount, rows, n_new, page_size, grown)
PyObject* pages_extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "pages_extend";
    if (!arity(what, n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tables t(what, a);
        const at::Tensor& rows = tensor(a[3], what, "rows");
        const int32_t* r = ints(what, "row numbers", rows, 1);
        const int64_t fresh = integer(a[4]), page = integer(a[5]);
        same_device(what, {&t.table, &t.lengths, &t.refcount, &rows});
        int32_t* grown = optional_ints(what, "grown", a[6], t.rows, t.table);
        Call c(t.table);
        const size_t bytes = smlm_pages_extend_workspace(rows.size(0), t.pages);
        checked(what, smlm_pages_extend_grown(t.t, t.stride, t.rows, t.blocks, t.l, t.r, t.pages, page, r, rows.size(0),
                                              fresh, grown, c.workspace(bytes), bytes, c.st, c.stream));
        Py_RETURN_NONE;
    });
}

// (table, lengths, refcount, pool, parents, children)
PyObject* pages_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "pages_fork";
    if (!arity(what, n, 6)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tables t(what, a);
        const at::Tensor &pool = tensor(a[3], what, "pool"), &from = tensor(a[4], what, "parents"),
                         &to = tensor(a[5], what, "children");
        const int32_t *p = ints(what, "row numbers", from, 1), *ch = ints(what, "row numbers", to, 1);
        same_device(what, {&t.table, &t.lengths, &t.refcount, &from, &to});
        const Pool pl(what, pool, t.refcount);
        const int64_t pairs = from.size(0);
        if (to.size(0) != pairs)
            refuse("%s: %lld parents, %lld children", what, (long long)pairs, (long long)to.size(0));
        Call c(t.table);
        const size_t bytes = smlm_pages_fork_workspace(pairs, t.rows, t.blocks, t.pages);
        checked(what, smlm_pages_fork(pl.p, pl.planes, pl.heads, pl.token_bytes, t.t, t.stride, t.rows, t.blocks, t.l, t.r,
                                      t.pages, pl.page, p, ch, pairs, c.workspace(bytes), bytes, c.st, c.stream));
        Py_RETURN_NONE;
    });
}

// (table, refcount, pool)
PyObject* pages_compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
    const char* what = "pages_compact";
    if (!arity(what, n, 3)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &table = tensor(a[0], what, "table"), &refcount = tensor(a[1], what, "refcount");
        int32_t *t = ints(what, "table", table, 2), *r = ints(what, "refcount", refcount, 1);
        same_device(what, {&table, &refcount});
        const Pool pl(what, tensor(a[2], what, "pool"), refcount);
        Call c(table);
        const size_t bytes = smlm_pages_compact_workspace(refcount.size(0));
        checked(what, smlm_pages_compact(pl.p, pl.planes, pl.heads, pl.token_bytes, t, row_stride(table), table.size(0),
                                         table.size(1), r, refcount.size(0), pl.page, c.workspace(bytes), bytes, c.st,
                                         c.stream));
        Py_RETURN_NONE;
    });
}

// (function of a device number that gives the address of its status word or None)
PyObject* init(PyObject*, PyObject* f) {
    Py_INCREF(f);
    Py_XSETREF(status_of_device, f);
    Py_RETURN_NONE;
}

// Whether SMLM_B200_CHECK=1 is set now (os.environ.get costs ten times as much as this call).
PyObject* checking(PyObject*, PyObject*) {
    const char* v = std::getenv("SMLM_B200_CHECK");
    return PyBool_FromLong(v && v[0] == '1' && !v[1]);
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"init", init, METH_O, nullptr},
                         {"checking", checking, METH_NOARGS, nullptr},
                         FAST(attention),
                         FAST(attention_launches),
                         FAST(append),
                         FAST(pages_free),
                         FAST(pages_trim),
                         FAST(pages_extend),
                         FAST(pages_fork),
                         FAST(pages_compact),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__paged() { return PyModule_Create(&module); }
