// front.cpp -- the torch front end of the batched attention operators (their Python names, arguments and
// documentation are in ops.py): the checks of the tensors, the outputs, and the calls of the C ABI.
//
// In C++ because they are called once per layer and step at sizes where the host bounds an eager call: a
// tensor's type, shape, strides, device and address take 0.6 us to ask for from Python and 0.05 here.
//
// The C entries are called through addresses that ops.py takes from the library it has loaded, so this
// module links to torch only.  Nothing is thrown past a function here: errors are Python exceptions.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>

#include <string>

#include "nmi_fp8_linear.h"

namespace {

struct Raised {};       // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const std::string& why) {
    PyErr_SetString(type, why.c_str());
    throw Raised{};
}
[[noreturn]] void bad_value(const std::string& why) { refuse(PyExc_ValueError, why); }

struct Owned {
    PyObject* p;
    explicit Owned(PyObject* o) : p(o) {
        if (!p) throw Raised{};
    }
    ~Owned() { Py_XDECREF(p); }
    Owned(const Owned&) = delete;
};

std::string num(int64_t n) { return std::to_string(n); }
std::string list(at::IntArrayRef x) {
    std::string s = "(";
    for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + num(x[i]);
    return s + ")";
}
std::string show(const at::Tensor& t) {
    return std::string(c10::toString(t.scalar_type())) + " " + list(t.sizes()) + " strides " + list(t.strides());
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
void on_device(const at::Tensor& t, const char* name, int64_t dev) {
    if (t.get_device() != dev) bad_value(std::string("all tensors must be on one GPU: ") + name + " is on " + t.device().str());
}

// Rows [T, >= cols] of bf16 on GPU `dev`.
struct Rows {
    void* p = nullptr;
    int64_t ld = 0;
};
Rows rows(const at::Tensor& t, int64_t T, int64_t cols, const char* name, int64_t dev) {
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.size(0) != T || t.size(1) < cols || t.stride(1) != 1)
        bad_value(std::string(name) + " must be a bf16 [" + num(T) + ", >= " + num(cols) + "] tensor with contiguous rows, got " +
                  show(t));
    on_device(t, name, dev);
    // (torch's stride of a dimension of one element has no meaning)
    return {t.data_ptr(), T > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8};
}
Rows rows(PyObject* o, int64_t T, int64_t cols, const char* name, int64_t dev) { return rows(tensor(o, name), T, cols, name, dev); }

// A contiguous vector of n values on GPU `dev`; nullptr where it is None.
template <class V>
V* vector(PyObject* o, int64_t n, at::ScalarType type, const char* name, int64_t dev) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        bad_value(std::string(name) + " must be a contiguous " + c10::toString(type) + " vector of " + num(n) + " values, got " +
                  show(t));
    on_device(t, name, dev);
    return static_cast<V*>(t.data_ptr());
}

int as_int(int64_t n, const char* name) {
    if (n < 0 || n > INT32_MAX) bad_value(std::string(name) + "=" + num(n) + " is out of range");
    return (int)n;
}

// Whether two tensors of one shape lie alike: their strides, but for dimensions of one element, whose strides have
// no meaning.
bool lie_alike(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

// Pages [n_pages, n_kv_heads, page_size, 128] of any strides with contiguous head vectors, K and V alike.
nmi_paged_kv paged_kv(PyObject* k_o, PyObject* v_o, PyObject* table_o, int64_t batch, PyObject* k_scale, PyObject* v_scale,
                      int64_t dev) {
    const at::Tensor &k = tensor(k_o, "k_pages"), &v = tensor(v_o, "v_pages"), &table = tensor(table_o, "page_table");
    if (k.dim() != 4 || k.size(3) != 128 || k.stride(3) != 1)
        bad_value("k_pages must be [n_pages, n_kv_heads, page_size, 128] with contiguous head vectors, got " + show(k));
    const bool e4m3 = k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kByte;
    if (!e4m3 && k.scalar_type() != at::kBFloat16)
        refuse(PyExc_TypeError, std::string("pages must be bfloat16, float8_e4m3fn or uint8 codes, got ") +
                                    c10::toString(k.scalar_type()));
    if (v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() || !lie_alike(k, v))
        bad_value("v_pages must be as k_pages (" + show(k) + "), got " + show(v));
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != batch ||
        (table.size(1) > 1 && table.stride(1) != 1))
        bad_value("page_table must be int32 [batch=" + num(batch) + ", max_pages] with contiguous rows, got " + show(table));
    on_device(k, "k_pages", dev);
    on_device(v, "v_pages", dev);
    on_device(table, "page_table", dev);
    if (!k.size(1)) bad_value("pages of no KV heads");
    if (!e4m3 && (k_scale != Py_None || v_scale != Py_None)) bad_value("a bf16 cache takes no scales");
    nmi_paged_kv c{};
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    // (strides of a dimension of one element have no meaning)
    c.page_stride = k.size(0) > 1 ? k.stride(0) : 128;
    c.head_stride = k.size(1) > 1 ? k.stride(1) : 128;
    c.token_stride = k.size(2) > 1 ? k.stride(2) : 128;
    c.page_table = static_cast<const int32_t*>(table.data_ptr());
    c.page_table_stride = batch > 1 ? table.stride(0) : table.size(1);
    c.k_scale = vector<float>(k_scale, k.size(1), at::kFloat, "k_scale", dev);
    c.v_scale = vector<float>(v_scale, k.size(1), at::kFloat, "v_scale", dev);
    c.kv_type = e4m3 ? NMI_KV_E4M3 : NMI_KV_BF16;
    c.n_pages = as_int(k.size(0), "n_pages");
    c.page_size = as_int(k.size(2), "page_size");
    c.max_pages = as_int(table.size(1), "max_pages");
    c.n_kv_heads = as_int(k.size(1), "n_kv_heads");
    return c;
}

// Query heads of q [T, n_heads * 128].
int64_t query_heads(const at::Tensor& q, int64_t n_kv) {
    if (q.dim() != 2 || !q.size(1) || q.size(1) % (n_kv * 128))
        bad_value("q must be [T, n_heads * 128], n_heads a multiple of " + num(n_kv) + ", got " + list(q.sizes()));
    return q.size(1) / 128;
}

void on_gpu(const at::Tensor& t) {
    if (t.get_device() < 0) bad_value("tensors must be on a GPU, got " + t.device().str());
}

PyObject* new_ref(PyObject* o) {
    Py_INCREF(o);
    return o;
}
// The tensor given for an output, or a new one [T, cols] beside `like`.
PyObject* output(PyObject* given, const at::Tensor& like, int64_t T, int64_t cols) {
    PyObject* o = given != Py_None ? new_ref(given) : THPVariable_Wrap(at::empty({T, cols}, like.options()));
    if (!o) throw Raised{};
    return o;
}

template <class F>
F entry(PyObject* address) {
    void* p = PyLong_AsVoidPtr(address);
    if (!p) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no entry point");
        throw Raised{};
    }
    return reinterpret_cast<F>(p);
}
void* stream_of(PyObject* o) {
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Raised{};
    return p;
}
// What the library reports, raised by _lib.check.
void check(PyObject* raise_error, int rc, const char* name) {
    if (rc != NMI_OK) Owned(PyObject_CallFunction(raise_error, "is", rc, name));
}
float scale_of(PyObject* o) {
    if (o == Py_None) return 0.08838834764831845f;              // 1 / sqrt(128)
    const double s = PyFloat_AsDouble(o);
    if (s == -1.0 && PyErr_Occurred()) throw Raised{};
    return (float)s;
}

template <PyObject* (*BODY)(PyObject* const*), Py_ssize_t ARGS>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != ARGS) return PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, ARGS);
    try {
        return BODY(args);
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// _lib.check, stream, entry, k, v, k_pages, v_pages, page_table, start_pos, cu_seqlens, q, inv_freq, interleaved, k_scale,
// v_scale, q_out, k_out -> (q_out, k_out)
PyObject* kv_append_paged(PyObject* const* a) {
    const at::Tensor &k = tensor(a[3], "k"), &start = tensor(a[8], "start_pos");
    const int64_t dev = k.get_device(), T = k.dim() ? k.size(0) : -1;
    if (start.dim() != 1) bad_value("start_pos must be an int32 vector [batch], got " + list(start.sizes()));
    const int64_t batch = start.size(0);
    const int32_t* start_p = vector<int32_t>(a[8], batch, at::kInt, "start_pos", dev);
    const nmi_paged_kv cache = paged_kv(a[5], a[6], a[7], batch, a[13], a[14], dev);
    const int64_t n_kv = cache.n_kv_heads;
    const Rows kr = rows(k, T, n_kv * 128, "k", dev), vr = rows(a[4], T, n_kv * 128, "v", dev);
    const int32_t* cu = vector<int32_t>(a[9], batch + 1, at::kInt, "cu_seqlens", dev);
    if (a[9] == Py_None && T != batch) bad_value(num(T) + " rows for " + num(batch) + " sequences: give cu_seqlens");
    PyObject *q_o = a[10], *q_out = a[15], *k_out = a[16];
    if (q_o == Py_None && q_out != Py_None) bad_value("q_out without q");
    const float* freq = nullptr;
    int64_t rotary = 0, H = 0;
    Rows qr, qor, kor;
    if (a[11] != Py_None) {
        rotary = 2 * tensor(a[11], "inv_freq").numel();
        freq = vector<float>(a[11], rotary / 2, at::kFloat, "inv_freq", dev);
        if (q_o != Py_None) {
            H = query_heads(tensor(q_o, "q"), n_kv);
            qr = rows(q_o, T, H * 128, "q", dev);
            if (q_out != Py_None) qor = rows(q_out, T, H * 128, "q_out", dev);
        }
        if (k_out != Py_None) kor = rows(k_out, T, n_kv * 128, "k_out", dev);
    } else if (q_o != Py_None || k_out != Py_None) {
        bad_value("q and k_out are for the rotation: give inv_freq");
    }
    on_gpu(k);
    const int interleaved = PyObject_IsTrue(a[12]);
    if (interleaved < 0) throw Raised{};
    Owned out(q_o == Py_None ? new_ref(Py_None) : output(q_out, THPVariable_Unpack(q_o), T, H * 128));
    if (q_o != Py_None && q_out == Py_None) qor = {THPVariable_Unpack(out.p).data_ptr(), H * 128};
    if (T && batch) {
        auto call = entry<decltype(&nmi_kv_append_paged)>(a[2]);
        void* stream = stream_of(a[1]);
        const int b = as_int(batch, "batch"), n = as_int(T, "tokens"), h = as_int(H, "n_heads"), r = as_int(rotary, "rotary_dim");
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = call(&cache, qr.p, qr.ld, kr.p, kr.ld, vr.p, vr.ld, qor.p, qor.ld, kor.p, kor.ld, cu, start_p, b, n, h, freq, r,
                  interleaved, stream);
        Py_END_ALLOW_THREADS;
        check(a[0], rc, "nmi_kv_append_paged");
    }
    return PyTuple_Pack(2, out.p, k_out);
}

// _lib.check, stream, entry, its workspace's size, workspace, kept, q, k_pages, v_pages, page_table, kv_lens, k_scale, v_scale,
// scale, out -> out.  workspace(device, bytes, stream) -> (tensor, key), kept[key] = tensor after the launch.
PyObject* sdpa_decode_paged(PyObject* const* a) {
    const at::Tensor& q = tensor(a[6], "q");
    const int64_t dev = q.get_device();
    if (q.dim() != 2) bad_value("q must be [batch, n_heads * 128], got " + list(q.sizes()));
    const int64_t batch = q.size(0), cols = q.size(1);
    const nmi_paged_kv cache = paged_kv(a[7], a[8], a[9], batch, a[11], a[12], dev);
    const int64_t H = query_heads(q, cache.n_kv_heads);
    const Rows qr = rows(q, batch, cols, "q", dev);
    tensor(a[10], "kv_lens");
    const int32_t* lens = vector<int32_t>(a[10], batch, at::kInt, "kv_lens", dev);
    Rows orow;
    if (a[14] != Py_None) orow = rows(a[14], batch, cols, "out", dev);
    on_gpu(q);
    const float scale = scale_of(a[13]);
    Owned out(output(a[14], q, batch, cols));
    if (a[14] == Py_None) orow = {THPVariable_Unpack(out.p).data_ptr(), cols};
    if (batch) {
        auto call = entry<decltype(&nmi_sdpa_decode_paged)>(a[2]);
        auto bytes = entry<decltype(&nmi_sdpa_decode_paged_workspace_bytes)>(a[3]);
        void* stream = stream_of(a[1]);
        const int b = as_int(batch, "batch"), h = as_int(H, "n_heads");
        const size_t need = bytes(b, h, cache.n_kv_heads);
        Owned device(PyObject_GetAttrString(a[6], "device")), n(PyLong_FromSize_t(need));
        PyObject* argv[] = {device.p, n.p, a[1]};
        Owned taken(PyObject_Vectorcall(a[4], argv, 3, nullptr));
        if (!PyTuple_Check(taken.p) || PyTuple_GET_SIZE(taken.p) != 2) bad_value("workspace: (tensor, key) expected");
        PyObject *ws = PyTuple_GET_ITEM(taken.p, 0), *key = PyTuple_GET_ITEM(taken.p, 1);
        void* ws_p = tensor(ws, "workspace").data_ptr();
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = call(&cache, qr.p, qr.ld, orow.p, orow.ld, lens, b, h, scale, ws_p, need, stream);
        Py_END_ALLOW_THREADS;
        if (key != Py_None && PyDict_SetItem(a[5], key, ws)) throw Raised{};
        check(a[0], rc, "nmi_sdpa_decode_paged");
    }
    return new_ref(out.p);
}

// _lib.check, stream, entry, q, k, v, cu_seqlens, n_heads, n_kv_heads, scale, out -> out
PyObject* sdpa_prefill_packed_bf16(PyObject* const* a) {
    const at::Tensor& q = tensor(a[3], "q");
    const int64_t dev = q.get_device(), T = q.dim() ? q.size(0) : -1;
    const long H = PyLong_AsLong(a[7]), n_kv = PyLong_AsLong(a[8]);
    if ((H == -1 || n_kv == -1) && PyErr_Occurred()) throw Raised{};
    if (H < 1 || n_kv < 1 || H > INT32_MAX || n_kv > INT32_MAX)
        bad_value("n_heads=" + num(H) + " n_kv_heads=" + num(n_kv) + " must be at least 1");
    const Rows qr = rows(q, T, H * 128, "q", dev), kr = rows(a[4], T, n_kv * 128, "k", dev);
    const Rows vr = rows(a[5], T, n_kv * 128, "v", dev);
    const at::Tensor& offsets = tensor(a[6], "cu_seqlens");
    if (offsets.dim() != 1 || offsets.size(0) < 1)
        bad_value("cu_seqlens must be an int32 vector [batch + 1], got " + list(offsets.sizes()));
    const int64_t batch = offsets.size(0) - 1;
    const int32_t* cu = vector<int32_t>(a[6], batch + 1, at::kInt, "cu_seqlens", dev);
    Rows orow;
    if (a[10] != Py_None) orow = rows(a[10], T, H * 128, "out", dev);
    on_gpu(q);
    const float scale = scale_of(a[9]);
    Owned out(output(a[10], q, T, H * 128));
    if (a[10] == Py_None) orow = {THPVariable_Unpack(out.p).data_ptr(), H * 128};
    if (T && batch) {
        auto call = entry<decltype(&nmi_sdpa_prefill_packed_bf16)>(a[2]);
        void* stream = stream_of(a[1]);
        const int b = as_int(batch, "batch"), n = as_int(T, "tokens");
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = call(qr.p, qr.ld, kr.p, kr.ld, vr.p, vr.ld, orow.p, orow.ld, cu, b, n, (int)H, (int)n_kv, scale, stream);
        Py_END_ALLOW_THREADS;
        check(a[0], rc, "nmi_sdpa_prefill_packed_bf16");
    }
    return new_ref(out.p);
}

template <PyObject* (*BODY)(PyObject* const*), Py_ssize_t ARGS>
PyCFunction method() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<BODY, ARGS>));
}
PyMethodDef methods[] = {{"kv_append_paged", method<kv_append_paged, 17>(), METH_FASTCALL, nullptr},
                         {"sdpa_decode_paged", method<sdpa_decode_paged, 15>(), METH_FASTCALL, nullptr},
                         {"sdpa_prefill_packed_bf16", method<sdpa_prefill_packed_bf16, 11>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "front", "torch front end of the batched attention operators", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_front() { return PyModule_Create(&module); }
