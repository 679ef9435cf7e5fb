// _ctm_lists: the short way from a Python list of tensors to the C entries over lists (ctm_grad_norms, ctm_grad_clip, ctm_sgd_step).  What those
// entries cost on the lists of an optimisation is mostly the host's reading of pointers, dtypes and layouts: ten Python attribute accesses per
// tensor are ~0.8 us, this module needs ~0.03 us.  It takes the plain case -- contiguous tensors of one dtype on one device -- and returns None for
// everything else, refused arguments included (the interpreter's lock is held all along: nobody changes a list meanwhile); the caller (_native.py) then goes its
// general way, which handles strided views and words the errors.
#include <torch/csrc/Device.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <cstring>
#include <vector>
#include "../../include/ctm_hip.h"

namespace {

using norms_fn = decltype(&ctm_grad_norms);
using clip_fn = decltype(&ctm_grad_clip);
using sgd_fn = decltype(&ctm_sgd_step);

// The arguments every call starts with: (entry, float64 context, complex128 context, device, stream)
struct Call {
    void* fn; ctm_ctx* ctx[2]; c10::Device device; void* stream;
    bool cplx = false;
    ctm_ctx* context() const { return ctx[cplx]; }
};

struct List {
    PyObject* seq = nullptr;
    Py_ssize_t n = 0;
    std::vector<const double*> ptr;
    std::vector<long long> numel;
    const at::Tensor& at(Py_ssize_t i) const { return THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq, i)); }
};

// false: not the plain case.  `like`: the list whose shapes and dtype this one has to have.  `written`: the call writes it -- memory that a tensor
// shares with its lazy clones until one of them is written becomes its own here.
bool read(Call& c, PyObject* seq, List& l, const List* like, bool written) {
    if (!PyList_CheckExact(seq) && !PyTuple_CheckExact(seq)) return false;
    l.seq = seq;
    l.n = PySequence_Fast_GET_SIZE(seq);
    if (l.n == 0 || (like && like->n != l.n)) return false;
    l.ptr.resize(l.n);
    l.numel.resize(l.n);
    for (Py_ssize_t i = 0; i < l.n; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
        if (!THPVariable_Check(o)) return false;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || t.layout() != at::kStrided || t.device() != c.device || !t.has_storage()) return false;
        const at::ScalarType st = t.scalar_type();
        if (st != at::kDouble && st != at::kComplexDouble) return false;
        if (i == 0 && !like) c.cplx = st == at::kComplexDouble;
        if ((st == at::kComplexDouble) != c.cplx || !t.is_contiguous() || t.is_conj() || t.is_neg()) return false;
        if (like && t.sizes() != like->at(i).sizes()) return false;
        l.ptr[i] = static_cast<const double*>(written ? t.mutable_data_ptr() : t.const_data_ptr());
        l.numel[i] = t.numel();
    }
    return c.context() != nullptr;
}

void changed(const List& l) {
    for (Py_ssize_t i = 0; i < l.n; ++i) {
        const at::Tensor& t = l.at(i);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
}

at::Tensor workspace(const Call& c, Py_ssize_t n) {
    return at::empty({(int64_t)CTM_GRAD_WS_DOUBLES(n)}, at::TensorOptions().dtype(at::kDouble).device(c.device));
}

// [N2, Ninf]: the head of the workspace
PyObject* norms_of(at::Tensor&& ws) {
    ws.unsafeGetTensorImpl()->set_sizes_contiguous({2});
    return THPVariable_Wrap(std::move(ws));
}

// What a call that did not succeed gives: an argument that the entry refused goes the general way (nothing was launched), any other status is
// returned as a number.
PyObject* failed(int st) {
    if (st == CTM_ERR_BADARG) Py_RETURN_NONE;
    return PyLong_FromLong(st);
}

bool call_of(PyObject* const* a, Call& c) {
    if (!THPDevice_Check(a[3])) return false;
    c.fn = PyLong_AsVoidPtr(a[0]);
    c.ctx[0] = (ctm_ctx*)PyLong_AsVoidPtr(a[1]);
    c.ctx[1] = (ctm_ctx*)PyLong_AsVoidPtr(a[2]);
    c.device = reinterpret_cast<THPDevice*>(a[3])->device;
    c.stream = PyLong_AsVoidPtr(a[4]);
    return !PyErr_Occurred();
}

PyObject* general_way() {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

#define ENTRY(min_args)                                                                                                    \
    if (nargs != min_args) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }              \
    Call c{nullptr, {nullptr, nullptr}, c10::Device(c10::kCPU), nullptr};                                                  \
    if (!call_of(a, c)) return general_way();                                                                              \
    try {
#define END_ENTRY                                                                                                          \
    } catch (const std::exception& e) { PyErr_SetString(PyExc_RuntimeError, e.what()); return nullptr; }                   \
    return general_way();

// (entry, ctx, ctx, device, stream, tensors)
PyObject* grad_norms(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ENTRY(6)
    List x;
    if (read(c, a[5], x, nullptr, false)) {
        at::Tensor ws = workspace(c, x.n);
        const int st = ((norms_fn)c.fn)(c.context(), c.stream, (int)x.n, x.ptr.data(), x.numel.data(), ws.mutable_data_ptr<double>(), ws.numel());
        return st == CTM_OK ? norms_of(std::move(ws)) : failed(st);
    }
    END_ENTRY
}

// (entry, ctx, ctx, device, stream, tensors, outputs or None, norm code, max_norm)
PyObject* grad_clip(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ENTRY(9)
    List x, y;
    if (read(c, a[5], x, nullptr, a[6] == Py_None) && (a[6] == Py_None || read(c, a[6], y, &x, true))) {
        const List& out = a[6] == Py_None ? x : y;
        const int code = (int)PyLong_AsLong(a[7]);
        const double bound = PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) return nullptr;
        at::Tensor ws = workspace(c, x.n);
        const int st = ((clip_fn)c.fn)(c.context(), c.stream, (int)x.n, x.ptr.data(), const_cast<double* const*>(out.ptr.data()), x.numel.data(), code,
                                       bound, ws.mutable_data_ptr<double>(), ws.numel());
        if (st != CTM_OK) return failed(st);
        changed(out);
        return norms_of(std::move(ws));
    }
    END_ENTRY
}

// (entry, ctx, ctx, device, stream, params, grads, buffers or None, lr, momentum, dampening, first, norm code, max_norm); True without a bound
PyObject* sgd_step(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ENTRY(14)
    List p, g, m;
    const bool buffers = a[7] != Py_None;
    if (read(c, a[5], p, nullptr, true) && read(c, a[6], g, &p, false) && (!buffers || read(c, a[7], m, &p, true))) {
        const double lr = PyFloat_AsDouble(a[8]), mu = PyFloat_AsDouble(a[9]), tau = PyFloat_AsDouble(a[10]), bound = PyFloat_AsDouble(a[13]);
        const int first = PyObject_IsTrue(a[11]), code = (int)PyLong_AsLong(a[12]);
        if (PyErr_Occurred()) return nullptr;
        at::Tensor ws;
        if (bound >= 0.0) ws = workspace(c, p.n);
        const int st = ((sgd_fn)c.fn)(c.context(), c.stream, (int)p.n, const_cast<double* const*>(p.ptr.data()), g.ptr.data(),
                                      buffers ? const_cast<double* const*>(m.ptr.data()) : nullptr, p.numel.data(), lr, mu, tau, first, code, bound,
                                      ws.defined() ? ws.mutable_data_ptr<double>() : nullptr, ws.defined() ? ws.numel() : 0);
        if (st != CTM_OK) return failed(st);
        changed(p);
        if (buffers) changed(m);
        if (ws.defined()) return norms_of(std::move(ws));
        Py_RETURN_TRUE;
    }
    END_ENTRY
}

PyMethodDef methods[] = {{"grad_norms", (PyCFunction)(void (*)(void))grad_norms, METH_FASTCALL, nullptr},
                         {"grad_clip", (PyCFunction)(void (*)(void))grad_clip, METH_FASTCALL, nullptr},
                         {"sgd_step", (PyCFunction)(void (*)(void))sgd_step, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ctm_lists", "Lists of tensors on their way to the native library", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (the module reads torch's own structures: only with the release that it was compiled against)
PyMODINIT_FUNC PyInit__ctm_lists() {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
    PyObject* str = version ? PyObject_Str(version) : nullptr;
    const char* v = str ? PyUnicode_AsUTF8(str) : nullptr;
    const bool same = v && !strcmp(v, CTM_TORCH_VERSION);
    if (v && !same) PyErr_Format(PyExc_ImportError, "compiled against torch " CTM_TORCH_VERSION ", not %s", v);
    Py_XDECREF(str);
    Py_XDECREF(version);
    Py_XDECREF(torch);
    return same ? PyModule_Create(&module) : nullptr;
}
