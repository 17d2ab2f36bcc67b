// SPDX-License-Identifier: Apache-2.0
//
// The calls on torch's CUDA tensors (layers.py, optim.py) over the C ABI: the checks of their arguments, the tensors
// of their results and the current stream, in C++ because a single token's product takes 7 us on the device and the
// same steps in Python take as long (a step over 300 tensors: 100 us).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <exception>
#include <sstream>
#include <stdexcept>
#include <string>

#include "oztt_cuda.h"

namespace {

// Refusals, raised as ValueError.
struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& text) { throw Refused(text); }

std::string text(const at::Tensor& t) {
    std::ostringstream s;
    s << '[';
    for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
    s << ']';
    return s.str();
}

// torch.OutOfMemoryError, as torch's own operations raise it.
void raise_out_of_memory(const char* text) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (kind) PyErr_SetString(kind, text);
    Py_XDECREF(kind);
    Py_XDECREF(torch);
}

// Runs f, raising what it throws.
template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        raise_out_of_memory(e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::bad_alloc&) {
        PyErr_SetString(PyExc_MemoryError, "host memory exhausted");
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// One call of the C ABI without the interpreter's lock; its codes as layers.py's callers know them.
template <class F>
void call(F&& f) {
    char err[1024];
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f(err, sizeof err);
    Py_END_ALLOW_THREADS;
    if (rc == OZTT_OK) return;
    if (rc == OZTT_EINVAL) refuse(err);
    if (rc == OZTT_ENOMEM) throw std::bad_alloc();
    throw std::runtime_error(err);
}

// A call's scratch memory, from torch's allocator on the current stream: its cache serves the call, and it frees what it
// holds before it reports that there is none. Given back after the call, to whatever the stream does next.
struct TorchScratch {
    c10::DataPtr memory;
    std::exception_ptr failure;
    static void* alloc(void* self, size_t bytes) noexcept {
        auto* s = static_cast<TorchScratch*>(self);
        try {
            s->memory = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
            return s->memory.get();
        } catch (...) {
            s->failure = std::current_exception();
            return nullptr;
        }
    }
};
// call() of a function that takes an allocator and its context
template <class F>
void call_with_scratch(F&& f) {
    TorchScratch scratch;
    try {
        call([&](char* err, size_t len) { return f(&TorchScratch::alloc, &scratch, err, len); });
    } catch (const std::bad_alloc&) {
        if (scratch.failure) std::rethrow_exception(scratch.failure);
        throw;
    }
}

const at::Tensor* tensor_or_none(PyObject* o, const char* who, const char* what) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) refuse(std::string(who) + ": " + what + " must be a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* who, const char* what) {
    const at::Tensor* t = tensor_or_none(o, who, what);
    if (!t) refuse(std::string(who) + ": " + what + " is missing");
    return *t;
}

int32_t format_of(const at::Tensor& t, const char* who) {
    if (!t.is_cuda()) refuse(std::string(who) + ": the tensors must be on a CUDA device");
    if (t.scalar_type() == at::kBFloat16) return OZTT_FMT_BF16;
    if (t.scalar_type() == at::kHalf) return OZTT_FMT_FP16;
    refuse(std::string(who) + ": the type must be torch.bfloat16 or torch.float16, not " + c10::toString(t.scalar_type()));
}
void same_kind(const at::Tensor& first, const at::Tensor* t, const char* who, const char* what) {
    if (t && (t->scalar_type() != first.scalar_type() || t->device() != first.device()))
        refuse(std::string(who) + ": " + what + " must be " + c10::toString(first.scalar_type()) + " on " + first.device().str());
}

// A matrix, or a vector as one row.
oztt_view view(const at::Tensor& t) {
    const bool matrix = t.dim() == 2;
    return {t.data_ptr(), matrix ? t.stride(0) : 0, t.stride(matrix ? 1 : 0)};
}

// A tensor whose memory holds its values: itself, or a copy where torch keeps a negation or a zero for later.
at::Tensor with_values(const at::Tensor& t) { return t.is_neg() || t._is_zerotensor() ? t.clone() : t; }

at::Tensor rows_of(const at::Tensor& given, int64_t rows, int64_t cols) {
    const at::Tensor t = with_values(given);
    return t.dim() == 2 ? t : t.reshape({rows, cols});
}

bool wants_gradient(std::initializer_list<const at::Tensor*> all) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : all)
        if (t && t->requires_grad()) return true;
    return false;
}

// A tangent of torch's forward mode would be lost without a trace: the products have no derivatives of that kind.
void refuse_tangents(const char* who, std::initializer_list<const at::Tensor*> all) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const at::Tensor* t : all)
        if (t && t->_fw_grad(0).defined())
            throw std::runtime_error(std::string(who) + ": forward-mode differentiation is not supported");
}

// Whether torch is recording what it dispatches (a tracer, a dispatch mode), or a tensor has no memory of its own to be
// worked on (a subclass that dispatches, a functional or fake tensor): such a call has to be dispatched itself, since a
// recorder would keep the results' allocation and never see what is written into them. What must not pass in silence
// either way is refused: tangents, and the wrapped tensors of torch.func, which may hide some.
bool is_dispatched(const char* who, std::initializer_list<const at::Tensor*> all) {
    refuse_tangents(who, all);
    constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
    for (const at::Tensor* t : all)
        if (t && t->key_set().has_any(wrapped))
            throw std::runtime_error(std::string(who) + ": the transforms of torch.func are not supported");
    if (c10::impl::dispatch_mode_enabled() || at::tracer::impl::is_dispatch_enabled()) return true;
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Python, c10::DispatchKey::Functionalize});
    for (const at::Tensor* t : all)
        if (t && t->key_set().has_any(keys)) return true;
    return false;
}

PyObject* wrapped(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

bool expect(Py_ssize_t got, Py_ssize_t wanted, const char* who) {
    if (got == wanted) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", who, wanted);
    return false;
}

// linear(x, weight, bias, residual, activation, save_pre, outermost) -> (y, pre or None). A call that a user makes
// (`outermost`) gives None where a gradient is wanted, and NotImplemented where it has to be dispatched: layers.py
// makes it again from there.
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (!expect(count, 7, "linear")) return nullptr;
    return guarded([&]() -> PyObject* {
        constexpr const char* who = "linear";
        const at::Tensor &x = tensor(args[0], who, "x"), &w = tensor(args[1], who, "weight");
        const at::Tensor *b = tensor_or_none(args[2], who, "bias"), *r = tensor_or_none(args[3], who, "residual");
        const bool save_pre = args[5] == Py_True, outermost = args[6] == Py_True;
        if (outermost && is_dispatched(who, {&x, &w, b, r})) Py_RETURN_NOTIMPLEMENTED;
        oztt_linear a{};
        a.format = format_of(x, who);
        same_kind(x, &w, who, "weight");
        same_kind(x, b, who, "bias");
        same_kind(x, r, who, "residual");
        a.activation = (int32_t)PyLong_AsLong(args[4]);
        const int64_t dim = x.dim();
        if (w.dim() != 2 || !dim || x.size(dim - 1) != w.size(1))
            refuse("linear: x " + text(x) + " does not match weight " + text(w));
        const int64_t n = w.size(0), k = w.size(1);
        if (b && (b->dim() != 1 || b->size(0) != n)) refuse("linear: bias " + text(*b) + " does not match weight " + text(w));
        int64_t m = 1;
        bool fits = !r || r->dim() == dim;
        for (int64_t i = 0; i + 1 < dim; ++i) {
            m *= x.size(i);
            fits = fits && (!r || r->size(i) == x.size(i));
        }
        if (r && !(fits && r->size(dim - 1) == n))
            refuse("linear: residual " + text(*r) + " does not match the output of x " + text(x) + " and weight " + text(w));
        if (outermost && wants_gradient({&x, &w, b, r})) Py_RETURN_NONE;
        at::NoGradGuard no_grad;
        const at::Tensor x2 = rows_of(x, m, k), w2 = with_values(w), b2 = b ? with_values(*b) : at::Tensor();
        const at::Tensor r2 = r ? rows_of(*r, m, n) : at::Tensor();
        at::Tensor y = at::empty({m, n}, x.options().requires_grad(false)), pre;
        if (save_pre) pre = at::empty_like(y);
        a.m = (uint64_t)m;
        a.n = (uint64_t)n;
        a.k = (uint64_t)k;
        a.x = view(x2);
        a.w = view(w2);
        if (b) a.bias = view(b2);
        if (r) a.residual = view(r2);
        a.y = view(y);
        if (save_pre) a.pre = view(pre);
        const int device = x.get_device();
        void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        call_with_scratch([&](oztt_allocator alloc, void* context, char* err, size_t len) {
            return oztt_linear_forward_in(device, &a, alloc, context, stream, err, len);
        });
        if (dim != 2) {
            auto shape = x.sizes().vec();
            shape.back() = n;
            y = y.view(shape);
            if (save_pre) pre = pre.view(shape);
        }
        return Py_BuildValue("(NN)", wrapped(y), wrapped(pre));
    });
}

// linear_backward(dy, x, weight, pre, activation, need_input, need_weight, need_bias, outermost) -> (dx, dw, db), or
// NotImplemented where a user's call has to be dispatched
PyObject* linear_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (!expect(count, 9, "linear_backward")) return nullptr;
    return guarded([&]() -> PyObject* {
        constexpr const char* who = "linear_backward";
        const at::Tensor &dy = tensor(args[0], who, "dy"), &x = tensor(args[1], who, "x"), &w = tensor(args[2], who, "weight");
        const at::Tensor* pre = tensor_or_none(args[3], who, "pre");
        if (args[8] == Py_True && is_dispatched(who, {&dy, &x, &w, pre})) Py_RETURN_NOTIMPLEMENTED;
        oztt_linear_grad a{};
        a.format = format_of(dy, who);
        same_kind(dy, &x, who, "x");
        same_kind(dy, &w, who, "weight");
        same_kind(dy, pre, who, "pre");
        a.activation = (int32_t)PyLong_AsLong(args[4]);
        const int64_t dim = x.dim();
        if (w.dim() != 2 || !dim || x.size(dim - 1) != w.size(1))
            refuse("linear_backward: x " + text(x) + " does not match weight " + text(w));
        const int64_t n = w.size(0), k = w.size(1);
        int64_t m = 1;
        bool fits = dy.dim() == dim && dy.size(dim - 1) == n;
        for (int64_t i = 0; i + 1 < dim; ++i) {
            m *= x.size(i);
            fits = fits && dy.size(i) == x.size(i);
        }
        if (!fits) refuse("linear_backward: dy " + text(dy) + " does not match x " + text(x) + " and weight " + text(w));
        if (a.activation != OZTT_ACT_NONE && !pre) refuse("linear_backward: the activation needs pre");
        if (pre && pre->sizes() != dy.sizes())
            refuse("linear_backward: pre " + text(*pre) + " does not match dy " + text(dy));
        at::NoGradGuard no_grad;
        const at::Tensor x2 = rows_of(x, m, k), w2 = with_values(w), dy2 = rows_of(dy, m, n);
        const at::Tensor pre2 = pre ? rows_of(*pre, m, n) : at::Tensor();
        const auto options = dy.options().requires_grad(false);
        at::Tensor dx, dw, db;
        if (args[5] == Py_True) dx = at::empty({m, k}, options);
        if (args[6] == Py_True) dw = at::empty({n, k}, options);
        if (args[7] == Py_True) db = at::empty({n}, options);
        a.m = (uint64_t)m;
        a.n = (uint64_t)n;
        a.k = (uint64_t)k;
        a.dy = view(dy2);
        a.x = view(x2);
        a.w = view(w2);
        if (pre) a.pre = view(pre2);
        if (dx.defined()) a.dx = view(dx);
        if (dw.defined()) a.dw = view(dw);
        if (db.defined()) a.db = view(db);
        if (dx.defined() || dw.defined() || db.defined()) {
            const int device = dy.get_device();
            void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
            call_with_scratch([&](oztt_allocator alloc, void* context, char* err, size_t len) {
                return oztt_linear_backward_in(device, &a, alloc, context, stream, err, len);
            });
        }
        if (dim != 2 && dx.defined()) dx = dx.view(x.sizes());
        return Py_BuildValue("(NNN)", wrapped(dx), wrapped(dw), wrapped(db));
    });
}

int32_t type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return OZTT_TYPE_BF16;
        case at::kHalf: return OZTT_TYPE_FP16;
        case at::kFloat: return OZTT_TYPE_FP32;
        default: return -1;
    }
}

// Whether a tensor is its memory: not one that dispatches elsewhere (a subclass, a wrapped, functional or fake tensor),
// nor one that keeps a negation or a zero for later.
bool is_memory(const at::Tensor& t) {
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                        c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
    return !t.key_set().has_any(keys);
}

// A tracer, or a mode that records programs or computes shapes alone, sees nothing of what is written here.
void refuse_recorders(const char* who) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    bool some = at::tracer::impl::is_dispatch_enabled();
    if (c10::impl::dispatch_mode_enabled())
        for (const auto key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
            some = some || TorchDispatchModeTLS::get_mode(key).has_value();
    if (some) throw std::runtime_error(std::string(who) + " cannot be traced or recorded");
}

// The items of a list or tuple of n (not to be looked at after the lock has been released).
PyObject** items(PyObject* o, Py_ssize_t n, const char* what) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) refuse(std::string("AdamW: ") + what + " must be a list or a tuple");
    if (PySequence_Fast_GET_SIZE(o) != n) refuse(std::string("AdamW: ") + what + " must be as many as params");
    return PySequence_Fast_ITEMS(o);
}

// The record of the moments (m, v, m_exp, v_exp) of `blocks` blocks, the exponents None with 32 bits. Their addresses
// are asked for in every call: a copy of an optimiser has other buffers than the original.
oztt_adamw_moments moments_of(PyObject* four, uint64_t blocks, int device) {
    if (!PyTuple_Check(four) || PyTuple_GET_SIZE(four) != 4) throw std::runtime_error("AdamW: the moments are four buffers");
    const auto buffer = [&](int i, bool wide, uint64_t count) -> void* {
        const at::Tensor* t = tensor_or_none(PyTuple_GET_ITEM(four, i), "AdamW", "a buffer of the moments");
        if (!t || !t->is_cuda() || t->get_device() != device || t->scalar_type() != (wide ? at::kFloat : at::kByte) ||
            (uint64_t)t->numel() != count || !t->is_contiguous())
            refuse("AdamW: a buffer of the moments is not what it was made as");
        return t->data_ptr();
    };
    oztt_adamw_moments m{};
    m.bits = PyTuple_GET_ITEM(four, 2) == Py_None ? 32 : 8;
    m.m = buffer(0, m.bits == 32, blocks * OZTT_ADAMW_BLOCK);
    m.v = buffer(1, m.bits == 32, blocks * OZTT_ADAMW_BLOCK);
    if (m.bits == 8) {
        m.m_exp = static_cast<uint8_t*>(buffer(2, false, blocks));
        m.v_exp = static_cast<uint8_t*>(buffer(3, false, blocks));
    }
    return m;
}

// adamw_step(table, params, masters, grads, grad_scale, moments, hyper, device): table a writable buffer of
// oztt_adamw_tensor, one for each parameter, with the count and type that it was made for; the addresses, which a
// program may change between steps, are filled in here. masters and grads may hold None; moments are the four
// buffers, hyper the bytes of oztt_adamw_hyper (with grad_scale filled in here).
PyObject* adamw_step(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (!expect(count, 8, "adamw_step")) return nullptr;
    Py_buffer table;
    if (PyObject_GetBuffer(args[0], &table, PyBUF_WRITABLE) != 0) return nullptr;
    PyObject* result = guarded([&]() -> PyObject* {
        refuse_recorders("AdamW.step");
        auto* t = static_cast<oztt_adamw_tensor*>(table.buf);
        const Py_ssize_t n = table.len / (Py_ssize_t)sizeof(oztt_adamw_tensor);
        PyObject **params = items(args[1], n, "params"), **masters = items(args[2], n, "masters"),
                 **grads = items(args[3], n, "grads");
        const int device = (int)PyLong_AsLong(args[7]);
        uint64_t blocks = 0;
        for (Py_ssize_t i = 0; i < n; ++i) blocks += (t[i].count + OZTT_ADAMW_BLOCK - 1) / OZTT_ADAMW_BLOCK;
        const oztt_adamw_moments moments = moments_of(args[5], blocks, device);
        for (Py_ssize_t i = 0; i < n; ++i) {
            const auto address = [&](const at::Tensor& x, const char* what) -> void* {
                const auto which = [&] { return std::string("AdamW: ") + what + " " + std::to_string(i); };
                if (!x.is_cuda() || x.get_device() != device) refuse(which() + " must be on the parameters' device");
                if ((uint64_t)x.numel() != t[i].count) refuse(which() + " has not its parameter's size");
                if (!x.is_contiguous()) refuse(which() + " must be contiguous");
                if (!is_memory(x)) refuse(which() + " has no memory of its own values");
                return x.data_ptr();
            };
            t[i].grad = nullptr;
            const at::Tensor* g = tensor_or_none(grads[i], "AdamW", "a gradient");
            if (!g) continue;
            t[i].grad_type = type_of(*g);
            if (t[i].grad_type < 0) refuse("AdamW: gradient " + std::to_string(i) + " must be BF16, FP16 or FP32");
            t[i].grad = address(*g, "gradient");
            const at::Tensor& p = tensor(params[i], "AdamW", "a parameter");
            if (type_of(p) != t[i].param_type) refuse("AdamW: parameter " + std::to_string(i) + " has changed its type");
            t[i].param = address(p, "parameter");
            const at::Tensor* w = tensor_or_none(masters[i], "AdamW", "a master");
            if (w && w->scalar_type() != at::kFloat) refuse("AdamW: master " + std::to_string(i) + " must be FP32");
            t[i].master = w ? static_cast<float*>(address(*w, "master")) : nullptr;
        }
        oztt_adamw_hyper hyper;
        if (PyBytes_GET_SIZE(args[6]) != sizeof hyper) throw std::runtime_error("adamw_step: a record of another size");
        std::memcpy(&hyper, PyBytes_AS_STRING(args[6]), sizeof hyper);
        if (const at::Tensor* s = tensor_or_none(args[4], "AdamW", "grad_scale")) {
            if (s->scalar_type() != at::kFloat || !s->is_cuda() || s->get_device() != device || s->numel() != 1 || !is_memory(*s))
                refuse("AdamW: grad_scale must be one FP32 number on the parameters' device");
            hyper.grad_scale = s->const_data_ptr<float>();
        }
        // what was saved for a backward pass that has not run is no longer what it was
        const auto written = [](PyObject* o) {
            if (o == Py_None) return;
            const at::Tensor& x = THPVariable_Unpack(o);
            if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
        };
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (grads[i] == Py_None) continue;
            written(params[i]);
            written(masters[i]);
        }
        for (Py_ssize_t i = 0; i < 4; ++i) written(PyTuple_GET_ITEM(args[5], i));
        void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        call([&](char* err, size_t len) { return oztt_adamw_step(device, t, (uint64_t)n, &moments, &hyper, stream, err, len); });
        Py_RETURN_NONE;
    });
    PyBuffer_Release(&table);
    return result;
}

// adamw_values(moments, blocks, device) -> (m, v): the values of 8-bit moments as BF16
PyObject* adamw_values(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (!expect(count, 3, "adamw_values")) return nullptr;
    return guarded([&]() -> PyObject* {
        refuse_recorders("AdamW.moments");
        const int64_t blocks = PyLong_AsLongLong(args[1]);
        const int device = (int)PyLong_AsLong(args[2]);
        const oztt_adamw_moments moments = moments_of(args[0], (uint64_t)blocks, device);
        const auto options = at::TensorOptions(at::kBFloat16).device(at::kCUDA, (c10::DeviceIndex)device);
        const at::Tensor m = at::empty({blocks * OZTT_ADAMW_BLOCK}, options), v = at::empty_like(m);
        void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        call([&](char* err, size_t len) {
            return oztt_adamw_values(device, &moments, (uint64_t)blocks, static_cast<uint16_t*>(m.data_ptr()),
                                     static_cast<uint16_t*>(v.data_ptr()), stream, err, len);
        });
        return Py_BuildValue("(NN)", wrapped(m), wrapped(v));
    });
}

// has_memory(tensor) -> bool
PyObject* has_memory(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (!expect(count, 1, "has_memory")) return nullptr;
    return guarded([&]() -> PyObject* { return PyBool_FromLong(is_memory(tensor(args[0], "AdamW", "a parameter"))); });
}

PyMethodDef methods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"linear_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear_backward)), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adamw_step)), METH_FASTCALL, nullptr},
    {"adamw_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adamw_values)), METH_FASTCALL, nullptr},
    {"has_memory", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(has_memory)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch() { return PyModule_Create(&module); }
