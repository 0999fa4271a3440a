// The Python side of the routed 8-bit operators: checks torch tensors, allocates results from torch's
// allocator on the current stream and calls the C-ABI.  It is compiled because a serving step makes
// several such calls of a few microseconds each: the same checks and the ctypes call took 13-23 us a
// call in Python, more than the kernels.  stlq_b200/operators.py documents the operators; the functions
// here are theirs, with the handle and the device before the other arguments.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../include/stlq_b200.h"

namespace {

// The library's entry points, by the addresses that Python found in the library it loaded.
struct Api {
    decltype(&stlq_b200_last_error) last_error;
    decltype(&stlq_b200_quantize_rows) quantize_rows;
    decltype(&stlq_b200_matmul_i8) matmul_i8;
    decltype(&stlq_b200_matmul_i8_grouped) matmul_i8_grouped;
    decltype(&stlq_b200_sort_by_expert_workspace) sort_workspace;
    decltype(&stlq_b200_sort_by_expert) sort;
    decltype(&stlq_b200_dispatch) dispatch;
    decltype(&stlq_b200_dispatch_i8) dispatch_i8;
    decltype(&stlq_b200_combine) combine;
    decltype(&stlq_b200_combine_backward) combine_backward;
} api{};
PyObject* failed = nullptr;  // stlq_b200.StlqB200Error

struct Refused : std::runtime_error {  // ValueError
    using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {  // StlqB200Error
    using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python error is set

std::string Shown(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ") " + c10::toString(t.scalar_type());
}

void Check(int rc, const char* what) {
    if (rc) throw Failed(std::string(what) + " failed (" + std::to_string(rc) + "): " + api.last_error());
}

// ---- arguments ---------------------------------------------------------------------------------

struct Args {
    PyObject* const* v;
    Py_ssize_t n;
    void* handle;
    int device;

    Args(PyObject* const* args, Py_ssize_t count, Py_ssize_t expected) : v(args), n(count) {
        if (count != expected) throw Refused("wrong number of arguments");
        if (!api.last_error) throw Failed("the library has not been given");
        handle = PyLong_AsVoidPtr(v[0]);
        device = static_cast<int>(Int(1));
        if (PyErr_Occurred()) throw Raised{};
        if (!handle) throw Refused("the handle is closed");
    }
    long long Int(int i) const {
        const long long x = PyLong_AsLongLong(v[i]);
        if (x == -1 && PyErr_Occurred()) throw Raised{};
        return x;
    }
    const at::Tensor& Tensor(int i, const char* name) const {
        if (!THPVariable_Check(v[i])) throw Refused(std::string(name) + " must be a tensor");
        return THPVariable_Unpack(v[i]);
    }
    const at::Tensor* Maybe(int i, const char* name) const { return v[i] == Py_None ? nullptr : &Tensor(i, name); }
    void* Stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
    at::Tensor Empty(at::IntArrayRef shape, at::ScalarType type) const {
        return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt);
    }
};

int FloatCode(at::ScalarType t) {
    return t == at::kFloat ? STLQ_B200_F32 : t == at::kBFloat16 ? STLQ_B200_BF16 : t == at::kHalf ? STLQ_B200_F16 : -1;
}
bool IsFloat(at::ScalarType t) { return FloatCode(t) >= 0; }
constexpr const char* kFloats = "float32, bfloat16 or float16";

void On(const Args& a, const char* name, const at::Tensor& t) {
    if (!t.is_cuda() || t.get_device() != a.device)
        throw Refused(std::string(name) + " must be on cuda:" + std::to_string(a.device) + ", got " + t.device().str());
    if (t.layout() != at::kStrided) throw Refused(std::string(name) + " must be a dense tensor");
    if (t._fw_grad(0).defined())  // it would be dropped without a word
        throw Refused(std::string(name) + " carries a forward-mode tangent, and these operators have no forward-mode derivatives");
}

// A matrix with contiguous rows on the device; its leading dimension.
int64_t Rows(const Args& a, const char* name, const at::Tensor& t, bool type_ok, const char* types) {
    if (t.dim() != 2 || !type_ok) throw Refused(std::string(name) + " must be a matrix of " + types + ", got " + Shown(t));
    On(a, name, t);
    const int64_t rows = t.size(0), cols = t.size(1);
    const int64_t ld = rows > 1 ? t.stride(0) : std::max<int64_t>(cols, 1);
    if ((cols > 1 && t.stride(1) != 1) || ld < cols)
        throw Refused("the rows of " + std::string(name) + " must be contiguous and not overlap");
    if (cols > 0x7fffffff) throw Refused(std::string(name) + " has rows of 2^31 elements or more");
    return ld;
}

// The same for rows that are quantised or exchanged.
int64_t LongRows(const Args& a, const char* name, const at::Tensor& t, bool type_ok, const char* types) {
    const int64_t ld = Rows(a, name, t, type_ok, types);
    if (t.size(1) > STLQ_B200_MAX_COLS) throw Refused(std::string(name) + " has rows of more than 2^31 - 4096 elements");
    return ld;
}

void Vector(const Args& a, const char* name, const at::Tensor& t, int64_t n, at::ScalarType type) {
    if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != type || !t.is_contiguous())
        throw Refused(std::string(name) + " must be contiguous " + c10::toString(type) + " of shape (" + std::to_string(n) + ",), got " + Shown(t));
    On(a, name, t);
}

struct Route {
    int64_t tokens;
    int topk, experts;
    const int32_t *position, *offsets;
};
Route Routing(const Args& a, int at) {
    const at::Tensor &p = a.Tensor(at, "position"), &o = a.Tensor(at + 1, "offsets");
    if (p.dim() != 2 || o.dim() != 1 || p.scalar_type() != at::kInt || o.scalar_type() != at::kInt || !p.is_contiguous() || !o.is_contiguous())
        throw Refused("position (tokens, topk) and offsets (experts + 1,) must be contiguous int32");
    On(a, "the routing", p);
    On(a, "the routing", o);
    if (p.size(1) < 1 || p.size(1) > STLQ_B200_MAX_TOPK || o.size(0) < 2 || o.size(0) > STLQ_B200_MAX_ROOT + 1)
        throw Refused("topk must be in [1, 64] and experts in [1, 65536]");
    return {p.size(0), static_cast<int>(p.size(1)), static_cast<int>(o.size(0) - 1), p.const_data_ptr<int32_t>(), o.const_data_ptr<int32_t>()};
}

void Mix(const Args& a, const at::Tensor& w, const Route& r) {
    if (w.dim() != 2 || w.size(0) != r.tokens || w.size(1) != r.topk || !IsFloat(w.scalar_type()) || !w.is_contiguous())
        throw Refused("weights must be contiguous floats of shape (" + std::to_string(r.tokens) + ", " + std::to_string(r.topk) + "), got " + Shown(w));
    On(a, "weights", w);
}

// int8 rows on 16-byte boundaries, as the products read them; `whole` is what is returned to Python.
struct Rows8 {
    at::Tensor whole;
    int64_t ld;
};
Rows8 Empty8(const Args& a, int64_t rows, int64_t cols) {
    const int64_t ld = (cols + 15) / 16 * 16;
    at::Tensor t = a.Empty({rows, ld}, at::kChar);
    return {ld == cols ? t : t.narrow(1, 0, cols), ld};
}

// `t` as a product reads it: on 16-byte boundaries, copied there if it is not.
at::Tensor Operand(const Args& a, const char* name, const at::Tensor& t, int64_t* ld) {
    *ld = Rows(a, name, t, t.scalar_type() == at::kChar, "int8");
    if (t.size(0) <= 1) *ld = (*ld + 15) / 16 * 16;  // one row: its stride is not used, and bytes past its end are not read
    if (*ld % 16 == 0 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0) return t;
    Rows8 r = Empty8(a, t.size(0), t.size(1));
    r.whole.copy_(t);
    *ld = r.ld;
    return r.whole;
}

PyObject* Wrap(const at::Tensor& t) {
    PyObject* p = THPVariable_Wrap(t);
    if (!p) throw Raised{};
    return p;
}
PyObject* Wrap(const at::Tensor& x, const at::Tensor& y) {
    PyObject *p = Wrap(x), *q = nullptr;
    try {
        q = Wrap(y);
    } catch (...) {
        Py_DECREF(p);
        throw;
    }
    PyObject* t = PyTuple_Pack(2, p, q);
    Py_DECREF(p);
    Py_DECREF(q);
    if (!t) throw Raised{};
    return t;
}

template <typename F>
PyObject* Guard(F&& f) {
    try {
        return f();
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const Failed& e) {
        PyErr_SetString(failed ? failed : PyExc_RuntimeError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// ---- operators ---------------------------------------------------------------------------------

// (handle, device, x)
PyObject* QuantizeRows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 3);
        const at::Tensor& x = a.Tensor(2, "x");
        const int64_t ldx = LongRows(a, "x", x, IsFloat(x.scalar_type()), kFloats);
        const int64_t rows = x.size(0), cols = x.size(1);
        const Rows8 q = Empty8(a, rows, cols);
        const at::Tensor scale = a.Empty({rows}, at::kFloat);
        Check(api.quantize_rows(static_cast<stlq_b200_kernels*>(a.handle), x.const_data_ptr(), FloatCode(x.scalar_type()), ldx, rows,
                                static_cast<int>(cols), q.whole.mutable_data_ptr<int8_t>(), q.ld, scale.mutable_data_ptr<float>(), a.Stream()),
              "stlq_b200_quantize_rows");
        return Wrap(q.whole, scale);
    });
}

PyObject* Product(const Args& a, const at::Tensor& q, const at::Tensor& qs, const at::Tensor& w, const at::Tensor& ws, const at::Tensor* bias,
                  const at::Tensor* offsets, int experts, int64_t n, PyObject* type, PyObject* into) {
    const int64_t rows = q.size(0), kdim = q.size(1);
    if (w.size(1) != kdim) throw Refused("w has " + std::to_string(w.size(1)) + " columns, q " + std::to_string(kdim));
    if (kdim > STLQ_B200_MAX_I8_K) throw Refused("at most 131071 columns, got " + std::to_string(kdim));
    Vector(a, "q_scale", qs, rows, at::kFloat);
    Vector(a, "w_scale", ws, experts * n, at::kFloat);
    if (bias) Vector(a, "bias", *bias, experts * n, at::kFloat);
    if (into != Py_None && !THPVariable_Check(into)) throw Refused("out must be a tensor");
    at::ScalarType kind = into == Py_None ? at::kBFloat16 : THPVariable_Unpack(into).scalar_type();
    if (type != Py_None) {
        if (!THPDtype_Check(type)) throw Refused("out_dtype must be a torch.dtype");
        const at::ScalarType asked = reinterpret_cast<THPDtype*>(type)->scalar_type;
        if (into != Py_None && asked != kind) throw Refused("out has another type than out_dtype");
        kind = asked;
    }
    if (!IsFloat(kind)) throw Refused("out_dtype must be float32, bfloat16 or float16");
    const at::Tensor out = into == Py_None ? a.Empty({rows, n}, kind) : THPVariable_Unpack(into);
    if (out.dim() != 2 || out.size(0) != rows || out.size(1) != n)
        throw Refused("out must have shape (" + std::to_string(rows) + ", " + std::to_string(n) + "), got " + Shown(out));
    const int64_t ldo = Rows(a, "out", out, true, kFloats);
    if (out.requires_grad() && c10::GradMode::is_enabled())
        throw Refused("out requires a gradient, which this product does not have: detach it, or call under torch.no_grad()");
    int64_t ldq, ldw;
    const at::Tensor qo = Operand(a, "q", q, &ldq), wo = Operand(a, "w", w, &ldw);
    auto* h = static_cast<stlq_b200_kernels*>(a.handle);
    const float* b = bias ? bias->const_data_ptr<float>() : nullptr;
    if (offsets)
        Check(api.matmul_i8_grouped(h, qo.const_data_ptr<int8_t>(), ldq, qs.const_data_ptr<float>(), wo.const_data_ptr<int8_t>(), ldw,
                                    ws.const_data_ptr<float>(), b, offsets->const_data_ptr<int32_t>(), experts, rows, static_cast<int>(n),
                                    static_cast<int>(kdim), out.mutable_data_ptr(), FloatCode(kind), ldo, a.Stream()),
              "stlq_b200_matmul_i8_grouped");
    else
        Check(api.matmul_i8(h, qo.const_data_ptr<int8_t>(), ldq, qs.const_data_ptr<float>(), wo.const_data_ptr<int8_t>(), ldw,
                            ws.const_data_ptr<float>(), b, rows, static_cast<int>(n), static_cast<int>(kdim), out.mutable_data_ptr(),
                            FloatCode(kind), ldo, a.Stream()),
              "stlq_b200_matmul_i8");
    // A backward pass that saved `out` has to see that it changed.
    if (into != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return Wrap(out);
}

// (handle, device, q, q_scale, w, w_scale, bias, out_dtype, out)
PyObject* Matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 9);
        const at::Tensor &q = a.Tensor(2, "q"), &w = a.Tensor(4, "w");
        if (q.dim() != 2 || w.dim() != 2) throw Refused("q and w must be matrices");
        if (w.size(0) > 0x7fffffff) throw Refused("w has 2^31 rows or more");
        return Product(a, q, a.Tensor(3, "q_scale"), w, a.Tensor(5, "w_scale"), a.Maybe(6, "bias"), nullptr, 1, w.size(0), args[7], args[8]);
    });
}

// (handle, device, q, q_scale, w, w_scale, offsets, bias, out_dtype, out)
PyObject* MatmulGrouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 10);
        const at::Tensor &q = a.Tensor(2, "q"), &ws = a.Tensor(5, "w_scale"), &offsets = a.Tensor(6, "offsets");
        const at::Tensor* bias = a.Maybe(7, "bias");
        at::Tensor w = a.Tensor(4, "w");
        if (q.dim() != 2 || w.dim() != 3) throw Refused("q must be a matrix and w have three dimensions (experts, n, cols)");
        const int64_t experts = w.size(0), channels = w.size(1), cols = w.size(2);
        if (experts < 1 || experts > STLQ_B200_MAX_EXPERTS) throw Refused("experts must be in [1, 1024], got " + std::to_string(experts));
        if (channels > 0x7fffffff / experts) throw Refused("w has 2^31 rows or more");
        Vector(a, "offsets", offsets, experts + 1, at::kInt);
        const auto per_channel = [&](const at::Tensor& t) { return t.dim() == 2 && t.size(0) == experts && t.size(1) == channels; };
        if (!per_channel(ws) || (bias && !per_channel(*bias))) throw Refused("w_scale and bias must have shape (experts, n)");
        if (!ws.is_contiguous() || (bias && !bias->is_contiguous())) throw Refused("w_scale and bias must be contiguous");
        // The experts' rows follow one another.
        if (experts > 1 && channels > 0 && w.stride(0) != channels * (channels > 1 ? w.stride(1) : w.stride(0))) w = w.contiguous();
        const int64_t ld = channels > 1 ? w.stride(1) : experts > 1 ? w.stride(0) : std::max<int64_t>(cols, 1);
        w = w.as_strided({experts * channels, cols}, {ld, cols > 1 ? w.stride(2) : 1});
        const at::Tensor flat = ws.view({-1}), flat_bias = bias ? bias->view({-1}) : at::Tensor();
        return Product(a, q, a.Tensor(3, "q_scale"), w, flat, bias ? &flat_bias : nullptr, &offsets, static_cast<int>(experts), channels, args[8], args[9]);
    });
}

// (handle, device, ids, experts) -> order, position, offsets
PyObject* Sort(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&]() -> PyObject* {
        const Args a(args, n, 4);
        const at::Tensor& ids = a.Tensor(2, "ids");
        const long long experts = a.Int(3);
        const bool wide = ids.scalar_type() == at::kLong;
        if (ids.dim() < 1 || ids.dim() > 2 || (!wide && ids.scalar_type() != at::kInt) || !ids.is_contiguous())
            throw Refused("ids must be contiguous int32 or int64 of shape (tokens, topk), got " + Shown(ids));
        On(a, "ids", ids);
        const int64_t tokens = ids.size(0), topk = ids.dim() == 2 ? ids.size(1) : 1;
        if (topk < 1 || topk > STLQ_B200_MAX_TOPK || experts < 1 || experts > STLQ_B200_MAX_ROOT)
            throw Refused("topk must be in [1, 64] and experts in [1, 65536]");
        size_t bytes = 0;
        if (api.sort_workspace(tokens, static_cast<int>(topk), static_cast<int>(experts), &bytes)) throw Refused(api.last_error());
        const at::Tensor order = a.Empty({tokens * topk}, at::kInt), position = a.Empty({tokens, topk}, at::kInt);
        const at::Tensor offsets = a.Empty({experts + 1}, at::kInt);
        at::Tensor space;
        if (bytes) space = a.Empty({static_cast<int64_t>(bytes)}, at::kByte);
        Check(api.sort(static_cast<stlq_b200_kernels*>(a.handle), ids.const_data_ptr(), wide ? STLQ_B200_I64 : STLQ_B200_I32, tokens,
                       static_cast<int>(topk), static_cast<int>(experts), order.mutable_data_ptr<int32_t>(), position.mutable_data_ptr<int32_t>(),
                       offsets.mutable_data_ptr<int32_t>(), bytes ? space.mutable_data_ptr() : nullptr, bytes, a.Stream()),
              "stlq_b200_sort_by_expert");
        PyObject* two = Wrap(position, offsets);
        PyObject* one = THPVariable_Wrap(order);
        PyObject* t = one ? PyTuple_Pack(3, one, PyTuple_GET_ITEM(two, 0), PyTuple_GET_ITEM(two, 1)) : nullptr;
        Py_XDECREF(one);
        Py_DECREF(two);
        if (!t) throw Raised{};
        return t;
    });
}

// (handle, device, x, position, offsets)
PyObject* Dispatch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 5);
        const at::Tensor& x = a.Tensor(2, "x");
        const int64_t size = x.element_size();
        const int64_t ldx = LongRows(a, "x", x, size == 1 || size == 2 || size == 4, "elements of 1, 2 or 4 bytes");
        const Route r = Routing(a, 3);
        if (r.tokens != x.size(0)) throw Refused("the routing has " + std::to_string(r.tokens) + " rows, x " + std::to_string(x.size(0)));
        const int64_t cols = x.size(1);
        const at::Tensor out = a.Empty({r.tokens * r.topk, cols}, x.scalar_type());
        Check(api.dispatch(static_cast<stlq_b200_kernels*>(a.handle), x.const_data_ptr(), static_cast<int>(size), ldx, r.tokens,
                           static_cast<int>(cols), r.topk, r.position, r.offsets, r.experts, out.mutable_data_ptr(), cols, a.Stream()),
              "stlq_b200_dispatch");
        return Wrap(out);
    });
}

// (handle, device, x, position, offsets)
PyObject* DispatchI8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 5);
        const at::Tensor& x = a.Tensor(2, "x");
        const int64_t ldx = LongRows(a, "x", x, IsFloat(x.scalar_type()), kFloats);
        const Route r = Routing(a, 3);
        if (r.tokens != x.size(0)) throw Refused("the routing has " + std::to_string(r.tokens) + " rows, x " + std::to_string(x.size(0)));
        const int64_t cols = x.size(1);
        const Rows8 q = Empty8(a, r.tokens * r.topk, cols);
        const at::Tensor scale = a.Empty({r.tokens * r.topk}, at::kFloat);
        Check(api.dispatch_i8(static_cast<stlq_b200_kernels*>(a.handle), x.const_data_ptr(), FloatCode(x.scalar_type()), ldx, r.tokens,
                              static_cast<int>(cols), r.topk, r.position, r.offsets, r.experts, q.whole.mutable_data_ptr<int8_t>(), q.ld,
                              scale.mutable_data_ptr<float>(), a.Stream()),
              "stlq_b200_dispatch_i8");
        return Wrap(q.whole, scale);
    });
}

// (handle, device, y, weights, position, offsets)
PyObject* Combine(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 6);
        const at::Tensor& y = a.Tensor(2, "y");
        const at::Tensor* w = a.Maybe(3, "weights");
        const int64_t ldy = LongRows(a, "y", y, IsFloat(y.scalar_type()), kFloats);
        const Route r = Routing(a, 4);
        if (y.size(0) != r.tokens * r.topk)
            throw Refused("y must have tokens * topk = " + std::to_string(r.tokens * r.topk) + " rows, got " + std::to_string(y.size(0)));
        if (w) Mix(a, *w, r);
        const int64_t cols = y.size(1);
        const at::Tensor out = a.Empty({r.tokens, cols}, y.scalar_type());
        Check(api.combine(static_cast<stlq_b200_kernels*>(a.handle), y.const_data_ptr(), FloatCode(y.scalar_type()), ldy, r.tokens,
                          static_cast<int>(cols), r.topk, w ? w->const_data_ptr() : nullptr, w ? FloatCode(w->scalar_type()) : STLQ_B200_F32,
                          r.position, r.offsets, r.experts, out.mutable_data_ptr(), cols, a.Stream()),
              "stlq_b200_combine");
        return Wrap(out);
    });
}

// (handle, device, dout, y, weights, position, offsets)
PyObject* CombineBackward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&] {
        const Args a(args, n, 7);
        const at::Tensor &dout = a.Tensor(2, "dout"), &y = a.Tensor(3, "y"), &w = a.Tensor(4, "weights");
        const Route r = Routing(a, 5);
        const int64_t ldd = LongRows(a, "dout", dout, IsFloat(dout.scalar_type()), kFloats);
        const int64_t ldy = LongRows(a, "y", y, y.scalar_type() == dout.scalar_type(), "dout's type");
        if (dout.size(0) != r.tokens || y.size(0) != r.tokens * r.topk || dout.size(1) != y.size(1))
            throw Refused("dout and y must have " + std::to_string(r.tokens) + " and " + std::to_string(r.tokens * r.topk) +
                          " rows of one length, got " + Shown(dout) + " and " + Shown(y));
        Mix(a, w, r);
        const int64_t cols = y.size(1);
        const at::Tensor dy = a.Empty({y.size(0), cols}, y.scalar_type()), dw = a.Empty({r.tokens, r.topk}, w.scalar_type());
        Check(api.combine_backward(static_cast<stlq_b200_kernels*>(a.handle), dout.const_data_ptr(), FloatCode(dout.scalar_type()), ldd,
                                   y.const_data_ptr(), ldy, r.tokens, static_cast<int>(cols), r.topk, w.const_data_ptr(),
                                   FloatCode(w.scalar_type()), r.position, r.offsets, r.experts, dy.mutable_data_ptr(), cols,
                                   dw.mutable_data_ptr(), a.Stream()),
              "stlq_b200_combine_backward");
        return Wrap(dy, dw);
    });
}

// (order, position, offsets) -> tokens, topk, experts
PyObject* CheckRouting(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return Guard([&]() -> PyObject* {
        if (n != 3) throw Refused("order, position and offsets are needed");
        for (int i = 0; i < 3; ++i)
            if (!THPVariable_Check(args[i])) throw Refused("order, position and offsets must be tensors");
        const at::Tensor &o = THPVariable_Unpack(args[0]), &p = THPVariable_Unpack(args[1]), &f = THPVariable_Unpack(args[2]);
        if (o.dim() != 1 || p.dim() != 2 || f.dim() != 1) throw Refused("order, position and offsets must have 1, 2 and 1 dimensions");
        for (const at::Tensor* t : {&o, &p, &f})
            if (t->scalar_type() != at::kInt || !t->is_contiguous()) throw Refused("order, position and offsets must be contiguous int32");
        const int64_t tokens = p.size(0), topk = p.size(1), experts = f.size(0) - 1;
        if (o.size(0) != tokens * topk) throw Refused("order must have tokens * topk = " + std::to_string(tokens * topk) + " elements");
        if (topk < 1 || topk > STLQ_B200_MAX_TOPK) throw Refused("topk must be in [1, 64], got " + std::to_string(topk));
        if (experts < 1 || experts > STLQ_B200_MAX_ROOT) throw Refused("experts must be in [1, 65536], got " + std::to_string(experts));
        PyObject* t = Py_BuildValue("LLL", static_cast<long long>(tokens), static_cast<long long>(topk), static_cast<long long>(experts));
        if (!t) throw Raised{};
        return t;
    });
}

// (StlqB200Error, addresses of the entry points in Api's order)
PyObject* Give(PyObject*, PyObject* const* args, Py_ssize_t n) {
    constexpr Py_ssize_t kCount = sizeof(Api) / sizeof(void*);
    if (n != kCount + 1) {
        PyErr_SetString(PyExc_ValueError, "wrong number of entry points");
        return nullptr;
    }
    void* at[kCount];
    for (Py_ssize_t i = 0; i < kCount; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i + 1]);
        if (PyErr_Occurred()) return nullptr;
    }
    static_assert(sizeof(at) == sizeof(Api));
    memcpy(static_cast<void*>(&api), at, sizeof(at));
    Py_INCREF(args[0]);
    Py_XDECREF(failed);
    failed = args[0];
    Py_RETURN_NONE;
}

#define STLQ_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {STLQ_METHOD("give", Give),
                         STLQ_METHOD("check_routing", CheckRouting),
                         STLQ_METHOD("quantize_rows", QuantizeRows),
                         STLQ_METHOD("matmul_i8", Matmul),
                         STLQ_METHOD("matmul_i8_grouped", MatmulGrouped),
                         STLQ_METHOD("sort_by_expert", Sort),
                         STLQ_METHOD("dispatch", Dispatch),
                         STLQ_METHOD("dispatch_i8", DispatchI8),
                         STLQ_METHOD("combine", Combine),
                         STLQ_METHOD("combine_backward", CombineBackward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", "Checks and calls of the routed 8-bit operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__operators() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "BUILT_FOR", STLQ_BUILT_FOR) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
