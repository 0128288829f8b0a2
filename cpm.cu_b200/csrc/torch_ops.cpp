// Python module cpmcu._ops: the operators on the caller's streams (part 4 of include/cpmcu_b200.h) for torch tensors.  Checks of arguments, outputs and
// workspaces of torch's allocator, and torch's current stream, in one call: through ctypes the same takes 4 to 6 us more, as long as the launch and
// longer than many of the kernels run (one token's product 7.9 us a call that way).  Refusals are ValueErrors, what the library reports is a
// RuntimeError, and torch's allocator without memory torch.OutOfMemoryError.
#include <Python.h>

#include <initializer_list>
#include <limits>
#include <string>

#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/cpmcu_b200.h"

namespace {

struct Raised {   // a Python exception to set
    PyObject* type;
    std::string text;
};
struct PythonError {};   // one that is set already

[[noreturn]] void refuse(const std::string& text) { throw Raised{PyExc_ValueError, text}; }

std::string shape_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}
const char* dtype_text(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return "torch.bfloat16";
        case at::kFloat: return "torch.float32";
        case at::kInt: return "torch.int32";
        case at::kByte: return "torch.uint8";
        default: return c10::toString(t);
    }
}

const at::Tensor& tensor_of(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor& matrix_of(PyObject* o, const char* what) {
    if (!THPVariable_Check(o) || THPVariable_Unpack(o).dim() != 2) refuse(std::string(what) + " must be a matrix");
    return THPVariable_Unpack(o);
}

// rows: any distance between the rows of a matrix; otherwise contiguous.  device < 0: any GPU.
void check(const at::Tensor& t, const char* what, at::ScalarType type, std::initializer_list<int64_t> shape, int device, bool rows = false) {
    if (t.scalar_type() != type || t.sizes() != at::IntArrayRef(shape)) {
        refuse(std::string(what) + " must be " + dtype_text(type) + " of shape " + shape_text(shape) + ", got " + dtype_text(t.scalar_type()) + " " + shape_text(t.sizes()));
    }
    if (!t.is_cuda() || (device >= 0 && t.get_device() != device)) {
        refuse(std::string(what) + " must be on " + (device >= 0 ? "cuda:" + std::to_string(device) : "the GPU") + ", got " + t.device().str());
    }
    if (t.is_contiguous()) return;
    if (!rows) refuse(std::string(what) + " must be contiguous");
    if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) {
        refuse(std::string(what) + " must have consecutive elements in rows that do not overlap");
    }
}
long long ld_of(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(1, t.size(1)); }

long long whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}
int small(PyObject* o, const char* what) {
    const long long v = whole(o);
    if (v < std::numeric_limits<int>::min() || v > std::numeric_limits<int>::max()) refuse(std::string(what) + " does not fit 32 bits");
    return static_cast<int>(v);
}
int small(int64_t v, const char* what) {
    if (v > std::numeric_limits<int>::max()) refuse(std::string(what) + " does not fit 32 bits");
    return static_cast<int>(v);
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError();
    return static_cast<float>(v);
}

// Makes a GPU current for a while.
struct Device {
    c10::cuda::OptionalCUDAGuard guard;
    explicit Device(int device) {
        if (c10::cuda::current_device() != device) guard.set_index(static_cast<c10::DeviceIndex>(device));
    }
};
// Straight from torch's allocator: the dispatcher's way there takes longer than the allocation.
at::Tensor empty(std::initializer_list<int64_t> shape, at::ScalarType type, int device) {
    const Device current(device);
    return at::detail::empty_generic(at::IntArrayRef(shape), c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

// Runs an entry point with GPU `device` current, on torch's current stream of it, without the interpreter's lock.  What torch throws in there is
// carried out of it as text: an exception must not pass the point where the lock is taken again.
template <typename F>
void run(int device, F&& call) {
    int code = -1;
    std::string text;
    Py_BEGIN_ALLOW_THREADS
    try {
        const Device current(device);
        code = call(static_cast<void*>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()));
        if (code < 0) text = cpmcu_last_error();
    } catch (const std::exception& e) {
        code = -1;
        text = e.what();
    }
    Py_END_ALLOW_THREADS
    if (code < 0) throw Raised{PyExc_RuntimeError, text};
}

// The rows of a layer and what is made of them before the product: arguments shared by linear and ffn.
struct Input {
    at::Tensor x, norm, delta, total, out;
    int rows = 0, device = 0;
    float eps = 0.f, delta_scale = 1.f;
    const void* pointer(const at::Tensor& t) const { return t.defined() ? t.data_ptr() : nullptr; }
};
Input input_of(PyObject* x, int width, int out, int device, PyObject* norm, PyObject* eps, PyObject* delta, PyObject* delta_scale, PyObject* y) {
    Input in;
    in.device = device;
    in.x = matrix_of(x, "x");
    const int64_t rows = in.x.size(0);
    in.rows = small(rows, "the number of rows");
    check(in.x, "x", at::kBFloat16, {rows, width}, device, true);
    if (norm != Py_None) {
        in.norm = tensor_of(norm, "norm_weight");
        check(in.norm, "norm_weight", at::kBFloat16, {width}, device);
        in.eps = real(eps);
    }
    if (delta != Py_None) {
        if (norm == Py_None) refuse("delta needs norm_weight");
        in.delta = tensor_of(delta, "delta");
        check(in.delta, "delta", at::kBFloat16, {rows, width}, device);
        in.delta_scale = real(delta_scale);
        in.total = empty({rows, width}, at::kBFloat16, device);
    }
    if (y != Py_None) {
        in.out = tensor_of(y, "out");
        check(in.out, "out", at::kBFloat16, {rows, out}, device, true);
    } else {
        in.out = empty({rows, out}, at::kBFloat16, device);
    }
    return in;
}
c10::DataPtr workspace_of(const Input& in, int out, int width, int inter, long& bytes) {
    const Device current(in.device);   // also of the question: the division of the work asks the GPU what it holds
    bytes = cpmcu_w8a8_workspace_bytes(in.rows, out, width, inter);
    if (bytes < 0) refuse(cpmcu_last_error());
    if (bytes == 0) return c10::DataPtr();
    return c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes));
}
PyObject* result_of(const Input& in) {
    PyObject* y = THPVariable_Wrap(in.out);
    if (!in.total.defined()) return y;
    PyObject* t = THPVariable_Wrap(in.total);
    PyObject* both = PyTuple_Pack(2, y, t);
    Py_DECREF(y);
    Py_DECREF(t);
    return both;
}

// Packed weights: their bytes, and the GPU they are on.
const at::Tensor& packed_of(PyObject* o, const char* what, int out, int width, bool gated, int device = -1) {
    const at::Tensor& t = tensor_of(o, what);
    const long bytes = cpmcu_w8a8_packed_bytes(out, width, gated);
    if (bytes < 0) refuse(cpmcu_last_error());
    check(t, what, at::kByte, {bytes}, device);
    return t;
}

void out_of_memory(const char* text) {   // torch.OutOfMemoryError
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_Clear();
    PyErr_SetString(type != nullptr ? type : PyExc_RuntimeError, text);
    Py_XDECREF(type);
    Py_XDECREF(torch);
}

template <Py_ssize_t N, typename F>
PyObject* guarded(Py_ssize_t n, F&& f) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "%zd arguments wanted, got %zd", N, n);
    try {
        return f();
    } catch (const Raised& e) {
        PyErr_SetString(e.type, e.text.c_str());
    } catch (const PythonError&) {
    } catch (const c10::OutOfMemoryError& e) {
        out_of_memory(e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// linear(x, packed weights, out, width, bias, norm_weight, eps, delta, delta_scale, out tensor)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded<10>(n, [&] {
        const int out = small(a[2], "out"), width = small(a[3], "width");
        const at::Tensor& packed = packed_of(a[1], "weight", out, width, false);
        const int device = packed.get_device();
        Input in = input_of(a[0], width, out, device, a[5], a[6], a[7], a[8], a[9]);
        at::Tensor bias;
        if (a[4] != Py_None) {
            bias = tensor_of(a[4], "bias");
            check(bias, "bias", at::kBFloat16, {out}, device);
        }
        long bytes;
        const c10::DataPtr ws = workspace_of(in, out, width, 0, bytes);
        if (in.rows > 0) {
            run(device, [&](void* stream) {
                return cpmcu_w8a8_linear(in.x.data_ptr(), ld_of(in.x), packed.data_ptr(), in.pointer(bias), in.pointer(in.norm), in.eps, in.pointer(in.delta), in.delta_scale,
                                         in.total.defined() ? in.total.data_ptr() : nullptr, in.out.data_ptr(), ld_of(in.out), in.rows, out, width,
                                         ws.get(), bytes, stream);
            });
        }
        return result_of(in);
    });
}

// ffn(x, packed gate/up weights, packed down weights, width, inter, norm_weight, eps, delta, delta_scale, out tensor)
PyObject* ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded<10>(n, [&] {
        const int width = small(a[3], "width"), inter = small(a[4], "inter");
        const at::Tensor& gate_up = packed_of(a[1], "gate_up", inter, width, true);
        const int device = gate_up.get_device();
        const at::Tensor& down = packed_of(a[2], "down", width, inter, false, device);
        Input in = input_of(a[0], width, width, device, a[5], a[6], a[7], a[8], a[9]);
        long bytes;
        const c10::DataPtr ws = workspace_of(in, width, width, inter, bytes);
        if (in.rows > 0) {
            run(device, [&](void* stream) {
                return cpmcu_w8a8_ffn(in.x.data_ptr(), ld_of(in.x), gate_up.data_ptr(), down.data_ptr(), in.pointer(in.norm), in.eps, in.pointer(in.delta), in.delta_scale,
                                      in.total.defined() ? in.total.data_ptr() : nullptr, in.out.data_ptr(), ld_of(in.out), in.rows, width, inter,
                                      ws.get(), bytes, stream);
            });
        }
        return result_of(in);
    });
}

// rotary_append(qkv, heads, kv_heads, dim, rot_dims, interleaved, inv_freq, factor, positions, k_cache, v_cache, slots, out tensor)
PyObject* rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded<13>(n, [&] {
        const at::Tensor& qkv = matrix_of(a[0], "qkv");
        const int64_t rows = qkv.size(0);
        const int heads = small(a[1], "heads"), kv_heads = small(a[2], "kv_heads"), dim = small(a[3], "dim"), rot = small(a[4], "rot_dims");
        if (heads < 0 || kv_heads < 0 || dim < 0 || rot < 0) refuse("sizes must not be negative");
        const int interleaved = PyObject_IsTrue(a[5]);
        if (interleaved < 0) throw PythonError();
        check(qkv, "qkv", at::kBFloat16, {rows, (heads + 2ll * kv_heads) * dim}, -1, true);
        const int device = qkv.get_device();
        const at::Tensor &inv_freq = tensor_of(a[6], "inv_freq"), &pos = tensor_of(a[8], "positions");
        check(inv_freq, "inv_freq", at::kFloat, {rot / 2}, device);
        check(pos, "positions", at::kInt, {rows}, device);
        void *k = nullptr, *v = nullptr;
        const int32_t* slots = nullptr;
        int cache_rows = 0;
        if (kv_heads > 0) {
            const at::Tensor &kc = matrix_of(a[9], "k_cache"), &vc = matrix_of(a[10], "v_cache"), &sl = tensor_of(a[11], "slots");
            cache_rows = small(kc.size(0), "the number of cache rows");
            check(kc, "k_cache", at::kBFloat16, {cache_rows, static_cast<int64_t>(kv_heads) * dim}, device);
            check(vc, "v_cache", at::kBFloat16, {cache_rows, static_cast<int64_t>(kv_heads) * dim}, device);
            check(sl, "slots", at::kInt, {rows}, device);
            k = kc.data_ptr();
            v = vc.data_ptr();
            slots = sl.data_ptr<int32_t>();
        }
        const int64_t q_cols = static_cast<int64_t>(heads) * dim;
        at::Tensor q;
        if (a[12] != Py_None) {
            q = tensor_of(a[12], "out");
            check(q, "out", at::kBFloat16, {rows, q_cols}, device, true);
        } else {
            q = empty({rows, q_cols}, at::kBFloat16, device);
        }
        const float factor = real(a[7]);
        const int count = small(rows, "the number of rows");
        run(device, [&](void* stream) {
            return cpmcu_rotary_append(qkv.data_ptr(), ld_of(qkv), count, heads, kv_heads, dim, rot, interleaved, inv_freq.data_ptr<float>(), factor,
                                       pos.data_ptr<int32_t>(), q.data_ptr(), ld_of(q), k, v, cache_rows, slots, stream);
        });
        return THPVariable_Wrap(q);
    });
}

PyMethodDef methods[] = {{"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
                         {"ffn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(ffn)), METH_FASTCALL, nullptr},
                         {"rotary_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary_append)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
