// What the CPython functions of native.cpp and native_paged.cpp share: arguments, streams, errors.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

#include "gpuk_b200.h"

namespace gpuk_native {

using at::Tensor;

inline void check(int status, const char *what) {
    TORCH_CHECK(status == GPUK_OK, "gpuk::", what, ": ", gpuk_status_string(status), ": ", gpuk_last_error());
}

inline const Tensor &tensor_arg(PyObject *o, const char *what) {
    TORCH_CHECK(THPVariable_Check(o), "gpuk: ", what, " must be a tensor");
    return THPVariable_Unpack(o);
}
inline int64_t int_arg(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
// A size as the C ABI takes it.
inline int int_size(int64_t v) {
    TORCH_CHECK(v >= 0 && v <= INT_MAX, "gpuk: a size of ", v, " is out of range");
    return static_cast<int>(v);
}
struct NoGil {
    PyThreadState *state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};
inline void expect_args(Py_ssize_t n, Py_ssize_t want, const char *what) { TORCH_CHECK(n == want, "gpuk::", what, " takes ", want, " arguments, got ", n); }
inline void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
inline Tensor empty_like_on(const Tensor &t, at::IntArrayRef sizes, at::ScalarType type) { return at::detail::empty_cuda(sizes, type, t.device(), std::nullopt); }

// A tensor whose operators would go straight to the CUDA kernels: of the class Tensor itself, dense and contiguous, no transform or lazy bit on it.
inline bool plain_class(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor &t = THPVariable_Unpack(o);
    static const c10::DispatchKeySet other({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                            c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched, c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                            c10::DispatchKey::ZeroTensor, c10::DispatchKey::NestedTensor});
    return !t.key_set().has_any(other);
}
inline bool plain(PyObject *o, int device) {
    if (!plain_class(o)) return false;
    const Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && (device < 0 || t.get_device() == device) && t.layout() == at::kStrided && t.is_contiguous();
}
// Tracing, a functional transform or a dispatch mode, which want to see what is computed.
inline bool watched() {
    const c10::impl::LocalDispatchKeySet tls = c10::impl::tls_local_dispatch_key_set();
    static const c10::DispatchKeySet front({c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Functionalize,
                                            c10::DispatchKey::Tracer, c10::DispatchKey::Python, c10::DispatchKey::PreDispatch});
    return tls.included_.has_any(front) || c10::impl::TorchDispatchModeTLS::any_modes_set();
}
// No mode that wants to see operators: those, and function modes.
inline bool no_modes() { return !watched() && at::impl::PythonTorchFunctionTLS::stack_len() == 0; }

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
constexpr PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)); }

// native_paged.cpp
PyObject *paged_plan(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *rope(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *rope_paged(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *paged_keep(PyObject *, PyObject *const *args, Py_ssize_t n);

}  // namespace gpuk_native
