// Python module _calls: the functions of torch_ops.h called without the dispatcher. Small calls of these operators take the
// host longer than the device, and of the 4.7 us that a call through torch.ops costs, 2 are argument parsing and dispatch.
// Each function returns True if it made the call. It returns False, and has done nothing, for arguments that are not plain
// tensors or parameters, where something waits for the call in the dispatcher (a dispatch or function mode, a tracer, a function
// transform, a profiler), and where the checks refused: the caller then takes the way through the dispatcher. A CUDA call that
// failed is a RuntimeError: the call is not made twice.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <array>
#include <string>
#include <utility>

#include "torch_ops.h"

namespace {

// Modes, tracers and transforms put dispatch keys of their own in front of the usual ones; profilers are called back.
bool watched() {
    const c10::DispatchKeySet keys = c10::impl::tls_local_dispatch_key_set().included_;
    return !c10::default_included_set.has_all(keys) || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           at::impl::torch_function_mode_enabled() || at::hasCallbacks();
}

template <typename F, size_t... I>
bool invoke(F* op, const std::array<at::Tensor*, sizeof...(I)>& t, std::index_sequence<I...>) {
    bool done = false;
    std::string failure;
    PyThreadState* state = PyEval_SaveThread();   // a launch can wait for room in the stream's queue
    try {
        op(*t[I]...);
        done = true;
    } catch (const tiledcuda::CudaFailure& e) {
        failure = e.what_without_backtrace();
    } catch (...) {
    }
    PyEval_RestoreThread(state);
    if (!failure.empty()) PyErr_SetString(PyExc_RuntimeError, failure.c_str());
    return done;
}

template <size_t kArgs, auto op>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    std::array<at::Tensor*, kArgs> t;
    bool plain = n == static_cast<Py_ssize_t>(kArgs) && !watched();
    for (size_t i = 0; plain && i < kArgs; ++i) {
        plain = THPVariable_CheckExact(args[i]);
        if (plain) t[i] = const_cast<at::Tensor*>(&THPVariable_Unpack(args[i]));   // the caller's frame holds the arguments
    }
    if (plain && invoke(op, t, std::make_index_sequence<kArgs>{})) Py_RETURN_TRUE;
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_FALSE;
}

template <size_t kArgs, auto op>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<kArgs, op>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    method<3, &tiledcuda::quantize_rows>("quantize_rows"),
    method<5, &tiledcuda::gemm_i8>("gemm_i8"),
    method<4, &tiledcuda::grouped_gemm>("grouped_gemm"),
    method<6, &tiledcuda::grouped_gemm_i8>("grouped_gemm_i8"),
    method<4, &tiledcuda::grouped_gemm_dgrad>("grouped_gemm_dgrad"),
    method<4, &tiledcuda::grouped_gemm_wgrad>("grouped_gemm_wgrad"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
