// Arguments of the native calls without a general path behind them: checks with their errors, rows that the kernels can read, streams, and
// what a backward pass may rely on.  Included by one source file each.
#ifndef MORTAR_TORCH_ARGS_H
#define MORTAR_TORCH_ARGS_H

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mortar_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_rc(int rc, const char *what) {
    if (rc == MORTAR_OK) return;
    TORCH_CHECK(rc != MORTAR_ERR_HIP, what, " failed (", rc, "): ", mortar_last_error());
    TORCH_CHECK_VALUE(false, what, " failed (", rc, "): ", mortar_last_error());
}

// Kinds of tensors whose values a kernel launched on their address would miss.
const c10::DispatchKeySet &riders() {
    using K = c10::DispatchKey;
    static const c10::DispatchKeySet keys({K::Python, K::PythonTLSSnapshot, K::FuncTorchGradWrapper, K::FuncTorchBatched, K::FuncTorchDynamicLayerFrontMode,
                                K::FuncTorchDynamicLayerBackMode, K::Batched, K::Functionalize, K::Conjugate, K::Negative, K::ZeroTensor, K::Tracer});
    return keys;
}

bool plain_values(const at::Tensor &t) { return !t.key_set().has_any(riders()) && t.layout() == at::kStrided; }
bool plain(const at::Tensor &t) { return !c10::impl::tls_local_dispatch_key_set().included_.has_any(riders()) && plain_values(t); }

// Argument `name` as a plain tensor on the GPU.
const at::Tensor &tensor_arg(PyObject *o, const char *what, const char *name) {
    TORCH_CHECK_TYPE(THPVariable_CheckExact(o) || THPVariable_Check(o), what, ": ", name, " must be a tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    TORCH_CHECK(plain(t), what, ": ", name, " must be a plain strided tensor, outside functional transforms and tracing");
    TORCH_CHECK(t.is_cuda(), what, ": tensor must live on a ROCm device (the MORTAR runtime has no CPU path)");
    TORCH_CHECK(!t._fw_grad(0).defined(), what, ": no forward-mode gradients");
    return t;
}
at::Tensor optional_arg(PyObject *o, const char *what, const char *name) { return o == Py_None ? at::Tensor() : tensor_arg(o, what, name); }

void same_device(const at::Tensor &a, const at::Tensor &b, const char *what, const char *name) {
    TORCH_CHECK_VALUE(a.device() == b.device(), what, ": ", name, " is on ", b.device(), ", x on ", a.device());
}

int type_code(at::ScalarType t) { return t == at::kBFloat16 ? MORTAR_BF16 : t == at::kHalf ? MORTAR_FP16 : t == at::kFloat ? MORTAR_FP32 : -1; }

// t [..., d] as rows [M, d] that the kernels can read: `unit` values per 16 bytes, tiles: 256 rows within 2 GiB; copied where strides or
// address do not allow it.
at::Tensor rows_of(const at::Tensor &t, int64_t d, int64_t unit, bool tiles = true) {
    at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, d});
    const bool one = r.size(0) <= 1;
    if ((d > 1 && r.stride(1) != 1) || (!one && (r.stride(0) % unit || r.stride(0) < d || (tiles && r.stride(0) * 256 * r.element_size() >= INT64_C(1) << 31))) ||
        !aligned16(r.const_data_ptr()))
        r = r.clone(at::MemoryFormat::Contiguous);
    return r;
}
int64_t ld_of(const at::Tensor &r) { return r.size(0) <= 1 ? r.size(1) : r.stride(0); }

at::Tensor empty_like_rows(const at::Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().requires_grad(false)); }
at::Tensor empty_bytes(const at::Tensor &like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }
float *floats(const at::Tensor &t) { return t.defined() ? static_cast<float *>(t.data_ptr()) : nullptr; }
const void *data(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *mut(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The gradient of a result as the backward reads it: values as they lie in memory, once.
at::Tensor plain_gradient(const at::Tensor &dy, const char *what) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), what, ": its gradients cannot be differentiated again (create_graph=True)");
    if (!dy.defined()) return dy;
    const at::Tensor g = dy.resolve_neg();                 // (the imaginary part of a conjugate is negated lazily)
    TORCH_CHECK(plain_values(g), what, ": its gradient must be a plain strided tensor");
    return g;
}

// A tensor kept from the forward, as it comes back: saved-tensor hooks may have brought it to another place and other strides, and no further.
const at::Tensor &kept(const at::Tensor &t, const at::Tensor &dy, at::IntArrayRef sizes, at::ScalarType type, const char *what) {
    TORCH_CHECK(t.defined() && plain_values(t) && t.device() == dy.device() && t.scalar_type() == type && t.sizes() == sizes, what,
                ": a tensor that was saved for the backward came back with another shape, type or device");
    return t;
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    return F(self, a, na);
    END_HANDLE_TH_ERRORS
}

#define MORTAR_METHOD(name, f, doc) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<f>)), METH_FASTCALL, doc}

}  // namespace

#endif
