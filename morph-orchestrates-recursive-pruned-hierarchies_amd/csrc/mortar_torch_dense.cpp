// Native calls of the dense operators: LayerNorm and the dense SwiGLU MLP with their autograd nodes, and the 8-bit dense layer.
// One Python call each: checks, allocation, stream, launches.  Unlike the calls of mortar_torch.cpp these have no general path behind
// them: what they do not take they refuse, with the error worded here.
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
c10::DispatchKeySet riders() {
    using K = c10::DispatchKey;
    return c10::DispatchKeySet({K::Python, K::PythonTLSSnapshot, K::FuncTorchGradWrapper, K::FuncTorchBatched, K::FuncTorchDynamicLayerFrontMode,
                                K::FuncTorchDynamicLayerBackMode, K::Batched, K::Functionalize, K::Conjugate, K::Negative, K::ZeroTensor, K::Tracer});
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

// ---- LayerNorm -------------------------------------------------------------------------------------------------------

// x as rows [M, d] of consecutive values; 16-byte units where d is whole ones.
at::Tensor norm_rows(const at::Tensor &x, int64_t d) {
    const int64_t unit = x.scalar_type() == at::kFloat ? 4 : 8;
    const at::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, d});
    const int64_t M = rows.size(0);
    return (d > 1 && rows.stride(1) != 1) || (M > 1 && rows.stride(0) < d) || (d % unit == 0 && M > 1 && rows.stride(0) % unit) ? rows.contiguous() : rows;
}

// y, and for the backward (stats) the rows and their mean and 1 / deviation.
at::Tensor norm_forward(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, double eps, bool keep, at::Tensor &rows, at::Tensor &stats) {
    const int64_t d = x.size(-1);
    const c10::DeviceGuard guard(x.device());
    at::Tensor y = empty_like_rows(x, x.sizes());
    if (x.numel() == 0) return y;
    const int64_t M = x.numel() / d;
    rows = norm_rows(x, d);
    if (keep) stats = at::empty({2, M}, x.options().dtype(at::kFloat).requires_grad(false));
    const bool w32 = x.scalar_type() != at::kFloat && ((w.defined() && w.scalar_type() == at::kFloat) || (b.defined() && b.scalar_type() == at::kFloat));
    check_rc(mortar_layernorm(data(rows), M, (int32_t)d, M > 1 ? rows.stride(0) : d, type_code(x.scalar_type()), data(w), data(b), w32, (float)eps, mut(y), d,
                              keep ? floats(stats) : nullptr, keep ? floats(stats) + M : nullptr, stream_of(x)),
             "mortar_layernorm");
    return y;
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const std::optional<at::Tensor> &w, const std::optional<at::Tensor> &b, double eps) {
        at::Tensor rows, stats;
        const at::Tensor wt = w ? *w : at::Tensor();
        at::Tensor y = norm_forward(x, wt, b ? *b : at::Tensor(), eps, true, rows, stats);
        ctx->save_for_backward({rows, wt, stats});
        ctx->saved_data["shape"] = x.sizes();
        ctx->saved_data["bias"] = b ? c10::IValue(b->scalar_type()) : c10::IValue();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(4);
        const at::Tensor dy = plain_gradient(grads[0], "layernorm");
        if (!dy.defined()) return out;
        const auto v = ctx->get_saved_variables();
        const at::Tensor &w = v[1];
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const int64_t d = shape.back();
        // (edges are counted over the tensors that are there)
        const bool has_b = !ctx->saved_data["bias"].isNone();
        const bool need_x = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(w.defined() ? 2 : 1);
        const c10::DeviceGuard guard(dy.device());
        const at::ScalarType bt = has_b ? ctx->saved_data["bias"].toScalarType() : dy.scalar_type();
        const at::ScalarType pt = w.defined() ? w.scalar_type() : bt;
        const auto params = dy.options().dtype(pt).requires_grad(false);
        if (dy.numel() == 0) {
            if (need_x) out[0] = at::empty(shape, dy.options().requires_grad(false));
            if (need_w) out[1] = at::zeros({d}, params);
            if (need_b) out[2] = at::zeros({d}, params);
            return out;
        }
        const int64_t M = dy.numel() / d;
        const char *what = "layernorm";
        const at::Tensor rows = norm_rows(kept(v[0], dy, {M, d}, dy.scalar_type(), what), d), stats = kept(v[2], dy, {2, M}, at::kFloat, what).contiguous();
        const at::Tensor wc = w.defined() ? kept(w, dy, {d}, pt, what).contiguous() : w;
        const at::Tensor g = dy.dim() == 2 ? dy.contiguous() : dy.reshape({-1, d}).contiguous();
        at::Tensor dx, dw, db, ws;
        if (need_x) dx = at::empty(shape, dy.options().requires_grad(false));
        if (need_w) dw = at::empty({d}, params);
        if (need_b) db = at::empty({d}, params);
        if (need_w || need_b) ws = empty_bytes(dy, mortar_layernorm_workspace_bytes(M, (int32_t)d));
        check_rc(mortar_layernorm_bwd(data(g), d, data(rows), M > 1 ? rows.stride(0) : d, M, (int32_t)d, type_code(dy.scalar_type()), data(wc),
                                      dy.scalar_type() != at::kFloat && pt == at::kFloat, floats(stats), floats(stats) + M, mut(dx), d, mut(dw), mut(db),
                                      floats(ws), stream_of(dy)),
                 "mortar_layernorm_bwd");
        out[0] = dx;
        out[1] = dw;
        out[2] = db;
        return out;
    }
};

// layernorm(x, weight, bias, eps) -> y
PyObject *py_layernorm(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "layernorm";
    TORCH_CHECK_TYPE(na == 4, "layernorm: 4 arguments");
    const at::Tensor x = tensor_arg(a[0], what, "x"), w = optional_arg(a[1], what, "weight"), b = optional_arg(a[2], what, "bias");
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK_TYPE(type_code(x.scalar_type()) >= 0, what, ": expected bfloat16, float16 or float32, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, what, ": expected a tensor [..., d] with d > 0");
    TORCH_CHECK_VALUE(eps >= 0, what, ": eps is negative");
    const int64_t d = x.size(-1);
    TORCH_CHECK_VALUE(d <= (1 << 30), what, ": rows of ", d, " values are too long");
    for (const auto &p : {std::make_pair(&w, "weight"), std::make_pair(&b, "bias")}) {
        if (!p.first->defined()) continue;
        same_device(x, *p.first, what, p.second);
        TORCH_CHECK_TYPE(p.first->scalar_type() == x.scalar_type() || p.first->scalar_type() == at::kFloat, what, ": ", p.second, " must have the type of x or float32");
        TORCH_CHECK_VALUE(p.first->dim() == 1 && p.first->size(0) == d, what, ": ", p.second, " must be [", d, "]");
    }
    TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), what, ": weight and bias must have the same type");
    at::Tensor y;
    const bool record = c10::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()));
    const at::Tensor wc = w.defined() ? w.contiguous() : w, bc = b.defined() ? b.contiguous() : b;
    if (record) {
        const auto given = [](const at::Tensor &t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; };
        y = LayerNormFn::apply(x, given(wc), given(bc), eps);
    } else {
        at::Tensor rows, stats;
        y = norm_forward(x, wc, bc, eps, false, rows, stats);
    }
    return THPVariable_Wrap(std::move(y));
}

// ---- the dense MLP ---------------------------------------------------------------------------------------------------

at::Tensor workspace(const at::Tensor &like, int64_t M, int64_t N, int64_t K) {
    const int64_t n = mortar_dense_workspace_bytes(M, N, K);
    return n ? empty_bytes(like, n) : at::Tensor();
}

struct MlpRows {
    at::Tensor x, wgu, wd, gu;
};

// y of x [..., d]; keep: the rows, the weights as read and the gate_up output stay in `r`.
at::Tensor mlp_forward(const at::Tensor &x, const at::Tensor &wgu, const at::Tensor &wd, bool keep, MlpRows &r) {
    const int64_t d = x.size(-1), f = wd.size(1), n = wd.size(0);
    const c10::DeviceGuard guard(x.device());
    at::DimVector shape(x.sizes());
    shape.back() = n;
    at::Tensor y = empty_like_rows(x, shape);
    r.wgu = rows_of(wgu, d, 8);
    if ((f + 256) * ld_of(r.wgu) >= INT64_C(1) << 30) r.wgu = r.wgu.contiguous();        // a gate row and its up row are addressed together: 2 GiB
    r.wd = rows_of(wd, f, 8);
    if (x.numel() == 0) return y;
    const int64_t M = x.numel() / d;
    const int type = type_code(x.scalar_type());
    void *st = stream_of(x);
    r.x = rows_of(x, d, 8);
    const at::Tensor h = empty_like_rows(x, {M, f});
    if (keep) r.gu = empty_bytes(x, 6 * M * f);
    check_rc(mortar_dense_gateup_swiglu(data(r.x), M, (int32_t)d, ld_of(r.x), data(r.wgu), ld_of(r.wgu), (int32_t)f, type, mut(h), f, mut(r.gu), st),
             "mortar_dense_gateup_swiglu");
    int32_t tile_n, tile_m, ranges;
    check_rc(mortar_dense_form_host(0, M, n, f, &tile_n, &tile_m, &ranges), "mortar_dense_form_host");
    const at::Tensor ws = ranges > 1 ? empty_bytes(x, ranges * M * n * 4) : at::Tensor();          // (few rows take none)
    check_rc(mortar_dense_linear(data(h), M, (int32_t)f, f, data(r.wd), ld_of(r.wd), (int32_t)n, type, mut(y), n, floats(ws), st), "mortar_dense_linear");
    return y;
}

struct DenseMlpFn : public torch::autograd::Function<DenseMlpFn> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &wgu, const at::Tensor &wd) {
        MlpRows r;
        at::Tensor y = mlp_forward(x, wgu, wd, true, r);
        ctx->save_for_backward({r.x, r.wgu, r.wd, r.gu});
        ctx->saved_data["shape"] = x.sizes();
        ctx->saved_data["d_ff"] = wd.size(1);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(3);
        const at::Tensor dy = plain_gradient(grads[0], "dense_mlp");
        if (!dy.defined()) return out;
        const auto v = ctx->get_saved_variables();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const int64_t d = shape.back(), f = ctx->saved_data["d_ff"].toInt(), n = dy.size(-1);
        const bool need_x = ctx->needs_input_grad(0), need_gu = ctx->needs_input_grad(1), need_dn = ctx->needs_input_grad(2);
        const c10::DeviceGuard guard(dy.device());
        at::Tensor dx, dgw, ddw;
        if (need_x) dx = at::empty(shape, dy.options().requires_grad(false));
        if (dy.numel() == 0) {
            if (need_gu) dgw = at::zeros({2 * f, d}, dy.options().requires_grad(false));
            if (need_dn) ddw = at::zeros({n, f}, dy.options().requires_grad(false));
        } else {
            const int64_t M = dy.numel() / n;
            const int type = type_code(dy.scalar_type());
            void *st = stream_of(dy);
            const auto matrix = [&](int i, int64_t rows, int64_t cols) { return rows_of(kept(v[i], dy, {rows, cols}, dy.scalar_type(), "dense_mlp"), cols, 8); };
            const at::Tensor x = matrix(0, M, d), wgu = matrix(1, 2 * f, d), wd = matrix(2, n, f), gu = kept(v[3], dy, {6 * M * f}, at::kByte, "dense_mlp").contiguous();
            const at::Tensor g = rows_of(dy, n, 8);
            const at::Tensor dgu = empty_like_rows(dy, {M, 2 * f}), h = need_dn ? empty_like_rows(dy, {M, f}) : at::Tensor();
            check_rc(mortar_dense_swiglu_bwd(data(g), M, (int32_t)n, ld_of(g), data(wd), ld_of(wd), (int32_t)f, type, data(gu), mut(dgu), 2 * f, mut(h), f, st),
                     "mortar_dense_swiglu_bwd");
            if (need_dn) {
                ddw = empty_like_rows(dy, {n, f});
                const at::Tensor ws = workspace(dy, n, f, M);
                check_rc(mortar_dense_linear_dw(data(g), M, (int32_t)n, ld_of(g), data(h), f, (int32_t)f, type, mut(ddw), f, floats(ws), st), "mortar_dense_linear_dw");
            }
            if (need_gu) {
                dgw = empty_like_rows(dy, {2 * f, d});
                const at::Tensor ws = workspace(dy, 2 * f, d, M);
                check_rc(mortar_dense_linear_dw(data(dgu), M, (int32_t)(2 * f), 2 * f, data(x), ld_of(x), (int32_t)d, type, mut(dgw), d, floats(ws), st),
                         "mortar_dense_linear_dw");
            }
            if (need_x) {
                const at::Tensor ws = workspace(dy, M, d, 2 * f);
                check_rc(mortar_dense_linear_dx(data(dgu), M, (int32_t)(2 * f), 2 * f, data(wgu), ld_of(wgu), (int32_t)d, type, mut(dx), d, floats(ws), st),
                         "mortar_dense_linear_dx");
            }
        }
        out[0] = dx;
        out[1] = dgw;
        out[2] = ddw;
        return out;
    }
};

// dense_mlp(x, w_gate_up, w_down) -> y
PyObject *py_dense_mlp(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "dense_mlp";
    TORCH_CHECK_TYPE(na == 3, "dense_mlp: 3 arguments");
    const at::Tensor x = tensor_arg(a[0], what, "x"), wgu = tensor_arg(a[1], what, "w_gate_up"), wd = tensor_arg(a[2], what, "w_down");
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, what, ": expected bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_TYPE(wgu.scalar_type() == x.scalar_type() && wd.scalar_type() == x.scalar_type(), what, ": the weights must have the type of x");
    same_device(x, wgu, what, "w_gate_up");
    same_device(x, wd, what, "w_down");
    TORCH_CHECK_VALUE(x.dim() >= 1 && wgu.dim() == 2 && wd.dim() == 2, what, ": expected x [..., d], w_gate_up [2 * d_ff, d], w_down [d_out, d_ff]");
    TORCH_CHECK_VALUE(x.size(-1) == wgu.size(1), what, ": x has ", x.size(-1), " features, w_gate_up expects ", wgu.size(1));
    TORCH_CHECK_VALUE(wgu.size(0) == 2 * wd.size(1), what, ": w_gate_up ", wgu.sizes(), " and w_down ", wd.sizes(), " do not chain");
    for (const int64_t v : {x.size(-1), wd.size(1), wd.size(0)})
        TORCH_CHECK_VALUE(v > 0 && v % 8 == 0 && v < (1 << 28), what, ": widths must be positive multiples of 8, got ", v);
    TORCH_CHECK_VALUE(x.numel() / x.size(-1) < (1 << 30), what, ": too many rows");
    at::Tensor y;
    if (c10::GradMode::is_enabled() && (x.requires_grad() || wgu.requires_grad() || wd.requires_grad())) {
        y = DenseMlpFn::apply(x, wgu, wd);
    } else {
        MlpRows r;
        y = mlp_forward(x, wgu, wd, false, r);
    }
    return THPVariable_Wrap(std::move(y));
}

// dense_mlp_covers(x, w_gate_up, w_down) -> whether dense_mlp takes these tensors, of fitting sizes and types, as they are and where the call
// stands: no subclass, transform, tracing, mode or forward-mode gradient that it would refuse, and matrices that the kernels can address.
PyObject *py_dense_mlp_covers(PyObject *, PyObject *const *a, Py_ssize_t na) {
    TORCH_CHECK_TYPE(na == 3, "dense_mlp_covers: 3 arguments");
    for (Py_ssize_t i = 0; i < 3; ++i) {
        if (!THPVariable_CheckExact(a[i])) Py_RETURN_FALSE;
        const at::Tensor &t = THPVariable_Unpack(a[i]);
        if (!plain(t) || !t.is_cuda() || t._fw_grad(0).defined()) Py_RETURN_FALSE;
    }
    const at::Tensor &x = THPVariable_Unpack(a[0]), &wgu = THPVariable_Unpack(a[1]), &wd = THPVariable_Unpack(a[2]);
    const int64_t d = wgu.size(1), f = wd.size(1), n = wd.size(0), span = INT64_C(1) << 30;        // (values of 16 bits in 2 GiB)
    return PyBool_FromLong(x.numel() < d * span && 256 * std::max({d, 2 * f, n}) < span && (f + 256) * d < span);
}

// ---- 8 bits ----------------------------------------------------------------------------------------------------------

void no_gradients(const at::Tensor &t, const char *what) {
    TORCH_CHECK(!(c10::GradMode::is_enabled() && t.requires_grad()), what, ": no gradients flow through 8-bit values (detach the input or call under no_grad)");
}
void check_k(int64_t K, const char *what) { TORCH_CHECK_VALUE(K > 0 && K % 16 == 0 && K < (1 << 28), what, ": in_features must be a positive multiple of 16, got ", K); }

// quantize_fp8(x) -> (codes float8_e4m3fn like x, scales fp32 [..., ceil(K / 128)], consecutive along the rows)
PyObject *py_quantize_fp8(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "quantize_fp8";
    TORCH_CHECK_TYPE(na == 1, "quantize_fp8: 1 argument");
    const at::Tensor x = tensor_arg(a[0], what, "x");
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16, what, ": expected bfloat16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1, what, ": expected a tensor [..., K]");
    no_gradients(x, what);
    const int64_t K = x.size(-1), kb = (K + 127) / 128;
    check_k(K, what);
    const int64_t M = x.numel() / K;
    const c10::DeviceGuard guard(x.device());
    at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));
    at::Tensor s = at::empty({kb, M}, x.options().dtype(at::kFloat).requires_grad(false));
    if (M) {
        const at::Tensor r = rows_of(x, K, 8, false);
        check_rc(mortar_fp8_quantize(static_cast<const uint16_t *>(data(r)), M, (int32_t)K, ld_of(r), static_cast<uint8_t *>(mut(q)), K, floats(s), 1, M, stream_of(x)),
                 "mortar_fp8_quantize");
    }
    at::DimVector shape(x.sizes());
    shape.back() = kb;
    s = M ? s.t().view(shape) : at::empty(shape, s.options());
    PyObject *pq = THPVariable_Wrap(std::move(q)), *ps = THPVariable_Wrap(std::move(s));
    return Py_BuildValue("(NN)", pq, ps);
}

// quantize_fp8_weight(w) -> (codes float8_e4m3fn [N, K], scales fp32 [ceil(N / 128), ceil(K / 128)])
PyObject *py_quantize_fp8_weight(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "quantize_fp8_weight";
    TORCH_CHECK_TYPE(na == 1, "quantize_fp8_weight: 1 argument");
    const at::Tensor w = tensor_arg(a[0], what, "w");
    TORCH_CHECK_TYPE(type_code(w.scalar_type()) >= 0, what, ": expected bfloat16, float16 or float32, got ", w.scalar_type());
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) > 0, what, ": expected a matrix [out_features, in_features]");
    no_gradients(w, what);
    const int64_t N = w.size(0), K = w.size(1);
    check_k(K, what);
    TORCH_CHECK_VALUE(N < (1 << 23), what, ": too many rows");
    const c10::DeviceGuard guard(w.device());
    const at::Tensor r = rows_of(w, K, w.scalar_type() == at::kFloat ? 4 : 8, false);
    at::Tensor q = at::empty({N, K}, w.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));
    at::Tensor s = at::empty({(N + 127) / 128, (K + 127) / 128}, w.options().dtype(at::kFloat).requires_grad(false));
    check_rc(mortar_fp8_quantize_weight(data(r), (int32_t)N, (int32_t)K, ld_of(r), type_code(w.scalar_type()), static_cast<uint8_t *>(mut(q)), K, floats(s),
                                        s.size(1), stream_of(w)),
             "mortar_fp8_quantize_weight");
    PyObject *pq = THPVariable_Wrap(std::move(q)), *ps = THPVariable_Wrap(std::move(s));
    return Py_BuildValue("(NN)", pq, ps);
}

// linear_fp8(x, wq, ws, x_scale) -> y bf16 [..., N]
PyObject *py_linear_fp8(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "linear_fp8";
    TORCH_CHECK_TYPE(na == 4, "linear_fp8: 4 arguments");
    const at::Tensor x = tensor_arg(a[0], what, "x"), wq = tensor_arg(a[1], what, "wq"), ws = tensor_arg(a[2], what, "ws");
    at::Tensor xs = optional_arg(a[3], what, "x_scale");
    const bool codes = x.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK_TYPE(codes || x.scalar_type() == at::kBFloat16, what, ": expected bfloat16 or float8_e4m3fn, got ", x.scalar_type());
    TORCH_CHECK_TYPE(codes == xs.defined(), what, ": x_scale goes with float8_e4m3fn x, and only with it");
    TORCH_CHECK_TYPE(wq.scalar_type() == at::kFloat8_e4m3fn && ws.scalar_type() == at::kFloat, what, ": wq must be float8_e4m3fn and ws float32");
    no_gradients(x, what);
    same_device(x, wq, what, "wq");
    same_device(x, ws, what, "ws");
    TORCH_CHECK_VALUE(x.dim() >= 1 && wq.dim() == 2 && x.size(-1) == wq.size(1), what, ": x ", x.sizes(), " does not fit wq ", wq.sizes());
    const int64_t K = wq.size(1), N = wq.size(0), kb = (K + 127) / 128;
    check_k(K, what);
    TORCH_CHECK_VALUE(N > 0 && N % 8 == 0 && N < (1 << 28), what, ": out_features must be a positive multiple of 8, got ", N);
    TORCH_CHECK_VALUE(ws.dim() == 2 && ws.size(0) == (N + 127) / 128 && ws.size(1) == kb, what, ": ws must be [", (N + 127) / 128, ", ", kb, "], got ", ws.sizes());
    TORCH_CHECK_VALUE(wq.stride(1) == 1 && (N == 1 || (wq.stride(0) % 16 == 0 && wq.stride(0) >= K)) && aligned16(wq.const_data_ptr()), what,
                      ": the rows of wq must be contiguous and 16-byte aligned");
    const int64_t M = x.numel() / K;
    TORCH_CHECK_VALUE(M < (1 << 30), what, ": too many rows");
    const c10::DeviceGuard guard(x.device());
    if (codes) {
        same_device(x, xs, what, "x_scale");
        TORCH_CHECK_TYPE(xs.scalar_type() == at::kFloat, what, ": x_scale must be float32");
        TORCH_CHECK_VALUE(xs.dim() == x.dim() && xs.size(-1) == kb && xs.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1), what,
                          ": x_scale must be [..., ", kb, "] with the rows of x, got ", xs.sizes(), " for ", x.sizes());
    }
    at::DimVector shape(x.sizes());
    shape.back() = N;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kBFloat16).requires_grad(false));
    if (M) {
        void *st = stream_of(x);
        const at::Tensor wsc = ws.stride(1) == 1 && ws.stride(0) >= kb ? ws : ws.clone(at::MemoryFormat::Contiguous);
        at::Tensor xr, buf;
        const void *xp;
        const float *sx = nullptr;
        int64_t ldx, s_m = 0, s_k = 0;
        if (codes) {
            xr = rows_of(x, K, 16);
            xs = xs.dim() == 2 ? xs : xs.reshape({-1, kb});
            if (xs.stride(0) >= (INT64_C(1) << 29) / M) xs = xs.t().clone(at::MemoryFormat::Contiguous).t();        // (rows within 2 GiB)
            xp = data(xr), ldx = ld_of(xr);
            sx = static_cast<const float *>(xs.const_data_ptr()), s_m = xs.stride(0), s_k = xs.stride(1);
        } else {
            xr = rows_of(x, K, 8, false);
            xp = data(xr), ldx = ld_of(xr);
            if (!mortar_fp8_quantizes_inside(M, K)) {
                buf = empty_bytes(x, M * K + M * kb * 4);        // codes, then scales (M K is a multiple of 16)
                uint8_t *q = static_cast<uint8_t *>(mut(buf));
                float *s = reinterpret_cast<float *>(q + M * K);
                check_rc(mortar_fp8_quantize(static_cast<const uint16_t *>(xp), M, (int32_t)K, ldx, q, K, s, 1, M, st), "mortar_fp8_quantize");
                xp = q, ldx = K, sx = s, s_m = 1, s_k = M;
            }
        }
        const int64_t n = mortar_fp8_workspace_bytes(M, N, K);
        const at::Tensor wk = n ? empty_bytes(x, n) : at::Tensor();
        check_rc(mortar_fp8_linear(xp, M, (int32_t)K, ldx, sx, s_m, s_k, static_cast<const uint8_t *>(data(wq)), N > 1 ? wq.stride(0) : K,
                                   static_cast<const float *>(data(wsc)), ws.size(0) > 1 ? wsc.stride(0) : kb, (int32_t)N, static_cast<uint16_t *>(mut(y)), N, floats(wk), st),
                 "mortar_fp8_linear");
    }
    return THPVariable_Wrap(std::move(y));
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    HANDLE_TH_ERRORS
    return F(self, a, na);
    END_HANDLE_TH_ERRORS
}

#define MORTAR_METHOD(name, f, doc) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<f>)), METH_FASTCALL, doc}
PyMethodDef methods[] = {MORTAR_METHOD("layernorm", py_layernorm, "LayerNorm of the rows of x, with its autograd node."),
                         MORTAR_METHOD("dense_mlp", py_dense_mlp, "The dense SwiGLU MLP of the rows of x, with its autograd node."),
                         MORTAR_METHOD("dense_mlp_covers", py_dense_mlp_covers, "Whether dense_mlp takes these tensors."),
                         MORTAR_METHOD("quantize_fp8", py_quantize_fp8, "e4m3 codes and scales of activations."),
                         MORTAR_METHOD("quantize_fp8_weight", py_quantize_fp8_weight, "e4m3 codes and block scales of a weight."),
                         MORTAR_METHOD("linear_fp8", py_linear_fp8, "x W^T in e4m3."),
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

int mortar_add_dense_methods(PyObject *module) { return PyModule_AddFunctions(module, methods); }
