// Native calls around the products of a training step: the norm of many gradients and their clipping, tokens to their experts' rows and back with
// the autograd nodes.  As in mortar_torch_dense.cpp one Python call each, and what they do not take they refuse.
#include "mortar_torch_args.h"

#include <array>
#include <vector>

#include <ATen/MemoryOverlap.h>
#include <c10/core/InferenceMode.h>
#include <torch/csrc/utils/object_ptr.h>

namespace {

// ---- gradients -------------------------------------------------------------------------------------------------------

// The tensors of a Python sequence (or a single one), which keeps them.
struct TensorList {
    THPObjectPtr sequence;
    std::vector<const at::Tensor *> all;
    size_t size() const { return all.size(); }
    const at::Tensor &operator[](size_t i) const { return *all[i]; }
};

TensorList tensor_list(PyObject *o, const char *what, const char *name) {
    TensorList v;
    v.sequence = THPVariable_Check(o) ? PyTuple_Pack(1, o) : PySequence_Fast(o, "expected a sequence of tensors");
    if (!v.sequence) throw python_error();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(v.sequence.get());
    v.all.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) v.all.push_back(&tensor_arg(PySequence_Fast_GET_ITEM(v.sequence.get(), i), what, name));
    return v;
}

void check_grads(const TensorList &v, const char *what) {
    const bool record = c10::GradMode::is_enabled();
    for (const at::Tensor *t : v.all) {
        TORCH_CHECK_TYPE(type_code(t->scalar_type()) >= 0, what, ": expected bfloat16, float16 or float32 gradients, got ", t->scalar_type());
        TORCH_CHECK_VALUE(t->device() == v[0].device(), what, ": gradients on ", t->device(), " and on ", v[0].device());
        TORCH_CHECK(!(record && t->requires_grad()), what, ": no gradients flow through this call (detach the tensors or call under no_grad)");
    }
}

// Memory of a tensor, from its first value to behind its last.
struct Span {
    uintptr_t begin, end;
    size_t i;
};

// Nothing that a launch writes is written twice, or read for another tensor.  drop: a gradient that is there twice is counted once (in place).  Tensors mostly
// come in the order of their addresses, results and gradients each: two lists that are merged.
void check_overlap(std::vector<mortar_grad_t> &list, bool drop, const char *what) {
    std::vector<Span> written, read;
    written.reserve(list.size());
    read.reserve(list.size());
    const auto size = [](int type) { return type == MORTAR_FP32 ? 4 : 2; };
    for (size_t i = 0; i < list.size(); ++i) {
        const mortar_grad_t &g = list[i];
        if (!g.n) continue;
        const uintptr_t s = reinterpret_cast<uintptr_t>(g.src), d = reinterpret_cast<uintptr_t>(g.dst);
        written.push_back({d, d + g.n * size(g.out_type), i});
        if (s != d || g.type != g.out_type) read.push_back({s, s + g.n * size(g.type), i});
    }
    const auto less = [](const Span &a, const Span &b) { return a.begin < b.begin; };
    for (std::vector<Span> *v : {&written, &read})
        if (!std::is_sorted(v->begin(), v->end(), less)) std::stable_sort(v->begin(), v->end(), less);
    uintptr_t end_written = 0, end_read = 0;
    const Span *last = nullptr;
    for (auto w = written.begin(), r = read.begin(); w != written.end() || r != read.end();) {
        const bool is_read = w == written.end() || (r != read.end() && r->begin < w->begin);
        const Span &s = is_read ? *r++ : *w++;
        if (!is_read && drop && last && s.begin == last->begin && s.end == last->end && list[s.i].type == list[last->i].type) {
            list[s.i].n = 0;
            continue;
        }
        TORCH_CHECK_VALUE(s.begin >= end_written && (is_read || s.begin >= end_read), what, ": results overlap each other or another gradient");
        if (is_read) end_read = std::max(end_read, s.end);
        else end_written = std::max(end_written, s.end), last = &s;
    }
}

// Where a tensor's values lie: runs of `run` bytes at `at` plus any sum of multiples of the strides, the largest one first.
struct Places {
    uintptr_t at;
    int64_t run;
    std::vector<std::pair<int64_t, int64_t>> dims;           // stride in bytes, size
    std::vector<int64_t> extent;                             // bytes from dimension d on, all of them in front
    size_t i;                                                // of the gradient, or of the result that it has
    bool result, copied;
    uintptr_t end() const { return at + extent[0]; }
    bool same(const Places &o) const { return at == o.at && run == o.run && dims == o.dims; }
};

Places places_of(const at::Tensor &t, size_t i, bool result, bool copied) {
    Places p{reinterpret_cast<uintptr_t>(t.const_data_ptr()), (int64_t)t.element_size(), {}, {}, i, result, copied};
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1 && t.stride(d)) p.dims.push_back({t.stride(d) * (int64_t)t.element_size(), t.size(d)});
    std::sort(p.dims.begin(), p.dims.end(), std::greater<>());
    for (; !p.dims.empty() && p.dims.back().first == p.run; p.dims.pop_back()) p.run *= p.dims.back().second;
    p.extent.assign(p.dims.size() + 1, p.run);
    for (size_t d = p.dims.size(); d-- > 0;) p.extent[d] = p.extent[d + 1] + (p.dims[d].second - 1) * p.dims[d].first;
    return p;
}

int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

// Whether values of a from dimension da on and of b from db on, which begin `off` bytes behind a's, share a byte: exactly, by the dimension of the largest
// stride, of which only the steps are tried that bring the rest of both together.
bool meet(const Places &a, size_t da, const Places &b, size_t db, int64_t off) {
    if (off >= a.extent[da] || off + b.extent[db] <= 0) return false;
    const int64_t sa = da < a.dims.size() ? a.dims[da].first : 0, sb = db < b.dims.size() ? b.dims[db].first : 0;
    if (!sa && !sb) return true;
    const bool ia = sa >= sb, ib = sb >= sa;                 // which of them steps (both with one stride: what counts is the difference)
    const int64_t s = std::max(sa, sb), ea = a.extent[da + ia], eb = b.extent[db + ib];
    const int64_t least = ia ? 1 - a.dims[da].second : 0, most = ib ? b.dims[db].second - 1 : 0;
    const int64_t from = std::max(least, floor_div(-eb - off, s) + 1), to = std::min(most, floor_div(ea - 1 - off, s));
    for (int64_t t = from; t <= to; ++t)
        if (meet(a, da + ia, b, db + ib, off + t * s)) return true;
    return false;
}

// The same for results that are copied to where they belong, and for gradients that are copied from where they are, which may be in place all the same.  all: the
// results and gradients.
void check_copied(std::vector<Places> all, const char *what) {
    std::sort(all.begin(), all.end(), [](const Places &a, const Places &b) { return a.at < b.at; });
    std::vector<const Places *> open;                        // those that reach behind where the next one begins
    for (const Places &p : all) {
        open.erase(std::remove_if(open.begin(), open.end(), [&](const Places *o) { return o->end() <= p.at; }), open.end());
        for (const Places *o : open) {
            if (!(o->result || p.result) || !(o->copied || p.copied) || (o->i == p.i && o->same(p))) continue;
            TORCH_CHECK_VALUE(!meet(*o, 0, p, 0, (int64_t)(p.at - o->at)), what, ": results overlap each other or another gradient");
        }
        open.push_back(&p);
    }
}

PyObject *empty_norm() {
    at::Tensor zero = at::zeros({}, at::TensorOptions().dtype(at::kFloat));
    return THPVariable_Wrap(std::move(zero));
}

// grad_norm(grads, largest) -> fp32 []
PyObject *py_grad_norm(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "grad_norm";
    TORCH_CHECK_TYPE(na == 2, "grad_norm: 2 arguments");
    const TensorList grads = tensor_list(a[0], what, "each gradient");
    check_grads(grads, what);
    if (!grads.size()) return empty_norm();
    const c10::DeviceGuard guard(grads[0].device());
    std::vector<at::Tensor> held;
    std::vector<mortar_grad_t> list;
    list.reserve(grads.size());
    for (const at::Tensor *g : grads.all) {
        const bool flat = g->is_non_overlapping_and_dense();
        if (!flat) held.push_back(g->contiguous());
        list.push_back({data(flat ? *g : held.back()), nullptr, g->numel(), type_code(g->scalar_type()), 0});
    }
    at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
    const at::Tensor ws = empty_bytes(norm, std::max<int64_t>(8, mortar_grad_workspace_bytes(list.data(), (int64_t)list.size())));
    check_rc(mortar_grad_norm(list.data(), (int64_t)list.size(), a[1] == Py_True, floats(norm), mut(ws), stream_of(norm)), "mortar_grad_norm");
    return THPVariable_Wrap(std::move(norm));
}

// grad_clip(grads, out, max_norm, largest) -> (results, norm fp32 []); out: a sequence of tensors, None (new ones) or True (in place, a gradient that is
// there twice counts once)
PyObject *py_grad_clip(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "clip_grads";
    TORCH_CHECK_TYPE(na == 4, "grad_clip: 4 arguments");
    const TensorList grads = tensor_list(a[0], what, "each gradient");
    const bool in_place = a[1] == Py_True, fresh = a[1] == Py_None;
    const double max_norm = PyFloat_AsDouble(a[2]);
    if (PyErr_Occurred()) throw python_error();
    check_grads(grads, what);
    TORCH_CHECK_VALUE(max_norm >= 0, what, ": max_norm is negative or NaN");
    TensorList out;
    std::vector<at::Tensor> made;                        // results of its own
    if (fresh) {
        made.reserve(grads.size());
        for (const at::Tensor *g : grads.all) {
            const c10::DeviceGuard guard(g->device());
            made.push_back(at::empty_like(*g, g->options().requires_grad(false)));
            out.all.push_back(&made.back());
        }
    } else {
        out = tensor_list(in_place ? a[0] : a[1], what, "each result");
        TORCH_CHECK_VALUE(out.size() == grads.size(), what, ": ", out.size(), " results for ", grads.size(), " gradients");
        check_grads(out, what);
    }
    for (size_t i = 0; i < out.size(); ++i) {
        TORCH_CHECK_VALUE(out[i].sizes() == grads[i].sizes() && out[i].device() == grads[i].device(), what, ": result ", i, " has another shape or device than its gradient");
        TORCH_CHECK_TYPE(out[i].scalar_type() == grads[i].scalar_type() || out[i].scalar_type() == at::kFloat, what, ": result ", i, " must have the type of its gradient or float32");
        TORCH_CHECK(fresh || !out[i].is_inference() || c10::InferenceMode::is_enabled(), what, ": result ", i, " is an inference tensor, which nothing may write outside of inference mode");
        TORCH_CHECK_VALUE(out[i].is_non_overlapping_and_dense() || at::has_internal_overlap(out[i]) != at::MemOverlap::Yes, what, ": result ", i, " refers to one place several times");
    }
    at::Tensor norm;
    if (grads.size()) {
        const c10::DeviceGuard guard(grads[0].device());
        std::vector<at::Tensor> held;                                // copies of gradients that do not fill their memory, and
        std::vector<std::pair<size_t, at::Tensor>> back;             // results that go to where they belong behind the launches
        std::vector<mortar_grad_t> list;
        std::vector<std::pair<size_t, bool>> entry;                  // of the list: which gradient it is, and whether it is one of those copies
        list.reserve(grads.size());
        entry.reserve(grads.size());
        for (size_t i = 0; i < grads.size(); ++i) {
            const at::Tensor &g = grads[i], &o = out[i];
            at::Tensor s = g, d = o;
            const bool copied = !g.is_non_overlapping_and_dense() || (o.strides() != g.strides() && !(g.is_contiguous() && o.is_contiguous()));
            if (copied) {
                const auto same = [&](const std::pair<size_t, at::Tensor> &b) {
                    const at::Tensor &t = grads[b.first];
                    return t.const_data_ptr() == g.const_data_ptr() && t.sizes() == g.sizes() && t.strides() == g.strides() && t.scalar_type() == g.scalar_type();
                };
                if (!g.numel() || (in_place && std::any_of(back.begin(), back.end(), same))) continue;
                s = g.clone(at::MemoryFormat::Contiguous);
                d = at::empty(o.sizes(), o.options().requires_grad(false));
                held.push_back(s);
                back.emplace_back(i, d);
            }
            list.push_back({data(s), mut(d), g.numel(), type_code(g.scalar_type()), type_code(o.scalar_type())});
            entry.emplace_back(i, copied);
        }
        check_overlap(list, in_place, what);
        if (!back.empty() && !fresh) {
            std::vector<Places> places;
            places.reserve(2 * list.size());
            for (size_t k = 0; k < list.size(); ++k) {
                if (!list[k].n) continue;
                const size_t i = entry[k].first;
                for (const bool result : {true, false}) places.push_back(places_of(result ? out[i] : grads[i], i, result, entry[k].second));
                if (places.back().same(places[places.size() - 2])) places.pop_back();
            }
            check_copied(std::move(places), what);
        }
        norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
        const at::Tensor ws = empty_bytes(norm, std::max<int64_t>(8, mortar_grad_workspace_bytes(list.data(), (int64_t)list.size())));
        check_rc(mortar_grad_clip(list.data(), (int64_t)list.size(), a[3] == Py_True, max_norm, floats(norm), mut(ws), stream_of(norm)), "mortar_grad_clip");
        const at::NoGradGuard no_grad;
        for (const auto &b : back) out[b.first].copy_(b.second);
        if (!fresh)
            for (const at::Tensor *o : out.all) torch::autograd::impl::bump_version(*o);
    }
    PyObject *results = fresh ? PyList_New((Py_ssize_t)out.size()) : PySequence_List(out.sequence.get());
    if (!results) throw python_error();
    for (size_t i = 0; i < made.size(); ++i) PyList_SET_ITEM(results, (Py_ssize_t)i, THPVariable_Wrap(std::move(made[i])));
    PyObject *n = norm.defined() ? THPVariable_Wrap(std::move(norm)) : empty_norm();
    return Py_BuildValue("(NN)", results, n);
}

// ---- experts ---------------------------------------------------------------------------------------------------------

// expert_sort(ids, n_experts) -> (position int32 [N, k], token int32 [N k], offsets int32 [n_experts + 1])
PyObject *py_expert_sort(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "expert_sort";
    TORCH_CHECK_TYPE(na == 2, "expert_sort: 2 arguments");
    const at::Tensor ids = tensor_arg(a[0], what, "ids");
    const long experts = PyLong_AsLong(a[1]);
    if (experts == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, what, ": ids must be int32 or int64, got ", ids.scalar_type());
    TORCH_CHECK_VALUE(ids.dim() == 2 && ids.size(1) > 0, what, ": expected ids [tokens, slots], got ", ids.sizes());
    TORCH_CHECK_VALUE(experts > 0 && experts <= 1024, what, ": 1 to 1024 experts, got ", experts);
    TORCH_CHECK_VALUE(ids.numel() <= (1 << 26) - 4, what, ": too many slots");
    const c10::DeviceGuard guard(ids.device());
    const at::Tensor c = ids.contiguous();
    const auto options = ids.options().dtype(at::kInt);
    at::Tensor position = at::empty(ids.sizes(), options), token = at::empty({ids.numel()}, options), offsets = at::empty({experts + 1}, options);
    const int64_t n = mortar_expert_sort_workspace_bytes(ids.numel(), (int32_t)experts);
    const at::Tensor ws = n ? empty_bytes(ids, n) : at::Tensor();
    check_rc(mortar_expert_sort(data(c), ids.scalar_type() == at::kLong, ids.size(0), (int32_t)ids.size(1), (int32_t)experts, static_cast<int32_t *>(mut(position)),
                                static_cast<int32_t *>(mut(token)), static_cast<int32_t *>(mut(offsets)), mut(ws), stream_of(ids)),
             "mortar_expert_sort");
    PyObject *p = THPVariable_Wrap(std::move(position)), *t = THPVariable_Wrap(std::move(token)), *o = THPVariable_Wrap(std::move(offsets));
    return Py_BuildValue("(NNN)", p, t, o);
}

// Positions [N, k], offsets [E + 1] and (where there are any) the rows' tokens [N k] of an order, as a launch reads them.
struct Order {
    at::Tensor position, offsets, token;
    int64_t N, k;
    const int32_t *pos() const { return static_cast<const int32_t *>(position.const_data_ptr()); }
    const int32_t *full() const { return static_cast<const int32_t *>(offsets.const_data_ptr()) + offsets.size(0) - 1; }
    const int32_t *tokens() const { return static_cast<const int32_t *>(data(token)); }
};

Order order_of(const at::Tensor &position, const at::Tensor &offsets, const at::Tensor &token) {
    return {position.contiguous(), offsets.contiguous(), token.defined() ? token.contiguous() : token, position.size(0), position.size(1)};
}

Order order_arg(PyObject *p, PyObject *t, PyObject *o, const at::Tensor &x, const char *what) {
    const at::Tensor position = tensor_arg(p, what, "position"), offsets = tensor_arg(o, what, "offsets"), token = optional_arg(t, what, "token");
    same_device(x, position, what, "position");
    same_device(x, offsets, what, "offsets");
    TORCH_CHECK_TYPE(position.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt, what, ": position and offsets must be int32");
    TORCH_CHECK_VALUE(position.dim() == 2 && position.size(1) > 0 && offsets.dim() == 1 && offsets.size(0) > 1, what, ": expected position [tokens, slots] and offsets [experts + 1]");
    TORCH_CHECK_VALUE(position.numel() <= (1 << 26) - 4, what, ": too many slots");
    if (token.defined()) {
        same_device(x, token, what, "token");
        TORCH_CHECK_TYPE(token.scalar_type() == at::kInt, what, ": token must be int32");
        TORCH_CHECK_VALUE(token.dim() == 1 && token.size(0) == position.numel(), what, ": expected token [", position.numel(), "], got ", token.sizes());
    }
    return order_of(position, offsets, token);
}

// Memory of rows [N k, d] by slot: without the rows' tokens a launch leaves what no position names as it was.
at::Tensor empty_slots(const at::Tensor &like, const Order &o, int64_t d) {
    return o.token.defined() ? empty_like_rows(like, {o.N * o.k, d}) : at::zeros({o.N * o.k, d}, like.options().requires_grad(false));
}

void check_rows(const at::Tensor &x, int64_t rows, const char *what, const char *name) {
    TORCH_CHECK_TYPE(type_code(x.scalar_type()) >= 0, what, ": expected bfloat16, float16 or float32, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == rows && x.size(1) > 0, what, ": expected ", name, " [", rows, ", d], got ", x.sizes());
    TORCH_CHECK_VALUE(x.size(1) < (1 << 28), what, ": rows of ", x.size(1), " values are too long");
}

// x [N, d] with consecutive values in its rows.
at::Tensor lines(const at::Tensor &x) { return x.size(1) > 1 && x.stride(1) != 1 ? x.contiguous() : x; }

at::Tensor dispatch(const at::Tensor &x, const Order &o) {
    const c10::DeviceGuard guard(x.device());
    const at::Tensor r = lines(x);
    at::Tensor xs = empty_slots(x, o, x.size(1));
    check_rc(mortar_expert_dispatch_rows(data(r), o.N, (int32_t)x.size(1), r.stride(0), type_code(x.scalar_type()), (int32_t)o.k, o.pos(), o.full(), o.tokens(), mut(xs),
                                         stream_of(x)),
             "mortar_expert_dispatch_rows");
    return xs;
}

at::Tensor combine(const at::Tensor &ys, const at::Tensor &w, const Order &o) {
    const c10::DeviceGuard guard(ys.device());
    const at::Tensor r = ys.contiguous(), wc = w.defined() ? w.contiguous() : w;
    at::Tensor y = empty_like_rows(ys, {o.N, ys.size(1)});
    check_rc(mortar_expert_combine(data(r), o.N, (int32_t)ys.size(1), type_code(ys.scalar_type()), (int32_t)o.k, o.pos(), o.full(), data(wc),
                                   w.defined() ? type_code(w.scalar_type()) : 0, mut(y), stream_of(ys)),
             "mortar_expert_combine");
    return y;
}

// What a node keeps of an order besides the saved tensors: tokens, slots, length of the offsets, whether there are tokens.
void keep_order(AutogradContext *ctx, const Order &o, bool tokens) { ctx->saved_data["order"] = std::vector<int64_t>{o.N, o.k, o.offsets.size(0), tokens}; }
// The order in a backward pass: positions, offsets and tokens from the saved tensor `first` on.
Order kept_order(const std::vector<int64_t> &n, const variable_list &v, size_t first, const at::Tensor &g, const char *what) {
    return order_of(kept(v[first], g, {n[0], n[1]}, at::kInt, what), kept(v[first + 1], g, {n[2]}, at::kInt, what),
                    n[3] ? kept(v[first + 2], g, {n[0] * n[1]}, at::kInt, what) : at::Tensor());
}

struct DispatchFn : public torch::autograd::Function<DispatchFn> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &position, const at::Tensor &offsets, const std::optional<at::Tensor> &token) {
        const Order o = order_of(position, offsets, token ? *token : at::Tensor());
        ctx->save_for_backward({position, offsets});
        keep_order(ctx, o, false);                       // (rows by slot are read only)
        return dispatch(x, o);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(4);
        const char *what = "expert_dispatch";
        const at::Tensor g = plain_gradient(grads[0], what);
        if (!g.defined()) return out;
        out[0] = combine(g, at::Tensor(), kept_order(ctx->saved_data["order"].toIntVector(), ctx->get_saved_variables(), 0, g, what));
        return out;
    }
};

struct CombineFn : public torch::autograd::Function<CombineFn> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &ys, const std::optional<at::Tensor> &weights, const at::Tensor &position, const at::Tensor &offsets,
                              const std::optional<at::Tensor> &token) {
        const at::Tensor w = weights ? *weights : at::Tensor();
        // (not needs_input_grad: that asks the backward pass that is running, if a forward is run again within one)
        const bool need_w = w.defined() && w.requires_grad();
        const Order o = order_of(position, offsets, token ? *token : at::Tensor());
        ctx->save_for_backward({need_w ? ys : at::Tensor(), w, position, offsets, o.token});
        keep_order(ctx, o, o.token.defined());
        ctx->saved_data["type"] = w.defined() ? c10::IValue(w.scalar_type()) : c10::IValue();
        return combine(ys, w, o);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(5);
        const char *what = "expert_combine";
        const at::Tensor g = plain_gradient(grads[0], what);
        if (!g.defined()) return out;
        const auto v = ctx->get_saved_variables();
        const auto n = ctx->saved_data["order"].toIntVector();
        const std::array<int64_t, 2> shape{n[0], n[1]};
        const int64_t d = g.size(1), slots = n[0] * n[1];
        const bool weighted = !ctx->saved_data["type"].isNone();
        // (edges are counted over the tensors that are there)
        const bool need_y = ctx->needs_input_grad(0), need_w = weighted && ctx->needs_input_grad(1);
        const Order o = kept_order(n, v, 2, g, what);
        const c10::DeviceGuard guard(g.device());
        at::Tensor w, ys, dys, dw;
        if (weighted) w = kept(v[1], g, shape, ctx->saved_data["type"].toScalarType(), what).contiguous();
        if (need_w) ys = kept(v[0], g, {slots, d}, g.scalar_type(), what).contiguous();
        if (need_y) dys = empty_slots(g, o, d);
        if (need_w) dw = at::empty(shape, w.options().requires_grad(false));
        const at::Tensor r = lines(g);
        check_rc(mortar_expert_combine_bwd_rows(data(r), r.stride(0), data(ys), o.N, (int32_t)d, type_code(g.scalar_type()), (int32_t)o.k, o.pos(), o.full(), o.tokens(),
                                                data(w), weighted ? type_code(w.scalar_type()) : 0, mut(dys), mut(dw), stream_of(g)),
                 "mortar_expert_combine_bwd_rows");
        out[0] = dys;
        out[1] = dw;
        return out;
    }
};

std::optional<at::Tensor> maybe(const at::Tensor &t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }

// expert_dispatch(x, position, token, offsets) -> xs [N k, d]
PyObject *py_expert_dispatch(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "expert_dispatch";
    TORCH_CHECK_TYPE(na == 4, "expert_dispatch: 4 arguments");
    const at::Tensor x = tensor_arg(a[0], what, "x");
    const Order o = order_arg(a[1], a[2], a[3], x, what);
    check_rows(x, o.N, what, "x");
    at::Tensor xs = c10::GradMode::is_enabled() && x.requires_grad() ? DispatchFn::apply(x, o.position, o.offsets, maybe(o.token)) : dispatch(x, o);
    return THPVariable_Wrap(std::move(xs));
}

// expert_combine(ys, weights, position, token, offsets) -> y [N, d]
PyObject *py_expert_combine(PyObject *, PyObject *const *a, Py_ssize_t na) {
    const char *what = "expert_combine";
    TORCH_CHECK_TYPE(na == 5, "expert_combine: 5 arguments");
    const at::Tensor ys = tensor_arg(a[0], what, "ys"), w = optional_arg(a[1], what, "weights");
    const Order o = order_arg(a[2], a[3], a[4], ys, what);
    check_rows(ys, o.N * o.k, what, "ys");
    if (w.defined()) {
        same_device(ys, w, what, "weights");
        TORCH_CHECK_TYPE(type_code(w.scalar_type()) >= 0, what, ": weights must be bfloat16, float16 or float32, got ", w.scalar_type());
        TORCH_CHECK_VALUE(w.sizes() == o.position.sizes(), what, ": weights must be ", o.position.sizes(), " like the positions, got ", w.sizes());
    }
    at::Tensor y;
    if (c10::GradMode::is_enabled() && (ys.requires_grad() || (w.defined() && w.requires_grad())))
        y = CombineFn::apply(ys, maybe(w), o.position, o.offsets, maybe(o.token));
    else
        y = combine(ys, w, o);
    return THPVariable_Wrap(std::move(y));
}

PyMethodDef methods[] = {MORTAR_METHOD("grad_norm", py_grad_norm, "The norm over the gradients of many tensors."),
                         MORTAR_METHOD("grad_clip", py_grad_clip, "Gradients clipped to a norm over all of them."),
                         MORTAR_METHOD("expert_sort", py_expert_sort, "Slots of tokens sorted by expert."),
                         MORTAR_METHOD("expert_dispatch", py_expert_dispatch, "Tokens to the rows of their experts."),
                         MORTAR_METHOD("expert_combine", py_expert_combine, "Rows of the experts back to their tokens."),
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

int mortar_add_train_methods(PyObject *module) { return PyModule_AddFunctions(module, methods); }
