// embedding, layer_norm, rms_norm and dropout as differentiable functions of torch tensors, in native code for the reason that layers.cpp gives.
//
// Each function takes calls in which nothing needs a decision and returns None for anything else before it has done anything; the caller says
// what is wrong.
#define FUNCTIONS_ARE "embedding, layer_norm, rms_norm and dropout"
#include "functions.h"

#include <ATen/EmptyTensor.h>
#include <ATen/detail/CUDAHooksInterface.h>

namespace {

constexpr int64_t MOST = 0x7fffffff;

// Memory on the current device.  (By way of torch's dispatcher it costs 0.4 us more, of a call of 3.5.)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
    static c10::Allocator* const allocator = at::detail::getCUDAHooks().getCUDADeviceAllocator();
    return Tensor(at::detail::empty_generic(sizes, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}
// The rows of a tensor's last dimension, back to back within themselves: where they lie, if that is so, else in a copy that is kept here.  (A view for
// the same costs a call half a microsecond each.)
struct Lines {
    Tensor copy;
    const void* at = nullptr;
    int64_t apart = 0;
    explicit Lines(const Tensor& t) {
        if (!t.defined()) return;
        const int64_t n = t.dim() > 0 ? t.size(-1) : 1;
        if (!t.is_neg() && t.is_contiguous()) {
            at = t.data_ptr();
            apart = n;
            return;
        }
        Tensor b = bare(t);
        if (b.dim() != 2) b = b.reshape({rows_of(b), n});
        copy = (n > 1 && b.stride(1) != 1) || (b.size(0) > 1 && b.stride(0) < n) ? b.contiguous() : b;
        at = copy.data_ptr();
        apart = copy.stride(0);
    }
};
// The values of a tensor in the row-major order of its shape.
struct Values {
    Tensor copy;
    const void* at = nullptr;
    explicit Values(const Tensor& t) {
        if (t.defined() && (t.is_neg() || !t.is_contiguous())) copy = dense(t);
        at = pointer(copy.defined() ? copy : t);
    }
};
// The places of the tensors of a context: `always` of them, then those of COUNT optional ones that there are.
template <int COUNT> struct Places {
    AutogradContext* ctx;
    int at[COUNT];
    Places(AutogradContext* c, int always) : ctx(c) {
        const int64_t has = ctx->saved_data["has"].toInt();
        for (int i = 0, next = always; i < COUNT; ++i) at[i] = has >> i & 1 ? next++ : -1;
    }
    bool wanted(int i) const { return at[i] >= 0 && ctx->needs_input_grad(at[i]); }
    torch::autograd::Edge edge(int i) const { return at[i] >= 0 ? torch::autograd::get_current_node()->next_edge(at[i]) : torch::autograd::Edge(); }
};
bool trained(const Maybe& t) { return t && t->requires_grad(); }

// ---- norms --------------------------------------------------------------------------------------

struct Normed {
    Tensor y, sum, stats;
};
Normed norm_forward(int kind, const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, double eps, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const Lines x2(x), r2(r);
    const Values w1(w), b1(b);
    const int64_t rows = rows_of(x);
    Normed f;
    f.y = fresh(x.sizes(), x.scalar_type());
    if (r.defined()) f.sum = fresh(x.sizes(), x.scalar_type());
    if (keep) f.stats = fresh({kind == MUON_HIP_NORM_LAYER ? 2 : 1, rows}, at::kFloat);
    muon_hip_norm p{};
    p.kind = kind;
    p.dtype = dtype_of(x);
    p.rows = (int)rows;
    p.n = (int)x.size(-1);
    p.x = x2.at;
    p.x_row = x2.apart;
    if (r.defined()) {
        p.residual = r2.at;
        p.res_row = r2.apart;
        p.sum = f.sum.data_ptr();
    }
    p.weight = w1.at;
    p.bias = b1.at;
    p.eps = eps;
    p.y = f.y.data_ptr();
    p.stats = (float*)pointer(f.stats);
    if (const int rc = muon_hip_norm_run(&p, stream_of(x))) raise("norm", rc);
    return f;
}

// Kept is what the gradients that can be asked for read: the normalised rows' input for all but the bias', the weight for the input's.
struct Norm : torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, const Maybe& r, int64_t kind, double eps) {
        const bool for_x = x.requires_grad() || trained(r), for_w = trained(w);
        const Normed f = norm_forward((int)kind, x, given(w), given(b), given(r), eps, for_x || for_w);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({for_x || for_w ? (r ? f.sum : x) : Tensor(), for_x ? given(w) : Tensor(), f.stats});
        ctx->saved_data["has"] = (int64_t)(w.has_value() + 2 * b.has_value() + 4 * r.has_value());
        ctx->saved_data["kind"] = kind;
        if (!r) return {f.y};
        if (!for_x) ctx->mark_non_differentiable({f.sum});
        return {f.y, f.sum};
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        refuse_recording();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &s = saved[0], &w = saved[1], &stats = saved[2], &dy = incoming[0], ds = incoming.size() > 1 ? incoming[1] : Tensor();
        const Places<3> more(ctx, 1);
        const bool want_x = ctx->needs_input_grad(0), want_r = more.wanted(2), want_w = more.wanted(0), want_b = more.wanted(1);
        variable_list grads(6);
        Tensor dx;
        if (!dy.defined() && !ds.defined()) return grads;
        const Tensor& like = dy.defined() ? dy : ds;
        {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(like.device());
            const int64_t n = like.size(-1);
            if (!dy.defined()) {  // of the sum alone
                if (want_w) grads[1] = at::zeros({n}, like.options());
                if (want_b) grads[2] = at::zeros({n}, like.options());
            } else if (want_x || want_r || want_w || want_b) {
                const bool for_x = want_x || want_r;
                const Tensor none, &s_read = for_x || want_w ? s : none, &stats_read = for_x || want_w ? stats : none;
                const Tensor &w_read = for_x ? w : none, &ds_read = for_x ? ds : none;
                muon_hip_norm_grad p{};
                p.kind = (int)ctx->saved_data["kind"].toInt();
                p.dtype = dtype_of(like);
                p.rows = (int)rows_of(dy);
                check_kept(s_read, {like.scalar_type()}, like.sizes(), like);
                check_kept(stats_read, {at::kFloat}, {p.kind == MUON_HIP_NORM_LAYER ? 2 : 1, (int64_t)p.rows}, like);
                check_kept(w_read, {like.scalar_type()}, {n}, like);
                refuse_freed(dy, s_read, stats_read, w_read, ds_read);
                const Lines dy2(dy), s2(s_read), ds2(ds_read);
                const Values w1(w_read), stats1(stats_read);
                p.n = (int)n;
                p.dy = dy2.at;
                p.dy_row = dy2.apart;
                p.s = s2.at;  // (nothing where the bias' gradient alone is asked for)
                p.s_row = s2.apart;
                p.stats = (const float*)stats1.at;
                p.ds = ds2.at;
                p.ds_row = ds2.apart;
                p.weight = w1.at;
                if (for_x) p.dx = (dx = fresh(like.sizes(), like.scalar_type())).data_ptr();
                if (want_w) p.dweight = (grads[1] = fresh({n}, like.scalar_type())).data_ptr();
                if (want_b) p.dbias = (grads[2] = fresh({n}, like.scalar_type())).data_ptr();
                const long need = muon_hip_norm_grad_workspace(&p);
                if (need < 0) raise("norm_grad", need);
                Tensor ws;
                if (need > 0) ws = fresh({need}, at::kByte);
                if (const int rc = muon_hip_norm_grad_run(&p, need > 0 ? ws.data_ptr() : nullptr, (size_t)need, stream_of(like))) raise("norm_grad", rc);
            }
        }
        if (at::GradMode::is_enabled()) {
            enum { X = 1, W = 2, R = 4 };
            const torch::autograd::edge_list edges{torch::autograd::get_current_node()->next_edge(0), more.edge(0), more.edge(2)};
            close_history(dx, X | W | R, edges, {dy, ds});
            close_history(grads[1], dy.defined() ? X | R : 0, edges, {dy});
            close_history(grads[2], 0, edges, {dy});
        }
        if (!dy.defined()) dx = ds;  // history and all
        if (want_x) grads[0] = dx;
        if (want_r) grads[3] = dx;
        return grads;
    }
};

// ---- embedding ------------------------------------------------------------------------------------

Tensor embedding_forward(const Tensor& weight, const Tensor& ids, double scale) {
    const c10::DeviceGuard guard(weight.device());
    const Lines w2(weight);
    const Tensor i1 = ids.contiguous();
    auto shape = ids.sizes().vec();
    shape.push_back(weight.size(1));
    const Tensor y = fresh(shape, weight.scalar_type());
    if (const int rc = muon_hip_embedding(i1.data_ptr(), ids.scalar_type() == at::kLong, (int)ids.numel(), w2.at, w2.apart, (int)weight.size(0),
                                          (int)weight.size(1), dtype_of(weight), scale, y.data_ptr(), stream_of(weight)))
        raise("embedding", rc);
    return y;
}
struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t skip) {
        ctx->save_for_backward({ids});
        ctx->saved_data["vocab"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["skip"] = skip;
        return embedding_forward(weight, ids, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        refuse_recording();
        const Tensor ids = ctx->get_saved_variables()[0], &dy = incoming[0];
        variable_list grads(4);
        if (!ctx->needs_input_grad(0)) return grads;
        {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(dy.device());
            const int64_t vocab = ctx->saved_data["vocab"].toInt(), n = dy.size(-1);
            check_kept(ids, {at::kLong, at::kInt}, dy.sizes().slice(0, dy.dim() - 1), dy);
            refuse_freed(dy, ids);
            const Lines dy2(dy);
            const Tensor i1 = ids.contiguous();
            grads[0] = fresh({vocab, n}, dy.scalar_type());
            const int tokens = (int)ids.numel(), dtype = dtype_of(dy);
            const long need = muon_hip_embedding_grad_workspace(tokens, (int)vocab, (int)n, dtype);
            if (need < 0) raise("embedding_grad", need);
            Tensor ws;
            if (need > 0) ws = fresh({need}, at::kByte);
            if (const int rc = muon_hip_embedding_grad(i1.data_ptr(), ids.scalar_type() == at::kLong, tokens, dy2.at, dy2.apart, (int)vocab, (int)n,
                                                       dtype, ctx->saved_data["scale"].toDouble(), (int)ctx->saved_data["skip"].toInt(),
                                                       grads[0].data_ptr(), need > 0 ? ws.data_ptr() : nullptr, (size_t)need, stream_of(dy)))
                raise("embedding_grad", rc);
        }
        if (at::GradMode::is_enabled()) close_history(grads[0], 0, {}, {dy});
        return grads;
    }
};

// ---- dropout --------------------------------------------------------------------------------------

Tensor dropout_forward(const Tensor& x, const Tensor& r, const Tensor& seed_at, double p, int64_t seed, int64_t site) {
    const c10::DeviceGuard guard(x.device());
    const Values x1(x), r1(r);
    const Tensor y = fresh(x.sizes(), x.scalar_type());
    if (const int rc = muon_hip_dropout(x1.at, r1.at, y.data_ptr(), x.numel(), dtype_of(x), p, (unsigned long long)seed, pointer(seed_at),
                                        (unsigned)site, stream_of(x)))
        raise("dropout", rc);
    return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& r, const Maybe& seed_at, double p, int64_t seed, int64_t site) {
        if (x.requires_grad()) ctx->save_for_backward({given(seed_at)});
        ctx->saved_data["has"] = (int64_t)(r.has_value() + 2 * seed_at.has_value());
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["site"] = site;
        return dropout_forward(x, given(r), given(seed_at), p, seed, site);
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        refuse_recording();
        const Tensor& dy = incoming[0];
        variable_list grads(6);
        if (ctx->needs_input_grad(0)) {
            {
                const at::AutoGradMode off(false);
                const Tensor seed_at = ctx->get_saved_variables()[0];
                if (seed_at.defined()) check_kept(seed_at, {at::kLong}, seed_at.numel() == 1 ? seed_at.sizes() : at::IntArrayRef({1}), dy);
                refuse_freed(dy, seed_at);
                grads[0] = dropout_forward(dy, Tensor(), seed_at, ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), ctx->saved_data["site"].toInt());
            }
            if (at::GradMode::is_enabled()) close_history(grads[0], 0, {}, {dy});
        }
        if (Places<2>(ctx, 1).wanted(0)) grads[1] = dy;
        return grads;
    }
};

// ---- calls ----------------------------------------------------------------------------------------

// args[i] as an optional tensor of x's type and device; false where something has to be decided.
bool optional(PyObject* o, const Tensor& x, Tensor& out) {
    if (o == Py_None) return true;
    if (!plain(o, &x)) return false;
    out = THPVariable_Unpack(o);
    return true;
}

// norm(kind, x, weight or None, bias or None, residual or None, eps): y, or (y, sum) with a residual
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    refuse_recording();
    if (count != 6 || !plain(args[1], nullptr)) Py_RETURN_NONE;
    Tensor t[4] = {THPVariable_Unpack(args[1])};
    for (int i = 1; i < 4; ++i)
        if (!optional(args[1 + i], t[0], t[i])) Py_RETURN_NONE;
    const Tensor& x = t[0];
    if (x.dim() < 1 || x.size(-1) > MOST || rows_of(x) > MOST || (t[3].defined() && t[3].sizes() != x.sizes())) Py_RETURN_NONE;
    for (int i = 1; i < 3; ++i)
        if (t[i].defined() && (t[i].dim() != 1 || t[i].size(0) != x.size(-1))) Py_RETURN_NONE;
    const long kind = PyLong_AsLong(args[0]);
    const double eps = PyFloat_AsDouble(args[5]);
    if (PyErr_Occurred()) return nullptr;
    if (!(eps >= 0)) Py_RETURN_NONE;
    variable_list out;
    {
        pybind11::gil_scoped_release no_gil;
        if (differentiated(t, 4)) out = Norm::apply(x, maybe(t[1]), maybe(t[2]), maybe(t[3]), (int64_t)kind, eps);
        else {
            const Normed f = norm_forward((int)kind, x, t[1], t[2], t[3], eps, false);
            out = {f.y, f.sum};
        }
    }
    if (!t[3].defined()) return THPVariable_Wrap(out[0]);
    PyObject *y = THPVariable_Wrap(out[0]), *sum = y ? THPVariable_Wrap(out[1]) : nullptr, *pair = sum ? PyTuple_Pack(2, y, sum) : nullptr;
    Py_XDECREF(y);
    Py_XDECREF(sum);
    return pair;
    END_HANDLE_TH_ERRORS
}
// embedding(ids, weight, scale, id without a gradient or -1)
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    refuse_recording();
    if (count != 4 || !present(args[0]) || !plain(args[1], nullptr)) Py_RETURN_NONE;
    const Tensor ids = THPVariable_Unpack(args[0]), weight = THPVariable_Unpack(args[1]);
    if ((ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || ids.device() != weight.device() || ids.numel() > MOST || weight.dim() != 2 ||
        weight.size(0) >= MOST || weight.size(1) > MOST)
        Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(args[2]);
    const long skip = PyLong_AsLong(args[3]);
    if (PyErr_Occurred()) return nullptr;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = differentiated(&weight, 1) ? Embedding::apply(weight, ids, scale, (int64_t)skip) : embedding_forward(weight, ids, scale);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
// dropout(x, residual or None, p, seed: a whole number or a tensor of one, site)
PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    refuse_recording();
    if (count != 5 || !plain(args[0], nullptr)) Py_RETURN_NONE;
    Tensor t[2] = {THPVariable_Unpack(args[0])}, seed_at;
    if (!optional(args[1], t[0], t[1]) || (t[1].defined() && t[1].sizes() != t[0].sizes())) Py_RETURN_NONE;
    if (!PyLong_Check(args[3])) {
        if (!present(args[3])) Py_RETURN_NONE;
        seed_at = THPVariable_Unpack(args[3]);
        if (seed_at.scalar_type() != at::kLong || seed_at.numel() != 1 || seed_at.device() != t[0].device()) Py_RETURN_NONE;
    }
    const double p = PyFloat_AsDouble(args[2]);
    const int64_t seed = seed_at.defined() ? 0 : (int64_t)PyLong_AsUnsignedLongLongMask(args[3]);
    const unsigned long site = PyLong_AsUnsignedLongMask(args[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!(p >= 0 && p <= 1)) Py_RETURN_NONE;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        if (differentiated(t, 2)) out = Dropout::apply(t[0], maybe(t[1]), maybe(seed_at), p, seed, (int64_t)site);
        else out = dropout_forward(t[0], t[1], seed_at, p, seed, (int64_t)site);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL, nullptr},
                         {"embedding", (PyCFunction)(void (*)(void))embedding, METH_FASTCALL, nullptr},
                         {"dropout", (PyCFunction)(void (*)(void))dropout, METH_FASTCALL, nullptr},
                         {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", ROWS_TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
