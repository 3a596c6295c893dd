// linear and gated_linear as differentiable functions of torch tensors: what stands between a call and the launches of libmuon_hip, forward
// and backward, in native code.  The same in Python (ctypes and torch.autograd.Function) costs 25 us for a call and 200 for a training step,
// more than the kernels of a layer of 500 tokens.
//
// Each function takes calls in which nothing needs a decision: plain tensors of one type on one GPU, of shapes that fit.  For anything else
// it returns None before it has done anything, and the caller says what is wrong.  What a thread does is looked at here: refuse_recording.
#define FUNCTIONS_ARE "linear and gated_linear"
#include "functions.h"

namespace {

// ---- products -----------------------------------------------------------------------------------

// One or two matrices as an operand; turned: the reduction runs down their columns.
void operand(const void** at, long* row, long* col, const Tensor& t0, const Tensor& t1, bool turned) {
    const Tensor* t[2] = {&t0, &t1};
    for (int i = 0; i < 2; ++i) {
        at[i] = t[i]->data_ptr();
        row[i] = t[i]->stride(turned ? 1 : 0);
        col[i] = t[i]->stride(turned ? 0 : 1);
    }
}
struct Product : muon_hip_product {
    Product(int kind_, const Tensor& like, int64_t m_, int64_t n_, int64_t k_) : muon_hip_product{} {
        kind = kind_;
        dtype = dtype_of(like);
        m = (int)m_;
        n = (int)n_;
        k = (int)k_;
    }
    void left(const Tensor& t0, const Tensor& t1, bool turned = false) { operand(a, a_row, a_col, t0, t1, turned); }
    void right(const Tensor& t0, const Tensor& t1, bool turned = false) { operand(b, b_row, b_col, t0, t1, turned); }
    void run(const Tensor& like) {
        const long need = muon_hip_product_workspace(this);
        if (need < 0) raise("product", need);
        Tensor ws;
        if (need > 0) ws = at::empty({need}, like.options().dtype(at::kByte));
        if (const int rc = muon_hip_product_run(this, need > 0 ? ws.data_ptr() : nullptr, (size_t)need, stream_of(like))) raise("product", rc);
    }
};

// t as a matrix of the rows of its last dimension: a view where there is one
Tensor matrix(const Tensor& t) {
    const Tensor b = bare(t);
    return b.dim() == 2 ? b : b.reshape({rows_of(b), b.size(-1)});
}
// Memory for a result of the shape of x but for its last dimension.
Tensor result(const Tensor& x, int64_t n) {
    auto shape = x.sizes().vec();
    shape.back() = n;
    return at::empty(shape, x.options());
}

// Memory for a factor that the backward pass multiplies by, in the form that the library keeps it in.
Tensor factor(const Tensor& like, int64_t m, int64_t n) {
    return at::empty({muon_hip_product_aux_bytes(dtype_of(like), (int)m, (int)n)}, like.options().dtype(at::kByte));
}

// What a factor kept for m x n values has to be, and a form of it that the library takes: hooks may have laid it elsewhere.
Tensor factor_back(const Tensor& d, const Tensor& like, int64_t m, int64_t n) {
    if (!d.defined()) return d;
    check_kept(d, {at::kByte}, {muon_hip_product_aux_bytes(dtype_of(like), (int)m, (int)n)}, like);
    refuse_freed(d);
    return d.is_contiguous() && ((uintptr_t)d.data_ptr() & 15) == 0 ? d : d.clone(at::MemoryFormat::Contiguous);
}
// What an input, of k columns and the leading shape of the incoming gradient, and a weight have to be.
void check_input(const Tensor& x, const Tensor& dy, int64_t k) {
    auto shape = dy.sizes().vec();
    shape.back() = k;
    check_kept(x, {dy.scalar_type()}, shape, dy);
}
void check_weight(const Tensor& w, const Tensor& dy, int64_t k) { check_kept(w, {dy.scalar_type()}, {dy.size(-1), k}, dy); }

// Results of a forward pass, and the factors of the backward pass where they are kept.
struct Forward {
    Tensor out, aux[2];
};
Forward linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = matrix(x), w2 = bare(w), b1 = dense(b), r2 = r.defined() ? matrix(r) : r;
    const int64_t m = x2.size(0), n = w2.size(0);
    Forward f;
    f.out = result(x, n);
    if (keep && act != MUON_HIP_ACT_NONE) f.aux[0] = factor(x, m, n);
    Product p(MUON_HIP_PRODUCT_LINEAR, x, m, n, x2.size(1));
    p.activation = act;
    p.left(x2, x2);
    p.right(w2, w2);
    p.bias[0] = pointer(b1);
    if (r2.defined()) {
        p.residual = r2.data_ptr();
        p.res_row = r2.stride(0);
        p.res_col = r2.stride(1);
    }
    p.out[0] = f.out.data_ptr();
    p.aux[0] = (void*)pointer(f.aux[0]);
    p.run(x);
    return f;
}
Forward gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int act, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = matrix(x), g2 = bare(wg), u2 = bare(wu), b0 = dense(bg), b1 = dense(bu);
    const int64_t m = x2.size(0), n = g2.size(0);
    Forward f;
    f.out = result(x, n);
    Product p(MUON_HIP_PRODUCT_GATED, x, m, n, x2.size(1));
    p.activation = act;
    p.left(x2, x2);
    p.right(g2, u2);
    p.bias[0] = pointer(b0);
    p.bias[1] = pointer(b1);
    p.out[0] = f.out.data_ptr();
    for (int i = 0; keep && i < 2; ++i) {
        f.aux[i] = factor(x, m, n);
        p.aux[i] = f.aux[i].data_ptr();
    }
    p.run(x);
    return f;
}

// dz = dy * d for up to two factors and their sums over the rows.  Without a factor dz is dy itself, where its rows are whole 16-byte pieces.
struct Incoming {
    Tensor dz[2], db[2];
};
Incoming act_grad(const Tensor& dy_, int factors, const Tensor& d0, const Tensor& d1, bool want_dz, bool want_db0, bool want_db1, int64_t m, int64_t n) {
    const Tensor dy = dense(dy_).view({m, n});
    const int64_t pitch = (n + 7) / 8 * 8;
    const bool make = want_dz && (factors > 0 || pitch != n || ((uintptr_t)dy.data_ptr() & 15) != 0);
    const bool want_db[2] = {want_db0, want_db1};
    Incoming g;
    for (int i = 0; i < (factors > 1 ? 2 : 1); ++i) {
        g.dz[i] = make ? at::empty({m, pitch}, dy.options()).narrow(1, 0, n) : dy;
        if (want_db[i]) g.db[i] = at::empty({n}, dy.options());
    }
    if (make || want_db0 || want_db1) {
        Tensor parts;
        if (want_db0 || want_db1)
            parts = at::empty({muon_hip_act_grad_partials((int)m, (int)n) * (factors > 1 ? 2 : 1)}, dy.options().dtype(at::kFloat));
        const int rc = muon_hip_act_grad(dy.data_ptr(), factors, pointer(d0), pointer(d1), make ? g.dz[0].data_ptr() : nullptr,
                                         make && factors > 1 ? g.dz[1].data_ptr() : nullptr, pitch, (void*)pointer(g.db[0]), (void*)pointer(g.db[1]),
                                         dtype_of(dy), (int)m, (int)n, (float*)pointer(parts), stream_of(dy));
        if (rc) raise("act_grad", rc);
    }
    return g;
}

// The second derivative of an activation without a curve is zero.
bool curved(int act) { return act != MUON_HIP_ACT_NONE && act != MUON_HIP_ACT_RELU; }

void note(AutogradContext* ctx, const Tensor& x, const Maybe& a, const Maybe& b, int64_t act) {
    ctx->saved_data["k"] = x.size(-1);
    ctx->saved_data["has"] = (int64_t)(a.has_value() + 2 * b.has_value());
    ctx->saved_data["act"] = act;
}
// Whether the optional tensors behind `first` others need a gradient.
struct Wanted {
    bool a, b;
    int64_t has;
    Wanted(AutogradContext* ctx, int first) {
        has = ctx->saved_data["has"].toInt();
        a = (has & 1) && ctx->needs_input_grad(first);
        b = (has & 2) && ctx->needs_input_grad(first + (has & 1));
    }
    // Where the inputs' own gradients go, one place for each that a call may have.
    torch::autograd::edge_list edges(int first) const {
        const auto node = torch::autograd::get_current_node();
        torch::autograd::edge_list all(first + 2);
        for (int i = 0; i < first; ++i) all[i] = node->next_edge(i);
        if (has & 1) all[first] = node->next_edge(first);
        if (has & 2) all[first + 1] = node->next_edge(first + (has & 1));
        return all;
    }
};

// What is kept for a backward pass is what the gradients that can be asked for read, so that a frozen weight does not hold its input, and an
// input that no gradient reads may change.  k is the kept operand's, everything else of the shapes the incoming gradient's.
struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act) {
        const bool for_x = x.requires_grad(), for_w = w.requires_grad(), for_b = b && b->requires_grad();
        Forward f = linear_forward(x, w, given(b), given(r), (int)act, for_x || for_w || for_b);
        ctx->save_for_backward({for_w ? x : Tensor(), for_x ? w : Tensor(), f.aux[0]});
        note(ctx, x, b, r, act);
        return f.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        refuse_recording();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor none, &dy = incoming[0];
        const Wanted more(ctx, 2);
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = more.a;
        const Tensor &x = want_w ? saved[0] : none, &w = want_x ? saved[1] : none;
        variable_list grads(5);
        {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(dy.device());
            if (want_x || want_w || want_b) {
                const int64_t m = rows_of(dy), n = dy.size(-1), k = ctx->saved_data["k"].toInt();
                check_input(x, dy, k);
                check_weight(w, dy, k);
                refuse_freed(dy, x, w);
                const Tensor d = factor_back(saved[2], dy, m, n);
                Incoming g = act_grad(dy, d.defined() ? 1 : 0, d, Tensor(), want_x || want_w, want_b, false, m, n);
                grads[2] = g.db[0];
                if (want_x) {
                    const Tensor w2 = bare(w);
                    grads[0] = result(dy, w2.size(1));
                    Product p(MUON_HIP_PRODUCT_LINEAR, dy, m, w2.size(1), n);
                    p.left(g.dz[0], g.dz[0]);
                    p.right(w2, w2, true);
                    p.out[0] = grads[0].data_ptr();
                    p.run(dy);
                }
                if (want_w) {
                    const Tensor x2 = matrix(x);
                    grads[1] = at::empty({n, x2.size(1)}, dy.options());
                    Product p(MUON_HIP_PRODUCT_LINEAR, dy, n, x2.size(1), m);
                    p.left(g.dz[0], g.dz[0], true);
                    p.right(x2, x2, true);
                    p.out[0] = grads[1].data_ptr();
                    p.run(dy);
                }
            }
            if (more.b) grads[3] = dy;
        }
        if (at::GradMode::is_enabled()) {  // (the residual's is the incoming one, history and all)
            enum { X = 1, W = 2, B = 4 };
            const auto edges = more.edges(2);
            const unsigned dz = curved((int)ctx->saved_data["act"].toInt()) ? X | W | B : 0;
            close_history(grads[0], dz | W, edges, {dy});
            close_history(grads[1], dz | X, edges, {dy});
            close_history(grads[2], dz, edges, {dy});
        }
        return grads;
    }
};

// The gate's gradients (wg, bg) read the factor t = u act'(g), those of the other projection (wu, bu) s = act(g), x's both.
struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& bg, const Maybe& bu, int64_t act) {
        const bool for_x = x.requires_grad(), for_wg = wg.requires_grad(), for_wu = wu.requires_grad();
        const bool for_g = for_x || for_wg || (bg && bg->requires_grad()), for_u = for_x || for_wu || (bu && bu->requires_grad());
        Forward f = gated_forward(x, wg, wu, given(bg), given(bu), (int)act, true);
        const Tensor none;
        ctx->save_for_backward({for_wg || for_wu ? x : none, for_x ? wg : none, for_x ? wu : none, for_u ? f.aux[0] : none, for_g ? f.aux[1] : none});
        note(ctx, x, bg, bu, act);
        return f.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        refuse_recording();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor none, &dh = incoming[0];
        const bool want_x = ctx->needs_input_grad(0), want_wg = ctx->needs_input_grad(1), want_wu = ctx->needs_input_grad(2);
        const Wanted more(ctx, 3);
        const bool want_g = want_x || want_wg || more.a, want_u = want_x || want_wu || more.b, two = want_g && want_u;
        const Tensor &x = want_wg || want_wu ? saved[0] : none, &wg = want_x ? saved[1] : none, &wu = want_x ? saved[2] : none;
        variable_list grads(6);
        if (want_g || want_u) {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(dh.device());
            const int64_t m = rows_of(dh), n = dh.size(-1), k = ctx->saved_data["k"].toInt();
            check_input(x, dh, k);
            check_weight(wg, dh, k);
            check_weight(wu, dh, k);
            refuse_freed(dh, x, wg, wu);
            const Tensor s = factor_back(want_u ? saved[3] : none, dh, m, n), t = factor_back(want_g ? saved[4] : none, dh, m, n);
            Incoming g = act_grad(dh, two ? 2 : 1, want_g ? t : s, two ? s : Tensor(), want_x || want_wg || want_wu, want_g ? more.a : more.b,
                                  two && more.b, m, n);
            const int u = two ? 1 : 0;  // which of them is the other projection's, where it is wanted
            if (more.a) grads[3] = g.db[0];
            if (more.b) grads[4] = g.db[u];
            if (want_x) {
                const Tensor g2 = bare(wg), u2 = bare(wu);
                grads[0] = result(dh, g2.size(1));
                Product p(MUON_HIP_PRODUCT_SUM, dh, m, g2.size(1), n);
                p.left(g.dz[0], g.dz[1]);
                p.right(g2, u2, true);
                p.out[0] = grads[0].data_ptr();
                p.run(dh);
            }
            if (want_wg || want_wu) {
                const Tensor x2 = matrix(x);
                const bool both = want_wg && want_wu;
                Product p(both ? MUON_HIP_PRODUCT_EACH : MUON_HIP_PRODUCT_LINEAR, dh, n, x2.size(1), m);
                if (want_wg) grads[1] = at::empty({n, x2.size(1)}, dh.options());
                if (want_wu) grads[2] = at::empty({n, x2.size(1)}, dh.options());
                const int first = want_wg ? 0 : u;
                p.left(g.dz[first], g.dz[both ? 1 : first], true);
                p.right(x2, x2, true);
                p.out[0] = grads[want_wg ? 1 : 2].data_ptr();
                p.out[1] = both ? grads[2].data_ptr() : nullptr;
                p.run(dh);
            }
        }
        if (at::GradMode::is_enabled()) {
            enum { X = 1, WG = 2, WU = 4, BG = 8, BU = 16 };
            const auto edges = more.edges(3);
            const unsigned of_g = X | WG | BG, of_u = X | WU | BU;
            const unsigned dg = of_u | (curved((int)ctx->saved_data["act"].toInt()) ? of_g : 0), du = of_g;
            close_history(grads[0], dg | du | WG | WU, edges, {dh});
            close_history(grads[1], dg | X, edges, {dh});
            close_history(grads[2], du | X, edges, {dh});
            close_history(grads[3], dg, edges, {dh});
            close_history(grads[4], du, edges, {dh});
        }
        return grads;
    }
};

// ---- calls ------------------------------------------------------------------------------------

// The tensors of a call, None as an undefined one; false where something has to be decided.
bool unpack(PyObject* const* args, int count, int needed, Tensor* out) {
    if (!plain(args[0], nullptr)) return false;
    out[0] = THPVariable_Unpack(args[0]);
    for (int i = 1; i < count; ++i) {
        if (i >= needed && args[i] == Py_None) continue;
        if (!plain(args[i], &out[0])) return false;
        out[i] = THPVariable_Unpack(args[i]);
    }
    return true;
}
// Whether x, weight and bias fit, and their sizes are ones that the entry points take.
bool fits(const Tensor& x, const Tensor& w, const Tensor& b) {
    constexpr int64_t most = 0x7fffffff;
    return x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1) && w.size(0) <= most && w.size(1) <= most && rows_of(x) <= most &&
           (!b.defined() || (b.dim() == 1 && b.size(0) == w.size(0)));
}
// linear(x, weight, bias or None, residual or None, activation code)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    refuse_recording();
    Tensor t[4];
    if (count != 5 || !unpack(args, 4, 2, t) || !fits(t[0], t[1], t[2])) Py_RETURN_NONE;
    if (t[3].defined()) {
        bool same = t[3].dim() == t[0].dim() && t[3].size(-1) == t[1].size(0);
        for (int64_t d = 0; same && d + 1 < t[0].dim(); ++d) same = t[3].size(d) == t[0].size(d);
        if (!same) Py_RETURN_NONE;
    }
    const long act = PyLong_AsLong(args[4]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        if (differentiated(t, 4)) out = Linear::apply(t[0], t[1], maybe(t[2]), maybe(t[3]), (int64_t)act);
        else out = linear_forward(t[0], t[1], t[2], t[3], (int)act, false).out;
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
// gated_linear(x, weight_gate, weight_up, bias_gate or None, bias_up or None, activation code)
PyObject* gated_linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    refuse_recording();
    Tensor t[5];
    if (count != 6 || !unpack(args, 5, 3, t) || !fits(t[0], t[1], t[3]) || !fits(t[0], t[2], t[4]) || t[1].size(0) != t[2].size(0)) Py_RETURN_NONE;
    const long act = PyLong_AsLong(args[5]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        if (differentiated(t, 5)) out = GatedLinear::apply(t[0], t[1], t[2], maybe(t[3]), maybe(t[4]), (int64_t)act);
        else out = gated_forward(t[0], t[1], t[2], t[3], t[4], (int)act, false).out;
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
PyMethodDef methods[] = {{"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
                         {"gated_linear", (PyCFunction)(void (*)(void))gated_linear, METH_FASTCALL, nullptr},
                         {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layers", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layers() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", LAYERS_TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
