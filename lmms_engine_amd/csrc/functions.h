// What the modules of autograd functions (layers.cpp, rows.cpp) share: how tensors reach the launches of libmuon_hip, what is refused, and
// histories that cannot be followed a second time.  FUNCTIONS_ARE names the functions of the module that includes this.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <ATen/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>

#include "../../include/muon_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject* error_type = nullptr;  // MuonHipError

[[noreturn]] void raise(const char* what, long code) {
    const std::string text = std::string(what) + " failed (code " + std::to_string(code) + "): " + muon_hip_last_error();
    python_error e;
    {
        pybind11::gil_scoped_acquire gil;
        PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, text.c_str());
        e.persist();
    }
    throw e;
}

// Tools that record the torch operations of a function, to run them again on other tensors, or that run it on tensors without values, see the
// allocation of a result and none of the launches that fill it: what they made would return memory that nothing has written.
void refuse_recording() {
    using c10::impl::TorchDispatchModeKey;
    bool on = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
    for (const auto key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
        on = on || c10::impl::TorchDispatchModeTLS::get_mode(key).has_value();
    TORCH_CHECK_NOT_IMPLEMENTED(!on, FUNCTIONS_ARE " cannot be recorded or run on tensors without values: their launches are no torch operations");
}

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? MUON_HIP_F32 : MUON_HIP_BF16; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

// t without its history, its values where its pointer says
Tensor bare(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor d = t.detach();
    return d.is_neg() ? d.resolve_neg() : d;
}
Tensor dense(const Tensor& t) { return t.defined() ? bare(t).contiguous() : t; }
int64_t rows_of(const Tensor& t) {
    int64_t m = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) m *= t.size(d);
    return m;
}
const void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Stands for the second derivatives that there are none of: whoever comes through here on the way to an input is told so.
struct Once : torch::autograd::Node {
    variable_list apply(variable_list&&) override {
        TORCH_CHECK(false, FUNCTIONS_ARE " can be differentiated once: their backward pass has none of its own");
    }
};
// Gradient `g` depends on the inputs whose bits are set in `on` (positions of `edges`; those that need no gradient have no edge) and on
// the incoming gradients.  Where one of them is differentiated, so would g be: its history leads to all of them, so that a loss that g is a
// part of raises for each of them and loses no term, and to no other.
void close_history(Tensor& g, unsigned on, const torch::autograd::edge_list& edges, std::initializer_list<Tensor> incoming) {
    if (!g.defined()) return;
    torch::autograd::edge_list next;
    for (size_t i = 0; i < edges.size(); ++i)
        if ((on >> i & 1) && edges[i].is_valid()) next.push_back(edges[i]);
    for (const Tensor& dy : incoming)
        if (dy.defined() && dy.requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(dy));
    if (next.empty()) return;
    const auto node = std::shared_ptr<Once>(new Once(), torch::autograd::deleteNode);
    node->set_next_edges(std::move(next));
    torch::autograd::impl::set_gradient_edge(g, {node, node->add_input_metadata(g)});
}

// Tensors that a call may lack travel as optionals, and a context numbers the tensors that there are: `has` holds a bit for each that a call
// may have, the first one's lowest.
typedef std::optional<Tensor> Maybe;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }

// Whether the program has freed the memory of a tensor and kept the tensor, as sharded training does: no version counter tells, and the address of what was
// freed is null, or a small number in a view, not that of nothing.
bool freed(const Tensor& t) { return t.defined() && t.has_storage() && t.numel() > 0 && !t.storage().data(); }
// Of what a backward pass reads, where it may have happened since the forward pass.
template <typename... Tensors>
void refuse_freed(const Tensors&... all) {
    const auto one = [](const Tensor& t) { TORCH_CHECK_VALUE(!freed(t), "the memory of a tensor of shape ", t.sizes(), " was freed before its backward pass"); };
    (one(all), ...);
}
// What was kept for a backward pass comes back through the program's hooks, if it has any: it has to be of the type and shape that it had, and where the incoming
// gradient is, before its address goes to a kernel.
void check_kept(const Tensor& t, std::initializer_list<at::ScalarType> types, at::IntArrayRef sizes, const Tensor& like) {
    if (!t.defined()) return;
    TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch(), "what was kept for a backward pass is no plain tensor");
    TORCH_CHECK_TYPE(std::find(types.begin(), types.end(), t.scalar_type()) != types.end(), "what was kept for a backward pass is ", t.scalar_type(), ", it was ",
                     *types.begin());
    TORCH_CHECK_VALUE(t.sizes() == sizes, "what was kept for a backward pass has shape ", t.sizes(), ", it had ", sizes);
    TORCH_CHECK_VALUE(t.device() == like.device(), "what was kept for a backward pass is on ", t.device(), ", the incoming gradient on ", like.device());
}
// A plain tensor on a GPU whose memory is there.
bool present(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.unsafeGetTensorImpl()->is_python_dispatch()) return false;
    return !freed(t);
}
// The same of x's type and device.
bool plain(PyObject* o, const Tensor* x) {
    if (!present(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    if (x) return t.scalar_type() == x->scalar_type() && t.device() == x->device();
    return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
// Whether the call has a history; a tangent of forward mode counts too, so that autograd refuses it.
bool differentiated(const Tensor* t, int count) {
    const bool backward = at::GradMode::is_enabled();
    for (int i = 0; i < count; ++i)
        if (t[i].defined() && ((backward && t[i].requires_grad()) || t[i]._fw_grad(0).defined())) return true;
    return false;
}

// set_error(type): what a refusal of the library is raised as
PyObject* set_error(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XDECREF(error_type);
    error_type = type;
    Py_RETURN_NONE;
}

}  // namespace
