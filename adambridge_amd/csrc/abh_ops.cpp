// abh_ops.cpp -- the host's side of the operators of a model of expert blocks, natively (Python module _ops).
//
// A call of one token costs what its host work costs: through Python's autograd functions and ctypes a layer norm of
// one row took 13 us, its training pass 100, for kernels of 4 and 8.  Here are the ordinary calls: plain contiguous
// tensors of the kernels' types on one GPU, in no trace, transform or mode.  Every other call returns None, before
// anything is done, and the Python functions (norms.py, experts.py, vocabulary.py) check it, lay it out or take torch
// operations.  The backward passes are here too; one that is itself differentiated, batched or observed calls the
// Python function of the same formula in torch operations that connect() was given.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cstdint>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/adambridge_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::tensor_list;

// ---------------------------------------------------------------- the library's entry points

struct Api {
    decltype(&adambridge_set_stream) set_stream;
    decltype(&adambridge_last_error) last_error;
    decltype(&adambridge_layer_norm) layer_norm;
    decltype(&adambridge_layer_norm_work) layer_norm_work;
    decltype(&adambridge_layer_norm_backward) layer_norm_backward;
    decltype(&adambridge_route_work) route_work;
    decltype(&adambridge_route) route;
    decltype(&adambridge_route_backward) route_backward;
    decltype(&adambridge_dispatch) dispatch;
    decltype(&adambridge_combine) combine;
    decltype(&adambridge_combine_backward) combine_backward;
    decltype(&adambridge_expert_mm) expert_mm;
    decltype(&adambridge_expert_mm_dx) expert_mm_dx;
    decltype(&adambridge_expert_mm_work) expert_mm_work;
    decltype(&adambridge_expert_mm_dw) expert_mm_dw;
    decltype(&adambridge_embed) embed;
    decltype(&adambridge_embed_work) embed_work;
    decltype(&adambridge_embed_backward) embed_backward;
    decltype(&adambridge_token_losses) token_losses;
    decltype(&adambridge_token_losses_work) token_losses_work;
    decltype(&adambridge_token_losses_backward) token_losses_backward;
    decltype(&adambridge_token_losses_backward_work) token_losses_backward_work;
    decltype(&adambridge_expert_mlp_work) expert_mlp_work;
    decltype(&adambridge_expert_mlp) expert_mlp;
};

Api api;
bool connected = false;
PyObject* twice = nullptr;   // the backward passes in torch operations, by name
PyObject* placing = nullptr; // the class of the modes that only place new tensors (a default device)

// The tensor's device current and its current stream the library's, for the scope.
struct On {
    c10::OptionalDeviceGuard guard;
    explicit On(const Tensor& t)
    {
        guard.reset_device(t.device());
        api.set_stream(c10::hip::getCurrentHIPStream(t.device().index()).stream());
    }
};

void check(int64_t rc, const char* what)
{
    TORCH_CHECK(rc >= 0, what, " rejected the call (code ", rc, ")", rc == ADAMBRIDGE_EHIP ? std::string(": ") + api.last_error() : "");
}

int32_t code(at::ScalarType t) { return t == at::kFloat ? ADAMBRIDGE_DT_F32 : ADAMBRIDGE_DT_BF16; }
bool type_ok(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* place(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::empty(sizes, like.options().dtype(type)); }
Tensor scratch(int64_t bytes, const Tensor& like) { return bytes ? fresh({(bytes + 3) / 4}, at::kInt, like) : Tensor(); }

// -------------------------------------------------------------------------- ordinary calls

bool observed()
{
    using Modes = at::impl::PythonTorchFunctionTLS;
    for (int64_t i = 0, n = Modes::stack_len(); i < n; ++i)   // (also without the GIL: a type's address, no reference)
        if ((PyObject*)Py_TYPE(Modes::get_stack_at(i)->ptr(getPyInterpreter())) != placing) return true;
    return torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// The tensor if it is one whose memory the kernels take as it is; nullptr for anything else.
const Tensor* plain(PyObject* o)
{
    if (Py_TYPE(o) != (PyTypeObject*)THPVariableClass && Py_TYPE(o) != (PyTypeObject*)ParameterClass) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || !t.has_storage() || t._is_zerotensor() || t.is_neg() ||
        !t.is_contiguous())
        return nullptr;
    return t._fw_grad(0).defined() ? nullptr : &t;
}

// A tensor or None; false for neither.
bool plain_or_none(PyObject* o, const Tensor*& t)
{
    t = o == Py_None ? nullptr : plain(o);
    return t || o == Py_None;
}

bool values(const Tensor* t, int64_t dim) { return t && t->dim() == dim && type_ok(t->scalar_type()) && t->numel() > 0; }
bool beside(const Tensor* t, const Tensor* x, at::ScalarType type) { return t && t->device() == x->device() && t->scalar_type() == type; }

bool wants_grad(std::initializer_list<const Tensor*> ts)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t && t->requires_grad()) return true;
    return false;
}

// Whether a backward pass may run the kernels: not one that is differentiated in turn or observed, nor one whose gradient
// is a batch, holds no memory of its own or carries a tangent (an operand after the operator may be a dual one; the
// torch operations carry it on).
bool plain_backward(const Tensor& g)
{
    return !at::GradMode::is_enabled() && !observed() && g.layout() == at::kStrided && g.is_cuda() && g.has_storage() &&
           !g._is_zerotensor() && !g.is_neg() && !g.key_set().has(c10::DispatchKey::Python) && !g._fw_grad(0).defined();
}

// Whether a saved tensor is one that the kernels take, once it is contiguous: of this type, in memory of its own beside the
// gradient.  A hook on saved tensors may give back any other.  One of other sizes is an error, also where torch operations
// follow: they would index it on the device.  (Sizes without numbers, of a trace, are left to those.)
bool restored(const Tensor& t, const Tensor& g, at::ScalarType type, at::IntArrayRef sizes)
{
    TORCH_CHECK(t.defined() && (t.unsafeGetTensorImpl()->has_symbolic_sizes_strides() || t.sizes() == sizes),
                "a saved tensor came back as another: expected sizes ", sizes, ", got ", t.defined() ? t.sizes() : at::IntArrayRef());
    return t.layout() == at::kStrided && t.device() == g.device() && t.scalar_type() == type && t.has_storage() && !t._is_zerotensor() &&
           !t.is_neg() && !t.key_set().has(c10::DispatchKey::Python) && !t._fw_grad(0).defined();
}

// A gradient's sizes (none has no dimension); nothing where they are a trace's.
at::IntArrayRef sizes_of(const Tensor& g)
{
    return g.unsafeGetTensorImpl()->has_symbolic_sizes_strides() ? at::IntArrayRef() : g.sizes();
}

// A backward pass in torch operations, by the Python function of that name.
template <class Arguments>
tensor_list in_torch(const char* name, const Arguments& arguments, size_t n)
{
    pybind11::gil_scoped_acquire gil;
    const pybind11::object got = pybind11::reinterpret_borrow<pybind11::dict>(twice)[name](*arguments());
    const pybind11::sequence all = pybind11::cast<pybind11::sequence>(got);
    tensor_list out(n);
    for (size_t i = 0; i < n && i < all.size(); ++i)
        if (!all[i].is_none()) out[i] = pybind11::cast<Tensor>(all[i]);
    return out;
}

pybind11::object or_none(const Tensor& t) { return t.defined() ? pybind11::cast(t) : pybind11::none(); }

// ------------------------------------------------------------------------------ layer norm

Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats)
{
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    Tensor y = fresh(x.sizes(), x.scalar_type(), x);
    if (stats) *stats = fresh({rows, 2}, at::kFloat, x);
    const at::ScalarType wt = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
    const On on(x);
    check(api.layer_norm(address(x), code(x.scalar_type()), address(w), address(b), code(wt), rows, cols, (float)eps, place(y),
                         stats ? stats->mutable_data_ptr<float>() : nullptr), "adambridge_layer_norm");
    return y;
}

struct LayerNorm : Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor wt = w.value_or(Tensor()), bt = b.value_or(Tensor());
        Tensor stats;
        Tensor y = norm_forward(x, wt, bt, eps, &stats);
        ctx->save_for_backward({x, wt, stats});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["given"] = (int64_t)(wt.defined() | bt.defined() << 1 |
                                             (int64_t)(wt.defined() ? wt : bt.defined() ? bt : x).scalar_type() << 8);
        return y;
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const int64_t given = ctx->saved_data["given"].toInt();
        const at::ScalarType wt = (at::ScalarType)(given >> 8);
        // only given tensors count among a function's edges
        const bool want_x = ctx->needs_input_grad(0), want_w = (given & 1) && ctx->needs_input_grad(1),
                   want_b = (given & 2) && ctx->needs_input_grad(1 + (given & 1));
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const int64_t cols = sizes.empty() ? 0 : sizes.back(), rows = cols ? grads[0].numel() / cols : 0;
        const bool whole = cols && restored(x, grads[0], grads[0].scalar_type(), sizes) & restored(stats, grads[0], at::kFloat, {rows, 2}) &
                                       (!w.defined() || restored(w, grads[0], wt, {cols}));
        if (!whole || !plain_backward(grads[0]))
            return in_torch("layer_norm", [&] {
                return pybind11::make_tuple(grads[0], x, or_none(w), ctx->saved_data["eps"].toDouble(), want_x, want_w, want_b,
                                            pybind11::reinterpret_borrow<pybind11::object>((PyObject*)torch::getTHPDtype(wt)));
            }, 4);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), xc = x.contiguous(), wc = w.defined() ? w.contiguous() : w, sc = stats.contiguous();
        tensor_list out(4);
        if (want_x) out[0] = fresh(sizes, g.scalar_type(), g);
        if (want_w) out[1] = fresh({cols}, wt, g);
        if (want_b) out[2] = fresh({cols}, wt, g);
        Tensor work;
        if (want_w || want_b) {
            const int64_t bytes = api.layer_norm_work(rows, cols, code(g.scalar_type()));
            check(bytes, "adambridge_layer_norm_work");
            work = scratch(bytes, g);
        }
        const On on(g);
        check(api.layer_norm_backward(address(g), address(xc), code(g.scalar_type()), address(wc), code(wt), sc.const_data_ptr<float>(),
                                      rows, cols, place(out[0]), place(out[1]), place(out[2]), place(work)),
              "adambridge_layer_norm_backward");
        return out;
    }
};

// layer_norm(x, weight or None, bias or None, eps)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 4 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *x = plain(args[0]), *w, *b;
    if (!x || x->dim() < 1 || !type_ok(x->scalar_type()) || x->numel() == 0) Py_RETURN_NONE;
    if (!plain_or_none(args[1], w) || !plain_or_none(args[2], b) || !PyFloat_Check(args[3])) Py_RETURN_NONE;
    const int64_t cols = x->size(-1);
    for (const Tensor* t : {w, b})
        if (t && (t->dim() != 1 || t->size(0) != cols || t->device() != x->device() || !type_ok(t->scalar_type()))) Py_RETURN_NONE;
    if ((w && b && w->scalar_type() != b->scalar_type()) || cols > (int64_t)1 << 30 || x->numel() / cols > (int64_t)1 << 30) Py_RETURN_NONE;
    const double eps = PyFloat_AS_DOUBLE(args[3]);
    if (wants_grad({x, w, b}))
        return THPVariable_Wrap(LayerNorm::apply(*x, w ? optional<Tensor>(*w) : std::nullopt, b ? optional<Tensor>(*b) : std::nullopt, eps));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(norm_forward(*x, w ? *w : Tensor(), b ? *b : Tensor(), eps, nullptr));
    END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------------------------- route

// weights, chosen, ends, order, position
tensor_list route_forward(const Tensor& logits, int64_t top_k, bool normalize)
{
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    tensor_list out = {fresh({tokens, top_k}, at::kFloat, logits), fresh({tokens, top_k}, at::kInt, logits), fresh({experts}, at::kInt, logits),
                       fresh({tokens * top_k}, at::kInt, logits), fresh({tokens, top_k}, at::kInt, logits)};
    const int64_t bytes = api.route_work(tokens, experts, top_k);
    check(bytes, "adambridge_route_work");
    Tensor work = scratch(bytes, logits);
    const On on(logits);
    check(api.route(address(logits), code(logits.scalar_type()), tokens, experts, top_k, normalize, out[0].mutable_data_ptr<float>(),
                    out[1].mutable_data_ptr<int32_t>(), out[2].mutable_data_ptr<int32_t>(), out[3].mutable_data_ptr<int32_t>(),
                    out[4].mutable_data_ptr<int32_t>(), place(work)), "adambridge_route");
    return out;
}

struct Route : Function<Route> {
    static tensor_list forward(AutogradContext* ctx, const Tensor& logits, int64_t top_k, bool normalize)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        tensor_list out = route_forward(logits, top_k, normalize);
        ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({out[0], out[1], normalize ? Tensor() : logits});
        ctx->saved_data["of"] = (int64_t)(normalize | (int64_t)logits.scalar_type() << 8 | logits.size(1) << 16);
        return out;
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        tensor_list out(3);
        if (!grads[0].defined()) return out;
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor &weights = saved[0], &chosen = saved[1], &logits = saved[2];
        const int64_t of = ctx->saved_data["of"].toInt(), experts = of >> 16;
        const bool normalize = of & 1;
        const at::ScalarType type = (at::ScalarType)(of >> 8 & 255);
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const bool whole = !sizes.empty() && restored(weights, grads[0], at::kFloat, sizes) & restored(chosen, grads[0], at::kInt, sizes) &
                                                 (normalize || restored(logits, grads[0], type, {sizes[0], experts}));
        if (!whole || !plain_backward(grads[0]))
            return in_torch("route", [&] {
                return pybind11::make_tuple(grads[0], weights, chosen, or_none(logits), experts, normalize,
                                            pybind11::reinterpret_borrow<pybind11::object>((PyObject*)torch::getTHPDtype(type)));
            }, 3);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), w = weights.contiguous(), c = chosen.contiguous(), l = normalize ? Tensor() : logits.contiguous();
        const int64_t tokens = sizes[0], top_k = sizes[1];
        out[0] = fresh({tokens, experts}, type, g);
        const On on(g);
        check(api.route_backward(w.const_data_ptr<float>(), c.const_data_ptr<int32_t>(), g.const_data_ptr<float>(), address(l),
                                 code(type), tokens, experts, top_k, normalize, place(out[0])), "adambridge_route_backward");
        return out;
    }
};

// route(logits, top_k, normalize): a tuple
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 3 || !connected || observed()) Py_RETURN_NONE;
    const Tensor* logits = plain(args[0]);
    if (!values(logits, 2) || !PyLong_CheckExact(args[1]) || !PyBool_Check(args[2])) Py_RETURN_NONE;
    const int64_t top_k = PyLong_AsLongLong(args[1]);
    if (top_k == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (api.route_work(logits->size(0), logits->size(1), top_k) < 0) Py_RETURN_NONE;   // sizes out of the kernels' range
    tensor_list out;
    if (wants_grad({logits})) {
        out = Route::apply(*logits, top_k, args[2] == Py_True);
    } else {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = route_forward(*logits, top_k, args[2] == Py_True);
    }
    PyObject* tuple = PyTuple_New(5);
    if (!tuple) return nullptr;
    for (Py_ssize_t i = 0; i < 5; ++i) PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap(out[(size_t)i]));
    return tuple;
    END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------------- dispatch and combine

// A position that fits tokens x top_k rows of cols values.
bool position_ok(const Tensor* position, const Tensor* x, int64_t tokens, int64_t cols)
{
    return beside(position, x, at::kInt) && position->dim() == 2 && position->size(0) == tokens && tokens > 0 && position->size(1) >= 1 &&
           position->size(1) <= 64 && position->numel() < (int64_t)1 << 31 && cols <= (int64_t)1 << 22;
}

Tensor run_dispatch(const Tensor& x, const Tensor& position)
{
    const int64_t tokens = x.size(0), cols = x.size(1), top_k = position.size(1);
    Tensor rows = fresh({tokens * top_k, cols}, x.scalar_type(), x);
    const On on(x);
    check(api.dispatch(address(x), code(x.scalar_type()), position.const_data_ptr<int32_t>(), tokens, top_k, cols, place(rows)), "adambridge_dispatch");
    return rows;
}

Tensor run_combine(const Tensor& rows, const Tensor& weights, const Tensor& position)
{
    const int64_t tokens = position.size(0), cols = rows.size(1), top_k = position.size(1);
    Tensor out = fresh({tokens, cols}, rows.scalar_type(), rows);
    const On on(rows);
    check(api.combine(address(rows), code(rows.scalar_type()), weights.defined() ? weights.const_data_ptr<float>() : nullptr,
                      position.const_data_ptr<int32_t>(), tokens, top_k, cols, place(out)), "adambridge_combine");
    return out;
}

struct Dispatch : Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({position});
        ctx->saved_data["top_k"] = position.size(1);
        return run_dispatch(x, position);
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const int64_t top_k = ctx->saved_data["top_k"].toInt();
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const bool whole = !sizes.empty() && restored(saved[0], grads[0], at::kInt, {sizes[0] / top_k, top_k});
        if (!whole || !plain_backward(grads[0]))
            return in_torch("dispatch", [&] { return pybind11::make_tuple(grads[0], saved[0]); }, 2);
        const at::AutoDispatchBelowADInplaceOrView below;
        return {run_combine(grads[0].contiguous(), Tensor(), saved[0].contiguous()), Tensor()};
    }
};

struct Combine : Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& position)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({weights.requires_grad() ? rows : Tensor(), weights, position});
        ctx->saved_data["top_k"] = position.size(1);
        return run_combine(rows, weights, position);
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor &rows = saved[0], &weights = saved[1], &position = saved[2];
        const bool want_rows = ctx->needs_input_grad(0), want_weights = ctx->needs_input_grad(1);
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const int64_t tokens = sizes.empty() ? 0 : sizes[0], cols = sizes.empty() ? 0 : sizes[1], top_k = ctx->saved_data["top_k"].toInt();
        const bool whole = tokens && restored(weights, grads[0], at::kFloat, {tokens, top_k}) & restored(position, grads[0], at::kInt, {tokens, top_k}) &
                                         (!want_weights || restored(rows, grads[0], grads[0].scalar_type(), {tokens * top_k, cols}));
        if (!whole || !plain_backward(grads[0]))
            return in_torch("combine", [&] {
                return pybind11::make_tuple(grads[0], or_none(rows), weights, position, want_rows, want_weights);
            }, 3);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), r = want_weights ? rows.contiguous() : Tensor(), w = weights.contiguous(), p = position.contiguous();
        tensor_list out(3);
        if (want_rows) out[0] = fresh({tokens * top_k, cols}, g.scalar_type(), g);
        if (want_weights) out[1] = fresh({tokens, top_k}, at::kFloat, g);
        const On on(g);
        check(api.combine_backward(address(g), address(r), code(g.scalar_type()), w.const_data_ptr<float>(),
                                   p.const_data_ptr<int32_t>(), tokens, top_k, cols, place(out[0]),
                                   out[1].defined() ? out[1].mutable_data_ptr<float>() : nullptr), "adambridge_combine_backward");
        return out;
    }
};

// dispatch(x, position)
PyObject* dispatch(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 2 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *x = plain(args[0]), *position = plain(args[1]);
    if (!values(x, 2) || !position_ok(position, x, x->size(0), x->size(1))) Py_RETURN_NONE;
    if (wants_grad({x})) return THPVariable_Wrap(Dispatch::apply(*x, *position));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(run_dispatch(*x, *position));
    END_HANDLE_TH_ERRORS
}

// combine(rows, weights, position)
PyObject* combine(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 3 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *rows = plain(args[0]), *weights = plain(args[1]), *position = plain(args[2]);
    if (!values(rows, 2) || !beside(weights, rows, at::kFloat) || weights->dim() != 2) Py_RETURN_NONE;
    if (!position_ok(position, rows, weights->size(0), rows->size(1)) || position->size(1) != weights->size(1) ||
        rows->size(0) != position->numel())
        Py_RETURN_NONE;
    if (wants_grad({rows, weights})) return THPVariable_Wrap(Combine::apply(*rows, *weights, *position));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(run_combine(*rows, *weights, *position));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------- expert_mm

Tensor run_experts(int32_t product, const Tensor& a, const Tensor& b, const Tensor& ends, at::IntArrayRef sizes, int64_t n, int64_t k)
{
    const int64_t rows = a.size(0), experts = ends.size(0);
    const int32_t type = code(a.scalar_type());
    const int64_t bytes = api.expert_mm_work(product, type, rows, experts, n, k);
    check(bytes, "adambridge_expert_mm_work");
    Tensor out = fresh(sizes, a.scalar_type(), a), work = scratch(bytes, a);
    const On on(a);
    const auto fn = product == ADAMBRIDGE_EXPERTS_Y ? api.expert_mm : product == ADAMBRIDGE_EXPERTS_DX ? api.expert_mm_dx : api.expert_mm_dw;
    check(fn(address(a), address(b), ends.const_data_ptr<int32_t>(), place(out), type, rows, experts, n, k, place(work)), "adambridge_expert_mm");
    return out;
}

struct ExpertMM : Function<ExpertMM> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& ends)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({weight.requires_grad() ? x : Tensor(), weight, ends});
        ctx->saved_data["of"] = (int64_t)(weight.size(0) | weight.size(2) << 16);
        return run_experts(ADAMBRIDGE_EXPERTS_Y, x, weight, ends, {x.size(0), weight.size(1)}, weight.size(1), weight.size(2));
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &ends = saved[2];
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const int64_t of = ctx->saved_data["of"].toInt(), experts = of & 0xffff, k = of >> 16;
        const int64_t rows = sizes.empty() ? 0 : sizes[0], n = sizes.empty() ? 0 : sizes[1];
        const at::ScalarType type = grads[0].scalar_type();
        const bool whole = n && restored(weight, grads[0], type, {experts, n, k}) & restored(ends, grads[0], at::kInt, {experts}) &
                                    (!want_w || restored(x, grads[0], type, {rows, k}));
        if (!whole || !plain_backward(grads[0]))
            return in_torch("expert_mm", [&] {
                return pybind11::make_tuple(grads[0], or_none(x), weight, ends, want_x, want_w);
            }, 3);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), e = ends.contiguous();
        tensor_list out(3);
        if (want_x) out[0] = run_experts(ADAMBRIDGE_EXPERTS_DX, g, weight.contiguous(), e, {rows, k}, n, k);
        if (want_w) out[1] = run_experts(ADAMBRIDGE_EXPERTS_DW, g, x.contiguous(), e, {experts, n, k}, n, k);
        return out;
    }
};

// expert_mm(x, weight, ends)
PyObject* expert_mm(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 3 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *x = plain(args[0]), *weight = plain(args[1]), *ends = plain(args[2]);
    if (!x || !type_ok(x->scalar_type()) || x->dim() != 2 || !weight || weight->dim() != 3 || !beside(weight, x, x->scalar_type()) ||
        weight->numel() == 0 || weight->size(2) != x->size(1))
        Py_RETURN_NONE;
    constexpr int64_t most = (int64_t)1 << 22;
    if (!beside(ends, x, at::kInt) || ends->dim() != 1 || ends->size(0) != weight->size(0) || x->size(0) > (int64_t)1 << 30 ||
        weight->size(0) > 4096 || weight->size(1) > most || weight->size(2) > most || at::autocast::is_autocast_enabled(at::kCUDA))
        Py_RETURN_NONE;
    if (wants_grad({x, weight})) return THPVariable_Wrap(ExpertMM::apply(*x, *weight, *ends));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(run_experts(ADAMBRIDGE_EXPERTS_Y, *x, *weight, *ends, {x->size(0), weight->size(1)},
                                        weight->size(1), weight->size(2)));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------ expert_mlp

// expert_mlp(x, logits, up, down, gate or None, top_k, silu, normalize), of a few tokens without gradients
PyObject* expert_mlp(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 8 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *x = plain(args[0]), *logits = plain(args[1]), *up = plain(args[2]), *down = plain(args[3]), *gate;
    if (!plain_or_none(args[4], gate) || !values(x, 2) || !values(logits, 2) || logits->device() != x->device() || !values(up, 3)) Py_RETURN_NONE;
    if (!beside(up, x, x->scalar_type()) || !beside(down, x, x->scalar_type()) || (gate && !beside(gate, x, x->scalar_type()))) Py_RETURN_NONE;
    if (!PyLong_CheckExact(args[5]) || !PyBool_Check(args[6]) || !PyBool_Check(args[7]) || at::autocast::is_autocast_enabled(at::kCUDA)) Py_RETURN_NONE;
    const int64_t tokens = x->size(0), hidden = x->size(1), experts = up->size(0), inter = up->size(1);
    if (logits->size(0) != tokens || logits->size(1) != experts || up->size(2) != hidden || (gate && gate->sizes() != up->sizes()) ||
        down->sizes() != at::IntArrayRef({experts, hidden, inter}) || wants_grad({x, logits, up, down, gate}))
        Py_RETURN_NONE;
    const int64_t top_k = PyLong_AsLongLong(args[5]);
    if (top_k == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const int32_t type = code(x->scalar_type());
    const int64_t bytes = api.expert_mlp_work(type, tokens, experts, top_k, inter, hidden);
    if (bytes < 0) Py_RETURN_NONE;   // more than a few tokens, or sizes out of the kernels' range
    const at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = fresh({tokens, hidden}, x->scalar_type(), *x), work = scratch(bytes, *x);
    {
        const On on(*x);
        check(api.expert_mlp(address(*x), address(*logits), code(logits->scalar_type()), address(*up), gate ? address(*gate) : nullptr, address(*down),
                             type, tokens, experts, top_k, inter, hidden, args[6] == Py_True ? ADAMBRIDGE_SILU : ADAMBRIDGE_GELU, args[7] == Py_True,
                             place(out), place(work)), "adambridge_expert_mlp");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------------------------- embed

Tensor embed_forward(const Tensor& ids, const Tensor& weight, double scale)
{
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(weight.size(1));
    Tensor y = fresh(sizes, weight.scalar_type(), weight);
    const On on(weight);
    check(api.embed(address(ids), (int32_t)ids.element_size(), ids.numel(), address(weight), code(weight.scalar_type()), weight.size(0),
                    weight.size(1), (float)scale, place(y)), "adambridge_embed");
    return y;
}

struct Embed : Function<Embed> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({ids});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["vocab"] = weight.size(0);
        ctx->saved_data["type"] = (int64_t)ids.scalar_type();
        return embed_forward(ids, weight, scale);
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor& ids = saved[0];
        const double scale = ctx->saved_data["scale"].toDouble();
        const int64_t padding = ctx->saved_data["padding"].toInt(), vocab = ctx->saved_data["vocab"].toInt();
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const bool whole = !sizes.empty() && restored(ids, grads[0], (at::ScalarType)ctx->saved_data["type"].toInt(), sizes.slice(0, sizes.size() - 1));
        if (!whole || !plain_backward(grads[0]))
            return in_torch("embed", [&] {
                return pybind11::make_tuple(grads[0], ids, vocab, scale,
                                            padding < 0 ? pybind11::object(pybind11::none()) : pybind11::object(pybind11::int_(padding)));
            }, 4);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), i = ids.contiguous();
        const int64_t tokens = i.numel(), hidden = sizes.back();
        const int64_t bytes = api.embed_work(tokens, vocab, hidden);
        check(bytes, "adambridge_embed_work");
        tensor_list out(4);
        out[1] = fresh({vocab, hidden}, g.scalar_type(), g);
        Tensor work = scratch(bytes, g);
        const On on(g);
        check(api.embed_backward(address(i), (int32_t)i.element_size(), tokens, address(g), code(g.scalar_type()), vocab, hidden, (float)scale,
                                 padding, place(out[1]), place(work)), "adambridge_embed_backward");
        return out;
    }
};

// embed(ids, weight, scale, padding_idx or None)
PyObject* embed(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 4 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *ids = plain(args[0]), *weight = plain(args[1]);
    if (!values(weight, 2) || !ids || ids->device() != weight->device() || !PyFloat_CheckExact(args[2])) Py_RETURN_NONE;
    if ((ids->scalar_type() != at::kLong && ids->scalar_type() != at::kInt) || (args[3] != Py_None && !PyLong_CheckExact(args[3]))) Py_RETURN_NONE;
    int64_t padding = -1;
    if (args[3] != Py_None) {
        padding = PyLong_AsLongLong(args[3]);
        if (padding == -1 && PyErr_Occurred()) PyErr_Clear();
        if (padding < 0 || padding >= weight->size(0)) Py_RETURN_NONE;
    }
    if (api.embed_work(ids->numel(), weight->size(0), weight->size(1)) < 0) Py_RETURN_NONE;   // sizes out of the kernels' range
    const double scale = PyFloat_AS_DOUBLE(args[2]);
    if (wants_grad({weight})) return THPVariable_Wrap(Embed::apply(*ids, *weight, scale, padding));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(embed_forward(*ids, *weight, scale));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------- token losses

Tensor losses_forward(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore, Tensor* stats)
{
    const int64_t rows = targets.numel(), vocab = weight.size(0), size = weight.size(1);
    const int32_t type = code(hidden.scalar_type());
    const int64_t bytes = api.token_losses_work(type, rows, vocab, size);
    check(bytes, "adambridge_token_losses_work");
    Tensor losses = fresh(targets.sizes(), at::kFloat, hidden), work = scratch(bytes, hidden);
    if (stats) *stats = fresh({rows, 2}, at::kFloat, hidden);
    const On on(hidden);
    check(api.token_losses(address(hidden), address(weight), type, targets.const_data_ptr<int64_t>(), rows, vocab, size, ignore,
                           losses.mutable_data_ptr<float>(), stats ? stats->mutable_data_ptr<float>() : nullptr, place(work)),
          "adambridge_token_losses");
    return losses;
}

struct TokenLosses : Function<TokenLosses> {
    static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        Tensor stats;
        Tensor losses = losses_forward(hidden, weight, targets, ignore, &stats);
        ctx->save_for_backward({hidden, weight, targets, stats});
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["vocab"] = weight.size(0);
        ctx->saved_data["size"] = weight.size(1);
        ctx->saved_data["type"] = (int64_t)hidden.scalar_type();
        return losses;
    }
    static tensor_list backward(AutogradContext* ctx, const tensor_list& grads)
    {
        const tensor_list saved = ctx->get_saved_variables();
        const Tensor &hidden = saved[0], &weight = saved[1], &targets = saved[2], &stats = saved[3];
        const int64_t ignore = ctx->saved_data["ignore"].toInt(), vocab = ctx->saved_data["vocab"].toInt(), size = ctx->saved_data["size"].toInt();
        const at::ScalarType type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const bool numbers = !grads[0].unsafeGetTensorImpl()->has_symbolic_sizes_strides();
        const at::IntArrayRef sizes = sizes_of(grads[0]);
        const int64_t rows = numbers ? grads[0].numel() : 0;
        std::vector<int64_t> with_size = sizes.vec();
        with_size.push_back(size);
        const bool whole = numbers && restored(hidden, grads[0], type, with_size) & restored(weight, grads[0], type, {vocab, size}) &
                                          restored(targets, grads[0], at::kLong, sizes) & restored(stats, grads[0], at::kFloat, {rows, 2});
        if (!whole || !plain_backward(grads[0]))
            return in_torch("token_losses", [&] {
                return pybind11::make_tuple(grads[0], hidden, weight, targets, ignore, want_h, want_w);
            }, 4);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].contiguous(), h = hidden.contiguous(), w = weight.contiguous(), t = targets.contiguous(), s = stats.contiguous();
        const int64_t bytes = api.token_losses_backward_work(code(type), rows, vocab, size);
        check(bytes, "adambridge_token_losses_backward_work");
        tensor_list out(4);
        if (want_h) out[0] = fresh(with_size, type, g);
        if (want_w) out[1] = fresh({vocab, size}, type, g);
        Tensor work = scratch(bytes, g);
        const On on(g);
        check(api.token_losses_backward(g.const_data_ptr<float>(), address(h), address(w), code(type), t.const_data_ptr<int64_t>(), rows, vocab,
                                        size, ignore, s.const_data_ptr<float>(), place(out[0]), place(out[1]), place(work)),
              "adambridge_token_losses_backward");
        return out;
    }
};

// token_losses(hidden, weight, targets, ignore_index)
PyObject* token_losses(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 4 || !connected || observed()) Py_RETURN_NONE;
    const Tensor *hidden = plain(args[0]), *weight = plain(args[1]), *targets = plain(args[2]);
    if (!values(weight, 2) || !hidden || hidden->dim() < 1 || !beside(hidden, weight, weight->scalar_type()) || !beside(targets, weight, at::kLong) ||
        !PyLong_CheckExact(args[3]) || at::autocast::is_autocast_enabled(at::kCUDA))
        Py_RETURN_NONE;
    if (hidden->size(-1) != weight->size(1) || targets->sizes() != hidden->sizes().slice(0, hidden->dim() - 1)) Py_RETURN_NONE;
    const int64_t ignore = PyLong_AsLongLong(args[3]);
    if (ignore == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (api.token_losses_work(code(weight->scalar_type()), targets->numel(), weight->size(0), weight->size(1)) < 0)
        Py_RETURN_NONE;   // sizes out of the kernels' range
    if (wants_grad({hidden, weight})) return THPVariable_Wrap(TokenLosses::apply(*hidden, *weight, *targets, ignore));
    const at::AutoDispatchBelowADInplaceOrView below;
    return THPVariable_Wrap(losses_forward(*hidden, *weight, *targets, ignore, nullptr));
    END_HANDLE_TH_ERRORS
}

// --------------------------------------------------------------------------------- connect

// connect(addresses by entry point, backward passes in torch operations by operator, the class of default devices' modes)
PyObject* connect(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    if (nargs != 3 || !PyDict_CheckExact(args[0]) || !PyDict_CheckExact(args[1]) || !PyType_Check(args[2])) {
        PyErr_SetString(PyExc_TypeError, "connect(addresses, backward passes, class of default devices' modes)");
        return nullptr;
    }
    Api found;
    const struct { void* at; const char* name; } entries[] = {
        {&found.set_stream, "adambridge_set_stream"}, {&found.last_error, "adambridge_last_error"},
        {&found.layer_norm, "adambridge_layer_norm"}, {&found.layer_norm_work, "adambridge_layer_norm_work"},
        {&found.layer_norm_backward, "adambridge_layer_norm_backward"}, {&found.route_work, "adambridge_route_work"},
        {&found.route, "adambridge_route"}, {&found.route_backward, "adambridge_route_backward"},
        {&found.dispatch, "adambridge_dispatch"}, {&found.combine, "adambridge_combine"},
        {&found.combine_backward, "adambridge_combine_backward"}, {&found.expert_mm, "adambridge_expert_mm"},
        {&found.expert_mm_dx, "adambridge_expert_mm_dx"}, {&found.expert_mm_work, "adambridge_expert_mm_work"},
        {&found.expert_mm_dw, "adambridge_expert_mm_dw"}, {&found.embed, "adambridge_embed"},
        {&found.embed_work, "adambridge_embed_work"}, {&found.embed_backward, "adambridge_embed_backward"},
        {&found.token_losses, "adambridge_token_losses"}, {&found.token_losses_work, "adambridge_token_losses_work"},
        {&found.token_losses_backward, "adambridge_token_losses_backward"},
        {&found.token_losses_backward_work, "adambridge_token_losses_backward_work"},
        {&found.expert_mlp_work, "adambridge_expert_mlp_work"}, {&found.expert_mlp, "adambridge_expert_mlp"}};
    for (const auto& e : entries) {
        PyObject* o = PyDict_GetItemString(args[0], e.name);
        void* const p = o ? PyLong_AsVoidPtr(o) : nullptr;
        if (!p) {
            if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "connect: no %s", e.name);
            return nullptr;
        }
        std::memcpy(e.at, &p, sizeof p);
    }
    Py_INCREF(args[1]);
    Py_XSETREF(twice, args[1]);
    Py_INCREF(args[2]);
    Py_XSETREF(placing, args[2]);
    api = found;
    connected = true;
    Py_RETURN_NONE;
}

#define ABH_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef kMethods[] = {
    {"connect", ABH_FAST(connect), "The library's entry points, and the backward passes in torch operations."},
    {"layer_norm", ABH_FAST(layer_norm), "layer_norm(x, weight, bias, eps); None if the call is not an ordinary one."},
    {"route", ABH_FAST(route), "route(logits, top_k, normalize), a tuple; None if the call is not an ordinary one."},
    {"dispatch", ABH_FAST(dispatch), "dispatch(x, position); None if the call is not an ordinary one."},
    {"combine", ABH_FAST(combine), "combine(rows, weights, position); None if the call is not an ordinary one."},
    {"expert_mm", ABH_FAST(expert_mm), "expert_mm(x, weight, ends); None if the call is not an ordinary one."},
    {"expert_mlp", ABH_FAST(expert_mlp), "expert_mlp(x, logits, up, down, gate, top_k, silu, normalize); None if the call is not an ordinary one."},
    {"embed", ABH_FAST(embed), "embed(ids, weight, scale, padding_idx); None if the call is not an ordinary one."},
    {"token_losses", ABH_FAST(token_losses), "token_losses(hidden, weight, targets, ignore_index); None if the call is not an ordinary one."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ops", "The host's side of an expert block's operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&kModule); }
