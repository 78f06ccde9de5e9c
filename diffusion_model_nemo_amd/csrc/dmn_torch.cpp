// torch side of the trained-block operators: argument checks, outputs and workspaces from torch's allocator, autograd nodes,
// and the walk over a parameter list, around the C-ABI's entry points (include/dmn.h), whose addresses `bind` receives from
// the library that Python has loaded. Compiled, because these calls are small: a training call of a narrow layer norm spent
// 105 us in Python's side of autograd and 25 us on the GPU. Host code only; streams arrive as handles.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/StreamGuard.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cstring>
#include <unordered_set>
#include <vector>

#include "../../include/dmn.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&dmn_last_error) last_error;
    decltype(&dmn_layer_norm_forward) ln_forward;
    decltype(&dmn_layer_norm_workspace_bytes) ln_workspace;
    decltype(&dmn_layer_norm_backward) ln_backward;
    decltype(&dmn_linear_forward_workspace_bytes) linear_forward_workspace;
    decltype(&dmn_linear_forward) linear_forward;
    decltype(&dmn_linear_backward_workspace_bytes) linear_backward_workspace;
    decltype(&dmn_linear_backward) linear_backward;
    decltype(&dmn_clip_grads_workspace_bytes) clip_workspace;
    decltype(&dmn_clip_grads) clip;
    decltype(&dmn_stream_is_capturing) is_capturing;
} api;
PyObject* error_class = nullptr;     // DmnError
PyObject* current_stream = nullptr;  // device index -> stream handle

constexpr size_t kEntries = sizeof(Api) / sizeof(void*);
void bind(const std::vector<uintptr_t>& entries, py::object error, py::object stream) {
    if (entries.size() != kEntries) throw py::value_error("wrong number of entry points");
    memcpy(&api, entries.data(), sizeof(api));
    error_class = error.release().ptr();
    current_stream = stream.release().ptr();
}

std::string failure(int rc) { return c10::str("libdmn_hip error ", rc, ": ", api.last_error()); }
void check(int rc) {
    if (rc == 0) return;
    const std::string text = failure(rc);
    py::gil_scoped_acquire gil;
    PyErr_SetString(error_class, text.c_str());
    throw py::error_already_set();
}
void check_backward(int rc) {   // on a thread of the autograd engine
    if (rc != 0) throw std::runtime_error(failure(rc));
}

int code_of(at::ScalarType t) { return t == at::kFloat ? DMN_DT_F32 : t == at::kBFloat16 ? DMN_DT_BF16 : t == at::kHalf ? DMN_DT_F16 : -1; }

void check_input(const Tensor& x, const char* what) {
    if (!x.is_cuda()) throw std::runtime_error(c10::str(what, " runs only on MI355X device tensors (no CPU implementation)"));
    if (code_of(x.scalar_type()) < 0 || x.layout() != at::kStrided)
        throw py::value_error(c10::str(what, ": dtype must be float32, bfloat16 or float16, got ", x.scalar_type(), " (", x.layout(), ")"));
}
// Only the reverse-mode nodes below know what the kernels compute. A dual tensor would come out without its tangent, which
// reads as a derivative of zero, and a trace would hold the allocation of the output and nothing else: both are refused.
void check_recorded(const char* what, std::initializer_list<const std::optional<Tensor>*> inputs) {
    if (torch::jit::tracer::isTracing()) throw std::runtime_error(c10::str(what, " cannot be traced: its kernels are not torch operators"));
    for (const auto* t : inputs)
        if (t->has_value() && (*t)->_fw_grad(0).defined())
            throw std::runtime_error(c10::str(what, " has no forward-mode derivative: an input is a dual tensor"));
}
// Contiguous, with the values that are in memory: a view with the negation bit (the imaginary part of a conjugate) is copied.
Tensor dense(const Tensor& t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }
// p on x's device, of `shape` and of x's type (or float32 where `or_float`); comes back contiguous
Tensor checked_param(const std::optional<Tensor>& p, const char* name, at::IntArrayRef shape, const Tensor& x, bool or_float, bool rows = false) {
    if (!p.has_value()) return Tensor();
    if (p->device() != x.device()) throw std::runtime_error(c10::str(name, " on ", p->device(), ", input on ", x.device()));
    if (p->sizes() != shape) throw py::value_error(c10::str(name, " must have shape ", shape, ", got ", p->sizes()));
    if (p->scalar_type() != x.scalar_type() && !(or_float && p->scalar_type() == at::kFloat))
        throw py::value_error(c10::str(name, " must be ", x.scalar_type(), or_float ? " or Float" : "", ", got ", p->scalar_type()));
    return rows ? *p : dense(*p);
}

// `t` as rows of contiguous elements `ld` apart, copied only where its strides do not allow that.
struct Rows {
    Tensor t;
    int64_t ld;
};
Rows rows_of(const Tensor& t, int64_t limit = INT64_MAX) {   // strides from `limit` on are copied too
    const int64_t width = t.size(-1);
    if (t.is_neg()) return {dense(t), width};
    if (t.is_contiguous()) return {t, width};
    if (t.dim() == 2 && (t.stride(1) == 1 || width == 1) && t.stride(0) >= width && t.stride(0) < limit) return {t, t.stride(0)};
    return {t.contiguous(), width};
}
constexpr int64_t kLinearStride = 1 << 20;   // dmn_linear_*: strides below it
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* handle(int64_t stream) { return (void*)(uintptr_t)stream; }

// Gradients that carry a graph of their own (create_graph) must not be differentiated again: the kernels are not recorded.
variable_list once_differentiable(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (auto& g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_(true));
    auto node = std::make_shared<torch::autograd::DelayedError>("the backward pass of this operator is not differentiable", (int64_t)some.size());
    some = (*node)(std::move(some));
    size_t i = 0;
    for (auto& g : grads)
        if (g.defined()) g = some[i++];
    return grads;
}

int64_t stream_handle(c10::DeviceIndex device) {   // of its current stream; with the GIL held
    const py::object h = py::reinterpret_steal<py::object>(PyObject_CallFunction(current_stream, "i", (int)device));
    if (!h) throw py::error_already_set();
    return h.cast<int64_t>();
}
bool is_capturing(const c10::Stream& s) {
    c10::StreamGuard guard(s);
    py::gil_scoped_acquire gil;
    return api.is_capturing(handle(stream_handle(s.device_index()))) != 0;
}

// Under capture the gradients of a leaf would be accumulated on the stream on which an eager graph that still lives first
// used the leaf; torch then touches that stream in the middle of the capture, and the process ends. The same holds for any node of
// an eager graph that the backward would pass through. Such a call is refused, however far behind the inputs (views, transposes,
// copies) the node lies; a stream that was forked into the same capture is none of these. `pass`: the nodes that the
// backward will run (null: all).
using ExecInfo = std::unordered_map<torch::autograd::Node*, torch::autograd::GraphTask::ExecInfo>;
void check_nodes(std::vector<std::shared_ptr<torch::autograd::Node>> todo, const c10::Device& device, const ExecInfo* pass) {
    const c10::Stream now = c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getStream(device);
    std::unordered_set<torch::autograd::Node*> seen;
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        if (pass && !pass->empty()) {
            const auto it = pass->find(node.get());
            if (it == pass->end() || !it->second.should_execute()) continue;
        }
        const auto stream = node->stream();
        if (stream.has_value() && *stream != now && !is_capturing(*stream))
            throw std::runtime_error("a graph is being captured while an eager graph over the same parameters or inputs, made on another stream, "
                                     "still lives: drop its results first (del loss, outputs), or warm up on the capturing stream");
        for (const auto& edge : node->next_edges()) todo.push_back(edge.function);
    }
}
void check_capture(int64_t stream, const Tensor& x, std::initializer_list<const Tensor*> inputs) {
    if (!api.is_capturing(handle(stream))) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> nodes;
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) nodes.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    check_nodes(std::move(nodes), x.device(), nullptr);
}
// The same for a backward pass that is captured while its forward was not (made eagerly on the capturing stream): asked before
// the gradients are handed on.
void check_captured_backward(int64_t stream, const c10::Device& device) {
    if (!api.is_capturing(handle(stream))) return;
    const auto self = torch::autograd::get_current_node();
    if (!self) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> nodes;
    for (const auto& edge : self->next_edges()) nodes.push_back(edge.function);
    check_nodes(std::move(nodes), device, torch::autograd::get_current_graph_task_exec_info());
}

// ---- layer norm --------------------------------------------------------------------------------------------------------

int affine_code(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    return code_of(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type());
}

Tensor layer_norm_run(const Rows& x, const Tensor& weight, const Tensor& bias, double eps, int64_t stream, Tensor* stats) {
    const int64_t width = x.t.size(-1), rows = x.t.numel() / width;
    Tensor y = new_like(x.t);
    if (stats) *stats = at::empty({rows, 2}, x.t.options().dtype(at::kFloat));
    check(api.ln_forward(x.t.data_ptr(), x.ld, ptr(weight), ptr(bias), y.data_ptr(), stats ? (float*)stats->data_ptr() : nullptr, rows, (int)width,
                         code_of(x.t.scalar_type()), affine_code(x.t, weight, bias), (float)eps, handle(stream)));
    return y;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps,
                          int64_t stream) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_);
        const Rows r = rows_of(x);
        Tensor stats;
        Tensor y = layer_norm_run(r, weight, bias, eps, stream, &stats);
        ctx->save_for_backward({r.t, weight, bias, stats});
        ctx->saved_data["stream"] = stream;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        {
            at::AutoGradMode off(false);
            const auto saved = ctx->get_saved_variables();
            const Rows x = rows_of(saved[0]), dy = rows_of(grads[0]);
            const Tensor &weight = saved[1], &bias = saved[2], &stats = saved[3];
            c10::DeviceGuard guard(x.t.device());
            check_captured_backward(ctx->saved_data["stream"].toInt(), x.t.device());
            const int64_t width = x.t.size(-1), rows = stats.size(0);
            const int code = code_of(x.t.scalar_type());
            size_t edge = 0;   // the node has an edge for every tensor that was given
            if (ctx->needs_input_grad(edge++)) out[0] = new_like(x.t);
            if (weight.defined() && ctx->needs_input_grad(edge++)) out[1] = new_like(weight);
            if (bias.defined() && ctx->needs_input_grad(edge++)) out[2] = new_like(bias);
            const size_t bytes = out[1].defined() || out[2].defined() ? api.ln_workspace(rows, (int)width, code) : 0;
            const Tensor ws = workspace(bytes, x.t);
            check_backward(api.ln_backward(dy.t.data_ptr(), dy.ld, x.t.data_ptr(), x.ld, ptr(weight), (const float*)stats.data_ptr(), ptr(out[0]),
                                           ptr(out[1]), ptr(out[2]), rows, (int)width, code, affine_code(x.t, weight, bias), ptr(ws), bytes,
                                           handle(ctx->saved_data["stream"].toInt())));
        }
        return once_differentiable(std::move(out));
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps, int64_t stream) {
    const std::optional<Tensor> x_(x);
    check_recorded("layer_norm", {&x_, &weight_, &bias_});
    check_input(x, "layer_norm");
    if (x.dim() == 0 || x.size(-1) == 0) throw py::value_error("layer_norm needs a last axis of at least one element");
    if (x.size(-1) > INT32_MAX) throw py::value_error("layer_norm: the last axis is too long");
    if (!(eps >= 0.0)) throw py::value_error(c10::str("eps must be >= 0, got ", eps));
    const at::IntArrayRef shape = x.sizes().slice(x.dim() - 1);
    Tensor weight = checked_param(weight_, "weight", shape, x, true), bias = checked_param(bias_, "bias", shape, x, true);
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
        throw py::value_error(c10::str("weight and bias must have one type, got ", weight.scalar_type(), " and ", bias.scalar_type()));
    c10::DeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()))) {
        check_capture(stream, x, {&x, &weight, &bias});
        return LayerNormNode::apply(x, given(weight), given(bias), eps, stream);
    }
    return layer_norm_run(rows_of(x), weight, bias, eps, stream, nullptr);
}

// ---- linear layer ------------------------------------------------------------------------------------------------------

Tensor linear_run(const Rows& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act, int64_t stream, Tensor* z) {
    const int64_t out = weight.size(0), width = weight.size(1), rows = x.t.numel() / width;
    const int code = code_of(x.t.scalar_type());
    auto shape = x.t.sizes().vec();
    shape.back() = out;
    Tensor y = at::empty(shape, x.t.options());
    if (z) *z = at::empty({rows, out}, act & DMN_LINEAR_EXACT ? x.t.options().dtype(at::kFloat) : x.t.options());
    const Rows r = residual.defined() ? rows_of(residual) : Rows{Tensor(), 0};
    const size_t bytes = api.linear_forward_workspace(x.t.data_ptr(), x.ld, weight.data_ptr(), rows, (int)width, (int)out, code);
    const Tensor ws = workspace(bytes, x.t);
    check(api.linear_forward(x.t.data_ptr(), x.ld, weight.data_ptr(), ptr(bias), ptr(r.t), r.ld, y.data_ptr(), z ? z->data_ptr() : nullptr, rows,
                             (int)width, (int)out, (int)act, code, ptr(ws), bytes, handle(stream)));
    return y;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_,
                          const std::optional<Tensor>& residual, int64_t act, int64_t stream) {
        const Tensor bias = or_none(bias_);
        const Rows r = rows_of(x, kLinearStride);
        // the value in front of the activation is all that the backward needs of the forward's results
        const bool want_z = (act & ~DMN_LINEAR_EXACT) != 0 && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()));
        Tensor z;
        Tensor y = linear_run(r, weight, bias, or_none(residual), act, stream, want_z ? &z : nullptr);
        // x for dW and the weight for dx alone: what is not needed is not kept, and may be overwritten before the backward
        ctx->save_for_backward({weight.requires_grad() ? r.t : Tensor(), x.requires_grad() ? weight : Tensor(), z});
        ctx->saved_data["x"] = x.sizes();
        ctx->saved_data["weight"] = weight.sizes();
        ctx->saved_data["act"] = act;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(6);
        {
            at::AutoGradMode off(false);
            const auto saved = ctx->get_saved_variables();
            const Tensor &weight = saved[1], &z = saved[2];
            const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
            const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
            check_captured_backward(ctx->saved_data["stream"].toInt(), grads[0].device());
            if (need_x || need_w || need_b) {
                const auto w_shape = ctx->saved_data["weight"].toIntVector();
                const int64_t n = w_shape[0], width = w_shape[1], rows = grads[0].numel() / n, act = ctx->saved_data["act"].toInt();
                const Rows x = need_w ? rows_of(saved[0], kLinearStride) : Rows{Tensor(), width}, dy = rows_of(grads[0], kLinearStride);
                c10::DeviceGuard guard(dy.t.device());
                const int code = code_of(dy.t.scalar_type());
                if (need_x) out[0] = at::empty(ctx->saved_data["x"].toIntVector(), dy.t.options());
                if (need_w) out[1] = at::empty(w_shape, dy.t.options());
                if (need_b) out[2] = at::empty({n}, dy.t.options());
                const size_t bytes = api.linear_backward_workspace(dy.t.data_ptr(), dy.ld, ptr(x.t), x.ld, ptr(weight), rows, (int)width, (int)n,
                                                                   (int)act, code);
                const Tensor ws = workspace(bytes, dy.t);
                check_backward(api.linear_backward(dy.t.data_ptr(), dy.ld, ptr(x.t), x.ld, ptr(weight), ptr(z), ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                                   rows, (int)width, (int)n, (int)act, code, ptr(ws), bytes,
                                                   handle(ctx->saved_data["stream"].toInt())));
            }
        }
        out = once_differentiable(std::move(out));
        // the residual's gradient is the incoming one; its edge stands behind those of x, weight and, if given, bias
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(ctx->saved_data["bias"].toBool() ? 3 : 2)) out[3] = grads[0];
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& weight_, const std::optional<Tensor>& bias_, int64_t act, const std::optional<Tensor>& residual_,
              int64_t stream) {
    const std::optional<Tensor> x_(x), w_(weight_);
    check_recorded("linear", {&x_, &w_, &bias_, &residual_});
    check_input(x, "linear");
    if (weight_.dim() != 2 || weight_.size(0) == 0 || weight_.size(1) == 0 || weight_.size(0) > INT32_MAX || weight_.size(1) > INT32_MAX)
        throw py::value_error(c10::str("weight must be [out, in], got ", weight_.sizes()));
    const int64_t out = weight_.size(0), width = weight_.size(1);
    if (x.dim() == 0 || x.size(-1) != width) throw py::value_error(c10::str("expected a last axis of ", width, ", got ", x.sizes()));
    auto shape = x.sizes().vec();
    shape.back() = out;
    Tensor weight = checked_param(weight_, "weight", weight_.sizes(), x, false);
    Tensor bias = checked_param(bias_, "bias", {out}, x, false), residual = checked_param(residual_, "residual", shape, x, false, true);
    c10::DeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()) ||
                                       (residual.defined() && residual.requires_grad()))) {
        check_capture(stream, x, {&x, &weight, &bias, &residual});
        return LinearNode::apply(x, weight, given(bias), given(residual), act, stream);
    }
    return linear_run(rows_of(x, kLinearStride), weight, bias, residual, act, stream, nullptr);
}

// ---- gradient clipping -------------------------------------------------------------------------------------------------

// The ordinary case of training.clip_grad_norm_: every gradient (and every tensor of `out`) dense, contiguous, of the three
// types and on one device. Anything else comes back as None, and Python takes it apart with its own words.
py::object clip_grads(const py::list& params, const py::object& out, bool inf_norm, double max_norm, double grad_scale) {
    if (torch::jit::tracer::isTracing()) throw std::runtime_error("clip_grad_norm_ cannot be traced: its kernels are not torch operators");
    const size_t n = params.size();
    const bool to_out = !out.is_none();
    py::list outs = to_out ? py::reinterpret_borrow<py::list>(out) : py::list();
    std::vector<DmnGradTensor> table;
    std::vector<Tensor> written;
    table.reserve(n);
    written.reserve(n);
    c10::Device device(c10::kCPU);
    for (size_t i = 0; i < n; ++i) {
        PyObject* p = params[i].ptr();
        if (!THPVariable_Check(p)) return py::none();
        const Tensor& g = THPVariable_Unpack(p).grad();
        if (!g.defined()) continue;
        const int code = code_of(g.scalar_type());
        if (table.empty()) device = g.device();
        if (code < 0 || !g.is_cuda() || g.device() != device || g.layout() != at::kStrided || !g.is_contiguous() || g.is_neg() || g.is_inference()) return py::none();
        Tensor o = g;
        if (to_out) {
            if (!THPVariable_Check(outs[i].ptr())) return py::none();
            o = THPVariable_Unpack(outs[i].ptr());
            if (code_of(o.scalar_type()) < 0 || o.device() != device || o.layout() != at::kStrided || !o.is_contiguous() || o.is_neg() || o.is_inference() ||
                o.sizes() != g.sizes())
                return py::none();
        }
        table.push_back({g.data_ptr(), o.data_ptr(), g.numel(), code, code_of(o.scalar_type())});
        written.push_back(std::move(o));
    }
    if (table.empty()) return py::none();
    c10::DeviceGuard guard(device);
    const at::TensorOptions on = at::TensorOptions().device(device);
    Tensor norm = at::empty({}, on.dtype(at::kFloat));
    const size_t bytes = api.clip_workspace((int)table.size());
    const Tensor ws = at::empty({(int64_t)bytes}, on.dtype(at::kByte));
    check(api.clip(table.data(), (int)table.size(), inf_norm, (float)max_norm, (float)grad_scale, (float*)norm.data_ptr(), ws.data_ptr(), bytes,
                   handle(stream_handle(device.index()))));
    for (const Tensor& t : written) t.unsafeGetTensorImpl()->bump_version();
    return py::reinterpret_steal<py::object>(THPVariable_Wrap(norm));
}

}  // namespace

PYBIND11_MODULE(_dmn_torch, m) {
    m.def("bind", &bind);
    m.def("layer_norm", torch::wrap_pybind_function_no_gil(layer_norm));
    m.def("linear", torch::wrap_pybind_function_no_gil(linear));
    m.def("clip_grads", torch::wrap_pybind_function(clip_grads));
}
