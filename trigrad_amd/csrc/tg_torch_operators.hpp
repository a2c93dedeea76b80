// tg_torch_operators.hpp -- the gated linear recurrence, its single step and the group norm for torch, without the interpreter between a
// call's steps: a step that answers for one token is 2 us of a kernel, and a training call on a short sequence was 140 us of Python.
//
// What is not the ordinary case (other types and devices, shapes that do not fit, subclasses, tangents, tracing) is left to the Python
// functions by returning None: they have the checks and the error texts.
#pragma once
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/ops/empty_like.h>

namespace {

struct OperatorLibrary {
    int (*recurrence_sizes)(const tg_recurrence *, int64_t *) = nullptr;
    int (*recurrence_forward)(const tg_recurrence *) = nullptr;
    int (*recurrence_backward)(const tg_recurrence *) = nullptr;
    int (*recurrence_step)(const void *, const void *, const tg_real *, void *, tg_real *, int64_t, int64_t, int64_t, int, int, int, int,
                           void *) = nullptr;
    int (*norm_sizes)(const tg_norm *, int64_t *) = nullptr;
    int (*norm_forward)(const tg_norm *) = nullptr;
    int (*norm_backward)(const tg_norm *) = nullptr;
    int (*attention_sizes)(const tg_attention *, int64_t *) = nullptr;
    int (*attention_forward)(const tg_attention *) = nullptr;
    int (*attention_backward)(const tg_attention *) = nullptr;
    int (*attention_step)(const tg_attention *) = nullptr;
    int (*adamw_step)(const tg_adamw *) = nullptr;
} operators;

struct Unlocked {  // the interpreter is others' while this lives
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

int type_code(at::ScalarType t) { return t == at::kFloat ? TG_TYPE_F32 : t == at::kHalf ? TG_TYPE_F16 : t == at::kBFloat16 ? TG_TYPE_BF16 : -1; }

// A tensor of the arguments, or an undefined one for None; false: not a case for this route.
bool take(PyObject *arg, bool optional, at::Tensor &t) {
    if (optional && arg == Py_None) return true;
    if (!THPVariable_Check(arg)) return false;
    t = THPVariable_Unpack(arg);
    return t.is_cuda() && !at::isTensorSubclassLike(t) && !t._fw_grad(0).defined();
}
bool take_code(PyObject *arg, int64_t below, int64_t &code) {
    if (!PyLong_CheckExact(arg)) return false;
    code = PyLong_AsLongLong(arg);
    if (PyErr_Occurred()) PyErr_Clear();
    return code >= 0 && code < below;
}
// Types and places that go together: `t` as `with`, or float32 where `wide`.
bool goes_with(const at::Tensor &t, const at::Tensor &with, bool wide) {
    return t.device() == with.device() && (t.scalar_type() == with.scalar_type() || (wide && t.scalar_type() == at::kFloat));
}
bool state_of(const at::Tensor &t, const at::Tensor &with, int64_t sequences, int64_t channels) {
    return t.device() == with.device() && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == sequences && t.size(1) == channels;
}
// Whether the bytes between a tensor's first and last element meet another's.
bool overlap(const at::Tensor &a, const at::Tensor &b) {
    const auto extent = [](const at::Tensor &t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); d++) last += (t.size(d) - 1) * t.stride(d);
        const char *first = static_cast<const char *>(t.data_ptr());
        return std::make_pair(first, first + (t.numel() ? (last + 1) * (int64_t)t.element_size() : 0));
    };
    const auto x = extent(a), y = extent(b);
    return x.first < y.second && y.first < x.second;
}
bool plain_call() { return !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer); }
const void *address(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *target(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
at::Tensor dense(const at::Tensor &t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }
at::Tensor room(const at::Tensor &like, int64_t bytes) { return bytes ? at::empty({bytes}, on(like, at::kByte)) : at::Tensor(); }

// While `stream` is captured: a leaf whose gradient accumulates on another stream, because an eager graph of it made there still lives.  The
// engine would join that stream into the capture, which invalidates it or ends the process.
void refuse_stale_leaves(void *stream, std::initializer_list<const at::Tensor *> inputs) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &status) != hipSuccess) {
        (void)hipGetLastError();
        return;
    }
    if (status != hipStreamCaptureStatusActive) return;
    for (const at::Tensor *t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto made_on = accumulator ? accumulator->stream() : std::nullopt;
        if (made_on && c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *made_on).stream() != stream)
            throw std::runtime_error("a call under capture has a leaf of a graph that was made on another stream and still lives: release that graph "
                                     "(its outputs, and what was computed from them) before the capture");
    }
}

// Gradients of gradients are refused where they are asked for, as torch's once_differentiable does.
variable_list once(const variable_list &grads, variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    bool asked = false;
    for (const at::Tensor &g : grads) asked = asked || (g.defined() && g.requires_grad());
    if (!asked) return out;
    variable_list fake;
    for (const at::Tensor &t : out) {
        fake.push_back(t.defined() ? t.detach() : t);
        if (t.defined()) fake.back().set_requires_grad(true);
    }
    auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                                 (int)fake.size());
    return (*error)(std::move(fake));
}

// ---- gated linear recurrence ---------------------------------------------------------

struct Sequences : torch::CustomClassHolder {
    tg_recurrence call = {};  // sizes and forms
    at::Tensor offsets, states, final, kept;
    int64_t backward_bytes = 0;
};

struct LinearRecurrence : torch::autograd::Function<LinearRecurrence> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &inputs, const at::Tensor &gates, const std::optional<at::Tensor> &initial,
                                 const c10::intrusive_ptr<Sequences> &s) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({inputs, gates, initial ? *initial : at::Tensor(), s->offsets, s->kept});
        ctx->saved_data["initial"] = initial.has_value();
        variable_list out;
        if (s->states.defined()) out.push_back(std::move(s->states));
        out.push_back(std::move(s->final));
        s->kept.reset();  // released with the node's saved tensors, not with the node
        s->offsets.reset();
        ctx->saved_data["states"] = out.size() == 2;
        ctx->saved_data["call"] = c10::IValue::make_capsule(s);
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const variable_list saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["call"].toCapsule();
        tg_recurrence r = static_cast<const Sequences *>(capsule.get())->call;
        const bool has_initial = ctx->saved_data["initial"].toBool(), has_states = ctx->saved_data["states"].toBool();
        const c10::DeviceGuard guard(saved[0].device());
        const at::Tensor inputs = dense(saved[0]), gates = dense(saved[1]),
                         initial = has_initial ? dense(saved[2]) : at::Tensor();
        const at::Tensor grad_states = has_states && grads[0].defined() ? dense(grads[0]) : at::Tensor(),
                         grad_final = grads.back().defined() ? dense(grads.back()) : at::Tensor();
        at::Tensor grad_inputs, grad_gates, grad_initial;
        {
            const at::NoGradGuard no_grad;
            if (ctx->needs_input_grad(0)) grad_inputs = at::empty_like(inputs);
            if (ctx->needs_input_grad(1)) grad_gates = at::empty_like(gates);
            if (has_initial && ctx->needs_input_grad(2)) grad_initial = at::empty_like(initial);
        }
        const at::Tensor workspace = room(inputs, static_cast<const Sequences *>(capsule.get())->backward_bytes);
        r.inputs = address(inputs);
        r.gates = address(gates);
        r.initial = static_cast<const float *>(address(initial));
        r.offsets = static_cast<const int32_t *>(address(saved[3]));
        r.states = nullptr;
        r.final = nullptr;
        r.kept = target(saved[4]);
        r.kept_bytes = saved[4].defined() ? saved[4].numel() : 0;
        r.workspace = target(workspace);
        r.workspace_bytes = workspace.defined() ? workspace.numel() : 0;
        r.stream = stream_of(inputs);
        r.grad_states = address(grad_states);
        r.grad_final = static_cast<const float *>(address(grad_final));
        r.grad_inputs = target(grad_inputs);
        r.grad_gates = target(grad_gates);
        r.grad_initial = static_cast<float *>(target(grad_initial));
        check(operators.recurrence_backward(&r), "tg_linear_recurrence_backward");
        return once(grads, {grad_inputs, grad_gates, grad_initial, at::Tensor()});
    }
};

// linear_recurrence(inputs, gates, initial, offsets, gate_form, input_form, reverse, return_states) -> (states or None, final), or None.  The
// forms are numbers.
PyObject *py_linear_recurrence(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    auto s = c10::make_intrusive<Sequences>();
    tg_recurrence &r = s->call;
    at::Tensor inputs, gates, initial;
    if (n != 8 || !plain_call() || !take(args[0], false, inputs) || !take(args[1], false, gates) || !take(args[2], true, initial) ||
        !take(args[3], true, s->offsets) || !take_code(args[4], 3, r.gate_form) || !take_code(args[5], 2, r.input_form) || !PyBool_Check(args[6]) ||
        !PyBool_Check(args[7]))
        Py_RETURN_NONE;
    const int64_t dims = s->offsets.defined() ? 2 : 3;
    if (type_code(inputs.scalar_type()) < 0 || inputs.dim() != dims || gates.dim() != dims || !goes_with(gates, inputs, true)) Py_RETURN_NONE;
    for (int64_t d = 0; d + 1 < dims; d++)
        if (gates.size(d) != inputs.size(d)) Py_RETURN_NONE;
    r.channels = inputs.size(dims - 1);
    r.gate_count = gates.size(dims - 1);
    if (r.gate_count < 1 || r.channels % r.gate_count != 0) Py_RETURN_NONE;
    r.sequences = inputs.size(0);
    r.length = inputs.size(dims - 2);
    if (s->offsets.defined()) {
        if (s->offsets.device() != inputs.device() || s->offsets.scalar_type() != at::kInt || s->offsets.dim() != 1 || s->offsets.size(0) < 2) Py_RETURN_NONE;
        r.sequences = s->offsets.size(0) - 1;
        r.length = inputs.size(0);
    }
    if (initial.defined() && !state_of(initial, inputs, r.sequences, r.channels)) Py_RETURN_NONE;
    r.type = type_code(inputs.scalar_type());
    r.gate_type = type_code(gates.scalar_type());
    r.reverse = args[6] == Py_True;
    const bool return_states = args[7] == Py_True;
    const bool for_backward = at::GradMode::is_enabled() && (inputs.requires_grad() || gates.requires_grad() || (initial.defined() && initial.requires_grad()));
    variable_list out;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(inputs.device());
        {
            const at::NoGradGuard no_grad;
            const at::Tensor x = dense(inputs), g = dense(gates), h = initial.defined() ? dense(initial) : initial;
            if (s->offsets.defined()) s->offsets = dense(s->offsets);
            r.inputs = address(x);
            r.gates = address(g);
            r.initial = static_cast<const float *>(address(h));
            r.offsets = static_cast<const int32_t *>(address(s->offsets));
            int64_t sizes[3];
            check(operators.recurrence_sizes(&r, sizes), "tg_linear_recurrence_sizes");
            if (return_states) s->states = at::empty(x.sizes(), x.options());
            s->final = at::empty({r.sequences, r.channels}, on(x, at::kFloat));
            if (for_backward) s->kept = room(x, sizes[0]);
            const at::Tensor workspace = room(x, sizes[1]);
            s->backward_bytes = sizes[2];
            r.states = target(s->states);
            r.final = static_cast<float *>(target(s->final));
            r.kept = target(s->kept);
            r.kept_bytes = sizes[0];
            r.workspace = target(workspace);
            r.workspace_bytes = sizes[1];
            r.stream = stream_of(x);
            check(operators.recurrence_forward(&r), "tg_linear_recurrence_forward");
        }
        if (for_backward) {
            refuse_stale_leaves(r.stream, {&inputs, &gates, &initial});
            out = LinearRecurrence::apply(inputs, gates, initial.defined() ? std::optional<at::Tensor>(initial) : std::nullopt, s);
        } else {
            if (return_states) out.push_back(s->states);
            out.push_back(s->final);
        }
    }
    PyObject *result = PyTuple_New(2);
    if (!result) return nullptr;
    if (return_states) {
        PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(out[0])));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(result, 0, Py_None);
    }
    PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(out.back())));
    return result;
    END_HANDLE_TH_ERRORS
}

// linear_recurrence_step(inputs, gates, state, gate_form, input_form, out or None) -> (states, new state), or None
PyObject *py_linear_recurrence_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor inputs, gates, state, out, states;
    int64_t gate_form, input_form;
    if (n != 6 || !plain_call() || !take(args[0], false, inputs) || !take(args[1], false, gates) || !take(args[2], false, state) ||
        !take_code(args[3], 3, gate_form) || !take_code(args[4], 2, input_form) || !take(args[5], true, out))
        Py_RETURN_NONE;
    if (!out.defined()) out = state;
    if (type_code(inputs.scalar_type()) < 0 || inputs.dim() != 2 || gates.dim() != 2 || !goes_with(gates, inputs, true) || gates.size(0) != inputs.size(0) ||
        gates.size(1) < 1 || inputs.size(1) % gates.size(1) != 0)
        Py_RETURN_NONE;
    for (const at::Tensor *t : {&state, &out})
        if (!state_of(*t, inputs, inputs.size(0), inputs.size(1)) || !t->is_contiguous() || t->is_neg()) Py_RETURN_NONE;
    if (at::GradMode::is_enabled() && (inputs.requires_grad() || gates.requires_grad() || state.requires_grad() || out.requires_grad())) Py_RETURN_NONE;
    // what is written may be the state itself and nothing else that is read
    if (overlap(out, inputs) || overlap(out, gates) || (out.data_ptr() != state.data_ptr() && overlap(out, state))) Py_RETURN_NONE;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(inputs.device());
        const at::NoGradGuard no_grad;
        const at::Tensor x = dense(inputs), g = dense(gates);
        states = at::empty(x.sizes(), x.options());
        check(operators.recurrence_step(address(x), address(g), static_cast<const float *>(address(state)), target(states), static_cast<float *>(target(out)),
                                        x.size(0), x.size(1), g.size(1), type_code(x.scalar_type()), type_code(g.scalar_type()), (int)gate_form,
                                        (int)input_form, stream_of(x)),
              "tg_linear_recurrence_step");
        if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    }
    PyObject *written = args[5] == Py_None ? args[2] : args[5];
    PyObject *result = PyTuple_New(2);
    if (!result) return nullptr;
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(states)));
    Py_INCREF(written);
    PyTuple_SET_ITEM(result, 1, written);
    return result;
    END_HANDLE_TH_ERRORS
}

// ---- group norm ------------------------------------------------------------------------

struct Normed : torch::CustomClassHolder {
    tg_norm call = {};
    at::Tensor y, statistics;
    int64_t backward_bytes = 0;
};

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const std::optional<at::Tensor> &weight,
                                 const std::optional<at::Tensor> &bias, const c10::intrusive_ptr<Normed> &s) {
        ctx->save_for_backward({x, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), s->statistics});
        ctx->saved_data["weight"] = weight.has_value();
        ctx->saved_data["bias"] = bias.has_value();
        variable_list out{std::move(s->y)};
        s->statistics.reset();
        ctx->saved_data["call"] = c10::IValue::make_capsule(s);
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const variable_list saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["call"].toCapsule();
        tg_norm c = static_cast<const Normed *>(capsule.get())->call;
        const bool has_weight = ctx->saved_data["weight"].toBool(), has_bias = ctx->saved_data["bias"].toBool();
        const c10::DeviceGuard guard(saved[0].device());
        const at::Tensor x = dense(saved[0]), weight = has_weight ? dense(saved[1]) : at::Tensor(),
                         bias = has_bias ? dense(saved[2]) : at::Tensor(), grad_y = dense(grads[0]);
        at::Tensor grad_x, grad_weight, grad_bias;
        {
            const at::NoGradGuard no_grad;
            if (ctx->needs_input_grad(0)) grad_x = at::empty_like(x);
            if (has_weight && ctx->needs_input_grad(1)) grad_weight = at::empty_like(weight);
            if (has_bias && ctx->needs_input_grad(has_weight ? 2 : 1)) grad_bias = at::empty_like(bias);
        }
        const at::Tensor workspace = room(x, static_cast<const Normed *>(capsule.get())->backward_bytes);
        c.x = address(x);
        c.weight = address(weight);
        c.bias = address(bias);
        c.y = nullptr;
        c.statistics = static_cast<float *>(target(saved[3]));
        c.workspace = target(workspace);
        c.workspace_bytes = workspace.defined() ? workspace.numel() : 0;
        c.stream = stream_of(x);
        c.grad_y = address(grad_y);
        c.grad_x = target(grad_x);
        c.grad_weight = target(grad_weight);
        c.grad_bias = target(grad_bias);
        check(operators.norm_backward(&c), "tg_group_norm_backward");
        return once(grads, {grad_x, grad_weight, grad_bias, at::Tensor()});
    }
};

// group_norm(x, num_groups, weight, bias, eps, activation) -> y, or None.  The activation is a number.
PyObject *py_group_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    auto s = c10::make_intrusive<Normed>();
    tg_norm &c = s->call;
    at::Tensor x, weight, bias;
    if (n != 6 || !plain_call() || !take(args[0], false, x) || !take_code(args[1], (int64_t)1 << 24, c.groups) || !take(args[2], true, weight) ||
        !take(args[3], true, bias) || !PyFloat_CheckExact(args[4]) || !take_code(args[5], 4, c.activation))
        Py_RETURN_NONE;
    c.eps = PyFloat_AS_DOUBLE(args[4]);
    if (type_code(x.scalar_type()) < 0 || x.dim() < 2 || !(c.eps >= 0.0)) Py_RETURN_NONE;
    c.channels = x.size(-1);
    if (c.groups < 1 || c.channels < 1 || c.channels % c.groups != 0) Py_RETURN_NONE;
    c.samples = x.size(0);
    c.positions = 1;
    for (int64_t d = 1; d + 1 < x.dim(); d++) c.positions *= x.size(d);
    for (const at::Tensor *t : {&weight, &bias})
        if (t->defined() && (!goes_with(*t, x, true) || t->dim() != 1 || t->size(0) != c.channels)) Py_RETURN_NONE;
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) Py_RETURN_NONE;
    c.type = type_code(x.scalar_type());
    c.weight_type = weight.defined() ? type_code(weight.scalar_type()) : bias.defined() ? type_code(bias.scalar_type()) : c.type;
    const bool for_backward = at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) ||
                                                             (bias.defined() && bias.requires_grad()));
    at::Tensor y;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(x.device());
        {
            const at::NoGradGuard no_grad;
            const at::Tensor in = dense(x), w = weight.defined() ? dense(weight) : weight, b = bias.defined() ? dense(bias) : bias;
            int64_t sizes[2];
            check(operators.norm_sizes(&c, sizes), "tg_group_norm_sizes");
            s->y = at::empty(in.sizes(), in.options());
            s->statistics = at::empty({c.samples, c.groups, 2}, on(in, at::kFloat));
            const at::Tensor workspace = room(in, sizes[0]);
            s->backward_bytes = sizes[1];
            c.x = address(in);
            c.weight = address(w);
            c.bias = address(b);
            c.y = target(s->y);
            c.statistics = static_cast<float *>(target(s->statistics));
            c.workspace = target(workspace);
            c.workspace_bytes = sizes[0];
            c.stream = stream_of(in);
            check(operators.norm_forward(&c), "tg_group_norm_forward");
        }
        if (for_backward) {
            refuse_stale_leaves(c.stream, {&x, &weight, &bias});
            y = GroupNorm::apply(x, weight.defined() ? std::optional<at::Tensor>(weight) : std::nullopt,
                                 bias.defined() ? std::optional<at::Tensor>(bias) : std::nullopt, s)[0];
        } else {
            y = s->y;
        }
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// refuse_stale_leaves(tensors or None ...): for calls that the Python functions make themselves
PyObject *py_refuse_stale_leaves(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t k = 0; k < n; k++) {
        if (!THPVariable_Check(args[k])) continue;
        const at::Tensor &t = THPVariable_Unpack(args[k]);
        if (t.is_cuda()) refuse_stale_leaves(stream_of(t), {&t});
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace
