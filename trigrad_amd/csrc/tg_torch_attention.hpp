// tg_torch_attention.hpp -- linear attention, its single step and the AdamW step for torch, without the interpreter between a call's steps: a step
// over 320 small tensors was 1.7 ms of Python around 27 us of kernels, and is 42 us here.
//
// What is not the ordinary case is left to the Python functions by returning None: they have the checks and the error texts.
#pragma once
#include "tg_torch_operators.hpp"

#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <vector>

namespace {

// ---- linear attention ------------------------------------------------------------------

// `t` with its last dimension dense; other dimensions keep their strides.
at::Tensor rows_as_they_lie(const at::Tensor &t) {
    const at::Tensor r = t.is_neg() ? t.resolve_neg() : t;
    return r.size(-1) == 1 || r.stride(-1) == 1 ? r : r.contiguous();
}
void strides_of(const at::Tensor &t, bool packed, int64_t out[3]) {  // of sequence, row and head
    const int64_t first = packed ? 0 : 1;
    out[0] = packed ? 0 : t.stride(0);
    out[1] = t.stride(first);
    out[2] = t.stride(first + 1);
}

struct Attended : torch::CustomClassHolder {
    tg_attention call = {};  // sizes and forms
    at::Tensor offsets, outputs, final, kept;
    int64_t backward_bytes = 0;
};

struct LinearAttention : torch::autograd::Function<LinearAttention> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &queries, const at::Tensor &keys, const at::Tensor &values, const at::Tensor &gates,
                                 const std::optional<at::Tensor> &initial, const c10::intrusive_ptr<Attended> &s) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({queries, keys, values, gates, initial ? *initial : at::Tensor(), s->offsets, s->kept});
        ctx->saved_data["initial"] = initial.has_value();
        variable_list out{std::move(s->outputs), std::move(s->final)};
        s->kept.reset();  // released with the node's saved tensors, not with the node
        s->offsets.reset();
        ctx->saved_data["call"] = c10::IValue::make_capsule(s);
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const variable_list saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["call"].toCapsule();
        tg_attention a = static_cast<const Attended *>(capsule.get())->call;
        const bool has_initial = ctx->saved_data["initial"].toBool(), packed = saved[5].defined();
        const c10::DeviceGuard guard(saved[2].device());
        const at::Tensor queries = rows_as_they_lie(saved[0]), keys = rows_as_they_lie(saved[1]), values = rows_as_they_lie(saved[2]), gates = dense(saved[3]),
                         initial = has_initial ? dense(saved[4]) : at::Tensor(), grad_outputs = grads[0].defined() ? rows_as_they_lie(grads[0]) : at::Tensor(),
                         grad_final = grads[1].defined() ? dense(grads[1]) : at::Tensor();
        at::Tensor grad_queries, grad_keys, grad_values, grad_gates, grad_initial;
        {
            const at::NoGradGuard no_grad;
            if (ctx->needs_input_grad(0)) grad_queries = at::empty(queries.sizes(), queries.options());
            if (ctx->needs_input_grad(1)) grad_keys = at::empty(keys.sizes(), keys.options());
            if (ctx->needs_input_grad(2)) grad_values = at::empty(values.sizes(), values.options());
            if (ctx->needs_input_grad(3)) grad_gates = at::empty(gates.sizes(), gates.options());
            if (has_initial && ctx->needs_input_grad(4)) grad_initial = at::empty(initial.sizes(), initial.options());
        }
        const at::Tensor workspace = room(values, static_cast<const Attended *>(capsule.get())->backward_bytes);
        a.queries = address(queries);
        a.keys = address(keys);
        a.values = address(values);
        a.gates = address(gates);
        a.initial = static_cast<const float *>(address(initial));
        a.offsets = static_cast<const int32_t *>(address(saved[5]));
        strides_of(queries, packed, a.query_strides);
        strides_of(keys, packed, a.key_strides);
        strides_of(values, packed, a.value_strides);
        a.outputs = nullptr;
        a.final = nullptr;
        a.kept = target(saved[6]);
        a.kept_bytes = saved[6].defined() ? saved[6].numel() : 0;
        a.workspace = target(workspace);
        a.workspace_bytes = workspace.defined() ? workspace.numel() : 0;
        a.stream = stream_of(values);
        a.grad_outputs = address(grad_outputs);
        if (grad_outputs.defined()) strides_of(grad_outputs, packed, a.grad_strides);
        a.grad_final = static_cast<const float *>(address(grad_final));
        a.grad_queries = target(grad_queries);
        a.grad_keys = target(grad_keys);
        a.grad_values = target(grad_values);
        a.grad_gates = target(grad_gates);
        a.grad_initial = static_cast<float *>(target(grad_initial));
        check(operators.attention_backward(&a), "tg_linear_attention_backward");
        return once(grads, {grad_queries, grad_keys, grad_values, grad_gates, grad_initial, at::Tensor()});
    }
};

bool take_scale(PyObject *arg, int64_t size, double &scale) {
    if (arg == Py_None)
        scale = 1.0 / std::sqrt((double)size);
    else if (PyFloat_CheckExact(arg))
        scale = PyFloat_AS_DOUBLE(arg);
    else
        return false;
    return true;
}

// Sizes of a call's tensors, whose rows have `dims` - 2 dimensions; false: not the ordinary case.
bool attention_sizes_of(tg_attention &a, const at::Tensor &queries, const at::Tensor &keys, const at::Tensor &values, const at::Tensor &gates, int64_t dims) {
    if (type_code(values.scalar_type()) < 0 || values.dim() != dims || keys.dim() != dims || queries.sizes() != keys.sizes() ||
        !goes_with(queries, values, false) || !goes_with(keys, values, false) || !goes_with(gates, values, true))
        return false;
    for (int64_t d = 0; d < dims - 2; d++)
        if (keys.size(d) != values.size(d)) return false;
    a.heads = values.size(dims - 2);
    a.key_heads = keys.size(dims - 2);
    a.key_size = keys.size(dims - 1);
    a.value_size = values.size(dims - 1);
    if (a.heads < 1 || a.key_heads < 1 || a.heads % a.key_heads != 0 || a.key_size < 1 || a.value_size < 1 || a.key_size > TG_ATTENTION_SIZE ||
        a.value_size > TG_ATTENTION_SIZE)
        return false;
    a.fixed_gates = gates.dim() == 1;
    if (a.fixed_gates) {
        if (gates.size(0) != a.heads) return false;
    } else {
        if (gates.dim() != dims - 1 || gates.size(dims - 2) != a.heads) return false;
        for (int64_t d = 0; d < dims - 2; d++)
            if (gates.size(d) != values.size(d)) return false;
    }
    a.type = type_code(values.scalar_type());
    a.gate_type = type_code(gates.scalar_type());
    return true;
}
bool states_of(const at::Tensor &t, const at::Tensor &with, const tg_attention &a) {
    return t.device() == with.device() && t.scalar_type() == at::kFloat && t.dim() == 4 && t.size(0) == a.sequences && t.size(1) == a.heads &&
           t.size(2) == a.key_size && t.size(3) == a.value_size;
}

// linear_attention(queries, keys, values, gates, initial, offsets, gate_form, scale) -> (outputs, final), or None.  The form is a number.
PyObject *py_linear_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    auto s = c10::make_intrusive<Attended>();
    tg_attention &a = s->call;
    at::Tensor queries, keys, values, gates, initial;
    if (n != 8 || !plain_call() || !take(args[0], false, queries) || !take(args[1], false, keys) || !take(args[2], false, values) ||
        !take(args[3], false, gates) || !take(args[4], true, initial) || !take(args[5], true, s->offsets) || !take_code(args[6], 3, a.gate_form) ||
        a.gate_form < TG_GATE_LOG)
        Py_RETURN_NONE;
    const bool packed = s->offsets.defined();
    if (!attention_sizes_of(a, queries, keys, values, gates, packed ? 3 : 4) || !take_scale(args[7], a.key_size, a.scale)) Py_RETURN_NONE;
    a.sequences = values.size(0);
    a.length = packed ? values.size(0) : values.size(1);
    if (packed) {
        if (s->offsets.device() != values.device() || s->offsets.scalar_type() != at::kInt || s->offsets.dim() != 1 || s->offsets.size(0) < 2) Py_RETURN_NONE;
        a.sequences = s->offsets.size(0) - 1;
    }
    if (initial.defined() && !states_of(initial, values, a)) Py_RETURN_NONE;
    bool for_backward = false;
    for (const at::Tensor *t : {&queries, &keys, &values, &gates, &initial}) for_backward = for_backward || (t->defined() && t->requires_grad());
    for_backward = for_backward && at::GradMode::is_enabled();
    variable_list out;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(values.device());
        {
            const at::NoGradGuard no_grad;
            const at::Tensor q = rows_as_they_lie(queries), k = rows_as_they_lie(keys), v = rows_as_they_lie(values), g = dense(gates),
                             h = initial.defined() ? dense(initial) : initial;
            if (packed) s->offsets = dense(s->offsets);
            a.queries = address(q);
            a.keys = address(k);
            a.values = address(v);
            a.gates = address(g);
            a.initial = static_cast<const float *>(address(h));
            a.offsets = static_cast<const int32_t *>(address(s->offsets));
            strides_of(q, packed, a.query_strides);
            strides_of(k, packed, a.key_strides);
            strides_of(v, packed, a.value_strides);
            int64_t sizes[4];
            check(operators.attention_sizes(&a, sizes), "tg_linear_attention_sizes");
            s->outputs = at::empty(v.sizes(), v.options());
            s->final = at::empty({a.sequences, a.heads, a.key_size, a.value_size}, on(v, at::kFloat));
            if (for_backward) s->kept = room(v, sizes[0]);
            const at::Tensor workspace = room(v, sizes[for_backward ? 2 : 1]);
            s->backward_bytes = sizes[3];
            a.outputs = target(s->outputs);
            a.final = static_cast<float *>(target(s->final));
            a.kept = target(s->kept);
            a.kept_bytes = s->kept.defined() ? sizes[0] : 0;
            a.workspace = target(workspace);
            a.workspace_bytes = sizes[for_backward ? 2 : 1];
            a.stream = stream_of(v);
            check(operators.attention_forward(&a), "tg_linear_attention_forward");
        }
        if (for_backward) {
            refuse_stale_leaves(a.stream, {&queries, &keys, &values, &gates, &initial});
            out = LinearAttention::apply(queries, keys, values, gates, initial.defined() ? std::optional<at::Tensor>(initial) : std::nullopt, s);
        } else {
            out = {s->outputs, s->final};
        }
    }
    PyObject *result = PyTuple_New(2);
    if (!result) return nullptr;
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(out[0])));
    PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(out[1])));
    return result;
    END_HANDLE_TH_ERRORS
}

// linear_attention_step(queries, keys, values, gates, state, gate_form, scale, out or None) -> (outputs, new state), or None
PyObject *py_linear_attention_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    tg_attention a = {};
    at::Tensor queries, keys, values, gates, state, out, outputs;
    if (n != 8 || !plain_call() || !take(args[0], false, queries) || !take(args[1], false, keys) || !take(args[2], false, values) ||
        !take(args[3], false, gates) || !take(args[4], false, state) || !take_code(args[5], 3, a.gate_form) || a.gate_form < TG_GATE_LOG ||
        !take(args[7], true, out))
        Py_RETURN_NONE;
    if (!out.defined()) out = state;
    if (!attention_sizes_of(a, queries, keys, values, gates, 3) || !take_scale(args[6], a.key_size, a.scale)) Py_RETURN_NONE;
    a.sequences = values.size(0);
    a.length = 1;
    for (const at::Tensor *t : {&state, &out})
        if (!states_of(*t, values, a) || !t->is_contiguous() || t->is_neg()) Py_RETURN_NONE;
    if (at::GradMode::is_enabled())
        for (const at::Tensor *t : {&queries, &keys, &values, &gates, &state, &out})
            if (t->requires_grad()) Py_RETURN_NONE;
    // what is written may be the state itself and nothing else that is read
    for (const at::Tensor *t : {&queries, &keys, &values, &gates})
        if (overlap(out, *t)) Py_RETURN_NONE;
    if (out.data_ptr() != state.data_ptr() && overlap(out, state)) Py_RETURN_NONE;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(values.device());
        const at::NoGradGuard no_grad;
        const at::Tensor q = rows_as_they_lie(queries), k = rows_as_they_lie(keys), v = rows_as_they_lie(values), g = dense(gates);
        outputs = at::empty(v.sizes(), v.options());
        a.queries = address(q);
        a.keys = address(k);
        a.values = address(v);
        a.gates = address(g);
        a.initial = static_cast<const float *>(address(state));
        a.outputs = target(outputs);
        a.final = static_cast<float *>(target(out));
        const std::pair<const at::Tensor *, int64_t *> strides[] = {{&q, a.query_strides}, {&k, a.key_strides}, {&v, a.value_strides}};
        for (const auto &[t, to] : strides) {
            to[0] = t->stride(0);
            to[2] = t->stride(1);
        }
        a.stream = stream_of(v);
        check(operators.attention_step(&a), "tg_linear_attention_step");
        if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    }
    PyObject *written = args[7] == Py_None ? args[4] : args[7];
    PyObject *result = PyTuple_New(2);
    if (!result) return nullptr;
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(outputs)));
    Py_INCREF(written);
    PyTuple_SET_ITEM(result, 1, written);
    return result;
    END_HANDLE_TH_ERRORS
}

// ---- AdamW -------------------------------------------------------------------------------

// The tensors of a list or tuple, and null for None.  A list is copied to a tuple that holds them for the call: other threads may change it meanwhile.
struct Tensors {
    std::vector<const at::Tensor *> at;
    THPObjectPtr held;

    bool empty() const { return at.empty(); }
    const at::Tensor *operator[](size_t i) const { return at[i]; }
    auto begin() const { return at.begin(); }
    auto end() const { return at.end(); }
};
// false: not a case for this route, as are tensors that are views with a negation still to be done, of another kind than torch's own, or on another
// device than a GPU.  That is all in a tensor's keys, which are those of the tensor before it as a rule.
bool take_tensors(PyObject *arg, size_t count, bool optional, Tensors &tensors) {
    if (optional && arg == Py_None) return true;
    const bool list = PyList_CheckExact(arg);
    if ((!list && !PyTuple_CheckExact(arg)) || (size_t)Py_SIZE(arg) != count) return false;
    if (list) {
        tensors.held = THPObjectPtr(PyList_AsTuple(arg));
        if (!tensors.held) throw python_error();
        arg = tensors.held.get();
    }
    auto &to = tensors.at;
    to.resize(count);
    c10::DispatchKeySet known;
    for (size_t i = 0; i < count; i++) {
        PyObject *item = PyTuple_GET_ITEM(arg, i);
        if (optional && item == Py_None) continue;
        if (!THPVariable_CheckTypeExact(Py_TYPE(item))) return false;  // a tensor or a parameter
        to[i] = &THPVariable_Unpack(item);
        const c10::DispatchKeySet keys = to[i]->key_set();
        if (keys == known) continue;
        if (!to[i]->is_cuda() || at::isTensorSubclassLike(*to[i]) || to[i]->is_neg()) return false;
        known = keys;
    }
    return true;
}

// A number, or a tensor of one float32 on the device.
bool take_single(PyObject *arg, const at::Tensor &with, double &number, at::Tensor &tensor) {
    if (THPVariable_Check(arg))
        return take(arg, false, tensor) && tensor.device() == with.device() && tensor.scalar_type() == at::kFloat && tensor.numel() == 1 && !tensor.is_neg();
    number = PyFloat_CheckExact(arg) ? PyFloat_AS_DOUBLE(arg) : PyLong_CheckExact(arg) ? PyLong_AsDouble(arg) : -1.0;
    if (PyErr_Occurred()) PyErr_Clear();
    return number >= 0.0;
}

struct Extent {
    const char *first, *last;
    bool written;
};
// Whether none of the extents that are written meets another.  Lists that lie one behind the other, as parts of a buffer each do, need no sorting.
bool apart(std::vector<std::vector<Extent>> &lists) {
    std::vector<Extent> whole;
    bool ascending = true;
    for (const auto &list : lists) {
        if (list.empty()) continue;
        for (size_t i = 1; i < list.size() && ascending; i++) ascending = list[i - 1].last <= list[i].first;
        whole.push_back({list.front().first, list.back().last, list.front().written});
    }
    const auto disjoint = [](std::vector<Extent> &extents) {
        std::sort(extents.begin(), extents.end(), [](const Extent &a, const Extent &b) { return a.first < b.first; });
        const char *end = nullptr, *end_written = nullptr;
        for (const Extent &e : extents) {
            if (e.first < end_written || (e.written && e.first < end)) return false;
            end = std::max(end, e.last);
            if (e.written) end_written = std::max(end_written, e.last);
        }
        return true;
    };
    if (ascending && disjoint(whole)) return true;
    whole.clear();
    for (const auto &list : lists) whole.insert(whole.end(), list.begin(), list.end());
    return disjoint(whole);
}

// adamw_step(params, grads, averages, squares, step, rate, beta1, beta2, eps, decay, copies, scales, grad_scale, maximize, seed) -> True, or None
PyObject *py_adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensors params, grads, averages, squares, copies, scales;
    at::Tensor step, rate, grad_scale;
    tg_adamw c = {};
    if (n != 15 || !plain_call() || (!PyList_CheckExact(args[0]) && !PyTuple_CheckExact(args[0])) || Py_SIZE(args[0]) == 0) Py_RETURN_NONE;
    const size_t count = (size_t)Py_SIZE(args[0]);
    if (!take_tensors(args[0], count, false, params) || !take_tensors(args[1], count, false, grads) || !take_tensors(args[2], count, false, averages) ||
        !take_tensors(args[3], count, false, squares) || !take_tensors(args[10], count, true, copies) || !take_tensors(args[11], count, true, scales) ||
        !take(args[12], true, grad_scale) || !take_single(args[4], *params[0], c.step, step) || !take_single(args[5], *params[0], c.rate, rate))
        Py_RETURN_NONE;
    double *const numbers[] = {&c.beta1, &c.beta2, &c.eps, &c.decay};
    for (int i = 0; i < 4; i++) {
        if (!PyFloat_CheckExact(args[6 + i])) Py_RETURN_NONE;
        *numbers[i] = PyFloat_AS_DOUBLE(args[6 + i]);
    }
    if (!(c.beta1 >= 0.0 && c.beta1 < 1.0 && c.beta2 >= 0.0 && c.beta2 < 1.0 && c.eps >= 0.0) || (!step.defined() && !(c.step >= 1.0)) ||
        !PyBool_Check(args[13]) || !PyLong_CheckExact(args[14]))
        Py_RETURN_NONE;
    c.maximize = args[13] == Py_True;
    c.seed = (int64_t)(PyLong_AsUnsignedLongLongMask(args[14]) & 0xFFFFFFFFu);
    const at::Tensor &like = *params[0];
    const c10::Device device = like.device();
    const auto single = [&](const at::Tensor &t) { return t.device() == device && t.scalar_type() == at::kFloat && t.numel() == 1 && !t.is_neg(); };
    if (grad_scale.defined() && !single(grad_scale)) Py_RETURN_NONE;
    const at::ScalarType state = scales.empty() ? at::kFloat : at::kFloat8_e4m3fn;
    const auto written = [&](const at::Tensor &t, at::ScalarType type) {
        return t.scalar_type() == type && t.device() == device && t.is_contiguous();
    };
    std::vector<std::vector<Extent>> extents(6);
    for (auto &e : extents) e.reserve(count);
    const auto extent = [](const void *first, int64_t bytes, bool written) {
        return Extent{static_cast<const char *>(first), static_cast<const char *>(first) + bytes, written};
    };
    std::vector<const void *> grad_at(count);
    std::vector<void *> param_at(count), average_at(count), square_at(count), copy_at(copies.empty() ? 0 : count), scale_at(scales.empty() ? 0 : count);
    std::vector<int64_t> sizes(count), grad_types(count), copy_types(copies.empty() ? 0 : count, -1);
    const bool recording = at::GradMode::is_enabled();
    for (size_t i = 0; i < count; i++) {
        const at::Tensor &p = *params[i], &g = *grads[i], &average = *averages[i], &square = *squares[i];
        if (!written(p, at::kFloat) || type_code(g.scalar_type()) < 0 || g.device() != device || g.sizes() != p.sizes() ||
            !g.is_contiguous() || !written(average, state) || !written(square, state) || average.sizes() != p.sizes() || square.sizes() != p.sizes() || (recording && p.requires_grad() && !p.is_leaf()))
            Py_RETURN_NONE;
        param_at[i] = target(p);
        grad_at[i] = address(g);
        average_at[i] = target(average);
        square_at[i] = target(square);
        sizes[i] = p.numel();
        grad_types[i] = type_code(g.scalar_type());
        if (!copies.empty() && copies[i]) {
            const at::Tensor &t = *copies[i];
            if ((!written(t, at::kHalf) && !written(t, at::kBFloat16)) || t.sizes() != p.sizes()) Py_RETURN_NONE;
            copy_at[i] = target(t);
            copy_types[i] = type_code(t.scalar_type());
        }
        if (!scales.empty()) {
            if (!scales[i]) Py_RETURN_NONE;
            const at::Tensor &t = *scales[i];
            if (!written(t, at::kFloat) || t.dim() != 2 || t.size(0) != (p.numel() + 255) / 256 || t.size(1) != 2) Py_RETURN_NONE;
            scale_at[i] = target(t);
        }
        if (sizes[i] == 0) continue;
        const int64_t state_bytes = sizes[i] * (scales.empty() ? 4 : 1);
        extents[0].push_back(extent(param_at[i], sizes[i] * 4, true));
        extents[1].push_back(extent(average_at[i], state_bytes, true));
        extents[2].push_back(extent(square_at[i], state_bytes, true));
        extents[3].push_back(extent(grad_at[i], sizes[i] * (grad_types[i] == TG_TYPE_F32 ? 4 : 2), false));
        if (!scales.empty()) extents[4].push_back(extent(scale_at[i], scales[i]->numel() * 4, true));
        if (!copies.empty() && copies[i]) extents[5].push_back(extent(copy_at[i], sizes[i] * 2, true));
    }
    for (const at::Tensor *t : {&step, &rate, &grad_scale})
        if (t->defined()) extents.push_back({extent(address(*t), 4, false)});
    if (!apart(extents)) Py_RETURN_NONE;
    c.params = reinterpret_cast<float *const *>(param_at.data());
    c.grads = grad_at.data();
    c.averages = average_at.data();
    c.squares = square_at.data();
    c.copies = copies.empty() ? nullptr : copy_at.data();
    c.scales = scales.empty() ? nullptr : reinterpret_cast<float *const *>(scale_at.data());
    c.sizes = sizes.data();
    c.grad_types = grad_types.data();
    c.copy_types = copies.empty() ? nullptr : copy_types.data();
    c.device_step = static_cast<const float *>(address(step));
    c.device_rate = static_cast<const float *>(address(rate));
    c.grad_scale = static_cast<const float *>(address(grad_scale));
    c.count = (int64_t)count;
    c.bits = scales.empty() ? 32 : 8;
    {
        const Unlocked unlocked;
        const c10::DeviceGuard guard(like.device());
        c.stream = stream_of(like);
        check(operators.adamw_step(&c), "tg_adamw_step");
        for (const auto *list : {&params, &averages, &squares, &copies, &scales})
            for (const at::Tensor *t : *list)
                if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// bind_operators(addresses of the library's entry points in OperatorLibrary's order)
PyObject *py_bind_operators(PyObject *, PyObject *args) {
    unsigned long long a[12];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9], &a[10], &a[11])) return nullptr;
    const auto set = [](auto &to, unsigned long long from) { to = reinterpret_cast<std::decay_t<decltype(to)>>(from); };
    set(operators.recurrence_sizes, a[0]);
    set(operators.recurrence_forward, a[1]);
    set(operators.recurrence_backward, a[2]);
    set(operators.recurrence_step, a[3]);
    set(operators.norm_sizes, a[4]);
    set(operators.norm_forward, a[5]);
    set(operators.norm_backward, a[6]);
    set(operators.attention_sizes, a[7]);
    set(operators.attention_forward, a[8]);
    set(operators.attention_backward, a[9]);
    set(operators.attention_step, a[10]);
    set(operators.adamw_step, a[11]);
    Py_RETURN_NONE;
}

}  // namespace
