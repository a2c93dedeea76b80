"""Linear attention with decays: `linear_attention` over whole sequences, with its gradient, and `linear_attention_step` for a single step.

    S_t = a_t S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   a = exp(gate) or sigmoid(gate)

It is `linear_recurrence` with a state of K x V values for a head: what a row adds is the product of its key and its value, and its query reads
the state.  A prompt, or what frames so far have left, is read by the one and carried on by the other:

    outputs, state = linear_attention(queries, keys, values, gates)
    for ...:
        outputs, state = linear_attention_step(query, key, value, gate, state)
"""
from typing import Optional, Tuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _C
from .util import create_check

check_tensor = create_check("cuda", None)

GATE_FORMS = {"log": 1, "logit": 2}
LARGEST_SIZE = 128  # of a key or value: TG_ATTENTION_SIZE


def _check(queries, keys, values, gates, initial, offsets, gate_form, initial_name="initial"):
    """-> (sequences, length) of checked arguments."""
    if gate_form not in GATE_FORMS:
        raise ValueError(f"gate_form must be one of {', '.join(GATE_FORMS)}, but got {gate_form}")
    if values.dtype not in _C.TYPE_CODES:
        raise TypeError(f"values must be of type {', '.join(map(str, _C.TYPE_CODES))}, but got {values.dtype}")
    real = _C.real_type(values.dtype)
    dims = 3 if offsets is not None else 4
    if values.dim() != dims:
        raise ValueError(f"values must have {dims} dimensions, but got {values.dim()}")
    check_tensor(values, "values", tuple(values.shape), values.dtype)
    rows, heads = values.shape[:-2], values.shape[-2]
    if keys.dim() != dims or keys.shape[:-2] != rows:
        raise ValueError(f"keys must be of shape {(*rows, 'G', 'K')}, but got {tuple(keys.shape)}")
    check_tensor(keys, "keys", tuple(keys.shape), values.dtype)
    check_tensor(queries, "queries", tuple(keys.shape), values.dtype)
    if heads < 1 or keys.shape[-2] < 1 or heads % keys.shape[-2] != 0:
        raise ValueError(f"the number of value heads must be a multiple of the number of key heads, but got {heads} and {keys.shape[-2]}")
    for name, size in (("keys", keys.shape[-1]), ("values", values.shape[-1])):
        if not 1 <= size <= LARGEST_SIZE:
            raise ValueError(f"{name} must have 1 to {LARGEST_SIZE} elements, but got {size}")
    check_tensor(gates, "gates", (heads,) if gates.dim() == 1 else (*rows, heads), real if gates.dtype == real else values.dtype)
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 2:
            raise ValueError(f"offsets must be of shape (S + 1,) with S >= 1, but got {tuple(offsets.shape)}")
        check_tensor(offsets, "offsets", tuple(offsets.shape), torch.int32)
        sequences, length = offsets.shape[0] - 1, values.shape[0]
    else:
        sequences, length = values.shape[:2]
    if initial is not None:
        check_tensor(initial, initial_name, (sequences, heads, keys.shape[-1], values.shape[-1]), real)
    for name, t in (("queries", queries), ("keys", keys), ("gates", gates), (initial_name, initial), ("offsets", offsets)):
        if t is not None and t.device != values.device:
            raise TypeError(f"{name} must be on {values.device}, but got {t.device}")
    return sequences, length


def _scale(scale, keys):
    return keys.shape[-1] ** -0.5 if scale is None else float(scale)


class LinearAttention(Function):
    @staticmethod
    def forward(ctx, queries, keys, values, gates, initial, offsets, gate_form, scale):
        sequences, length = _check(queries, keys, values, gates, initial, offsets, gate_form)
        ctx.set_materialize_grads(False)  # an output the loss does not use arrives as None instead of a zero tensor
        ctx.form = (sequences, length, GATE_FORMS[gate_form], _scale(scale, keys))
        ctx.has = (initial is not None, offsets is not None)
        if any(ctx.needs_input_grad):
            _C.refuse_stale_leaves(queries, keys, values, gates, initial)
        queries, keys, values = (_C.rows_as_they_lie(t) for t in (queries, keys, values))
        gates, initial, offsets = (None if t is None else _C.dense(t) for t in (gates, initial, offsets))
        outputs, final, kept = _C.linear_attention_forward(queries, keys, values, gates, initial, offsets, *ctx.form, any(ctx.needs_input_grad))
        if kept is not None:
            ctx.save_for_backward(queries, keys, values, gates, kept, *(t for t in (initial, offsets) if t is not None))
        return outputs, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_outputs, grad_final):
        queries, keys, values, gates, kept, *more = ctx.saved_tensors
        initial, offsets = more[0] if ctx.has[0] else None, more[-1] if ctx.has[1] else None
        # saved tensors may come back laid out anew
        queries, keys, values = (_C.rows_as_they_lie(t) for t in (queries, keys, values))
        grads = _C.linear_attention_backward(queries, keys, values, gates, initial, offsets, kept, grad_outputs, grad_final, *ctx.form,
                                             ctx.needs_input_grad[:5])
        return (*grads, None, None, None)


def linear_attention(
    queries: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    gates: torch.Tensor,
    initial: Optional[torch.Tensor] = None,
    offsets: Optional[torch.Tensor] = None,
    gate_form: str = "log",
    scale: Optional[float] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    S_t = a_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t along every sequence and for every head.
        queries, keys : (S, T, G, K), or (T, G, K) with offsets; float32, float16 or bfloat16 (float64: the double library).  Their last
            dimension is read as it lies where it is dense, whatever the other strides: parts of one projection need no copy
        values : (S, T, H, V), or (T, H, V) with offsets, H a multiple of G: a key head is that of H / G successive value heads.  K and V
            are at most 128
        gates : (S, T, H), or (T, H) with offsets, or (H,), a fixed decay for each head.  The values' type or float32
        initial : (S, H, K, V) float32, the states before the first step (default: zeros)
        offsets : (S + 1,) int32, not decreasing: sequence s is the rows offsets[s] to offsets[s + 1] - 1.  Sequences may be empty, and
            rows in front of offsets[0] or behind offsets[S] belong to none: their outputs and gradients are zeros
        gate_form : "log" a = exp(gate), "logit" a = sigmoid(gate)
        scale : default 1 / sqrt(K)

    Gates are decays, a <= 1; minus infinity is a = 0, where the sequence begins anew.  A value that is not finite makes outputs of its
    sequence and head that are not, those of up to 63 rows in front of it too; what is finite beside it has all its terms.  States are float32 and all sums
    are, whatever the types; outputs and gradients are rounded to theirs once.  Beside that a term of an output in bfloat16 is off by up to 2^-16 of itself, one of
    anything in float16 by 2^-22, or by 2^-39 of the largest in its row or column.  The call can be
    captured into a graph, with its backward pass; under capture a leaf of a graph that was made on another stream and still lives is refused.

    Returns:
        outputs : as values
        final : (S, H, K, V) float32, the state behind the last step of each sequence
    """
    module = _C.operators_by_torch_module(values)
    if module is not None:
        out = module.linear_attention(queries, keys, values, gates, initial, offsets, GATE_FORMS.get(gate_form), scale)
        if out is not None:
            return out
    return LinearAttention.apply(queries, keys, values, gates, initial, offsets, gate_form, scale)


def linear_attention_step(
    queries: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    gates: torch.Tensor,
    state: torch.Tensor,
    gate_form: str = "log",
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    One step of S sequences, without gradients.
        queries, keys : (S, G, K), values : (S, H, V), gates : (S, H) or (H,), as in `linear_attention`
        state : (S, H, K, V) float32, contiguous; becomes the new state if `out` is None
        out : where the new state is written instead, as state

    Returns:
        outputs : as values
        state : the new state (`state` itself, or `out`)
    """
    module = _C.operators_by_torch_module(values)
    if module is not None:
        result = module.linear_attention_step(queries, keys, values, gates, state, GATE_FORMS.get(gate_form), scale, out)
        if result is not None:
            return result
    if values.dim() != 3 or keys.dim() != 3 or queries.dim() != 3:
        raise ValueError(f"queries, keys and values must have 3 dimensions, but got {queries.dim()}, {keys.dim()} and {values.dim()}")
    _check(queries[:, None], keys[:, None], values[:, None], gates if gates.dim() == 1 else gates[:, None], state, None, gate_form, "state")
    new_state = state if out is None else out
    check_tensor(new_state, "out", tuple(state.shape), state.dtype)
    if new_state.device != values.device:
        raise TypeError(f"out must be on {values.device}, but got {new_state.device}")
    for name, t in (("state", state), ("out", new_state)):
        if not t.is_contiguous() or t.is_neg():
            raise ValueError(f"{name} must be contiguous, with no negation still to be done")
    for name, t in (("queries", queries), ("keys", keys), ("values", values), ("gates", gates)):
        if _C.overlap(new_state, t):
            raise ValueError(f"{name} must not overlap the state that is written")
    if new_state.data_ptr() != state.data_ptr() and _C.overlap(new_state, state):
        raise ValueError("out must be state itself or not overlap it")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (queries, keys, values, gates, state, new_state)):
        raise RuntimeError("linear_attention_step has no gradient: use linear_attention, or torch.no_grad()")
    queries, keys, values = (_C.rows_as_they_lie(t) for t in (queries, keys, values))
    outputs = _C.linear_attention_step(queries, keys, values, _C.dense(gates), state, new_state, GATE_FORMS[gate_form], _scale(scale, keys))
    if not new_state.is_inference():
        torch.autograd.graph.increment_version(new_state)
    return outputs, new_state
