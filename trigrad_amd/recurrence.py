"""The gated linear recurrence as an operator of its own: `linear_recurrence` over whole sequences, with its gradient, and
`linear_recurrence_step` for a single step.

    h_t = a_t h_{t-1} + u_t,   a = gate, exp(gate) or sigmoid(gate),   u = x or (1 - a) x

Compositing is this recurrence: an image that `render` returns holds premultiplied colours and, in channel 3, the
transmittance that is left, so slabs of a scene that are rendered apart, nearest first in `slabs` (L, H, W, 4), become one image
as the last state from the farthest slab to the nearest:

    colours, transmittance = slabs[None, ..., :3].reshape(1, L, -1), slabs[None, ..., 3].reshape(1, L, -1)
    _, image = linear_recurrence(colours, transmittance, background.reshape(1, -1), reverse=True, return_states=False)
"""
from typing import Optional, Tuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _C
from .util import create_check

check_tensor = create_check("cuda", None)

GATE_FORMS = {"value": 0, "log": 1, "logit": 2}
INPUT_FORMS = {"plain": 0, "complement": 1}


def _check(inputs, gates, initial, offsets, gate_form, input_form, initial_name="initial"):
    """-> (sequences, length) of checked arguments."""
    if gate_form not in GATE_FORMS:
        raise ValueError(f"gate_form must be one of {', '.join(GATE_FORMS)}, but got {gate_form}")
    if input_form not in INPUT_FORMS:
        raise ValueError(f"input_form must be one of {', '.join(INPUT_FORMS)}, but got {input_form}")
    if inputs.dtype not in _C.TYPE_CODES:
        raise TypeError(f"inputs must be of type {', '.join(map(str, _C.TYPE_CODES))}, but got {inputs.dtype}")
    real = _C.real_type(inputs.dtype)
    dims = 2 if offsets is not None else 3
    if inputs.dim() != dims:
        raise ValueError(f"inputs must have {dims} dimensions, but got {inputs.dim()}")
    channels = inputs.shape[-1]
    check_tensor(inputs, "inputs", tuple(inputs.shape), inputs.dtype)
    if gates.dim() != dims or gates.shape[:-1] != inputs.shape[:-1]:
        raise ValueError(f"gates must be of shape {(*inputs.shape[:-1], 'G')}, but got {tuple(gates.shape)}")
    if gates.shape[-1] < 1 or channels % gates.shape[-1] != 0:
        raise ValueError(f"the number of channels must be a multiple of the number of gates, but got {channels} and {gates.shape[-1]}")
    check_tensor(gates, "gates", tuple(gates.shape), real if gates.dtype == real else inputs.dtype)
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 2:
            raise ValueError(f"offsets must be of shape (S + 1,) with S >= 1, but got {tuple(offsets.shape)}")
        check_tensor(offsets, "offsets", tuple(offsets.shape), torch.int32)
        sequences, length = offsets.shape[0] - 1, inputs.shape[0]
    else:
        sequences, length = inputs.shape[:2]
    if initial is not None:
        check_tensor(initial, initial_name, (sequences, channels), real)
    for name, t in (("gates", gates), (initial_name, initial), ("offsets", offsets)):
        if t is not None and t.device != inputs.device:
            raise TypeError(f"{name} must be on {inputs.device}, but got {t.device}")
    return sequences, length


class LinearRecurrence(Function):
    @staticmethod
    def forward(ctx, inputs, gates, initial, offsets, gate_form, input_form, reverse, return_states):
        sequences, length = _check(inputs, gates, initial, offsets, gate_form, input_form)
        ctx.set_materialize_grads(False)  # an output the loss does not use arrives as None instead of a zero tensor
        ctx.form = (sequences, length, GATE_FORMS[gate_form], INPUT_FORMS[input_form], bool(reverse))
        ctx.has = (initial is not None, offsets is not None)
        if any(ctx.needs_input_grad):
            _C.refuse_stale_leaves(inputs, gates, initial)
        inputs, gates, initial, offsets = (None if t is None else _C.dense(t) for t in (inputs, gates, initial, offsets))
        states, final, kept = _C.linear_recurrence_forward(inputs, gates, initial, offsets, *ctx.form, return_states,
                                                           any(ctx.needs_input_grad))
        if kept is not None:
            ctx.save_for_backward(inputs, gates, kept, *(t for t in (initial, offsets) if t is not None))
        return states, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_states, grad_final):
        inputs, gates, kept, *more = ctx.saved_tensors
        initial, offsets = more[0] if ctx.has[0] else None, more[-1] if ctx.has[1] else None
        grads = _C.linear_recurrence_backward(inputs, gates, initial, offsets, kept, grad_states, grad_final, *ctx.form, *ctx.needs_input_grad[:3])
        return (*grads, None, None, None, None, None)


def linear_recurrence(
    inputs: torch.Tensor,
    gates: torch.Tensor,
    initial: Optional[torch.Tensor] = None,
    offsets: Optional[torch.Tensor] = None,
    gate_form: str = "value",
    input_form: str = "plain",
    reverse: bool = False,
    return_states: bool = True,
) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """
    h_t = a_t h_{t-1} + u_t along every sequence and in every channel.
        inputs : (S, T, D), or (T, D) with offsets; float32, float16 or bfloat16 (float64: the double library)
        gates : (S, T, G), or (T, G) with offsets, D a multiple of G: a gate is that of D / G successive channels.  The inputs' type
            or float32
        initial : (S, D) float32, the states before the first step (default: zeros)
        offsets : (S + 1,) int32, not decreasing: sequence s is the rows offsets[s] to offsets[s + 1] - 1.  Sequences may be empty, and
            rows in front of offsets[0] or behind offsets[S] belong to none: their states and gradients are zeros
        gate_form : "value" a = gate, "log" a = exp(gate), "logit" a = sigmoid(gate)
        input_form : "plain" u = x, "complement" u = (1 - a) x
        reverse : every sequence from its last row to its first
        return_states : False: only the final state is of interest, no others are written

    Gates are decays, |a| <= 1.  Larger ones are computed as long as no product of successive gates of a sequence leaves the range of
    float32, which is formed for all but the shortest.  States are summed in float32 whatever the types.  The call can be captured into
    a graph, with its backward pass; under capture a leaf of a graph that was made on another stream and still lives is refused.

    Returns:
        states : as inputs, or None
        final : (S, D) float32, the state behind the last step of each sequence
    """
    module = _C.operators_by_torch_module(inputs)
    if module is not None:
        out = module.linear_recurrence(inputs, gates, initial, offsets, GATE_FORMS.get(gate_form), INPUT_FORMS.get(input_form), reverse, return_states)
        if out is not None:
            return out
    return LinearRecurrence.apply(inputs, gates, initial, offsets, gate_form, input_form, reverse, return_states)


def linear_recurrence_step(
    inputs: torch.Tensor,
    gates: torch.Tensor,
    state: torch.Tensor,
    gate_form: str = "value",
    input_form: str = "plain",
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    One step h = a h + u of S sequences, without gradients.
        inputs : (S, D), gates : (S, G), as in `linear_recurrence`
        state : (S, D) float32, contiguous; becomes the new state if `out` is None
        out : where the new state is written instead, as state

    Returns:
        states : (S, D) in the inputs' type
        state : the new state in float32 (`state` itself, or `out`)
    """
    module = _C.operators_by_torch_module(inputs)
    if module is not None:
        result = module.linear_recurrence_step(inputs, gates, state, GATE_FORMS.get(gate_form), INPUT_FORMS.get(input_form), out)
        if result is not None:
            return result
    if inputs.dim() != 2:
        raise ValueError(f"inputs must have 2 dimensions, but got {inputs.dim()}")
    _check(inputs[:, None], gates[:, None], state, None, gate_form, input_form, "state")
    new_state = state if out is None else out
    check_tensor(new_state, "out", tuple(state.shape), state.dtype)
    for name, t in (("state", state), ("out", new_state)):
        if not t.is_contiguous() or t.is_neg():
            raise ValueError(f"{name} must be contiguous, with no negation still to be done")
    if new_state.device != inputs.device:
        raise TypeError(f"out must be on {inputs.device}, but got {new_state.device}")
    for name, t in (("inputs", inputs), ("gates", gates)):
        if _C.overlap(new_state, t):
            raise ValueError(f"{name} must not overlap the state that is written")
    if new_state.data_ptr() != state.data_ptr() and _C.overlap(new_state, state):
        raise ValueError("out must be state itself or not overlap it")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (inputs, gates, state, new_state)):
        raise RuntimeError("linear_recurrence_step has no gradient: use linear_recurrence, or torch.no_grad()")
    states = _C.linear_recurrence_step(_C.dense(inputs), _C.dense(gates), state, new_state, GATE_FORMS[gate_form], INPUT_FORMS[input_form])
    if not new_state.is_inference():
        torch.autograd.graph.increment_version(new_state)
    return states, new_state
