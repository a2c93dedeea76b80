"""Group norm with an activation for tensors whose channels lie last, as an image that `render` returns has them."""
import operator
from typing import Optional

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _C
from .util import create_check

check_tensor = create_check("cuda", None)

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


class GroupNorm(Function):
    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, activation):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, but got {activation}")
        if x.dtype not in _C.TYPE_CODES:
            raise TypeError(f"x must be of type {', '.join(map(str, _C.TYPE_CODES))}, but got {x.dtype}")
        check_tensor(x, "x", tuple(x.shape), x.dtype)
        if x.dim() < 2:
            raise ValueError(f"x must have at least 2 dimensions, but got {x.dim()}")
        channels = x.shape[-1]
        num_groups = operator.index(num_groups)
        if num_groups < 1 or channels < 1 or channels % num_groups != 0:
            raise ValueError(f"the number of channels must be a multiple of the number of groups, but got {channels} and {num_groups}")
        if not eps >= 0.0:
            raise ValueError(f"eps must not be negative, but got {eps}")
        real = _C.real_type(x.dtype)
        for name, t in (("weight", weight), ("bias", bias)):
            if t is not None:
                check_tensor(t, name, (channels,), real if t.dtype == real else x.dtype)
                if t.device != x.device:
                    raise TypeError(f"{name} must be on {x.device}, but got {t.device}")
        if weight is not None and bias is not None and weight.dtype != bias.dtype:
            raise TypeError(f"bias must be of type {weight.dtype}, but got {bias.dtype}")
        if any(ctx.needs_input_grad):
            _C.refuse_stale_leaves(x, weight, bias)
        x, weight, bias = (None if t is None else _C.dense(t) for t in (x, weight, bias))
        y, statistics = _C.group_norm_forward(x, num_groups, weight, bias, eps, ACTIVATIONS[activation])
        ctx.form = (num_groups, eps, ACTIVATIONS[activation])
        ctx.has = (weight is not None, bias is not None)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(x, statistics, *(t for t in (weight, bias) if t is not None))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, statistics, *more = ctx.saved_tensors
        weight = more[0] if ctx.has[0] else None
        bias = more[-1] if ctx.has[1] else None
        num_groups, eps, activation = ctx.form
        need_x, _, need_weight, need_bias = ctx.needs_input_grad[:4]
        grads = _C.group_norm_backward(grad_y, x, num_groups, weight, bias, statistics, eps, activation, need_x, need_weight, need_bias)
        return grads[0], None, grads[1], grads[2], None, None


def group_norm(
    x: torch.Tensor,
    num_groups: int,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    activation: str = "none",
) -> torch.Tensor:
    """
    act((x - mean) / sqrt(variance + eps) * weight + bias), mean and variance over a sample's positions and the channels of a group.
        x : (N, ..., C), channels last; float32, float16 or bfloat16 (float64: the double library).  (N, C) is a norm by token
        num_groups : a divisor of C; a group is C / num_groups successive channels
        weight, bias : (C,) of x's type or float32
        activation : "none", "relu", "silu" or "gelu" (by the error function)

    Sums and statistics are float32 whatever the types.  The call can be captured into a graph, with its backward pass; under capture a
    leaf of a graph that was made on another stream and still lives is refused.  Returns y as x.
    """
    module = _C.operators_by_torch_module(x)
    if module is not None:
        y = module.group_norm(x, num_groups, weight, bias, eps, ACTIVATIONS.get(activation))
        if y is not None:
            return y
    return GroupNorm.apply(x, num_groups, weight, bias, eps, activation)
