"""AdamW for what `render` and the operators have gradients of: `adamw_step`, one step over many tensors, and `AdamW`, the optimizer that keeps their
averages, in float32 or in 8 bits.

    m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

    optimizer = AdamW([{"params": [vertices], "lr": 1e-4}, {"params": [colors, opacities]}], lr=1e-2)
"""
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _C

BLOCK = 256  # successive elements of a tensor that share the scales of its averages in 8 bits
COPY_TYPES = (torch.float16, torch.bfloat16)
STATE_TYPE = torch.float8_e4m3fn


def scales_of(tensor: torch.Tensor) -> torch.Tensor:
    """The scales of `tensor`'s averages in 8 bits before the first step: (blocks of 256 elements, 2), zeros."""
    return torch.zeros((-(-tensor.numel() // BLOCK), 2), dtype=torch.float32, device=tensor.device)


def _written(name, t, like, dtypes, shape=None):
    """Checks a tensor that the step writes: as `like`, in memory as its elements are."""
    if t.device != like.device:
        raise TypeError(f"{name} must be on {like.device}, but got {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be of type {' or '.join(map(str, dtypes))}, but got {t.dtype}")
    if tuple(t.shape) != tuple(like.shape if shape is None else shape):
        raise ValueError(f"{name} must be of shape {tuple(like.shape if shape is None else shape)}, but got {tuple(t.shape)}")
    if not t.is_contiguous() or t.is_neg():
        raise ValueError(f"{name} must be contiguous, with no negation still to be done")


def _single(name, value, device):
    """A number, or a tensor of one float32 on the device."""
    if not isinstance(value, torch.Tensor):
        return float(value)
    if value.device != device or value.dtype != torch.float32 or value.numel() != 1 or value.is_neg():
        raise TypeError(f"{name} must be a number or a tensor of one float32 on {device}")
    return value


def _refuse_overlaps(lists):
    """Raises for memory that two of the tensors share, one of them written."""
    extents = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), written) for written, tensors in lists for t in tensors if t.numel())
    end, end_written = 0, 0  # of what is read, of what is written
    for first, last, written in extents:
        if first < end_written or (written and first < end):
            raise ValueError("a tensor that is written must not overlap another one or be there twice")
        end = max(end, last)
        end_written = max(end_written, last) if written else end_written


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    step: Union[int, torch.Tensor],
    lr: Union[float, torch.Tensor] = 1e-3,
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    copies: Optional[Sequence[Optional[torch.Tensor]]] = None,
    scales: Optional[Sequence[torch.Tensor]] = None,
    grad_scale: Optional[torch.Tensor] = None,
    maximize: bool = False,
    seed: int = 0,
) -> None:
    """
    One step of AdamW over all tensors of `params`, in place and outside of any graph.
        params : float32 (or all float64: the double library), contiguous, on one device
        grads : as params; float32, float16 or bfloat16
        exp_avgs, exp_avg_sqs : as params, the averages of the gradients and of their squares; or, with scales, float8_e4m3fn, the averages and
            the square roots of the squares' in units of the block's scales
        step : the number of this step, from 1, or a tensor of one float32 that the device reads it from
        lr : the learning rate, or a tensor of one float32
        copies : tensors in float16 or bfloat16 (or None) that receive the new params, for the programs that compute in 16 bits
        scales : for averages in 8 bits, of each tensor as `scales_of` makes them: (blocks of 256 elements, 2) float32, a block's largest
            average and its largest root of squares, divided by 448
        grad_scale : a tensor of one float32 (float64) that the gradients are multiplied with, as clipping and loss scaling leave one
        maximize : the gradients' opposite
        seed : an integer that is another one in every step, for averages in 8 bits: of its two neighbours in 8 bits a value becomes one by a random
            number that is mixed of the seed and its place, the nearer one more often, so that small changes are not lost.  To the seed the number of
            the step is added where step is a tensor, so that a captured step has other ones in every replay

    A gradient that is not finite makes its element so, and an infinite one with averages in 8 bits its block, whose scale it is.

    A tensor that is written may not overlap any other.  The call can be captured into a graph, with step and lr as tensors.
    """
    module = _C.operators_by_torch_module(params[0] if len(params) else None)
    if module is not None and module.adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, *betas, eps, weight_decay, copies, scales, grad_scale, maximize, seed):
        return
    for name, tensors in (("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs), ("copies", copies), ("scales", scales)):
        if tensors is not None and len(tensors) != len(params):
            raise ValueError(f"{name} must have {len(params)} tensors, but got {len(tensors)}")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must be at least 0 and below 1, but got {tuple(betas)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, but got {eps}")
    if not isinstance(step, torch.Tensor) and not step >= 1:
        raise ValueError(f"step must be at least 1, but got {step}")
    if not params:
        return
    device, real = params[0].device, params[0].dtype
    if device.type != "cuda":
        raise TypeError(f"params must be on cuda, but got {device.type}")
    if real not in (torch.float32, torch.float64):
        raise TypeError(f"params must be of type {torch.float32} or {torch.float64}, but got {real}")
    if real == torch.float64 and (copies is not None or scales is not None):
        raise TypeError("copies and averages in 8 bits go with params in float32")
    step, lr = _single("step", step, device), _single("lr", lr, device)
    if grad_scale is not None and (grad_scale.device != device or grad_scale.dtype != real or grad_scale.numel() != 1 or grad_scale.is_neg()):
        raise TypeError(f"grad_scale must be a tensor of one {real} on {device}")
    averages = (STATE_TYPE,) if scales is not None else (real,)
    gradient_types = (torch.float64,) if real == torch.float64 else (torch.float32, torch.float16, torch.bfloat16)
    dense = []
    for i, (p, g) in enumerate(zip(params, grads)):
        _written(f"params[{i}]", p, params[0], (real,), p.shape)
        if g.device != device or g.dtype not in gradient_types:
            raise TypeError(f"grads[{i}] must be on {device} and of type {' or '.join(map(str, gradient_types))}, but got {g.device} and {g.dtype}")
        if g.shape != p.shape:
            raise ValueError(f"grads[{i}] must be of shape {tuple(p.shape)}, but got {tuple(g.shape)}")
        _written(f"exp_avgs[{i}]", exp_avgs[i], p, averages)
        _written(f"exp_avg_sqs[{i}]", exp_avg_sqs[i], p, averages)
        if copies is not None and copies[i] is not None:
            _written(f"copies[{i}]", copies[i], p, COPY_TYPES)
        if scales is not None:
            _written(f"scales[{i}]", scales[i], p, (torch.float32,), (-(-p.numel() // BLOCK), 2))
        if p.requires_grad and not p.is_leaf and torch.is_grad_enabled():
            raise RuntimeError(f"params[{i}] is computed from others: a step changes leaves")
        dense.append(_C.dense(g.detach()))
    written = [*params, *exp_avgs, *exp_avg_sqs, *(t for t in copies or () if t is not None), *(scales or ())]
    _refuse_overlaps([(True, written), (False, [*dense, *(t for t in (grad_scale, step, lr) if isinstance(t, torch.Tensor))])])
    _C.adamw_step(params, dense, exp_avgs, exp_avg_sqs, copies, scales, step, lr, grad_scale, 8 if scales is not None else 32, seed=int(seed) & 0xFFFFFFFF,
                  maximize=bool(maximize), beta1=float(b1), beta2=float(b2), eps=float(eps), decay=float(weight_decay))
    torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])


class AdamW(torch.optim.Optimizer):
    """
    AdamW over groups of parameters, each group a few launches.
        params, lr, betas, eps, weight_decay, maximize : as torch.optim.AdamW takes them; lr may be a tensor of one float32
        state_bits : 32, or 8: averages in 8 bits with two float32 for every 256 elements, 2.03 bytes a parameter instead of 8
        capturable : steps are counted on the device, so that a step can be captured into a graph (with lr as a tensor where it is to change).
            Tensors that have had gradients in the same steps share a count, and a graph counts for those together that did when it was captured.
            A first step is not captured, nor any without capturable
        seed : of the random numbers that averages in 8 bits are rounded with, together with a step's number and the number of the call in it (one for
            each group, device, type and count)

    Parameters are dense in memory, in whatever order of their dimensions.  Those in float16 or bfloat16 are rounded copies of ones in float32 that the state
    keeps ("master").
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, state_bits=32, capturable=False, seed=0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, but got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, but got {lr}")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must not be negative, but got {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize, state_bits=state_bits,
                                      capturable=capturable, seed=seed))

    def _new_state(self, p, group, first):
        """The state of a parameter before its first step; `first`: the count of those on its device that begin with it."""
        state = {"step": first}
        if p.dtype in COPY_TYPES:
            state["master"] = p.detach().to(torch.float32, copy=True)
        if group["state_bits"] == 8:
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.uint8, requires_grad=False).view(STATE_TYPE) for _ in range(2))
            state["scales"] = scales_of(p)
        else:
            real = state.get("master", p).dtype
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros_like(p, dtype=real, requires_grad=False) for _ in range(2))
        return state

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[torch.Tensor] = None):
        """One step of every parameter that has a gradient.  grad_scale: as `adamw_step` takes it, for parameters of all types."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number = 0  # of the step's calls
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            capturing = any(p.is_cuda for p in params[:1]) and torch.cuda.is_current_stream_capturing()
            if capturing:
                self._refuse_what_no_replay_counts(params)
            firsts = {}  # by device
            states = [self.state[p] for p in params]
            for p, state in zip(params, states):
                if not state:
                    if p.grad.is_sparse:
                        raise RuntimeError("gradients must be dense")
                    if p.device not in firsts:
                        firsts[p.device] = torch.zeros(1, dtype=torch.float32, device=p.device) if group["capturable"] else 0
                    state.update(self._new_state(p, group, firsts[p.device]))
            calls = {}  # parameters of the same device, type and count together
            counted = {}  # states by their count on the device
            for p, state in zip(params, states):
                count = state["step"]
                if isinstance(count, torch.Tensor):
                    same = id(count)
                    counted.setdefault(same, []).append(state)
                else:
                    same = state["step"] = count + 1
                together = calls.setdefault((p.device, state.get("master", p).dtype, same), ([], []))
                together[0].append(p)
                together[1].append(state)
            if counted:
                self._count(group, counted, capturing)
            for together in calls.values():
                self._step_together(group, *together, grad_scale, number)
                number += 1
        return loss

    def _refuse_what_no_replay_counts(self, params):
        for p in params:
            state = self.state.get(p)
            if not state:
                raise RuntimeError("a parameter's first step cannot be captured: its averages would begin anew in every replay")
            if not isinstance(state["step"], torch.Tensor):
                raise RuntimeError("a step that is captured has to be counted on the device: the optimizer must be capturable")

    def _count(self, group, counted, capturing):
        """Counts a step on the device, once whatever calls read the count.  One that others of the group share, who do not step now, stays theirs, and those who
        do go on with a copy."""
        waiting = {id(self.state[p]["step"]) for p in group["params"] if p.grad is None and self.state.get(p)}
        for same, states in counted.items():
            count = states[0]["step"]
            if same in waiting:
                if capturing:
                    raise RuntimeError("a parameter that has no gradient now is counted with others that have one: make a step without capture first")
                count = count.clone()
                for state in states:
                    state["step"] = count
            count.add_(1.0)

    def _step_together(self, group, params: List[torch.Tensor], states, grad_scale, number):
        count = states[0]["step"]
        eight = group["state_bits"] == 8
        if params[0].dtype == torch.float64 and grad_scale is not None and grad_scale.dtype == torch.float32:
            grad_scale = grad_scale.double()
        low = any("master" in s for s in states)
        lists = [[s.get("master", p) for s, p in zip(states, params)], [p.grad for p in params], [s["exp_avg"] for s in states],
                 [s["exp_avg_sq"] for s in states], [p if "master" in s else None for s, p in zip(states, params)] if low else None]
        if not all(map(torch.Tensor.is_contiguous, params)):  # in memory all of a parameter's tensors lie as it does
            orders = [sorted(range(p.dim()), key=lambda d: -p.stride(d)) for p in params]
            lists = [None if ts is None else [None if t is None else t.permute(o) for t, o in zip(ts, orders)] for ts in lists]
        adamw_step(*lists[:4], count, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                   copies=lists[4], scales=[s["scales"] for s in states] if eight else None, grad_scale=grad_scale, maximize=group["maximize"],
                   seed=group["seed"] + (count if isinstance(count, int) else 0) + (number << 24))

    def load_state_dict(self, state_dict):
        """As torch's, with every tensor of the state in the type that it was saved in."""
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        placed = {}  # counts that several parameters share stay shared
        for i, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    key = (id(value), p.device)
                    if key not in placed:
                        placed[key] = value.detach().to(p.device, copy=True)
                    self.state[p][name] = placed[key]
