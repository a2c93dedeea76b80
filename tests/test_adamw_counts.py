"""How the optimizer counts steps: once each for every parameter that has a gradient, whatever it shares a call or a count with."""
import copy

import pytest
import torch

U = 2.0 ** -24
KINDS = [{}, {"capturable": True}]


@pytest.fixture
def calls(monkeypatch):
    """What the optimizer calls the step with, in place of the step: dicts, on any device."""
    import trigrad_amd
    made = []

    def step(params, grads, exp_avgs, exp_avg_sqs, step, **kw):
        count = step if not isinstance(step, torch.Tensor) else step.device if step.device.type == "meta" else step.item()
        made.append(dict(kw, params=params, step=count, devices={t.device for t in (*params, *((step,) if isinstance(step, torch.Tensor) else ()))}))
    monkeypatch.setattr(trigrad_amd.adamw, "adamw_step", step)
    return made


def leaf(dtype=torch.float32, device="cpu", grad=True):
    p = torch.zeros(4, dtype=dtype, device=device, requires_grad=True)
    p.grad = torch.ones_like(p) if grad else None
    return p


def counts_of(calls, p):
    return [c["step"] for c in calls if any(t is p for t in c["params"])]


@pytest.mark.parametrize("kwargs", KINDS)
def test_types_that_begin_together(calls, kwargs):
    import trigrad_amd
    params = [leaf(), leaf(torch.float64), leaf()]
    optimizer = trigrad_amd.AdamW(params, **kwargs)
    for _ in range(3):
        optimizer.step()
    assert len(calls) == 6
    for p in params:
        assert counts_of(calls, p) == [1, 2, 3]
    loaded = trigrad_amd.AdamW(params, **kwargs)
    loaded.load_state_dict(copy.deepcopy(optimizer.state_dict()))
    loaded.step()
    for p in params:
        assert counts_of(calls, p) == [1, 2, 3, 4]


def test_devices_of_a_group(calls):
    import trigrad_amd
    params = [leaf(), leaf(device="meta")]
    optimizer = trigrad_amd.AdamW(params, capturable=True)
    for _ in range(2):
        optimizer.step()
    assert counts_of(calls, params[0]) == [1, 2]
    assert all(len(c["devices"]) == 1 for c in calls) and len(calls) == 4


@pytest.mark.parametrize("kwargs", KINDS)
def test_a_step_without_a_gradient(calls, kwargs):
    """Such a parameter is where it was: its next step has the next number."""
    import trigrad_amd
    a, b, c = leaf(), leaf(), leaf()
    optimizer = trigrad_amd.AdamW([a, b, c], **kwargs)
    for skipped in ((), (b,), (b, c), (), (a,), ()):
        for p in (a, b, c):
            p.grad = None if any(p is s for s in skipped) else torch.ones_like(p)
        optimizer.step()
    assert counts_of(calls, a) == [1, 2, 3, 4, 5] and counts_of(calls, b) == [1, 2, 3, 4] and counts_of(calls, c) == [1, 2, 3, 4, 5]
    assert [optimizer.state[p]["step"] for p in (a, b, c)] == [5, 4, 5]


@pytest.mark.gpu
@pytest.mark.parametrize("kwargs", KINDS)
def test_optimizer_is_torchs(cuda, kwargs):
    """A group of two types in which parameters skip steps, saved and loaded half way, beside torch's."""
    import trigrad_amd
    g = torch.Generator().manual_seed(0)
    values = [torch.randn(300, generator=g), torch.randn(200, generator=g, dtype=torch.float64), torch.randn(100, generator=g)]
    mine, theirs = ([t.to(cuda).requires_grad_() for t in values] for _ in range(2))
    a, b = trigrad_amd.AdamW(mine, lr=1e-2, **kwargs), torch.optim.AdamW(theirs, lr=1e-2, foreach=False)
    for turn in range(10):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            there = (turn + i) % 3 > 0 or turn < 2
            p.grad = torch.randn(p.shape, generator=g, dtype=p.dtype).to(cuda) if there else None
            q.grad = None if p.grad is None else p.grad.clone()
        a.step()
        b.step()
        if turn == 5:
            state = copy.deepcopy(a.state_dict())
            a = trigrad_amd.AdamW(mine, lr=5.0, **kwargs)
            a.load_state_dict(state)
    for p, q in zip(mine, theirs):  # a change is at most ten rates, rounded like the param in each of ten steps, on either side
        half = U if p.dtype == torch.float32 else 2.0 ** -53
        assert ((p - q).abs() <= 2 * 10 * half * (4 * q.abs() + 16 * 0.1)).all()


@pytest.mark.gpu
def test_captures_that_would_not_count_are_refused(cuda):
    """A count that the host has is the same in every replay, and a state that a graph makes is made anew."""
    import trigrad_amd
    for kwargs, warm, match in (({}, True, "capturable"), ({"capturable": True}, False, "first step"), ({"capturable": True}, True, "others")):
        params = [torch.ones(50, device=cuda, requires_grad=True) for _ in range(2)]
        for p in params:
            p.grad = torch.ones_like(p)
        optimizer = trigrad_amd.AdamW(params, **kwargs)
        if warm:
            optimizer.step()
        if match == "others":
            params[1].grad = None
        before = [p.detach().clone() for p in params]
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=match):
            with torch.cuda.graph(graph):
                optimizer.step()
        assert all(torch.equal(p, q) for p, q in zip(params, before))
        optimizer.step()  # and nothing is left of it
        assert [int(optimizer.state[p].get("step", 0)) for p in params] == [2 if warm else 1, 1 if match == "others" else 2 if warm else 1]


@pytest.mark.parametrize("kwargs", KINDS)
def test_calls_of_a_step_have_seeds_of_their_own(calls, kwargs):
    """Equal places of two groups are not rounded with the same random numbers; one group's are those of its seed and count."""
    import trigrad_amd
    groups = [{"params": [leaf(), leaf()]}, {"params": [leaf()]}, {"params": [leaf()], "seed": 7}]
    optimizer = trigrad_amd.AdamW(groups, state_bits=8, seed=5, **kwargs)
    for _ in range(3):
        optimizer.step()
    seeds = [c["seed"] & 0xFFFFFFFF for c in calls]
    assert len(set(seeds)) == (3 if kwargs else 9) and len(set(seeds[:3])) == 3
    assert seeds[::3] == ([5, 5, 5] if kwargs else [6, 7, 8])


def test_grad_scale_of_two_types(calls):
    """One in float32, as clipping leaves it, is for the float64 parameters too."""
    import trigrad_amd
    optimizer = trigrad_amd.AdamW([leaf(), leaf(torch.float64)])
    scale = torch.tensor([0.3])
    optimizer.step(grad_scale=scale)
    assert [c["grad_scale"].dtype for c in calls] == [torch.float32, torch.float64]
    assert calls[0]["grad_scale"] is scale and calls[1]["grad_scale"].item() == scale.item()


@pytest.mark.gpu
def test_steps_of_two_types_with_a_grad_scale(cuda):
    import trigrad_amd
    mine, theirs = ([torch.ones(100, dtype=t, device=cuda, requires_grad=True) for t in (torch.float32, torch.float64)] for _ in range(2))
    a, b = trigrad_amd.AdamW(mine, lr=1e-2), torch.optim.AdamW(theirs, lr=1e-2, foreach=False)
    scale = torch.tensor([0.25], device=cuda)
    for turn in range(3):
        for p, q in zip(mine, theirs):
            p.grad = torch.full_like(p, turn + 1.0)
            q.grad = p.grad * 0.25
        a.step(grad_scale=scale)
        b.step()
    for p, q in zip(mine, theirs):  # as in the test beside torch's
        half = U if p.dtype == torch.float32 else 2.0 ** -53
        assert ((p - q).abs() <= 2 * 3 * half * (4 * q.abs() + 16 * 0.03)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_that_lie_otherwise(cuda, dtype, bits):
    """Channels last, or turned, as torch's takes them: the steps of a contiguous parameter with the same values in the same places in memory."""
    import trigrad_amd
    g = torch.Generator().manual_seed(3)
    x = torch.randn((6, 5, 4, 3), generator=g).to(cuda, dtype)
    for turn in (lambda t: t.contiguous(memory_format=torch.channels_last), lambda t: t.permute(3, 0, 2, 1).contiguous().permute(1, 3, 2, 0)):
        p = turn(x).requires_grad_()
        order = sorted(range(4), key=lambda d: -p.stride(d))
        q = p.detach().permute(order).clone(memory_format=torch.contiguous_format).requires_grad_()
        assert not p.is_contiguous()
        a, b = (trigrad_amd.AdamW([t], lr=1e-2, state_bits=bits) for t in (p, q))
        for n in range(3):
            grad = torch.randn(x.shape, generator=g).to(cuda, dtype)
            p.grad = turn(grad) if n else grad  # a gradient may lie otherwise than its parameter
            q.grad = grad.permute(order).contiguous()
            a.step()
            b.step()
            if n == 1:
                state = copy.deepcopy(a.state_dict())
                a = trigrad_amd.AdamW([p], lr=1e-2, state_bits=bits)
                a.load_state_dict(state)
        assert torch.equal(p.permute(order), q) and p.stride() == turn(x).stride()
    hole = torch.zeros((8, 8), device=cuda)[:, :4].requires_grad_()
    hole.grad = torch.ones_like(hole)
    with pytest.raises(ValueError, match="contiguous"):
        trigrad_amd.AdamW([hole]).step()
