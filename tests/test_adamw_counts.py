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
