"""The operators one after another, as a program that looks at frames has them."""
import numpy as np
import pytest
import torch

U = 2.0 ** -24


@pytest.mark.gpu
def test_states_over_rendered_frames(cuda):
    """Frames that `render` returns, a state for each pixel and colour carried from one to the next by single steps, and the last one normalised: as the recurrence
    over all frames at once has it."""
    import scenes as S
    import trigrad_amd
    W, H, frames = 48, 40, 6
    scene = S.random_soup(300, W, H, seed=9, sigma_px=6.0)
    d = {k: torch.from_numpy(v).to(cuda) for k, v in scene.items() if isinstance(v, np.ndarray)}
    with torch.no_grad():
        images = torch.stack([trigrad_amd.render(d["vertices"], d["indices"], d["colors"] * (0.5 + 0.1 * f), d["opacities"], W, H)[0] for f in range(frames)])
        colours, gates = images[..., :3].reshape(frames, H * W, 3), images[..., 3:].reshape(frames, H * W, 1)  # a gate for a pixel's colours
        state, before = torch.zeros((H * W, 3), device=cuda), []
        for x, g in zip(colours, gates):
            h, state = trigrad_amd.linear_recurrence_step(x, g, state, input_form="complement")
            before.append(h)
        states, final = trigrad_amd.linear_recurrence(colours.transpose(0, 1), gates.transpose(0, 1), input_form="complement")
        largest = colours.abs().max().item()
        for f in range(frames):  # a step is two roundings of values that are no larger than the colours
            assert (before[f] - states[:, f]).abs().max().item() <= 4 * (f + 1) * U * largest
        assert (state - final).abs().max().item() <= 4 * frames * U * largest
        y = trigrad_amd.group_norm(state.view(1, H, W, 3), 1, activation="silu")
        z = state.double()
        z = (z - z.mean()) / (z.var(unbiased=False) + 1e-5).sqrt()
        want = (z * torch.sigmoid(z)).view(1, H, W, 3)
        # sums of 5760 values over a workgroup's threads and lanes: at most 64 additions in a row, times the distance of the largest from the mean
        assert (y.double() - want).abs().max().item() <= 1.2 * (64 + 8) * 4 * U * (1 + z.abs().max().item()) ** 2


def _training_calls(cuda, seed):
    """[(leaves, call)]: a recurrence over chunks, one over packed sequences, a norm that is streamed and one that is held."""
    import trigrad_amd
    rng = torch.Generator().manual_seed(seed)

    def leaf(*shape):
        return torch.rand(shape, generator=rng).to(cuda).requires_grad_()
    cuts = torch.tensor([0, 100, 100, 4000], dtype=torch.int32, device=cuda)
    return [([leaf(1, 9000, 64), leaf(1, 9000, 64), leaf(1, 64)], lambda x, g, h: trigrad_amd.linear_recurrence(x, g, h)),
            ([leaf(4000, 24), leaf(4000, 8), leaf(3, 24)], lambda x, g, h: trigrad_amd.linear_recurrence(x, g, h, cuts, "logit", "complement")),
            ([leaf(1, 40000, 32), leaf(32), leaf(32)], lambda x, w, b: (trigrad_amd.group_norm(x, 8, w, b, activation="silu"),)),
            ([leaf(500, 256), leaf(256), leaf(256)], lambda x, w, b: (trigrad_amd.group_norm(x, 4, w, b, activation="gelu"),))]


def _with_gradients(leaves, call):
    out = call(*leaves)
    return [*(t.detach() for t in out), *torch.autograd.grad(sum(t.square().sum() for t in out), leaves)]


@pytest.fixture(params=["module", "python"])
def route(request, monkeypatch):
    from trigrad_amd import _C
    monkeypatch.setattr(_C, "ONE_CALL_OPERATORS", request.param == "module")


@pytest.mark.gpu
def test_saved_tensors_kept_on_the_host_and_recomputed(cuda, route):
    """What a program saves memory with: saved tensors that wait in host memory, and a forward pass that is run again for the backward one."""
    from torch.utils.checkpoint import checkpoint
    for leaves, call in _training_calls(cuda, 1):
        want = _with_gradients(leaves, call)
        with torch.autograd.graph.save_on_cpu():
            moved = _with_gradients(leaves, call)
        again = _with_gradients(leaves, lambda *t: checkpoint(call, *t, use_reentrant=False))
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, moved, again))


@pytest.mark.gpu
def test_calls_of_several_threads(cuda, route):
    """Threads with streams of their own, each with all of the calls, as often as to overlap."""
    import threading
    calls = _training_calls(cuda, 2)
    want = [_with_gradients(*c) for c in calls]
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = [([t.detach().clone().requires_grad_() for t in leaves], call) for leaves, call in calls]
            for _ in range(8):
                got = [_with_gradients(*c) for c in mine]
                torch.cuda.current_stream().synchronize()
                wrong.extend(not torch.equal(p, q) for a, b in zip(want, got) for p, q in zip(a, b))
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(wrong) == 3 * 8 * sum(len(w) for w in want) and not any(wrong)
