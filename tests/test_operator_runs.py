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
