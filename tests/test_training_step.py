"""Linear attention, the norm by head and the AdamW step one after another, as a program that learns from frames has them."""
import numpy as np
import pytest
import torch

from attention_reference import TYPES, U, reference

HEADS, SIZE = 4, 16
WIDTH = HEADS * SIZE


def frames_of(cuda, count, scene_seed=9):
    """Frames that `render` returns, as rows of patches: (patches, count, 48)."""
    import scenes as S
    import trigrad_amd
    scene = S.random_soup(300, 48, 40, seed=scene_seed, sigma_px=6.0)
    d = {k: torch.from_numpy(v).to(cuda) for k, v in scene.items() if isinstance(v, np.ndarray)}
    with torch.no_grad():
        images = [trigrad_amd.render(d["vertices"], d["indices"], d["colors"] * (0.4 + 0.02 * f), d["opacities"], 48, 40)[0][..., :3] for f in range(count)]
    patches = torch.stack(images, 1).reshape(10, 4, count, 12, 4, 3).permute(0, 3, 2, 1, 4, 5).reshape(120, count, 48)
    return patches[:8].contiguous()


def weights_of(cuda, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = {"project": (48, 3 * WIDTH + HEADS), "norm": (WIDTH,), "bias": (WIDTH,), "out": (WIDTH, 48)}
    return {n: (torch.randn(s, generator=g) * (0.2 if len(s) > 1 else 0.1) + (1.0 if n == "norm" else 0.0)).to(cuda).requires_grad_() for n, s in shapes.items()}


def forward(w, frames, attention, norm):
    rows = frames[:, :-1] @ w["project"]
    q, k, v = (rows[..., i * WIDTH:(i + 1) * WIDTH].unflatten(-1, (HEADS, SIZE)) for i in range(3))
    o = attention(q, k, v, rows[..., 3 * WIDTH:])
    y = norm(o.reshape(-1, WIDTH), w["norm"], w["bias"]).reshape(*frames.shape[:1], -1, WIDTH)
    return (y @ w["out"] - frames[:, 1:]).square().mean()


def own(w, frames):
    import trigrad_amd
    return forward(w, frames, lambda q, k, v, g: trigrad_amd.linear_attention(q, k, v, g, gate_form="logit")[0],
                   lambda x, a, b: trigrad_amd.group_norm(x, HEADS, a, b, activation="silu"))


def plain(w, frames):
    def attention(q, k, v, g):
        B, T = q.shape[:2]
        flat = [t.reshape(B * T, *t.shape[2:]) for t in (q, k, v, g)]
        return reference(*flat, None, list(range(0, B * T + 1, T)), "logit")[0].reshape(v.shape)

    def norm(x, a, b):
        h = x.view(-1, HEADS, SIZE)
        z = ((h - h.mean(-1, keepdim=True)) / (h.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()).view(x.shape) * a + b
        return z * torch.sigmoid(z)
    return forward(w, frames, attention, norm)


@pytest.mark.gpu
def test_training_steps(cuda):
    """Three steps in float32 beside the same in 64 bits: gradients, and what the optimizer makes of them."""
    import trigrad_amd
    frames = frames_of(cuda, 40)
    w = weights_of(cuda)
    d = {n: t.detach().double().requires_grad_() for n, t in w.items()}
    mine = trigrad_amd.AdamW(list(w.values()), lr=1e-2)
    theirs = torch.optim.AdamW(list(d.values()), lr=1e-2, foreach=False)
    for turn in range(3):
        mine.zero_grad()
        theirs.zero_grad()
        loss, want = own(w, frames), plain(d, frames.double())
        loss.backward()
        want.backward()
        # a thousand products and sums in a row at most, of terms that are no larger than eight times what they add up to in norm
        assert abs(loss.item() - want.item()) <= 8 * 1000 * U * want.item()
        for n in w:
            assert (w[n].grad - d[n].grad).norm() <= 8 * 1000 * U * d[n].grad.norm(), (turn, n)
        mine.step()
        theirs.step()
        # a gradient's relative error moves a weight by that part of the rate; those near zero may change sign: the rest of the rate for at most that many
        for n in w:
            assert (w[n] - d[n]).norm() <= 3 * (turn + 1) * 1e-2 * (8 * 1000 * U) ** 0.5 * d[n].numel() ** 0.5, (turn, n)
        with torch.no_grad():  # go on from the same weights, so that steps are compared and not where they lead
            for n in w:
                d[n].copy_(w[n])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_step(cuda, bits):
    """Forward and backward pass and the step in one graph, beside eager work: as the eager steps, bit by bit."""
    import trigrad_amd
    batches = [frames_of(cuda, 40, seed) for seed in (9, 10, 11)]
    results = []
    for captured in (False, True):
        w = weights_of(cuda, 1)
        optimizer = trigrad_amd.AdamW(list(w.values()), lr=1e-2, capturable=True, state_bits=bits)
        frames, losses = batches[0].clone(), []

        def step():
            optimizer.zero_grad(set_to_none=True)
            loss = own(w, frames)
            loss.backward()
            optimizer.step()
            return loss.detach()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
            step()
        torch.cuda.synchronize()
        if captured:
            optimizer.zero_grad(set_to_none=True)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = step()
        for batch in batches + batches:
            frames.copy_(batch)
            if captured:
                graph.replay()
                losses.append(held.clone())
            else:
                losses.append(step())
            torch.cuda.synchronize()
            torch.randn(1000, device=cuda).sum().item()
        results.append([*losses, *(t.detach() for t in w.values())])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_frames_one_by_one(cuda):
    """What a model has read of frames in one call is carried on row by row: as over all of them at once, in 16 bits."""
    import trigrad_amd
    frames = frames_of(cuda, 40)
    with torch.no_grad():
        w = weights_of(cuda)
        rows = (frames @ w["project"]).to(torch.bfloat16)
        q, k, v = (rows[..., i * WIDTH:(i + 1) * WIDTH].unflatten(-1, (HEADS, SIZE)) for i in range(3))
        gates = rows[..., 3 * WIDTH:]
        every, last = trigrad_amd.linear_attention(q, k, v, gates, gate_form="logit")
        some, state = trigrad_amd.linear_attention(*(t[:, :25] for t in (q, k, v, gates)), gate_form="logit")
        for t in range(25, 40):
            y, state = trigrad_amd.linear_attention_step(q[:, t], k[:, t], v[:, t], gates[:, t], state, gate_form="logit")
            some = torch.cat([some, y[:, None]], 1)
        sizes = torch.cat([trigrad_amd.linear_attention(q.abs(), k.abs(), v.abs(), gates, gate_form="logit")[0]])
        assert ((every.float() - some.float()).abs() <= 2.02 * TYPES[torch.bfloat16] * (every.float().abs() + sizes.float())).all()
        assert ((state - last).abs() <= 256 * U * trigrad_amd.linear_attention(q.abs(), k.abs(), v.abs(), gates, gate_form="logit")[1]).all()
