"""Channels-last group norm with an activation against its definition in 64 bits, forward and backward, and its refusals.

Tolerances, with u = 2^-24: a sum over n values is off by at most L u times the sum of their magnitudes, L the longest chain of additions
(at most 64 + n / 64: a thread's share, the tree over a workgroup, the workgroups' sums).  The statistics come from sums of x - p and
(x - p)^2 around some value p of the group, so the variance is off by 2 (L + 4) u (1 + z^2) of itself, z the largest distance of a value from
the mean in standard deviations, and the mean by (L + 2) u (1 + z) standard deviations and u of itself.  These go through the formulas to first order; exponentials and
error functions are taken to be good to 16 u, and the activations' second derivatives are at most 1.  Beside that an output is rounded once."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24


def _activation(kind, z):
    """(y, slope) in 64 bits."""
    if kind == "relu":
        return z.clamp_min(0.0), (z > 0.0).double()
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return z, torch.ones_like(z)


def reference(x, groups, weight, bias, eps, activation, grad_y=None):
    """-> {name: (value, bound)}"""
    N, C = x.shape[0], x.shape[-1]
    x64 = x.detach().double().cpu().reshape(N, -1, groups, C // groups)
    S = x64.shape[1]
    w = weight.detach().double().cpu().view(groups, -1) if weight is not None else torch.ones((groups, C // groups), dtype=torch.float64)
    b = bias.detach().double().cpu().view(groups, -1) if bias is not None else torch.zeros((groups, C // groups), dtype=torch.float64)
    avg = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mean = avg(x64)
    var = avg((x64 - mean) ** 2)
    rstd = (var + eps) ** -0.5
    L = 64 + S * (C // groups) / 64
    z_max = ((x64 - mean).abs().amax((1, 3), keepdim=True) * rstd).clamp_min(1.0)
    d_rstd = (L + 4) * U * (1 + z_max ** 2) + 4 * U  # of itself
    d_mean = ((L + 2) * U * (1 + z_max) / rstd + U * mean.abs())
    hat = (x64 - mean) * rstd
    d_hat = hat.abs() * (d_rstd + 3 * U) + d_mean * rstd
    z = hat * w + b
    d_z = w.abs() * d_hat + 4 * U * ((hat * w).abs() + b.abs())
    y, slope = _activation(activation, z)
    d_y = (1.2 * d_z + 16 * U * y.abs() + d_z ** 2) if activation != "none" else d_z
    out = {"y": (y.reshape(x.shape), d_y.reshape(x.shape))}
    if grad_y is None:
        return out
    dy = grad_y.double().cpu().reshape(x64.shape)
    d_slope = {"none": torch.zeros_like(z), "relu": (z.abs() <= d_z).double()}.get(activation, d_z + 16 * U * (1 + z.abs()))
    dz, d_dz = dy * slope, dy.abs() * (d_slope + 2 * U * slope.abs())
    dh, d_dh = dz * w, d_dz * w.abs() + 2 * U * (dz * w).abs()
    m1, m2 = avg(dh), avg(dh * hat)
    d_m1 = avg(d_dh) + (L + 2) * U * avg(dh.abs())
    d_m2 = avg(d_dh * hat.abs() + dh.abs() * d_hat) + (L + 3) * U * avg((dh * hat).abs())
    dx = rstd * (dh - m1 - hat * m2)
    d_dx = rstd * (d_dh + d_m1 + hat.abs() * d_m2 + d_hat * m2.abs() + (d_rstd + 6 * U) * (dh.abs() + m1.abs() + (hat * m2).abs()))
    Lw = 64 + N * S / 64
    flat = lambda t: t.sum((0, 1)).reshape(C)  # noqa: E731
    out["grad_x"] = (dx.reshape(x.shape), d_dx.reshape(x.shape))
    out["grad_weight"] = (flat(dz * hat), flat(d_dz * hat.abs() + dz.abs() * d_hat) + (Lw + 2) * U * flat((dz * hat).abs()))
    out["grad_bias"] = (flat(dz), flat(d_dz) + (Lw + 1) * U * flat(dz.abs()))
    return out


def assert_near(name, got, wanted):
    want, bound = wanted
    assert got.shape == want.shape, name
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float64 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    allowed = (bound + want.abs()) * half + bound + tiny + 1e-30
    off = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(off).all(), f"{name}: not finite"
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} of the bound at {np.unravel_index(int((off / allowed).argmax()), off.shape)}"


def make(cuda, seed, shape, dtype=torch.float32, second=None, offset=1.0):
    rng = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = torch.randn(shape, generator=rng) * torch.exp(0.5 * torch.randn((C,), generator=rng)) + offset * torch.randn((C,), generator=rng)
    w, b = 1.0 + 0.3 * torch.randn((C,), generator=rng), 0.3 * torch.randn((C,), generator=rng)
    dy = torch.randn(shape, generator=rng)
    return x.to(dtype).to(cuda), w.to(second or dtype).to(cuda), b.to(second or dtype).to(cuda), dy.to(dtype).to(cuda)


def run_and_check(x, groups, w, b, dy, activation="none", eps=1e-5):
    import trigrad_amd
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = trigrad_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], eps, activation)
    assert y.dtype == x.dtype and y.shape == x.shape
    there = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("grad_x", "grad_weight", "grad_bias"), leaves) if t is not None], torch.autograd.grad(y, there, dy)))
    want = reference(x, groups, w, b, eps, activation, dy)
    assert_near("y", y, want["y"])
    for name, got in grads.items():
        assert_near(name, got, want[name])
    return [y.detach(), *grads.values()]


TYPES = {"f32": (torch.float32, None), "bf16": (torch.bfloat16, None), "f16": (torch.float16, None),
         "bf16_f32": (torch.bfloat16, torch.float32), "f16_f32": (torch.float16, torch.float32), "f64": (torch.float64, None)}


@pytest.fixture(params=["module", "python"])
def route(request, monkeypatch):
    """Calls by the torch module, which takes the ordinary ones, and all of them by the Python functions."""
    from trigrad_amd import _C
    monkeypatch.setattr(_C, "ONE_CALL_OPERATORS", request.param == "module")


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("types", sorted(TYPES))
def test_types_and_activations(types, activation, cuda, route):
    for seed, (shape, groups) in enumerate([((2, 9, 11, 24), 4), ((50, 64), 8), ((1, 700, 40), 5)]):
        x, w, b, dy = make(cuda, seed, shape, *TYPES[types])
        run_and_check(x, groups, w, b, dy, activation)
        run_and_check(x, groups, None, None, dy, activation)


@pytest.mark.gpu
@pytest.mark.parametrize("channels,groups", [(1, 1), (2, 2), (3, 1), (4, 2), (6, 3), (8, 8), (15, 5), (32, 32), (33, 3), (64, 1), (64, 4), (96, 2),
                                             (120, 8), (130, 13), (256, 32), (260, 4), (320, 32), (513, 3), (1024, 1), (2056, 8)])
def test_channels_and_groups(channels, groups, cuda):
    for seed, (rows, dtype) in enumerate([((2, 33), torch.float32), ((3, 130), torch.bfloat16)]):
        x, w, b, dy = make(cuda, seed + channels, (*rows, channels), dtype, torch.float32)
        run_and_check(x, groups, w, b, dy, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("samples,positions", [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (2, 257), (1, 1000), (5, 1023), (1, 4097), (1, 20000), (300, 3), (3000, 1),
                                               (70, 16), (9, 150)])
def test_sizes(samples, positions, cuda):
    for seed, (channels, groups, dtype) in enumerate([(16, 4, torch.float32), (40, 5, torch.bfloat16), (256, 8, torch.float16), (7, 7, torch.float32)]):
        if samples * positions * channels > 2_000_000:
            continue
        x, w, b, dy = make(cuda, seed + positions, (samples, positions, channels), dtype)
        run_and_check(x, groups, w, b, dy, ("none", "gelu", "silu", "relu")[seed])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 300000, 8), 2), ((2, 3000, 512), 16), ((4000, 1, 1024), 16), ((20, 64, 64, 32), 8), ((1, 40000, 33), 11)])
def test_large(shape, groups, cuda):
    x, w, b, dy = make(cuda, 5, shape, torch.bfloat16, torch.float32)
    run_and_check(x, groups, w, b, dy, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("types,samples,channels,groups", [
    ("bf16", 5, 520, 1), ("bf16", 9000, 520, 1), ("bf16", 3, 1024, 2), ("f16", 3, 4104, 1), ("bf16", 700, 8192, 1), ("bf16_f32", 7, 8200, 1), ("f16", 2, 16384, 1),
    ("bf16", 2, 16392, 1), ("bf16", 33, 1001, 1), ("f16_f32", 3, 4094, 1), ("bf16", 2, 4097, 1), ("f32", 5, 260, 1), ("f32", 9, 12300, 3), ("f32", 2, 16384, 1),
    ("f32", 2, 16388, 1), ("f32", 3, 4095, 1), ("f64", 4, 130, 1), ("f64", 2, 4100, 1), ("f64", 2, 8192, 1), ("f64", 3, 2049, 1)])
def test_wide_tokens(types, samples, channels, groups, cuda):
    """Samples of one position whose groups are wider than a wave: around a thread's accesses, a workgroup's, and what it can hold."""
    dtype, second = TYPES[types]
    x, w, b, dy = make(cuda, 8, (samples, channels), dtype, second)
    run_and_check(x, groups, w, b, dy, "silu")
    run_and_check(x[1:], groups, w, None, dy[1:], "none")
    if dtype != torch.float64:  # storage that begins off a vector's alignment
        flat = torch.zeros((x.numel() + 1,), dtype=dtype, device=cuda)
        flat[1:] = x.flatten()
        run_and_check(flat[1:].view(x.shape), groups, w, b, dy, "gelu")


@pytest.mark.gpu
def test_only_weight_only_bias_and_partial_gradients(cuda, route):
    import trigrad_amd
    x, w, b, dy = make(cuda, 2, (2, 50, 48))
    full = run_and_check(x, 6, w, b, dy, "silu")
    run_and_check(x, 6, w, None, dy, "silu")
    run_and_check(x, 6, None, b, dy, "silu")
    for k in range(3):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        (one,) = torch.autograd.grad(trigrad_amd.group_norm(leaves[0], 6, leaves[1], leaves[2], activation="silu"), leaves[k], dy)
        assert torch.equal(one, full[1 + k])
    assert not trigrad_amd.group_norm(x, 6, w, b).requires_grad


@pytest.mark.gpu
def test_far_from_zero_and_constant(cuda):
    """A mean of a thousand deviations keeps the variance; a constant group has none, and its output is the bias."""
    import trigrad_amd
    for shape in ((2, 500, 32), (1, 30000, 16), (600, 1, 64)):
        x, w, b, dy = make(cuda, 3, shape)
        x = 0.5 * x + 500.0
        run_and_check(x, 4, w, b, dy, "none")
        y = trigrad_amd.group_norm(torch.full(shape, 7.25, device=cuda), 4, w, b)
        assert torch.equal(y, b.expand(shape))


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    import trigrad_amd
    for activation in ("none", "silu", "gelu"):
        x, w, b, _ = make(cuda, 4, (2, 3, 6), torch.float64)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        assert torch.autograd.gradcheck(lambda x, w, b: trigrad_amd.group_norm(x, 2, w, b, activation=activation), leaves)


@pytest.mark.gpu
def test_strides_and_alignment(cuda, route):
    import trigrad_amd
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, dy = make(cuda, 6, (2, 31, 24), dtype)
        run_and_check(x[..., :12], 3, w[:12], b[12:], dy[..., 4:16], "silu")
        run_and_check(x.transpose(0, 1), 4, w, b, dy.transpose(0, 1), "silu")
        flat = torch.randn((2 * 31 * 24 + 1,)).to(dtype).to(cuda)
        run_and_check(flat[1:].view(2, 31, 24), 4, w[::2].repeat_interleave(2), b, flat[:-1].view(2, 31, 24), "silu")
        # an image stored channels first, as another library hands it over, and a gradient that arrives expanded
        first = torch.randn((2, 24, 5, 7)).to(dtype).to(cuda).permute(0, 2, 3, 1)
        run_and_check(first, 4, w, b, first * 0.5, "gelu")
        leaf = x.detach().requires_grad_()
        (got,) = torch.autograd.grad(trigrad_amd.group_norm(leaf, 4, w, b, activation="silu").sum(), leaf)
        assert_near("grad_x", got, reference(x, 4, w, b, 1e-5, "silu", torch.ones_like(x))["grad_x"])


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_group(cuda):
    import trigrad_amd
    for shape in ((3, 200, 32), (1, 30000, 32), (500, 1, 32)):
        x, w, b, dy = make(cuda, 6, shape)
        clean = trigrad_amd.group_norm(x, 4, w, b, activation="relu")
        for value in (float("nan"), float("inf")):
            bad = x.clone()
            bad[0, 0, 9] = value  # the second group of the first sample
            y = trigrad_amd.group_norm(bad, 4, w, b, activation="relu")
            assert torch.isnan(y[0, :, 8:16]).all()
            y[0, :, 8:16] = clean[0, :, 8:16]
            assert torch.equal(y, clean)


@pytest.mark.gpu
def test_saturated_activations(cuda):
    """Far out the activations are 0 or z and their slopes 0 or 1: nothing overflows."""
    x, w, b, dy = make(cuda, 7, (2, 100, 16))
    b = torch.where(torch.arange(16, device=cuda) % 2 == 0, 300.0, -300.0)
    for activation in ("relu", "silu", "gelu"):
        y, dx, dw, db = run_and_check(x, 4, w, b, dy, activation)
        assert not y[..., 1::2].any() or activation == "silu" and y[..., 1::2].abs().max() < 1e-30


@pytest.mark.gpu
def test_empty_inputs(cuda, route):
    import trigrad_amd
    for shape in ((0, 5, 8), (3, 0, 8), (0, 8)):
        x = torch.zeros(shape, device=cuda, requires_grad=True)
        w, b = (torch.ones((8,), device=cuda, requires_grad=True) for _ in range(2))
        y = trigrad_amd.group_norm(x, 2, w, b)
        assert y.shape == x.shape
        grads = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
        assert torch.equal(grads[1], torch.zeros_like(w)) and torch.equal(grads[2], torch.zeros_like(b))


@pytest.mark.gpu
def test_same_bits_every_time(cuda):
    for shape, groups in (((1, 50000, 32), 8), ((3000, 1, 512), 8), ((6, 900, 64), 4)):
        x, w, b, dy = make(cuda, 6, shape, torch.bfloat16)
        import trigrad_amd
        first = None
        for _ in range(5):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = trigrad_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu")
            got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            first = first or got
            assert all(torch.equal(p, q) for p, q in zip(first, got))


@pytest.mark.gpu
def test_other_streams_and_graphs(cuda, route):
    """Two captured graphs on two streams, replayed together with eager calls between, every replay checked."""
    import trigrad_amd
    graphs = []
    for k, (shape, groups) in enumerate([((1, 40000, 32), 8), ((700, 1, 256), 4)]):
        x, w, b, dy = make(cuda, k, shape)
        leaves = [t.requires_grad_() for t in (x, w, b)]

        def step(leaves=leaves, dy=dy, groups=groups):
            y = trigrad_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu")
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        graphs.append((graph, out, step, leaves, stream))
    for turn in range(4):
        for _, _, _, leaves, _ in graphs:
            with torch.no_grad():
                leaves[0].mul_(1.0 + 0.5 * torch.rand_like(leaves[0]))
        torch.cuda.synchronize()
        for graph, _, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, step, _, _ in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_of_the_same_leaves(cuda, route):
    import trigrad_amd
    x, w, b, dy = make(cuda, 1, (2, 50, 32))
    leaf = w.requires_grad_()
    eager = trigrad_amd.group_norm(x, 4, leaf, b, activation="silu")
    want = torch.autograd.grad(eager, leaf, dy, retain_graph=True)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = torch.autograd.grad(trigrad_amd.group_norm(x, 4, leaf, b, activation="silu"), leaf, dy)[0]
        return graph, out
    with pytest.raises(RuntimeError, match="made on another stream"):
        capture()
    del eager
    graph, out = capture()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_backward_twice_and_after_a_change(cuda, route):
    import trigrad_amd
    x, w, b, dy = make(cuda, 1, (2, 300, 16))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = trigrad_amd.group_norm(*leaves[:1], 4, *leaves[1:], activation="silu")
    first, second = (torch.autograd.grad(y, leaves, dy, retain_graph=True) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    with torch.no_grad():
        w.add_(0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    assert torch.equal(trigrad_amd.group_norm(x, np.int64(4)), trigrad_amd.group_norm(x, 4))


@pytest.mark.gpu
def test_more_elements_than_31_bits_count(cuda):
    """2^31 elements and some in samples of 2^20: the last sample against the definition."""
    import trigrad_amd
    samples, positions, channels = 2 ** 11 + 2, 2 ** 12, 256
    x = torch.empty((samples, positions, channels), dtype=torch.bfloat16, device=cuda)
    for p in range(0, samples, 256):
        x[p:p + 256].normal_()
    leaf = x.requires_grad_()
    y = trigrad_amd.group_norm(leaf, 4, activation="silu")
    (got,) = torch.autograd.grad(y, leaf, x.detach())
    want = reference(x[-1:], 4, None, None, 1e-5, "silu", x.detach()[-1:])
    assert_near("y", y[-1:], want["y"])
    assert_near("grad_x", got[-1:], want["grad_x"])


@pytest.mark.gpu
def test_more_workgroups_than_22_bits_count(cuda):
    """Rows of an odd number of channels that no workgroup holds, in 18 workgroups each: the first and last rows against the definition."""
    import trigrad_amd
    samples, channels = 2 ** 18, 4353
    x = torch.empty((samples, channels), dtype=torch.bfloat16, device=cuda)
    for p in range(0, samples, 1 << 14):
        x[p:p + (1 << 14)].normal_()
    leaf = x.requires_grad_()
    y = trigrad_amd.group_norm(leaf, 1)
    (got,) = torch.autograd.grad(y, leaf, x.detach())
    for part in (slice(0, 3), slice(samples // 2, samples // 2 + 2), slice(samples - 3, samples)):
        want = reference(x[part], 1, None, None, 1e-5, "none", x.detach()[part])
        assert_near("y", y[part], want["y"])
        assert_near("grad_x", got[part], want["grad_x"])


@pytest.mark.gpu
def test_a_negation_still_to_be_done(cuda, route):
    """Tensors whose values are the negatives of what is in memory, as a conjugate's imaginary part."""
    import trigrad_amd
    x, w, b, dy = make(cuda, 7, (2, 9, 8))
    y = run_and_check(x, 2, w, b, dy, "silu")
    leaves = [torch._neg_view(-t).requires_grad_() for t in (x, w, b)]
    again = trigrad_amd.group_norm(leaves[0], 2, *leaves[1:], activation="silu")
    assert torch.equal(y[0], again)
    for want, got in zip(y[1:], torch.autograd.grad(again, leaves, torch._neg_view(-dy))):
        assert torch.equal(want, got)


@pytest.mark.gpu
def test_run_of_operators(cuda, oracle):
    """Slabs of a scene rendered apart, composited, a recurrence over their features, its states normalised by head and by frame: the image is
    that of the slabs one by one, and the gradient reaches the scene's colours."""
    import scenes as S
    import trigrad_amd
    W, H, L = 64, 48, 5
    scene = S.random_soup(400, W, H, seed=4, sigma_px=6.0)
    d = {k: torch.from_numpy(v).to(cuda) for k, v in scene.items() if isinstance(v, np.ndarray)}
    colors = d["colors"].clone().requires_grad_()
    order = d["vertices"][d["indices"].long(), 2].mean(1).argsort()
    slabs = torch.stack([trigrad_amd.render(d["vertices"], part.contiguous(), colors, d["opacities"], W, H)[0]
                         for part in d["indices"][order].chunk(L)])
    flat = slabs[None].reshape(1, L, -1, 4)
    _, image = trigrad_amd.linear_recurrence(flat[..., :3].reshape(1, L, -1), flat[..., 3], reverse=True, return_states=False)
    want = torch.zeros((H, W, 3), dtype=torch.float64, device=cuda)
    for slab in reversed(slabs.detach().double().unbind(0)):
        want = want * slab[..., 3:] + slab[..., :3]
    assert (image.detach().double().view(H, W, 3) - want).abs().max() <= 16 * L * U
    (through,) = torch.autograd.grad(image.square().sum(), colors, retain_graph=True)
    plain = torch.zeros((H, W, 3), device=cuda)
    for slab in reversed(slabs.unbind(0)):
        plain = plain * slab[..., 3:] + slab[..., :3]
    (beside,) = torch.autograd.grad(plain.square().sum(), colors, retain_graph=True)
    assert through.abs().max() > 0 and torch.allclose(through, beside, rtol=1e-4, atol=1e-5 * beside.abs().max().item())
    # rows of the image as sequences of features, a gate by head, normalised by head and then by frame
    rng = torch.Generator().manual_seed(0)
    lift = torch.randn((3, 32), generator=rng).to(cuda)
    features = image.view(H, W, 3) @ lift
    gates = torch.randn((H, W, 4), generator=rng).to(cuda)
    states, _ = trigrad_amd.linear_recurrence(features, gates, gate_form="logit", input_form="complement")
    heads = trigrad_amd.group_norm(states.reshape(-1, 32), 4, activation="silu").view(1, H, W, 32)
    out = trigrad_amd.group_norm(heads, 8, activation="gelu")
    assert out.shape == (1, H, W, 32)
    (grad,) = torch.autograd.grad(out.square().mul(torch.rand(out.shape, generator=rng).to(cuda)).sum(), colors)
    assert torch.isfinite(grad).all() and grad.abs().max() > 0


def test_refusals_without_gpu():
    import trigrad_amd
    x = torch.zeros((2, 3, 8))
    f = trigrad_amd.group_norm
    with pytest.raises(TypeError, match="x must be on cuda, but got cpu"):
        f(x, 2)
    with pytest.raises(ValueError, match="activation must be one of none, relu, silu, gelu, but got tanh"):
        f(x, 2, activation="tanh")
    with pytest.raises(TypeError, match="x must be of type"):
        f(x.int(), 2)


@pytest.mark.gpu
def test_refusals(cuda, route):
    import trigrad_amd
    f = trigrad_amd.group_norm
    x, w, b, _ = make(cuda, 1, (2, 3, 8))
    for bad, error, match in (
            (lambda: f(x, 3), ValueError, "multiple of the number of groups, but got 8 and 3"),
            (lambda: f(x, 0), ValueError, "multiple of the number of groups"),
            (lambda: f(x[0, 0], 2), ValueError, "x must have at least 2 dimensions, but got 1"),
            (lambda: f(x, 2, w[:4]), ValueError, "weight must be of shape"),
            (lambda: f(x, 2, w, b.half()), TypeError, "bias must be of type torch.float32"),
            (lambda: f(x.bfloat16(), 2, w.bfloat16(), b), TypeError, "bias must be of type torch.bfloat16, but got torch.float32"),
            (lambda: f(x, 2, w.cpu()), TypeError, "weight must be on cuda"),
            (lambda: f(x, 2, eps=-1.0), ValueError, "eps must not be negative"),
            (lambda: f(x, 2, eps=float("nan")), ValueError, "eps must not be negative")):
        with pytest.raises(error, match=match):
            bad()
    leaf = x.detach().requires_grad_()
    (grad,) = torch.autograd.grad(f(leaf, 2).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("bits", [32, 64])
def test_native_refusals(bits):
    import ctypes as C
    from trigrad_amd import _lib
    lib = _lib.load(bits)
    kind = 3 if bits == 64 else 0
    good = dict(samples=2, positions=5, channels=8, groups=4, type=kind, weight_type=kind, eps=1e-5)
    sizes = (C.c_int64 * 2)()

    def call(name, **kw):
        n = _lib.Norm(**{**good, **kw})
        return getattr(lib, name)(C.byref(n), *([sizes] if name.endswith("sizes") else []))
    assert call("tg_group_norm_sizes") == 0 and min(sizes) >= 0
    for kw in (dict(samples=-1), dict(positions=-1), dict(channels=0), dict(groups=3), dict(groups=0), dict(type=9), dict(weight_type=2 if bits == 64 else 1),
               dict(type=0 if bits == 64 else 3), dict(activation=4), dict(activation=-1), dict(eps=-1.0), dict(eps=float("nan")),
               dict(samples=1 << 31), dict(samples=1 << 20, positions=1 << 21), dict(channels=1 << 24, groups=1)):
        for name in ("tg_group_norm_sizes", "tg_group_norm_forward", "tg_group_norm_backward"):
            assert call(name, **kw) == -1, (name, kw)
    for name in ("tg_group_norm_forward", "tg_group_norm_backward"):
        assert call(name, grad_x=64) == -1 and name.encode() in lib.tg_last_error()
        assert call(name, samples=0) == 0 and call(name, positions=0) == 0
        assert getattr(lib, name)(None) == -1
