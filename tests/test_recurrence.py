"""The gated linear recurrence against its definition in 64 bits, step by step, forward and backward; the single step; refusals.

Tolerances: with a relative error of K for each step (a gate's exponential or logistic function 5 units of 2^-24, the product with the
input 1, the step's multiply-add 1, the products of gates that join pieces of a sequence 1 a step, the rest for the joints), the error of
a state obeys E_t = |a| (E_{t-1} + K M_{t-1}) + K |u_t|, where M_t = |a| M_{t-1} + |u_t| is the same recurrence of magnitudes; the
gradients' errors obey the same recurrence backwards.  Beside that an output is rounded once to its type, half a step."""
import numpy as np
import pytest
import torch

K = 12 * 2.0 ** -24


def _gate(form, g):
    if form == "value":
        return g, 1.0 - g, torch.ones_like(g)
    if form == "log":
        return torch.exp(g), -torch.expm1(g), torch.exp(g)
    return torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(g) * torch.sigmoid(-g)


def _sequences(inputs, offsets):
    """The index tuples of every sequence's rows."""
    if offsets is None:
        return [(s, slice(None)) for s in range(inputs.shape[0])]
    cuts = offsets.tolist()
    return [(slice(p, q),) for p, q in zip(cuts, cuts[1:])]


def reference(inputs, gates, initial, offsets, gate_form, input_form, reverse, grad_states=None, grad_final=None):
    """-> {name: (value, bound on the kernels' error before the last rounding)} in 64 bits, from the definition, on the CPU."""
    x_, g_ = inputs.detach().double().cpu(), gates.detach().double().cpu()
    R, D = x_.shape[-1] // g_.shape[-1], x_.shape[-1]
    cuts = _sequences(x_, offsets)
    S = len(cuts)
    h0 = initial.detach().double().cpu() if initial is not None else torch.zeros((S, D), dtype=torch.float64)
    zeros = lambda t: (torch.zeros_like(t), torch.zeros_like(t))  # noqa: E731
    out = {"states": zeros(x_), "final": zeros(h0), "grad_inputs": zeros(x_), "grad_gates": zeros(g_), "grad_initial": zeros(h0)}
    dh_ = grad_states.double().cpu() if grad_states is not None else torch.zeros_like(x_)
    df = grad_final.double().cpu() if grad_final is not None else torch.zeros_like(h0)
    for s, at in enumerate(cuts):
        x, g, dh = x_[at], g_[at], dh_[at]
        T, G = g.shape
        a, rest, slope = _gate(gate_form, g)
        wide, wide_rest = a.repeat_interleave(R, -1), rest.repeat_interleave(R, -1)
        u = x if input_form == "plain" else wide_rest * x
        order = range(T - 1, -1, -1) if reverse else range(T)
        h, m, e = h0[s], h0[s].abs(), torch.zeros(D, dtype=torch.float64)
        states, errors, before, before_e, before_m = (torch.zeros_like(x) for _ in range(5))
        for t in order:
            before[t], before_e[t], before_m[t] = h, e, m
            e = wide[t].abs() * (e + K * m) + K * u[t].abs()
            m = wide[t].abs() * m + u[t].abs()
            h = wide[t] * h + u[t]
            states[t], errors[t] = h, e
        out["states"][0][at], out["states"][1][at] = states, errors
        out["final"][0][s], out["final"][1][s] = h, e
        lam, lam_m, lam_e = df[s], df[s].abs(), torch.zeros(D, dtype=torch.float64)
        dx, dx_e = torch.zeros_like(x), torch.zeros_like(x)
        da, da_e = torch.zeros_like(x), torch.zeros_like(x)
        for t in reversed(order):
            lam, lam_m, lam_e = lam + dh[t], lam_m + dh[t].abs(), lam_e + K * (lam_m + dh[t].abs())
            scale = 1.0 if input_form == "plain" else wide_rest[t]
            dx[t], dx_e[t] = lam * scale, (lam_e + K * lam_m) * abs(scale)
            there = before[t] if input_form == "plain" else before[t] - x[t]
            size = before_m[t] if input_form == "plain" else before_m[t] + x[t].abs()
            da[t] = lam * there
            da_e[t] = lam_e * size + lam_m * (before_e[t] + K * size)
            lam, lam_m, lam_e = wide[t] * lam, wide[t].abs() * lam_m, wide[t].abs() * (lam_e + K * lam_m)
        # a sum over the R channels of a gate: four in a lane, a tree over a wave, then the waves' sums
        depth = (16 + R / 64) * 2.0 ** -24
        magnitude = (da.abs() + da_e).reshape(T, G, R).sum(-1)
        out["grad_inputs"][0][at], out["grad_inputs"][1][at] = dx, dx_e
        out["grad_gates"][0][at] = da.reshape(T, G, R).sum(-1) * slope
        out["grad_gates"][1][at] = (da_e.reshape(T, G, R).sum(-1) + (depth + K) * magnitude) * slope.abs()
        out["grad_initial"][0][s], out["grad_initial"][1][s] = lam, lam_e
    return out


def assert_near(name, got, wanted):
    want, bound = wanted
    assert got.shape == want.shape, name
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float64 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # half a step of numbers below the normal ones
    allowed = (bound + want.abs()) * half + bound + tiny + 1e-30
    off = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(off).all(), f"{name}: not finite"
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} of the bound at {np.unravel_index(int((off / allowed).argmax()), off.shape)}"


def make(cuda, seed, rows, channels, gates, dtype=torch.float32, gate_dtype=None, gate_form="value", sequences=None, initial=True):
    rng = torch.Generator().manual_seed(seed)
    x = torch.randn((*rows, channels), generator=rng)
    g = torch.randn((*rows, gates), generator=rng)
    g = {"value": lambda: torch.sigmoid(g + 1.5), "log": lambda: -torch.exp(1.5 * g - 3.0), "logit": lambda: 1.5 * g + 2.0}[gate_form]()
    h0 = torch.randn((sequences if sequences is not None else rows[0], channels), generator=rng) if initial else None
    real = torch.float64 if dtype == torch.float64 else torch.float32
    return (x.to(dtype).to(cuda), g.to(gate_dtype or dtype).to(cuda), None if h0 is None else h0.to(real).to(cuda), rng)


def run_and_check(x, g, h0, offsets=None, gate_form="value", input_form="plain", reverse=False, return_states=True, use_final=True, rng=None):
    import trigrad_amd
    x, g = x.detach().requires_grad_(), g.detach().requires_grad_()
    h0 = h0.detach().requires_grad_() if h0 is not None else None
    states, final = trigrad_amd.linear_recurrence(x, g, h0, offsets, gate_form, input_form, reverse, return_states)
    dh = torch.randn(x.shape, generator=rng).to(x.dtype).to(x.device) if return_states else None
    df = torch.randn(final.shape, generator=rng).to(final.dtype).to(x.device) if use_final or not return_states else None
    ends = [(o, d) for o, d in ((states, dh), (final, df)) if d is not None]
    leaves = [t for t in (x, g, h0) if t is not None]
    grads = torch.autograd.grad([o for o, _ in ends], leaves, [d for _, d in ends])
    want = reference(x, g, h0, None if offsets is None else offsets.cpu(), gate_form, input_form, reverse, dh, df)
    if return_states:
        assert states.dtype == x.dtype
        assert_near("states", states, want["states"])
    else:
        assert states is None
    assert_near("final", final, want["final"])
    for name, got, leaf in zip(("grad_inputs", "grad_gates", "grad_initial"), grads, leaves):
        assert got.dtype == leaf.dtype
        assert_near(name, got, want[name])
    return states, final, grads


TYPES = {"f32": (torch.float32, None), "bf16": (torch.bfloat16, None), "f16": (torch.float16, None),
         "bf16_f32": (torch.bfloat16, torch.float32), "f16_f32": (torch.float16, torch.float32), "f64": (torch.float64, None)}


@pytest.fixture(params=["module", "python"])
def route(request, monkeypatch):
    """Calls by the torch module, which takes the ordinary ones, and all of them by the Python functions."""
    from trigrad_amd import _C
    monkeypatch.setattr(_C, "ONE_CALL_OPERATORS", request.param == "module")


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("input_form", ["plain", "complement"])
@pytest.mark.parametrize("gate_form", ["value", "log", "logit"])
@pytest.mark.parametrize("types", sorted(TYPES))
def test_forms_and_types(types, gate_form, input_form, reverse, cuda, route):
    dtype, gate_dtype = TYPES[types]
    for seed, (rows, channels, gates) in enumerate([((3, 37), 24, 24), ((2, 70), 40, 10), ((1, 300), 6, 2)]):
        x, g, h0, rng = make(cuda, seed, rows, channels, gates, dtype, gate_dtype, gate_form, initial=seed != 1)
        run_and_check(x, g, h0, None, gate_form, input_form, reverse, rng=rng)


LENGTHS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 1025]


@pytest.mark.gpu
@pytest.mark.parametrize("length", LENGTHS)
def test_lengths(length, cuda):
    for seed, (S, channels, gates, dtype) in enumerate([(1, 64, 64, torch.float32), (3, 20, 5, torch.bfloat16), (2, 130, 1, torch.float16)]):
        x, g, h0, rng = make(cuda, seed + length, (S, length), channels, gates, dtype)
        run_and_check(x, g, h0, input_form="complement" if seed == 1 else "plain", reverse=seed == 2, rng=rng)


@pytest.mark.gpu
@pytest.mark.parametrize("channels,gates", [(1, 1), (2, 2), (2, 1), (3, 1), (5, 5), (6, 2), (12, 3), (15, 3), (33, 33), (64, 2), (96, 1),
                                            (100, 4), (129, 43), (256, 1), (257, 257), (260, 1), (384, 3), (520, 2), (1000, 1), (1028, 4), (1280, 320)])
def test_channels_and_shared_gates(channels, gates, cuda):
    for seed, (rows, dtype) in enumerate([((2, 45), torch.float32), ((1, 150), torch.bfloat16)]):
        x, g, h0, rng = make(cuda, seed + channels, rows, channels, gates, dtype, gate_form="logit")
        run_and_check(x, g, h0, gate_form="logit", input_form="complement", reverse=seed == 1, rng=rng)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels,gates,dtype", [((1, 9001), 8, 8, torch.float32), ((2, 4500), 64, 64, torch.bfloat16),
                                                       ((1, 6000), 128, 2, torch.float16), ((1, 5000), 1, 1, torch.float32),
                                                       ((3, 2200), 260, 65, torch.bfloat16)])
def test_long_sequences(rows, channels, gates, dtype, cuda):
    x, g, h0, rng = make(cuda, 7, rows, channels, gates, dtype, torch.float32, "log")
    run_and_check(x, g, h0, gate_form="log", rng=rng)
    run_and_check(x, g, None, gate_form="log", input_form="complement", reverse=True, rng=rng)


def _offsets(rng, total, sequences, first=0, pad=0):
    cuts = rng.integers(first, total - pad + 1, sequences + 1)
    cuts.sort()
    cuts[0], cuts[-1] = first, total - pad
    return torch.from_numpy(cuts.astype(np.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("total,sequences,first,pad", [(1, 1, 0, 0), (40, 7, 0, 3), (700, 1, 5, 9), (700, 90, 0, 0), (1500, 900, 3, 0), (5200, 6, 0, 600),
                                                       (64, 3, 64, 0)])
def test_packed_sequences(total, sequences, first, pad, reverse, cuda):
    """Sequences end to end, many of them empty, rows of none in front and behind."""
    cuts = _offsets(np.random.default_rng(total), total, sequences, first, pad)
    for seed, (channels, gates, dtype) in enumerate([(12, 12, torch.float32), (40, 5, torch.bfloat16), (3, 1, torch.float32), (300, 1, torch.float16)]):
        x, g, h0, rng = make(cuda, seed, (total,), channels, gates, dtype, sequences=sequences)
        run_and_check(x, g, h0, cuts.to(cuda), input_form="complement" if seed % 2 else "plain", reverse=reverse, rng=rng)
        run_and_check(x, g, None, cuts.to(cuda), reverse=reverse, use_final=False, rng=rng)


@pytest.mark.gpu
def test_sequence_ends_on_every_row_of_a_piece(cuda):
    """Sequences of one to three rows around each other: an end and a start in every place that a thread's, a wave's or a workgroup's rows end at."""
    lengths = [1, 2, 3, 0, 1, 1, 0, 0, 2, 5, 4, 0, 8, 7, 9, 16, 15, 17, 31, 64, 63, 65, 1] * 12
    cuts = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32))
    for channels, gates in ((4, 4), (64, 1), (1, 1)):
        x, g, h0, rng = make(cuda, channels, (int(cuts[-1]),), channels, gates, torch.float32, sequences=len(lengths))
        run_and_check(x, g, h0, cuts.to(cuda), rng=rng)


@pytest.mark.gpu
def test_only_the_final_state(cuda, route):
    """The compositing call: no states out, no gradient of them in; a short axis and very many channels, three to a gate."""
    for rows, channels, gates in (((1, 8), 3 * 5000, 5000), ((4, 3), 600, 200), ((1, 700), 12, 12)):
        x, g, h0, rng = make(cuda, 3, rows, channels, gates)
        run_and_check(x, g, h0, reverse=True, return_states=False, rng=rng)


@pytest.mark.gpu
def test_gradients_that_are_asked_for(cuda, route):
    import trigrad_amd
    x, g, h0, rng = make(cuda, 5, (2, 90), 24, 6)
    _, _, full = run_and_check(x, g, h0, use_final=False, rng=torch.Generator().manual_seed(9))
    dh = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(cuda)
    for k in range(3):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, g, h0))]
        states, _ = trigrad_amd.linear_recurrence(*leaves)
        (one,) = torch.autograd.grad(states, leaves[k], dh)
        assert torch.equal(one, full[k])
    states, final = trigrad_amd.linear_recurrence(x, g, h0)
    assert not states.requires_grad and not final.requires_grad


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """torch.autograd.gradcheck in float64 (differences of the forward pass), as the components' derivatives are checked."""
    import trigrad_amd
    cuts = torch.tensor([0, 3, 3, 8], dtype=torch.int32, device=cuda)
    for gate_form in ("value", "log", "logit"):
        for input_form in ("plain", "complement"):
            x, g, h0, _ = make(cuda, 2, (2, 5), 6, 3, torch.float64, None, gate_form)
            leaves = [t.requires_grad_() for t in (x, g, h0)]
            assert torch.autograd.gradcheck(lambda *t: trigrad_amd.linear_recurrence(*t, None, gate_form, input_form, True), leaves)
            x, g, h0, _ = make(cuda, 2, (9,), 4, 2, torch.float64, None, gate_form, sequences=3)
            leaves = [t.requires_grad_() for t in (x, g, h0)]
            assert torch.autograd.gradcheck(lambda *t: trigrad_amd.linear_recurrence(*t, cuts, gate_form, input_form), leaves)


@pytest.mark.gpu
def test_strides_and_alignment(cuda, route):
    """Views: channels taken out of wider rows, rows transposed, storage that begins off a vector's alignment."""
    import trigrad_amd
    for dtype in (torch.float32, torch.bfloat16):
        rng = torch.Generator().manual_seed(1)
        image = torch.rand((6, 50, 4), generator=rng).to(dtype).to(cuda)
        run_and_check(image[..., :3], image[..., 3:], None, reverse=True, rng=rng)
        x, g, h0, rng = make(cuda, 4, (40, 3), 16, 16, dtype)
        run_and_check(x.transpose(0, 1), g.transpose(0, 1), h0[:3], rng=rng)
        flat = torch.randn((2 * 40 * 16 + 1,), generator=rng).to(dtype).to(cuda)
        gate = torch.rand((2 * 40 * 16 + 1,), generator=rng).to(dtype).to(cuda)
        run_and_check(flat[1:].view(2, 40, 16), gate[1:].view(2, 40, 16), None, rng=rng)
        # a gradient that arrives expanded
        leaf = x.detach().requires_grad_()
        states, _ = trigrad_amd.linear_recurrence(leaf, g)
        (got,) = torch.autograd.grad(states.sum(), leaf)
        want = reference(x, g, None, None, "value", "plain", False, torch.ones_like(x))
        assert_near("grad_inputs", got, want["grad_inputs"])


@pytest.mark.gpu
def test_a_negation_still_to_be_done(cuda, route):
    """Tensors whose values are the negatives of what is in memory, as a conjugate's imaginary part."""
    import trigrad_amd
    x, g, h0, rng = make(cuda, 5, (2, 40), 6, 3)
    ends = [torch.randn(s, generator=rng).to(cuda) for s in ((2, 40, 6), (2, 6))]
    plain = [t.clone().requires_grad_() for t in (x, g, h0)]
    negated = [torch._neg_view(-t).requires_grad_() for t in (x, g, h0)]
    results = []
    for leaves, given in ((plain, ends), (negated, [torch._neg_view(-t) for t in ends])):
        out = trigrad_amd.linear_recurrence(*leaves)
        results.append([*out, *torch.autograd.grad(out, leaves, given)])
    assert all(torch.equal(want, got) for want, got in zip(*results))
    with torch.no_grad():
        want = trigrad_amd.linear_recurrence_step(x[:, 0], g[:, 0], h0.clone())
        got = trigrad_amd.linear_recurrence_step(negated[0][:, 0], negated[1][:, 0], h0.clone())
        assert all(torch.equal(*pair) for pair in zip(want, got))
        with pytest.raises(ValueError, match="no negation"):
            trigrad_amd.linear_recurrence_step(x[:, 0], g[:, 0], torch._neg_view(h0))


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_nothing_leaks_across_sequences(reverse, cuda):
    """NaN and infinities in one sequence, and in rows that belong to none, leave the others' states and gradients as they are."""
    import trigrad_amd
    cuts = torch.tensor([2, 30, 30, 95, 400, 1300], dtype=torch.int32, device=cuda)
    for channels, gates in ((8, 8), (64, 4)):
        x, g, h0, rng = make(cuda, 8, (1310,), channels, gates, sequences=5)
        dh, df = torch.randn(x.shape, generator=rng).to(cuda), torch.randn(h0.shape, generator=rng).to(cuda)

        def run(x, g, h0, dh):
            leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
            out = trigrad_amd.linear_recurrence(*leaves, cuts, reverse=reverse)
            return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (dh, df)))
        clean = run(x, g, h0, dh)
        bad = [t.clone() for t in (x, g, h0, dh)]
        for t in bad[:2] + bad[3:]:
            t[95:400] = float("nan")
            t[:2], t[1300:] = float("inf"), float("-inf")
        bad[0][200] = float("inf")
        dirty = run(*bad)
        rows = torch.ones(1310, dtype=torch.bool, device=cuda)
        rows[95:400] = False
        for k in (0, 2, 3):
            assert torch.equal(clean[k][rows], dirty[k][rows])
        for k in (0, 2, 3):
            assert not dirty[k][:2].any() and not dirty[k][1300:].any()
        others = [0, 1, 2, 4]
        for k in (1, 4):
            assert torch.equal(clean[k][others], dirty[k][others])
        assert torch.isnan(dirty[0][300]).all() and torch.isnan(dirty[1][3]).all()


@pytest.mark.gpu
def test_nan_is_kept_from_where_it_enters(cuda):
    import trigrad_amd
    x, g, h0, _ = make(cuda, 8, (1, 3000), 8, 8)
    x[0, 1200, 3] = float("nan")
    states, final = trigrad_amd.linear_recurrence(x, g, h0)
    bad = torch.isnan(states[0])
    assert not bad[:1200].any() and bad[1200:, 3].all() and not bad[:, :3].any() and not bad[:, 4:].any()
    assert torch.isnan(final[0, 3])


@pytest.mark.gpu
def test_gates_of_zero_one_and_more(cuda):
    """Gates of 0 forget, gates of 1 sum up (exact in small integers), gates above 1 grow, also from states that are 0 for long."""
    import trigrad_amd
    T = 3000
    x = torch.randint(-3, 4, (1, T, 16), generator=torch.Generator().manual_seed(3)).float().to(cuda)
    states, final = trigrad_amd.linear_recurrence(x, torch.ones_like(x))
    assert torch.equal(states, x.cumsum(1)) and torch.equal(final, x.sum(1))
    states, _ = trigrad_amd.linear_recurrence(x, torch.zeros_like(x))
    assert torch.equal(states, x)
    x = torch.zeros((1, T, 16), device=cuda)
    x[0, T - 20] = 1.0
    states, final = trigrad_amd.linear_recurrence(x, torch.full_like(x, 2.0))
    want = torch.zeros_like(x)
    want[0, T - 20:] = (1 << torch.arange(20, device=cuda)).float()[:, None]
    assert torch.equal(states, want) and torch.equal(final, want[:, -1])


@pytest.mark.gpu
def test_empty_inputs(cuda, route):
    import trigrad_amd
    for shape, gates in (((0, 5, 8), 8), ((3, 0, 8), 2), ((2, 4, 0), 0)):
        x = torch.zeros(shape, device=cuda, requires_grad=True)
        if shape[2] == 0:
            with pytest.raises(ValueError, match="multiple of the number of gates"):
                trigrad_amd.linear_recurrence(x, torch.zeros((*shape[:2], gates), device=cuda))
            continue
        g = torch.zeros((*shape[:2], gates), device=cuda, requires_grad=True)
        h0 = torch.randn((shape[0], shape[2]), device=cuda).requires_grad_()
        states, final = trigrad_amd.linear_recurrence(x, g, h0)
        assert states.shape == x.shape and torch.equal(final, h0)
        grads = torch.autograd.grad([states, final], [x, g, h0], [torch.zeros_like(states), torch.ones_like(final)])
        assert torch.equal(grads[2], torch.ones_like(h0))
        assert torch.equal(trigrad_amd.linear_recurrence(x, g)[1], torch.zeros_like(h0))
    x = torch.zeros((0, 8), device=cuda)
    states, final = trigrad_amd.linear_recurrence(x, x, None, torch.zeros(4, dtype=torch.int32, device=cuda))
    assert states.shape == (0, 8) and torch.equal(final, torch.zeros((3, 8), device=cuda))


@pytest.mark.gpu
def test_same_bits_every_time(cuda):
    """Sums do not depend on which workgroup comes first."""
    for rows, channels, gates, cuts in (((1, 9000), 192, 192, None), ((1, 5000), 1024, 1, None), ((9000,), 96, 8, _offsets(np.random.default_rng(1), 9000, 40))):
        x, g, h0, _ = make(cuda, 6, rows, channels, gates, torch.bfloat16, sequences=None if cuts is None else 40)
        cuts = None if cuts is None else cuts.to(cuda)
        first = None
        for _ in range(5):
            import trigrad_amd
            leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
            out = trigrad_amd.linear_recurrence(*leaves, cuts)
            got = [*out, *torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])]
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.gpu
def test_other_streams_and_graphs(cuda, route):
    """Two captured graphs on two streams, replayed in turn with eager calls between, every replay checked."""
    import trigrad_amd
    graphs = []
    for k, (rows, channels, gates) in enumerate([((1, 5000), 64, 64), ((2, 3000), 256, 2)]):
        x, g, h0, rng = make(cuda, k, rows, channels, gates)
        dh = torch.randn(x.shape, generator=rng).to(cuda)
        leaves = [t.requires_grad_() for t in (x, g, h0)]

        def step(leaves=leaves, dh=dh):
            states, final = trigrad_amd.linear_recurrence(*leaves)
            return [states.detach(), final.detach(), *torch.autograd.grad(states, leaves, dh)]
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
        for graph, out, step, leaves, stream in graphs:
            with torch.no_grad():
                leaves[0].add_(0.25)
        torch.cuda.synchronize()
        for graph, _, _, _, stream in graphs:  # both under way at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, out, step, leaves, stream in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_of_the_same_leaves(cuda, route):
    """The engine would join the eager graph's stream into the capture: refused, and taken once that graph is gone."""
    import trigrad_amd
    x, g, _, _ = make(cuda, 1, (2, 50), 32, 32)
    leaf = x.requires_grad_()
    eager = trigrad_amd.linear_recurrence(leaf, g)[0]
    want = torch.autograd.grad(eager, leaf, torch.ones_like(eager), retain_graph=True)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            states, _ = trigrad_amd.linear_recurrence(leaf, g)
            out = torch.autograd.grad(states, leaf, torch.ones_like(states))[0]
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
    x, g, h0, _ = make(cuda, 1, (2, 300), 16, 16)
    leaves = [t.requires_grad_() for t in (x, g, h0)]
    states, final = trigrad_amd.linear_recurrence(*leaves)
    first = torch.autograd.grad([states, final], leaves, [torch.ones_like(states), torch.ones_like(final)], retain_graph=True)
    second = torch.autograd.grad([states, final], leaves, [torch.ones_like(states), torch.ones_like(final)], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.no_grad():
        g.add_(0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(states, leaves, torch.ones_like(states))
    # a state that a step writes over is a change too
    _, final = trigrad_amd.linear_recurrence(*leaves)
    kept = final.square()
    with torch.no_grad():
        trigrad_amd.linear_recurrence_step(x[:, 0], g[:, 0], final.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


@pytest.mark.gpu
def test_offsets_beyond_the_rows_end_at_them(cuda):
    import trigrad_amd
    x, g, h0, _ = make(cuda, 1, (100,), 8, 8, sequences=4)
    for given, meant in (([0, 40, 130, 150, 150], [0, 40, 100, 100, 100]), ([-7, 3, 3, 90, 1000], [0, 3, 3, 90, 100])):
        a, b = (trigrad_amd.linear_recurrence(x, g, h0, torch.tensor(c, dtype=torch.int32, device=cuda)) for c in (given, meant))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_more_elements_than_31_bits_count(cuda):
    """2^31 elements and some: the last rows against the definition, started far enough before them that what is in front is forgotten."""
    import trigrad_amd
    rows, channels, tail = 2 ** 20 + 77, 2048, 400
    x = torch.empty((1, rows, channels), dtype=torch.bfloat16, device=cuda)
    g = torch.full((1, rows, 1), 0.5, dtype=torch.bfloat16, device=cuda)
    for p in range(0, rows, 1 << 18):
        x[:, p:p + (1 << 18)].normal_()
    states, final = trigrad_amd.linear_recurrence(x, g)
    want = reference(x[:, -tail:], g[:, -tail:], None, None, "value", "plain", False)
    assert_near("states", states[:, -200:], tuple(t[:, -200:] for t in want["states"]))
    assert_near("final", final, want["final"])
    del states
    leaf = x.requires_grad_()
    states, _ = trigrad_amd.linear_recurrence(leaf, g)
    (got,) = torch.autograd.grad(states, leaf, x.detach())
    want = reference(x[:, -tail:], g[:, -tail:], None, None, "value", "plain", False, x.detach()[:, -tail:])
    assert_near("grad_inputs", got[:, -tail:], want["grad_inputs"])


@pytest.mark.gpu
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("sequences,channels,gates", [(1, 1, 1), (1, 1024, 1024), (3, 30, 10), (7, 129, 129), (33, 256, 2), (2, 260, 1)])
def test_step(sequences, channels, gates, types, cuda, route):
    """One step is a sequence of one row, in place or beside the state."""
    import trigrad_amd
    dtype, gate_dtype = TYPES[types]
    for gate_form in ("value", "log", "logit"):
        for input_form in ("plain", "complement"):
            x, g, state, _ = make(cuda, channels, (sequences,), channels, gates, dtype, gate_dtype, gate_form)
            want = reference(x[:, None], g[:, None], state, None, gate_form, input_form, False)
            beside, before = torch.empty_like(state), state.clone()
            h, new = trigrad_amd.linear_recurrence_step(x, g, state, gate_form, input_form, out=beside)
            assert new is beside and torch.equal(state, before) and h.dtype == dtype
            assert_near("state", new, want["final"])
            assert_near("states", h[:, None], want["states"])
            h2, new = trigrad_amd.linear_recurrence_step(x, g, state, gate_form, input_form)
            assert new is state and torch.equal(state, beside) and torch.equal(h, h2)


@pytest.mark.gpu
def test_step_after_step_is_the_sequence(cuda, route):
    import trigrad_amd
    x, g, h0, _ = make(cuda, 1, (4, 30), 96, 12, torch.bfloat16, torch.float32, "logit")
    want = reference(x, g, h0, None, "logit", "complement", False)
    state = h0.clone()
    with torch.no_grad():
        h = [trigrad_amd.linear_recurrence_step(x[:, t], g[:, t], state, "logit", "complement")[0] for t in range(30)]
    assert_near("states", torch.stack(h, 1), want["states"])
    assert_near("final", state, want["final"])
    # the prompt as a sequence, then one step from its final state
    _, state = trigrad_amd.linear_recurrence(x[:, :29], g[:, :29], h0, gate_form="logit", input_form="complement")
    trigrad_amd.linear_recurrence_step(x[:, 29], g[:, 29], state, "logit", "complement")
    assert_near("final", state, want["final"])


def test_refusals_without_gpu():
    import trigrad_amd
    from trigrad_amd import _C
    x, g = torch.zeros((2, 3, 8)), torch.zeros((2, 3, 4))
    f = trigrad_amd.linear_recurrence
    with pytest.raises(TypeError, match="inputs must be on cuda, but got cpu"):
        f(x, g)
    with pytest.raises(ValueError, match="gate_form must be one of value, log, logit, but got exp"):
        f(x, g, gate_form="exp")
    with pytest.raises(ValueError, match="input_form must be one of plain, complement, but got sqrt"):
        f(x, g, input_form="sqrt")
    with pytest.raises(TypeError, match="inputs must be of type"):
        f(x.int(), g)
    with pytest.raises(ValueError, match="inputs must have 3 dimensions, but got 2"):
        f(x[0], g[0])
    with pytest.raises(ValueError, match="inputs must have 2 dimensions, but got 3"):
        f(x, g, None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="inputs must have 2 dimensions, but got 3"):
        trigrad_amd.linear_recurrence_step(x, g, torch.zeros((2, 8)))
    assert set(_C.TYPE_CODES.values()) == {0, 1, 2, 3}


@pytest.mark.gpu
def test_refusals(cuda, route):
    import trigrad_amd
    f, step = trigrad_amd.linear_recurrence, trigrad_amd.linear_recurrence_step
    x, g, h0, _ = make(cuda, 1, (2, 3), 8, 4)
    cuts = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    for bad, error, match in (
            (lambda: f(x, g[:, :2]), ValueError, "gates must be of shape"),
            (lambda: f(x, torch.zeros((2, 3, 3), device=cuda)), ValueError, "multiple of the number of gates, but got 8 and 3"),
            (lambda: f(x, g.cpu()), TypeError, "gates must be on cuda"),
            (lambda: f(x, g.half()), TypeError, "gates must be of type torch.float32"),
            (lambda: f(x.bfloat16(), g.half()), TypeError, "gates must be of type torch.bfloat16"),
            (lambda: f(x, g, h0[:1]), ValueError, "initial must be of shape"),
            (lambda: f(x.bfloat16(), g, h0.bfloat16()), TypeError, "initial must be of type torch.float32"),
            (lambda: f(x[0], g[0], None, cuts.long()), TypeError, "offsets must be of type torch.int32"),
            (lambda: f(x[0], g[0], None, cuts.cpu()), TypeError, "offsets must be on cuda"),
            (lambda: f(x[0], g[0], None, cuts[:1]), ValueError, "offsets must be of shape"),
            (lambda: f(x[0], g[0], h0, cuts), ValueError, "initial must be of shape"),
            (lambda: step(x[:, 0], g[:, 0], h0[:, :4]), ValueError, "state must be of shape"),
            (lambda: step(x[:, 0], g[:, 0], h0.half()), TypeError, "state must be of type torch.float32"),
            (lambda: step(x[:, 0], g[:, 0], torch.zeros((8, 2), device=cuda).t()), ValueError, "state must be contiguous"),
            (lambda: step(x[:, 0], g[:, 0], h0, out=h0[:1]), ValueError, "out must be of shape"),
            (lambda: step(x[:, 0], g[:, 0], h0, out=x.view(-1)[:16].view(2, 8)), ValueError, "inputs must not overlap"),
            (lambda: step(x[:, 0], g[:, 0], h0, out=g.view(-1)[:16].view(2, 8)), ValueError, "gates must not overlap"),
            (lambda: step(x[:1, 0], g[:1, 0], h0.view(-1)[:8].view(1, 8), out=h0.view(-1)[4:12].view(1, 8)), ValueError, "out must be state itself"),
            (lambda: step(x[:, 0].requires_grad_(), g[:, 0], h0), RuntimeError, "linear_recurrence_step has no gradient")):
        with pytest.raises(error, match=match):
            bad()
    # a gradient of the gradient is refused, not wrong
    leaf = x.detach().requires_grad_()
    states, _ = f(leaf, g)
    (grad,) = torch.autograd.grad(states.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("bits", [32, 64])
def test_native_refusals(bits):
    """The C entry points reject bad arguments before any device work."""
    import ctypes as C
    from trigrad_amd import _lib
    lib = _lib.load(bits)
    kind = 3 if bits == 64 else 0
    good = dict(sequences=2, length=5, channels=8, gate_count=4, type=kind, gate_type=kind)
    sizes = (C.c_int64 * 3)()

    def call(name, **kw):
        r = _lib.Recurrence(**{**good, **kw})
        return getattr(lib, name)(C.byref(r), *([sizes] if name.endswith("sizes") else []))
    assert call("tg_linear_recurrence_sizes") == 0 and min(sizes) >= 0
    for kw in (dict(sequences=-1), dict(length=-1), dict(channels=-8), dict(gate_count=3), dict(gate_count=0), dict(type=7), dict(gate_type=2 if bits == 64 else 1),
               dict(type=0 if bits == 64 else 3), dict(gate_form=3), dict(gate_form=-1), dict(input_form=2), dict(sequences=1 << 30, length=1 << 30),
               dict(length=1 << 31, offsets=64), dict(channels=1 << 31, gate_count=1)):
        for name in ("tg_linear_recurrence_sizes", "tg_linear_recurrence_forward", "tg_linear_recurrence_backward"):
            assert call(name, **kw) == -1, (name, kw)
    for name in ("tg_linear_recurrence_forward", "tg_linear_recurrence_backward"):
        assert call(name) == -1 and name.encode() in lib.tg_last_error()  # null pointers
        assert call(name, channels=0, gate_count=0) == 0 and call(name, sequences=0) == 0  # nothing to do
        assert getattr(lib, name)(None) == -1
    assert call("tg_linear_recurrence_backward", length=5000, inputs=64, gates=64, kept=64, kept_bytes=1 << 30) == -2
    assert lib.tg_linear_recurrence_step(None, None, None, None, None, 2, 8, 4, kind, kind, 0, 0, None) == -1
    assert lib.tg_linear_recurrence_step(None, None, None, None, None, 2, 8, 3, kind, kind, 0, 0, None) == -1
    assert lib.tg_linear_recurrence_step(None, None, None, None, None, 0, 8, 4, kind, kind, 0, 0, None) == 0
