"""The gated linear recurrence over axes of many chunks: the states that chunks start from, composed over long runs of chunks, and tensors off a
vector's alignment there.

Gates of exactly 0 and 1 on small integers are exact in 32 bits, however the pieces are joined, so these results have to be equal.  For
other gates the tolerance is that of test_recurrence.py, a relative error of K for each step carried along by the recurrences themselves, computed here by
doubling in 64 bits."""
import numpy as np
import pytest
import torch

from test_recurrence import K, _gate, _offsets, assert_near


def _doubled(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 0 from 0, in 64 bits."""
    a, u, width = a.clone(), u.clone(), 1
    while width < len(u):
        u[width:] = u[width:] + a[width:] * u[:-width]
        a[width:] = a[width:] * a[:-width]
        width *= 2
    return u


def reference(x, g, h0, offsets, gate_form, input_form, reverse, dh, df):
    """-> {name: (value, bound before the last rounding)}; (S, T, D) or packed, all sequences end to end as one axis."""
    S, D = h0.shape
    R = D // g.shape[-1]
    rows = x.numel() // D
    place = torch.arange(rows, device=x.device)
    if offsets is None:
        begin, end = (torch.arange(S, device=x.device) + k for k in (0, 1))
        begin, end = begin * (rows // S), end * (rows // S)
    else:
        begin, end = offsets[:-1].long(), offsets[1:].long()
    of = torch.searchsorted(end, place, right=True).clamp_max(S - 1)
    inside = ((place >= begin[of]) & (place < end[of]))[:, None]
    first, last = (place == begin[of])[:, None] & inside, (place == end[of] - 1)[:, None] & inside
    if reverse:
        first, last = last, first
    order = (lambda t: t.flip(0)) if reverse else (lambda t: t)
    back = (lambda t: t) if reverse else (lambda t: t.flip(0))
    step = -1 if reverse else 1
    before = lambda t, start: torch.where(first, start, t.roll(step, 0))  # noqa: E731
    after = lambda t, start: torch.where(last, start, t.roll(-step, 0))  # noqa: E731
    x, dh = (torch.where(inside, t.detach().double().reshape(rows, D), 0.0) for t in (x, dh))
    a, rest, slope = (torch.where(inside, t, 0.0) for t in _gate(gate_form, g.detach().double().reshape(rows, -1)))
    a, rest = a.repeat_interleave(R, -1), rest.repeat_interleave(R, -1)
    h0, df = h0.detach().double(), df.double()
    start, final = h0[of], df[of]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    u = x if input_form == "plain" else rest * x
    through = torch.where(first, zero, a)
    forward = lambda u: order(_doubled(order(through), order(u)))  # noqa: E731
    h = forward(u + torch.where(first, a * start, zero))
    m = forward(u.abs() + torch.where(first, a.abs() * start.abs(), zero))
    hb, mb = before(h, start), before(m, start.abs())
    e = forward(K * (a.abs() * mb + u.abs()))
    eb = before(e, zero)
    through = torch.where(inside, after(a, zero), zero)
    backward = lambda u: back(_doubled(back(through), back(u)))  # noqa: E731
    lam = backward(dh + torch.where(last, final, zero))
    lam_m = backward(dh.abs() + torch.where(last, final.abs(), zero))
    lam_e = backward(K * (lam_m + through.abs() * after(lam_m, zero)))
    scale = 1.0 if input_form == "plain" else rest
    there, size = (hb, mb) if input_form == "plain" else (hb - x, mb + x.abs())
    da, da_e = lam * there, lam_e * size + lam_m * (eb + K * size)
    by_gate = lambda t: t.reshape(rows, -1, R).sum(-1)  # noqa: E731
    ends = lambda t, none: torch.where((begin == end)[:, None], none, t[(begin if reverse else end - 1).clamp(0, rows - 1)])  # noqa: E731
    starts = lambda t, none: torch.where((begin == end)[:, None], none, t[(end - 1 if reverse else begin).clamp(0, rows - 1)])  # noqa: E731
    cpu = lambda *t: tuple(v.cpu() for v in t)  # noqa: E731
    return {"states": cpu(torch.where(inside, h, zero), e), "final": cpu(ends(h, h0), ends(e, zero)),
            "grad_inputs": cpu(torch.where(inside, lam, zero) * scale, (lam_e + K * lam_m) * abs(scale)),
            "grad_gates": cpu(by_gate(da) * slope, (by_gate(da_e) + (K + (16 + R / 64) * 2.0 ** -24) * by_gate(da.abs() + da_e)) * slope.abs()),
            "grad_initial": cpu(starts(a * lam, df), starts(a.abs() * (lam_e + K * lam_m), zero))}


def run(x, g, h0, offsets, gate_form, input_form, reverse, dh, df):
    import trigrad_amd
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    out = trigrad_amd.linear_recurrence(*leaves, offsets, gate_form, input_form, reverse)
    grads = torch.autograd.grad(out, leaves, [dh, df])
    return dict(zip(("states", "final", "grad_inputs", "grad_gates", "grad_initial"), (*out, *grads)))


def check(*args, exact=False):
    want = reference(*args)
    for name, got in run(*args).items():
        value, bound = want[name]
        got = got.detach().cpu().reshape(value.shape)
        if exact:
            assert torch.equal(got, value.to(got.dtype)), name
        else:
            assert_near(name, got, (value, bound))


def whole_numbers(rng, shape, most=1):
    return torch.randint(-most, most + 1, shape, generator=rng, device=rng.device).float()


# Chunks of 64 rows forward and 32 backward at 64 lanes a row: 1094 and 2188 chunks, 3282 and 6563 (runs that are read again in both
# directions), 704 and 1407 with chunks that a sequence ends in; 32 lanes a row.
LONG = [(1, 70001, 128, 128), (1, 210000, 128, 32), (2, 22507, 128, 1), (1, 70001, 48, 48), (1, 40000, 9, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("sequences,length,channels,gates", LONG)
def test_starting_states_of_long_runs_are_exact(sequences, length, channels, gates, reverse, cuda):
    """Sums since the last gate of 0, of which there is one in about 30000 rows: up to 26 runs of chunks lie between.  |h| and |l| stay far
    below 2^11, so that their products, over four channels and more, are whole numbers below 2^24."""
    rng = torch.Generator(cuda).manual_seed(length + channels)
    x, dh = (whole_numbers(rng, (sequences, length, channels)) for _ in range(2))
    h0, df = (whole_numbers(rng, (sequences, channels), 7) for _ in range(2))
    g = (torch.rand((sequences, length, gates), generator=rng, device=cuda) > 3e-5).float()
    check(x, g, h0, None, "value", "plain", reverse, dh, df, exact=True)
    check(x.bfloat16(), g, h0, None, "value", "plain", reverse, dh.bfloat16(), df, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("length,channels,gates,cuts", [(70001, 128, 128, [0, 31000, 31000, 70000]), (210000, 128, 32, [5, 6, 150001, 209990]),
                                                        (210000, 130, 130, [0, 210000])])
def test_starting_states_of_long_packed_sequences_are_exact(length, channels, gates, cuts, reverse, cuda):
    rng = torch.Generator(cuda).manual_seed(length + channels)
    x, dh = (whole_numbers(rng, (length, channels)) for _ in range(2))
    h0, df = (whole_numbers(rng, (len(cuts) - 1, channels), 7) for _ in range(2))
    g = (torch.rand((length, gates), generator=rng, device=cuda) > 3e-5).float()
    check(x, g, h0, torch.tensor(cuts, dtype=torch.int32, device=cuda), "value", "plain", reverse, dh, df, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("gate_form,input_form", [("log", "plain"), ("logit", "complement")])
def test_slow_decays(gate_form, input_form, reverse, cuda):
    """Decays over about ten thousand rows, of values that are all positive: the states are sums, and the tolerance a part of them."""
    rng = torch.Generator(cuda).manual_seed(3)
    for length, channels, gates, cuts in ((70001, 128, 128, None), (210000, 128, 4, None), (150001, 64, 64, [3, 60000, 60000, 150000])):
        rows, sequences = ((1, length), 1) if cuts is None else ((length,), len(cuts) - 1)
        x, dh = (torch.rand((*rows, channels), generator=rng, device=cuda) for _ in range(2))
        h0, df = (100.0 * torch.rand((sequences, channels), generator=rng, device=cuda) for _ in range(2))
        g = torch.rand((*rows, gates), generator=rng, device=cuda)
        g = -2e-4 * g if gate_form == "log" else 8.5 + g
        check(x, g, h0, None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device=cuda), gate_form, input_form, reverse, dh, df)


@pytest.mark.gpu
@pytest.mark.parametrize("channels,gates", [(64, 64), (64, 1), (128, 1), (96, 4), (384, 1)])
@pytest.mark.parametrize("inputs_off,gradients_off", [(False, True), (True, False), (True, True)])
def test_alignment_on_long_axes(channels, gates, inputs_off, gradients_off, cuda):
    """A forward pass of wide accesses and a backward one whose gradient begins off alignment, and the reverse: another split of the columns, the same
    kept states."""
    def off(t, shifted):
        flat = torch.empty((t.numel() + 1,), dtype=t.dtype, device=cuda)[int(shifted):][:t.numel()]
        return flat.copy_(t.flatten()).view(t.shape)
    rng = torch.Generator(cuda).manual_seed(channels)
    for dtype, length in ((torch.bfloat16, 9000), (torch.float32, 20011)):
        x, dh = (torch.randn((1, length, channels), generator=rng, device=cuda).to(dtype) for _ in range(2))
        g = torch.sigmoid(torch.randn((1, length, gates), generator=rng, device=cuda) + 3.0).to(dtype)
        h0, df = (torch.randn((1, channels), generator=rng, device=cuda) for _ in range(2))
        for cuts in (None, torch.from_numpy(_offsets(np.random.default_rng(1), length, 1, 3, 9).numpy()).to(cuda)):
            shape = (1, length) if cuts is None else (length,)
            check(off(x, inputs_off).view(*shape, -1), off(g, inputs_off).view(*shape, -1), h0, cuts, "value", "complement", False,
                  off(dh, gradients_off).view(*shape, -1), df)
