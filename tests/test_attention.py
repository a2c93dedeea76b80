"""Linear attention and its single step against the definition in 64 bits, and what they refuse."""
import itertools

import pytest
import torch

from attention_reference import TYPES, U, assert_near, reference, with_bounds

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(cuda, seed, rows, key_heads, shared, K, V, dtype, gate_form="log", gate_type=F32, fixed=False, sequences=None, spread=1.5, mean=None):
    """q, k, v, gates (rows first), and the initial states of `sequences`."""
    g = torch.Generator().manual_seed(seed)
    heads = key_heads * shared

    def normal(*shape):
        return torch.randn(shape, generator=g)
    gates = normal(*((heads,) if fixed else (rows, heads))) * spread
    gates = -(gates + (-2.5 if mean is None else mean)).exp() if gate_form == "log" else gates + (2.0 if mean is None else mean)
    parts = [normal(rows, key_heads, K).to(dtype), normal(rows, key_heads, K).to(dtype), normal(rows, heads, V).to(dtype), gates.to(gate_type)]
    initial = normal(sequences, heads, K, V) if sequences else None
    return [t.to(cuda) for t in parts], None if initial is None else initial.to(cuda)


def check(cuda, parts, initial, cuts, gate_form, dense=None, final_too=True, seed=0, scale=None, grads_of=None):
    """Outputs and all gradients of a call; dense: (B, T) instead of offsets."""
    import trigrad_amd
    g = torch.Generator().manual_seed(1000 + seed)
    shape = (lambda t: t.view(*dense, *t.shape[1:])) if dense else (lambda t: t)
    leaves = [t.detach().requires_grad_() for t in (shape(parts[0]), shape(parts[1]), shape(parts[2]), parts[3] if parts[3].dim() == 1 else shape(parts[3]))]
    if initial is not None:
        leaves.append(initial.detach().requires_grad_())
    offsets = None if dense else torch.tensor(cuts, dtype=torch.int32, device=cuda)
    o, f = trigrad_amd.linear_attention(*leaves[:4], leaves[4] if initial is not None else None, offsets, gate_form, scale)
    grad_o = torch.randn(o.shape, generator=g).to(cuda, o.dtype)
    grad_f = torch.randn(f.shape, generator=g).to(cuda) if final_too else None
    grads = torch.autograd.grad([o, f] if final_too else [o], leaves, [grad_o, grad_f] if final_too else [grad_o])
    wanted = with_bounds(*parts, initial, cuts, gate_form, grad_o.reshape(parts[2].shape), grad_f, scale)
    rows = max(b - a for a, b in zip(cuts, cuts[1:])) * (len(cuts) if parts[3].dim() == 1 else 1)
    for name, got, (value, magnitude) in zip(("outputs", "final", "dq", "dk", "dv", "dgates", "dinitial"), (o, f, *grads), wanted):
        assert_near(name, got, value, magnitude, rows, parts[2].dtype)
    return o, f, grads


SIZES = [(1, 1), (5, 7), (16, 16), (24, 40), (32, 32), (33, 64), (64, 33), (64, 64), (72, 128), (100, 72), (128, 128), (127, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_sizes_of_heads(cuda, dtype, K, V):
    parts, initial = make(cuda, K * 131 + V, 2 * 77, 2, 1, K, V, dtype, sequences=2)
    check(cuda, parts, initial, [0, 77, 154], "log", dense=(2, 77))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700, 2100])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_lengths(cuda, dtype, length):
    parts, _ = make(cuda, length, length, 1, 2, 40, 48, dtype, "logit", dtype if length % 2 else F32)
    check(cuda, parts, None, [0, length], "logit", dense=(1, length), final_too=length % 3 != 0)


@pytest.mark.gpu
@pytest.mark.parametrize("gate_form,fixed,shared,initial,wide", list(itertools.product(["log", "logit"], [False, True], [1, 4], [False, True], [False, True])))
def test_forms(cuda, gate_form, fixed, shared, initial, wide):
    parts, h0 = make(cuda, 7 * shared + fixed, 3 * 150, 2, shared, 64, 64, BF16, gate_form, F32 if wide else BF16, fixed, 3 if initial else None)
    check(cuda, parts, h0, [0, 150, 300, 450], gate_form, dense=(3, 150), seed=shared)


@pytest.mark.gpu
@pytest.mark.parametrize("cuts", [[0, 0], [0, 0, 300, 300], [0, 1, 2, 3, 300], [17, 17, 64, 130, 290], [0, 300], [300, 300, 300], [5, 69, 133, 133, 261]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_sequences(cuda, dtype, cuts):
    """Empty sequences, sequences of one row, rows in front of the first and behind the last, which hold NaN."""
    parts, initial = make(cuda, sum(cuts), 300, 2, 2, 32, 48, dtype, sequences=len(cuts) - 1)
    clean = [t.clone() for t in parts]
    for t, fill in zip(parts, (float("nan"), float("inf"), float("nan"), float("nan"))):
        t[:cuts[0]] = fill
        t[cuts[-1]:] = fill
    import trigrad_amd
    leaves = [t.detach().requires_grad_() for t in parts] + [initial.requires_grad_()]
    offsets = torch.tensor(cuts, dtype=torch.int32, device=cuda)
    o, f = trigrad_amd.linear_attention(*leaves[:4], leaves[4], offsets)
    grad_o, grad_f = torch.ones_like(o), torch.ones_like(f)
    grad_o[:cuts[0]] = float("nan")
    grad_o[cuts[-1]:] = float("nan")
    grads = torch.autograd.grad([o, f], leaves, [grad_o, grad_f])
    for t in (o, *grads[:4]):
        assert not t[:cuts[0]].any() and not t[cuts[-1]:].any()
    inside = torch.zeros(300, dtype=torch.bool, device=cuda)
    inside[cuts[0]:cuts[-1]] = True
    zeros = [torch.where(inside.view(-1, *(1,) * (t.dim() - 1)), t, torch.zeros_like(t)) for t in clean]
    wanted = with_bounds(*zeros, initial, cuts, "log", inside[:, None, None] * torch.ones_like(o), grad_f)
    for name, got, (value, magnitude) in zip(("outputs", "final", "dq", "dk", "dv", "dgates", "dinitial"), (o, f, *grads), wanted):
        assert_near(name, got, value, magnitude, 300, dtype)


@pytest.mark.gpu
def test_many_sequences_and_heads(cuda):
    """As many as that a workgroup goes through a whole sequence, training and not."""
    parts, initial = make(cuda, 3, 40 * 200, 16, 1, 16, 16, BF16, sequences=40)
    o, f, _ = check(cuda, parts, initial, list(range(0, 8001, 200)), "log", dense=(40, 200))
    import trigrad_amd
    with torch.no_grad():
        again = trigrad_amd.linear_attention(*(t.view(40, 200, *t.shape[1:]) for t in parts), initial)
    assert torch.equal(again[0], o) and torch.equal(again[1], f)


@pytest.mark.gpu
def test_nothing_at_all(cuda):
    import trigrad_amd
    for batch, length in ((0, 5), (3, 0), (0, 0)):
        q, k, v = (torch.zeros((batch, length, 2, 8), device=cuda, requires_grad=True) for _ in range(3))
        gates, initial = torch.zeros((2,), device=cuda, requires_grad=True), torch.randn((batch, 2, 8, 8), device=cuda).requires_grad_()
        o, f = trigrad_amd.linear_attention(q, k, v, gates, initial)
        assert o.shape == v.shape and torch.equal(f, initial)
        grads = torch.autograd.grad(f.sum() + o.sum(), (q, k, v, gates, initial))
        assert [g.shape for g in grads] == [t.shape for t in (q, k, v, gates, initial)]
        assert not grads[3].any() and torch.equal(grads[4], torch.ones_like(initial))
        state = torch.zeros((0, 2, 8, 8), device=cuda)
        row = torch.zeros((0, 2, 8), device=cuda)
        assert trigrad_amd.linear_attention_step(row, row, row, torch.zeros((0, 2), device=cuda), state)[0].shape == (0, 2, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gates_of_minus_infinity_begin_anew(cuda, dtype):
    """What lies in front of such a row has no part in what follows, whatever it is."""
    import trigrad_amd
    parts, initial = make(cuda, 5, 300, 2, 1, 32, 32, dtype, sequences=1)
    resets = [0, 63, 64, 65, 170]
    for form, low in (("log", -torch.inf), ("logit", -torch.inf)):
        gates = parts[3].clone() if form == "log" else -parts[3]
        gates[resets] = low
        check(cuda, [*parts[:3], gates], initial, [0, 300], form, dense=(1, 300))
        args = [t[None] for t in (*parts[:3], gates)]
        o, f = trigrad_amd.linear_attention(*args, initial, gate_form=form)
        other = [t.clone() for t in args]
        for t in other[:3]:
            t[:, :170] *= 3.0
        p, g = trigrad_amd.linear_attention(*other, initial * 1e6, gate_form=form)
        assert torch.equal(o[:, 192:], p[:, 192:]) and torch.equal(f, g)  # 192: the next chunk of either number of rows


@pytest.mark.gpu
def test_fast_and_slow_decays(cuda):
    """From decays that leave nothing of a row in the next to ones that leave all of it."""
    for mean, spread in ((-40.0, 0.0), (-9.0, 1.0), (3.0, 1.0), (5.0, 0.0)):
        for dtype in (F32, BF16):
            parts, initial = make(cuda, 11, 500, 2, 1, 32, 32, dtype, spread=spread, mean=mean, sequences=1)
            check(cuda, parts, initial, [0, 500], "log", dense=(1, 500))


@pytest.mark.gpu
def test_a_sequence_that_is_not_finite_spoils_no_other(cuda):
    import trigrad_amd
    parts, _ = make(cuda, 2, 3 * 130, 2, 1, 32, 32, BF16)
    args = [t.view(3, 130, *t.shape[1:]) for t in parts]
    want = trigrad_amd.linear_attention(*args)
    for which in range(4):
        for value in (float("nan"), float("inf")):
            spoiled = [t.clone() for t in args]
            spoiled[which][1, 70] = value
            got = trigrad_amd.linear_attention(*spoiled)
            for w, g in zip(want, got):
                assert torch.equal(w[[0, 2]], g[[0, 2]])
            assert torch.equal(want[0][1, :64], got[0][1, :64])  # and no row in front of its chunk


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(32, 64), (24, 40), (13, 9)])
def test_strides(cuda, K, V):
    """Parts of one projection, heads in front of rows, a head for all, storages off alignment: the same results as dense tensors have, bit by bit."""
    import trigrad_amd
    g = torch.Generator().manual_seed(3)
    B, T, H = 2, 140, 4
    for dtype in (F32, BF16):
        gates = (-torch.rand((B, T, H), generator=g)).to(cuda)
        fused = torch.randn((B, T, 2 * H * K + H * V + 1), generator=g).to(cuda, dtype)
        views = [fused[..., :H * K].unflatten(-1, (H, K)), fused[..., H * K:2 * H * K].unflatten(-1, (H, K)), fused[..., 2 * H * K:-1].unflatten(-1, (H, V))]
        turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in views]
        across = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in views]
        shifted = []
        for t in views:
            room = torch.empty((t.numel() + 1,), dtype=dtype, device=cuda)
            shifted.append(room[1:].view(t.shape).copy_(t))
        one_key = [views[0], views[1][:, :, :1].expand(-1, -1, H, -1), views[2]]

        def results(parts):
            leaves = [t.detach().requires_grad_() for t in (*parts, gates)]
            o, f = trigrad_amd.linear_attention(*leaves)
            return [o, f, *torch.autograd.grad((o.float().square().sum() + f.square().sum()), leaves)]
        want = results([t.contiguous() for t in views])
        for other in (views, turned, across, shifted):
            got = results(other)
            # what lies off alignment is read and written otherwise, and computed alike
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        a, b = results(one_key), results([t.contiguous() for t in one_key])
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        grads = torch.autograd.grad(trigrad_amd.linear_attention(*views, gates.requires_grad_())[0].transpose(1, 2).sum(), gates)  # a gradient of strides of its own
        assert grads[0].isfinite().all()


@pytest.mark.gpu
def test_negated_views(cuda):
    import trigrad_amd
    z = torch.randn((1, 40, 2, 16), dtype=torch.complex64, device=cuda)
    x = torch.randn((1, 40, 2, 16), device=cuda)
    gates = -torch.rand((1, 40, 2), device=cuda)
    neg = z.conj().imag
    assert neg.is_neg()
    for at in range(3):
        args = [neg if i == at else x for i in range(3)]
        plain = [t.resolve_neg().contiguous() for t in args]
        for a, b in zip(trigrad_amd.linear_attention(*args, gates), trigrad_amd.linear_attention(*plain, gates)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_that_are_none(cuda):
    """Offsets beyond the rows count as their ends; decreasing ones read and write nothing outside."""
    import trigrad_amd
    parts, _ = make(cuda, 4, 200, 1, 1, 16, 16, F32)
    want = trigrad_amd.linear_attention(*parts, offsets=torch.tensor([0, 90, 200], dtype=torch.int32, device=cuda))
    got = trigrad_amd.linear_attention(*parts, offsets=torch.tensor([-50, 90, 1 << 30], dtype=torch.int32, device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for cuts in ([200, 0, 200, 0, 200, 0], [0, 200, 0, 200, 100], [500, -500, 50]):
        leaves = [t.detach().requires_grad_() for t in parts]
        o, f = trigrad_amd.linear_attention(*leaves, offsets=torch.tensor(cuts * 20, dtype=torch.int32, device=cuda))
        torch.autograd.grad(o.sum() + f.sum(), leaves)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_that_change_between_the_passes(cuda):
    """What the forward call made of them no longer fits; nothing outside is read or written, and calls that follow are right."""
    import trigrad_amd
    parts, _ = make(cuda, 4, 200, 2, 1, 16, 16, F32)
    for changed in ([200, 200, 200], [0, 0, 0], [0, 10, 5], [-7, 1 << 30, 3]):
        leaves = [t.detach().requires_grad_() for t in parts]
        offsets = torch.tensor([0, 90, 200], dtype=torch.int32, device=cuda)
        o, f = trigrad_amd.linear_attention(*leaves, offsets=offsets)
        offsets.data.copy_(torch.tensor(changed, dtype=torch.int32))
        torch.autograd.grad(o.sum() + f.sum(), leaves)
        torch.cuda.synchronize()
    check(cuda, parts, None, [0, 90, 200], "log")


@pytest.mark.gpu
def test_elements_beyond_32_bits(cuda):
    """Rows whose places pass 2^31 elements: the last ones as from the state in front of them."""
    import trigrad_amd
    T, H, D = 600_000, 32, 128
    g = torch.Generator(cuda).manual_seed(0)
    q = torch.randn((1, T, 1, D), generator=g, device=cuda, dtype=BF16)
    v = torch.randn((1, T, H, D), generator=g, device=cuda, dtype=BF16)
    gates = torch.full((H,), -0.01, device=cuda)
    assert v.numel() > 1 << 31
    o, f = trigrad_amd.linear_attention(q, q, v, gates)
    cut = T - 700
    _, state = trigrad_amd.linear_attention(q[:, :cut], q[:, :cut], v[:, :cut], gates)
    tail, last = trigrad_amd.linear_attention(q[:, cut:], q[:, cut:], v[:, cut:], gates, state)
    # the states' parts of a chunk are rounded in other places: half a step of the outputs each, and of their terms
    size = tail.float().square().mean().sqrt()
    assert (o[:, cut:].float() - tail.float()).abs().max() <= 8 * TYPES[BF16] * max(size, tail.float().abs().max())
    assert (f - last).abs().max() <= 256 * U * 200 * last.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_are_the_sequence(cuda, dtype):
    import trigrad_amd
    for K, V, G, R, form, fixed in ((64, 64, 2, 1, "log", False), (24, 40, 1, 3, "logit", True), (128, 128, 2, 2, "logit", False), (7, 5, 2, 1, "log", False)):
        parts, initial = make(cuda, K + V, 3 * 20, G, R, K, V, dtype, form, fixed=fixed, sequences=3)
        args = [t.view(3, 20, *t.shape[1:]) if t.dim() > 1 else t for t in parts]
        o, f = trigrad_amd.linear_attention(*args, initial, gate_form=form)
        state, spare = initial.clone(), torch.empty_like(initial)
        value = with_bounds(*parts, initial, [0, 20, 40, 60], form, torch.zeros_like(parts[2]), None)
        for t in range(20):
            row = [a[:, t] for a in args[:3]] + [args[3] if fixed else args[3][:, t]]
            if t % 2:
                y, got = trigrad_amd.linear_attention_step(*row, state, gate_form=form, out=spare)
                assert got is spare
                state, spare = spare, state
            else:
                y, got = trigrad_amd.linear_attention_step(*row, state, gate_form=form)
                assert got is state
            assert_near("outputs", y, value[0][0].view(3, 20, -1, V)[:, t], value[0][1].view(3, 20, -1, V)[:, t], 20, dtype)
        assert_near("final", state, value[1][0], value[1][1], 20, dtype)
        assert_near("final", f, value[1][0], value[1][1], 20, dtype)
        assert o.dtype == dtype and state.dtype == F32


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads", [(1, 1), (1, 16), (300, 5)])
@pytest.mark.parametrize("K,V", [(1, 1), (128, 128), (64, 100), (100, 64), (30, 126), (17, 3)])
def test_step_sizes(cuda, batch, heads, K, V):
    import trigrad_amd
    for dtype in (F32, F16, BF16):
        parts, initial = make(cuda, K, batch, heads, 1, K, V, dtype, sequences=batch)
        value = with_bounds(*parts, initial, list(range(batch + 1)), "log", torch.zeros_like(parts[2]), None) if batch < 10 else None
        y, state = trigrad_amd.linear_attention_step(*parts, initial.clone())
        a = parts[3].double().exp()[..., None, None]
        want = a * initial.double() + parts[1].double()[..., :, None] * parts[2].double()[..., None, :]
        sizes = a * initial.double().abs() + (parts[1].double()[..., :, None] * parts[2].double()[..., None, :]).abs()
        assert ((state.double() - want).abs() <= 8 * U * sizes).all()
        read = (parts[0].double()[..., None] * want).sum(-2) * K ** -0.5
        limit = (K + 16) * U * (parts[0].double().abs()[..., None] * sizes).sum(-2) * K ** -0.5 + 1.01 * TYPES[dtype] * read.abs() + (2.0 ** -25 if dtype == F16 else 0.0)  # halves have no steps below 2^-24
        assert ((y.double() - read).abs() <= limit).all()
        if value is not None:
            assert_near("outputs", y, *value[0], 1, dtype)


@pytest.mark.gpu
def test_step_with_strides_and_states_off_alignment(cuda):
    import trigrad_amd
    fused = torch.randn((5, 3, 4, 20), device=cuda)
    q, k, v = (fused[:, i] for i in range(3))
    gates = -torch.rand((4, 5), device=cuda).t()
    room = torch.randn((5 * 4 * 400 + 1,), device=cuda)
    state = room[1:].view(5, 4, 20, 20)
    before = state.clone()
    y, _ = trigrad_amd.linear_attention_step(q, k, v, gates, state)
    z, other = trigrad_amd.linear_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), gates.contiguous(), before)
    assert torch.equal(state, other)
    assert ((y - z).abs() <= 64 * U * 20 * z.abs().max()).all()  # sums of 20 in another order


@pytest.mark.gpu
def test_gradients_that_are_wanted(cuda):
    """Each gradient alone is what it is with all others; a state that is shared by broadcasting gets the sum."""
    import trigrad_amd
    parts, initial = make(cuda, 8, 2 * 100, 2, 2, 32, 32, BF16, sequences=2)
    args = [t.view(2, 100, *t.shape[1:]) for t in parts] + [initial]

    def grads(wanted, ends):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(args)]
        o, f = trigrad_amd.linear_attention(*leaves)
        loss = sum(t.float().square().sum() for t, n in ((o, "o"), (f, "f")) if n in ends)
        return torch.autograd.grad(loss, [leaves[i] for i in wanted])
    for ends in ("of", "o", "f"):
        every = grads([0, 1, 2, 3, 4], ends)
        for i in range(5):
            if ends == "f" and i == 0:
                continue
            assert torch.equal(grads([i], ends)[0], every[i])
    assert not grads([0, 1], "f")[0].any()  # no query reads the final state
    shared = initial[:1].detach().requires_grad_()
    o, f = trigrad_amd.linear_attention(*args[:4], shared.expand(2, -1, -1, -1))
    (one,) = torch.autograd.grad(o.float().sum() + f.sum(), shared)
    both = initial[:1].expand(2, -1, -1, -1).contiguous().requires_grad_()
    o, f = trigrad_amd.linear_attention(*args[:4], both)
    (two,) = torch.autograd.grad(o.float().sum() + f.sum(), both)
    assert ((one - two.sum(0, keepdim=True)).abs() <= 2 * U * two.abs().sum(0, keepdim=True)).all()


@pytest.mark.gpu
def test_gradients_against_differences(cuda):
    """Along random directions, by the float kernels: a central difference of width h is off by h^2 and by the outputs' roundings over h."""
    import trigrad_amd
    parts, initial = make(cuda, 21, 200, 2, 2, 24, 40, F32, "logit", sequences=1)
    args = [t[None] for t in parts] + [initial]
    g = torch.Generator(cuda).manual_seed(1)
    weight, weight_f = torch.randn((1, 200, 4, 40), generator=g, device=cuda), torch.randn((1, 4, 24, 40), generator=g, device=cuda)

    def loss(args):
        o, f = trigrad_amd.linear_attention(*args, gate_form="logit")
        return (o * weight).sum(dtype=torch.float64) + (f * weight_f).sum(dtype=torch.float64)
    leaves = [t.detach().requires_grad_() for t in args]
    grads = torch.autograd.grad(loss(leaves), leaves)
    h = 2.0 ** -7
    for i in range(5):
        d = torch.randn(args[i].shape, generator=g, device=cuda)
        ends = [loss([t + s * h * d if j == i else t for j, t in enumerate(args)]) for s in (1, -1)]
        slope, want = (ends[0] - ends[1]) / (2 * h), (grads[i].double() * d).sum()
        # the loss is at most of third order in one input's direction but the gates', whose third derivative is below the loss's terms
        terms = sum((a.double().abs() * b.double().abs()).sum() for a, b in zip((grads[i],), (d,)))
        assert (slope - want).abs() <= 4 * h * h * terms + 1e-3 * terms / args[i].numel() ** 0.5


@pytest.mark.gpu
def test_double_precision(cuda):
    """float64 by the double library: differences, and the definition to its precision."""
    import trigrad_amd
    torch.manual_seed(0)
    f64 = dict(dtype=torch.float64, device=cuda)
    q, k = (torch.randn((1, 7, 1, 3), **f64).requires_grad_() for _ in range(2))
    v = torch.randn((1, 7, 2, 2), **f64).requires_grad_()
    initial = torch.randn((1, 2, 3, 2), **f64).requires_grad_()
    for form, gates in (("log", -torch.rand((1, 7, 2), **f64)), ("logit", torch.randn((2,), **f64))):
        gates.requires_grad_()
        assert torch.autograd.gradcheck(lambda *a: trigrad_amd.linear_attention(*a, gate_form=form), (q, k, v, gates, initial))
        o, f = trigrad_amd.linear_attention(q, k, v, gates, initial, gate_form=form)
        ro, rf = reference(q[0], k[0], v[0], gates if gates.dim() == 1 else gates[0], initial, [0, 7], form)
        assert (o[0] - ro).abs().max() < 1e-13 and (f - rf).abs().max() < 1e-13
        state = initial.detach().clone()
        for t in range(7):
            y, _ = trigrad_amd.linear_attention_step(q[:, t].detach(), k[:, t].detach(), v[:, t].detach(), (gates if gates.dim() == 1 else gates[:, t]).detach(), state, form)
            assert (y - o[:, t]).abs().max() < 1e-13
        assert (state - f).abs().max() < 1e-13
    cuts = torch.tensor([1, 3, 3, 6], dtype=torch.int32, device=cuda)
    assert torch.autograd.gradcheck(lambda *a: trigrad_amd.linear_attention(*a, offsets=cuts), (q[0].detach().requires_grad_(), k[0].detach().requires_grad_(),
                                                                                                 v[0].detach().requires_grad_(), -torch.rand((7, 2), **f64).requires_grad_()))


@pytest.mark.gpu
def test_python_functions_and_torch_module_agree(cuda, monkeypatch):
    import trigrad_amd
    from trigrad_amd import _C
    for packed, fixed in ((False, False), (True, False), (False, True)):
        parts, initial = make(cuda, 6, 200, 2, 2, 40, 32, BF16, "logit", fixed=fixed, sequences=2)
        cuts = torch.tensor([3, 90, 190], dtype=torch.int32, device=cuda) if packed else None
        shape = (lambda t: t) if packed else (lambda t: t.view(2, 100, *t.shape[1:]) if t.dim() > 1 else t)
        results = []
        for route in (True, False):
            monkeypatch.setattr(_C, "ONE_CALL_OPERATORS", route)
            leaves = [shape(t).detach().requires_grad_() for t in parts] + [initial.detach().requires_grad_()]
            o, f = trigrad_amd.linear_attention(*leaves[:4], leaves[4], cuts, "logit", 0.3)
            grads = torch.autograd.grad(o.float().square().sum() + f.square().sum(), leaves)
            y, s = trigrad_amd.linear_attention_step(*(t[:2] for t in parts[:3]), parts[3] if fixed else parts[3][:2], initial.clone(), "logit", 0.3)
            results.append([o, f, *grads, y, s])
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_captured_forward_and_backward(cuda):
    """Replays with new inputs, eager work in between, beside another graph: as the eager calls, bit by bit."""
    import trigrad_amd
    parts, initial = make(cuda, 9, 2 * 300, 2, 2, 32, 32, BF16, sequences=2)
    cuts = torch.tensor([0, 170, 590], dtype=torch.int32, device=cuda)
    calls = [([t.view(2, 300, *t.shape[1:]) for t in parts] + [initial], None), ([*parts, initial], cuts)]
    graphs = []
    for args, offsets in calls:
        leaves = [t.detach().clone().requires_grad_() for t in args]
        state = initial.clone()

        def work(leaves=leaves, offsets=offsets, state=state):
            o, f = trigrad_amd.linear_attention(*leaves[:4], leaves[4], offsets)
            grads = torch.autograd.grad(o.float().square().sum() + f.square().sum(), leaves)
            rows = [t.detach().reshape(-1, *t.shape[-2:])[:2] for t in leaves[:3]]
            y, new = trigrad_amd.linear_attention_step(*rows, leaves[3].detach().reshape(-1, 4)[:2], state, out=torch.empty_like(state))
            return [o, f, *grads, y, new]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = work()
        graphs.append((graph, leaves, work, held))
    g = torch.Generator(cuda).manual_seed(0)
    for turn in range(3):
        for graph, leaves, work, held in graphs:
            with torch.no_grad():
                for t in leaves[:3]:
                    t.copy_(torch.randn(t.shape, generator=g, device=cuda))
            graph.replay()
        torch.cuda.synchronize()
        for graph, leaves, work, held in graphs:
            got = [t.clone() for t in held]
            assert all(torch.equal(a, b) for a, b in zip(got, work())), turn


@pytest.mark.gpu
def test_two_captured_graphs_at_once(cuda):
    """Their replays overlap on two streams; each has workspaces of its own."""
    import trigrad_amd
    calls, streams, graphs, results = [], [torch.cuda.Stream() for _ in range(2)], [], []
    for seed, (batch, length) in enumerate(((1, 3000), (3, 1500))):
        parts, initial = make(cuda, 40 + seed, batch * length, 2, 2, 40, 72, BF16, sequences=batch)
        leaves = [t.view(batch, length, *t.shape[1:]).detach().requires_grad_() for t in parts] + [initial.requires_grad_()]
        g = torch.Generator().manual_seed(seed)
        calls.append((leaves, [torch.randn(batch, length, 4, 72, generator=g).to(cuda, BF16), torch.randn(batch, 4, 40, 72, generator=g).to(cuda)]))

    def run(leaves, grads):
        out = trigrad_amd.linear_attention(*leaves)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, grads)]
    for call, stream in zip(calls, streams):
        with torch.cuda.stream(stream):
            run(*call)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            results.append(run(*call))
    wanted = [run(*call) for call in calls]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got, want in zip(results, wanted) for a, b in zip(got, want))
        torch.randn(1000, device=cuda).sum().item()


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_is_refused(cuda):
    import trigrad_amd
    parts, _ = make(cuda, 9, 100, 1, 1, 16, 16, F32)
    leaves = [t[None].detach().requires_grad_() for t in parts]
    alive = trigrad_amd.linear_attention(*leaves)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(graph):
            trigrad_amd.linear_attention(*leaves)
    assert alive[0].isfinite().all()


@pytest.mark.gpu
def test_calls_on_other_streams(cuda):
    import trigrad_amd
    parts, initial = make(cuda, 10, 2 * 500, 2, 1, 64, 64, BF16, sequences=2)
    args = [t.view(2, 500, *t.shape[1:]) for t in parts] + [initial]

    def work():
        leaves = [t.detach().requires_grad_() for t in args]
        o, f = trigrad_amd.linear_attention(*leaves)
        return [o, f, *torch.autograd.grad(o.float().sum() + f.sum(), leaves)]
    want = work()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append(work())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))


def test_entry_points_without_a_gpu():
    import trigrad_amd
    x, gates = torch.zeros((1, 4, 2, 8)), torch.zeros((1, 4, 2))
    with pytest.raises(TypeError, match="must be on cuda"):
        trigrad_amd.linear_attention(x, x, x, gates)
    with pytest.raises(TypeError, match="must be on cuda"):
        trigrad_amd.linear_attention_step(x[0], x[0], x[0], gates[0], torch.zeros((4, 2, 8, 8)))
    with pytest.raises(ValueError, match="gate_form"):
        trigrad_amd.linear_attention(x, x, x, gates, gate_form="value")
    with pytest.raises(ValueError, match="dimensions"):
        trigrad_amd.linear_attention(x[0], x[0], x[0], gates)
    with pytest.raises(TypeError, match="must be of type"):
        trigrad_amd.linear_attention(x.int(), x.int(), x.int(), gates)


def test_library_refuses_on_the_host():
    """Sizes, types and missing pointers, before any device is touched; what a call needs of memory."""
    import ctypes as C
    from trigrad_amd import _lib
    lib, sizes = _lib.load(32), (C.c_int64 * 4)()
    good = dict(sequences=2, length=100, heads=4, key_heads=2, key_size=64, value_size=64, type=2, gate_type=0, gate_form=1, scale=1.0)

    def asked(**changed):
        return lib.tg_linear_attention_sizes(C.byref(_lib.Attention(**{**good, **changed})), sizes)
    assert asked() == 0 and sizes[0] > 0 and sizes[3] > 0
    for changed in (dict(key_heads=3), dict(key_size=129), dict(value_size=0), dict(key_size=0), dict(heads=0), dict(type=3), dict(type=7), dict(gate_type=1), dict(gate_form=0),
                    dict(gate_form=3), dict(sequences=-1), dict(length=-1), dict(sequences=1 << 40), dict(heads=1 << 17, key_heads=1), dict(length=1 << 33)):
        assert asked(**changed) == -1, changed
        assert lib.tg_linear_attention_forward(C.byref(_lib.Attention(**{**good, **changed}))) == -1
        assert lib.tg_linear_attention_backward(C.byref(_lib.Attention(**{**good, **changed}))) == -1
    assert lib.tg_linear_attention_sizes(None, sizes) == -1 and lib.tg_linear_attention_forward(None) == -1 and lib.tg_linear_attention_step(None) == -1
    assert lib.tg_linear_attention_forward(C.byref(_lib.Attention(**good))) == -1  # null pointers
    assert lib.tg_linear_attention_step(C.byref(_lib.Attention(**good))) == -1  # more than a row
    # sequences and heads of which a grid has no room for
    many = dict(good, sequences=1 << 23, length=1, heads=2, key_heads=2, key_size=1, value_size=1)
    some = {name: 16 for name in ("queries", "keys", "values", "gates", "initial", "outputs", "final")}
    assert lib.tg_linear_attention_step(C.byref(_lib.Attention(**many, **some))) == -1 and b"too many" in lib.tg_last_error()
    double = _lib.load(64)
    for types, sequences, code in ((dict(type=3, gate_type=3), 1 << 25, -1), (dict(type=3, gate_type=3), (1 << 25) - 1, 0)):
        assert double.tg_linear_attention_sizes(C.byref(_lib.Attention(**{**many, **types, "sequences": sequences})), sizes) == code
    some = {name: 16 for name in ("queries", "keys", "values", "gates", "outputs", "final")}  # not touched
    asked()
    if sizes[1]:
        assert lib.tg_linear_attention_forward(C.byref(_lib.Attention(**good, **some, workspace=16, workspace_bytes=sizes[1] - 1))) == -2
    assert lib.tg_linear_attention_forward(C.byref(_lib.Attention(**good, **some, kept=16, kept_bytes=sizes[0] - 1))) == -2
    assert lib.tg_linear_attention_backward(C.byref(_lib.Attention(**good, **some, kept=16, kept_bytes=sizes[0], workspace=16, workspace_bytes=sizes[3] - 1))) == -2
    assert lib.tg_linear_attention_backward(C.byref(_lib.Attention(**good, **some, workspace=16, workspace_bytes=sizes[3]))) == -1  # nothing kept
    assert lib.tg_linear_attention_forward(C.byref(_lib.Attention(**good, **some, kept=24, kept_bytes=sizes[0], workspace=16, workspace_bytes=sizes[2]))) == -2
    assert lib.tg_linear_attention_backward(C.byref(_lib.Attention(**good, **some, kept=16, kept_bytes=sizes[0], workspace=24, workspace_bytes=sizes[3]))) == -2


@pytest.mark.gpu
def test_refusals(cuda):
    import trigrad_amd
    parts, initial = make(cuda, 1, 20, 2, 2, 16, 8, F32, sequences=2)
    q, k, v, gates = (t.view(2, 10, *t.shape[1:]) for t in parts)
    call = trigrad_amd.linear_attention
    for bad, error in (((q[..., :8], k, v, gates), ValueError), ((q, k[:, :9], v, gates), ValueError), ((q, k, v, gates[..., :3]), ValueError),
                       ((q.half(), k, v, gates), TypeError), ((q, k, v, gates.half()), TypeError), ((q, k, v[:, :, :3], gates[..., :3]), ValueError),
                       ((q, k, v, gates, initial.half()), TypeError), ((q, k, v, gates, initial[:1]), ValueError), ((q.cpu(), k, v, gates), TypeError),
                       ((q, k, v, gates.cpu()), TypeError), ((torch.zeros((2, 10, 2, 129), device=cuda),) * 2 + (v, gates), ValueError)):
        with pytest.raises(error):
            call(*bad)
    with pytest.raises(TypeError):
        call(*parts, None, torch.tensor([0, 20], device=cuda))
    with pytest.raises(ValueError):
        call(*parts, None, torch.tensor([0], dtype=torch.int32, device=cuda))
    row = [t[:, 0] for t in (q, k, v, gates)]
    step = trigrad_amd.linear_attention_step
    with pytest.raises(ValueError, match="contiguous"):
        step(*row, initial.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="overlap"):
        step(initial.view(2, -1)[:, :32].view(2, 2, 16), row[1], row[2], row[3], initial)
    room = torch.zeros((initial.numel() + 64,), device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        step(*row, room[:-64].view(initial.shape), out=room[64:].view(initial.shape))
    with pytest.raises(ValueError):
        step(*row, initial, out=initial[:1].clone())
    with pytest.raises(RuntimeError, match="no gradient"):
        step(row[0].requires_grad_(), *row[1:], initial)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, gates)]
    o, _ = call(*leaves)
    first = torch.autograd.grad(o.square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        first[0].sum().backward()
