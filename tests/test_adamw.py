"""The AdamW step and the optimizer against their formulas, in 64 bits or operation by operation, and what they refuse."""
import copy
import io

import numpy as np
import pytest
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
B1, B2, EPS, DECAY, LR = 0.9, 0.999, 1e-8, 0.02, 3e-3


def make(cuda, sizes, seed=0, grad_types=(torch.float32,), offset=0):
    """Lists of params, gradients and averages; offset: elements that their storages begin off alignment."""
    g = torch.Generator().manual_seed(seed)

    def place(t):
        room = torch.empty((t.numel() + offset,), dtype=t.dtype, device=cuda)
        return room[offset:].view(t.shape).copy_(t)
    lists = [[], [], [], []]
    for i, n in enumerate(sizes):
        shape = (n,) if isinstance(n, int) else n
        values = [torch.randn(shape, generator=g) for _ in range(4)]
        values[1] = (values[1] * 0.1).to(grad_types[i % len(grad_types)])
        values[3] = values[3].square() * 0.01
        for to, t in zip(lists, values):
            to.append(place(t))
    return lists


def expected(p, g, m, v, step, lr=LR, grad_scale=1.0, maximize=False, b1=B1, b2=B2, eps=EPS, decay=DECAY):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * (-grad_scale if maximize else grad_scale)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    change = lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p * (1 - lr * decay) - change, m, v, change


def assert_step(before, after, step, **kw):
    """A factor that is rounded to float32, products and sums: four roundings of each term of an average, twelve of what is subtracted."""
    for i, (p, g, m, v) in enumerate(zip(*before)):
        want, wm, wv, change = expected(p, g, m, v, step, **kw)
        scale = abs(kw.get("grad_scale", 1.0))
        terms = B1 * m.double().abs() + (1 - B1) * g.double().abs() * scale
        assert ((after[2][i].double() - wm).abs() <= 4 * U * terms + 2.0 ** -140).all(), i
        assert ((after[3][i].double() - wv).abs() <= 6 * U * wv + 2.0 ** -140).all(), i
        spread = terms / wm.abs().clamp_min(1e-300)  # the average's terms may cancel, what its error is of
        assert ((after[0][i].double() - want).abs() <= 4 * U * p.double().abs() + (12 + 4 * spread) * U * change.abs()).all(), i


SIZES = [1, 3, 64, 255, 256, 257, 1000, 4095, 4096, 4097, 8192, 100003, (17, 33), (0,), (5, 0), (3, 4, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("grad_type", [torch.float32, torch.float16, torch.bfloat16])
def test_step(cuda, grad_type, offset):
    import trigrad_amd
    lists = make(cuda, SIZES, 1, (grad_type,), offset)
    before = [[t.clone() for t in l] for l in lists]
    versions = [t._version for t in lists[0]]
    assert trigrad_amd.adamw_step(*lists, 7, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY) is None
    assert_step(before, lists, 7)
    assert all(torch.equal(a, b) for a, b in zip(before[1], lists[1]))
    assert all(t._version > n for t, n in zip(lists[0], versions))


@pytest.mark.gpu
@pytest.mark.parametrize("step,maximize,scale", [(1, False, None), (2, True, None), (100000, False, 0.25), (3, True, -3.0)])
def test_step_numbers(cuda, step, maximize, scale):
    import trigrad_amd
    lists = make(cuda, [300, 5000], 2)
    before = [[t.clone() for t in l] for l in lists]
    trigrad_amd.adamw_step(*lists, step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, maximize=maximize,
                           grad_scale=None if scale is None else torch.tensor([scale], device=cuda))
    assert_step(before, lists, step, maximize=maximize, grad_scale=1.0 if scale is None else scale)


@pytest.mark.gpu
def test_many_tensors_of_mixed_types(cuda):
    """More than a launch has room for, gradients of three types and copies of two, or none."""
    import trigrad_amd
    sizes = [1 + 37 * i % 6000 for i in range(300)]
    lists = make(cuda, sizes, 3, (torch.float32, torch.bfloat16, torch.float16, torch.bfloat16))
    kinds = (None, torch.float16, torch.bfloat16)
    copies = [None if kinds[i % 3] is None else torch.zeros(n, dtype=kinds[i % 3], device=cuda) for i, n in enumerate(sizes)]
    before = [[t.clone() for t in l] for l in lists]
    trigrad_amd.adamw_step(*lists, 5, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, copies=copies)
    assert_step(before, lists, 5)
    for p, c in zip(lists[0], copies):
        assert c is None or torch.equal(c, p.to(c.dtype))


@pytest.mark.gpu
def test_step_and_rate_on_the_device(cuda):
    """Numbers that the device reads are the same as the host's, to the rounding of the rate."""
    import trigrad_amd
    for step in (1, 2, 1000, 10 ** 6):
        first, second = make(cuda, [5000, 33], 4), make(cuda, [5000, 33], 4)
        trigrad_amd.adamw_step(*first, step, lr=0.25, weight_decay=0.125)
        trigrad_amd.adamw_step(*second, torch.tensor([float(step)], device=cuda), lr=torch.tensor([0.25], device=cuda), weight_decay=0.125)
        for a, b in zip(first, second):
            for x, y in zip(a, b):  # a power of a beta in 64 bits on either side: its error of 1e-16 counts 1e3 times in 1 - b^t, below a rounding
                assert ((x - y).abs() <= 2 * U * (x.abs() + 0.25 * 12)).all()
        assert all(torch.equal(a, b) for i in (2, 3) for a, b in zip(first[i], second[i]))


# ---- 8 bits, operation by operation in float32 -----------------------------------------------

F = np.float32


def values8(codes):
    return codes.float().cpu().numpy()


def mixed(places, seed):
    x = (places.astype(np.uint64) * 0x9E3779B1 + ((seed * 0x85EBCA6B + 0xC2B2AE35) & 0xFFFFFFFF)) & 0xFFFFFFFF
    x = ((x ^ x >> 16) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ x >> 15) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ x >> 16


def neighbour(x, noise, least):
    """(values in units of the block's scale, scale) of one block."""
    largest = np.abs(x).max()
    if largest < F(2.0) ** -110:
        return np.zeros_like(x), F(0)
    y = np.minimum(np.abs(x) * ((F(1) / largest) * F(448)), F(448))
    bits = (y.view(np.uint32) + (noise.astype(np.uint32) << np.uint32(4))) & np.uint32(0xFFF00000)
    small = np.floor(y * F(512) + noise.astype(F) * F(2.0 ** -16))
    if least:
        small = np.where(y > 0, np.maximum(small, F(1)), small)
    z = np.where(y >= F(2.0 ** -6), bits.view(F), small * F(2.0 ** -9))
    return np.copysign(z, x), largest * F(1 / F(448))


def step8(p, g, m8, r8, scales, step, seed, place, lr=LR):
    """One tensor's step in float32, block by block -> p, values of the averages, scales."""
    out = [[], [], [], []]
    n1, n2 = F(1 - B1), F(1 - B2)
    for b in range(scales.shape[0]):
        at = slice(256 * b, min(256 * b + 256, len(p)))
        m = values8(m8)[at] * scales[b, 0] * F(B1) + g[at] * n1
        root = values8(r8)[at] * scales[b, 1]
        root = np.sqrt((root * root) * F(B2) + (g[at] * g[at]) * n2)
        rate, unbias = F(lr / (1 - B1 ** step)), F(1 / np.sqrt(1 - B2 ** step))
        out[0].append(p[at] * F(1 - lr * DECAY) - rate * (m / (root * unbias + F(EPS))))
        noise = mixed(np.arange(at.start, at.stop) + 256 * place, seed)
        for to, x, bits, least in ((1, m, noise & 0xFFFF, False), (2, root, noise >> 16, True)):
            value, scale = neighbour(x, bits, least)
            out[to].append(value)
            out[3].append(scale)
    return [np.concatenate(o) if o and o[0].ndim else np.array(o, F) for o in out[:3]] + [np.array(out[3], F).reshape(-1, 2)]


def make8(cuda, sizes, seed, offset=0, grad_type=torch.float32):
    p, g, m, v = make(cuda, sizes, seed, (grad_type,), offset)
    lists = [p, g, [], []]
    scales = []
    for a, b in zip(m, v):
        blocks = -(-a.numel() // 256)
        s = torch.rand((blocks, 2), device=cuda) * 1e-3
        scales.append(s)
        for to, t in zip(lists[2:], (a, b)):
            room = torch.empty((t.numel() + offset,), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
            to.append(room[offset:].view(t.shape).copy_((t * 100).abs().clamp_max(448) if to is lists[3] else (t * 100).clamp(-448, 448)))
    return lists, scales


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
def test_averages_in_8_bits(cuda, offset):
    """The same bits as the formula's operations one by one have, whatever the alignment and the tensor's place in the list."""
    import trigrad_amd
    sizes = [1, 255, 256, 257, 5000, 0, 12345]
    lists, scales = make8(cuda, sizes, 5, offset)
    before, scales_before = [[t.clone() for t in l] for l in lists], [s.cpu().numpy() for s in scales]
    for t in (lists[1][4], before[1][4]):
        t[300:812] = 0.0  # blocks whose gradient is zero, one of them with averages of zero
    for l in (lists, before):
        for which in (2, 3):
            l[which][4][512:768] = 0.0
    trigrad_amd.adamw_step(*lists, 9, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, scales=scales, seed=1234567)
    place = 0
    for i, n in enumerate(sizes):
        if n:
            p, m, r, s = step8(*(t.cpu().numpy() for t in (before[0][i], before[1][i])), before[2][i], before[3][i], scales_before[i], 9, 1234567, place)
            assert np.array_equal(lists[0][i].cpu().numpy(), p)
            assert np.array_equal(values8(lists[2][i]), m) and np.array_equal(values8(lists[3][i]), r)
            assert np.array_equal(scales[i].cpu().numpy(), s)
        place += -(-n // 256)


@pytest.mark.gpu
def test_rounding_to_8_bits_has_no_bias(cuda):
    """The mean over many seeds is the value: off by at most six standard deviations of a mean, where one rounding's is at most half a step."""
    import trigrad_amd
    n, seeds = 256, 4000
    g = torch.randn(n, device=cuda)
    g[0] = 5.0
    total, want = torch.zeros(n, device=cuda, dtype=torch.float64), None
    for seed in range(seeds):
        p, m, v = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(
            n, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scales = torch.zeros((1, 2), device=cuda)
        trigrad_amd.adamw_step([p], [g], [m], [v], 1, scales=[scales], seed=seed)
        total += m.double() * scales[0, 0].double()
        want = 0.1 * g.double()
    step = torch.maximum(want.abs() / 8, torch.full_like(want, 0.5 / 448 / 512))  # of neighbours: an eighth of a power of two below, or 2^-9 of the scale
    assert ((total / seeds - want).abs() <= 6 * 0.5 * step / seeds ** 0.5 + 2.0 ** -16 * step + 4 * U * want.abs()).all()


@pytest.mark.gpu
def test_averages_in_8_bits_follow_small_changes(cuda):
    """A constant gradient for 4000 steps: the average of its square is a thousandth nearer in each, which rounding to nearest would lose."""
    import trigrad_amd
    p = torch.zeros(1024, device=cuda, requires_grad=True)
    g = torch.linspace(0.5, 1.5, 1024, device=cuda)
    optimizer = trigrad_amd.AdamW([p], lr=0.0, state_bits=8)
    for _ in range(4000):
        p.grad = g
        optimizer.step()
    s = optimizer.state[p]
    root = s["exp_avg_sq"].float() * s["scales"][:, 1].repeat_interleave(256)
    # 1 - 0.999^4000 = 0.982 of the square; a value is within a step (an eighth at most) and the mean of all of them within 3 %
    assert ((root / g - 0.991).abs() <= 0.13).all() and abs((root / g).mean().item() - 0.991) <= 0.03


@pytest.mark.gpu
def test_values_that_are_not_finite(cuda):
    """They spoil their own elements, in 8 bits an infinite one its block."""
    import trigrad_amd
    for value in (float("nan"), float("inf")):
        lists = make(cuda, [1000], 6)
        clean = [[t.clone() for t in l] for l in lists]
        lists[1][0][333] = value
        for l in (lists, clean):
            trigrad_amd.adamw_step(*l, 1)
        keep = torch.arange(1000, device=cuda) != 333
        assert all(torch.equal(a[0][keep], b[0][keep]) for a, b in zip(lists, clean))
        assert not lists[2][0][333].isfinite()
        lists, scales = make8(cuda, [1000], 6)
        other, other_scales = make8(cuda, [1000], 6)
        for a, b in zip(other_scales, scales):
            a.copy_(b)
        lists[1][0][333] = value
        trigrad_amd.adamw_step(*lists, 1, scales=scales)
        trigrad_amd.adamw_step(*other, 1, scales=other_scales)
        keep = keep if value != value else torch.arange(1000, device=cuda) // 256 != 1
        assert all(torch.equal(a[0].float()[keep], b[0].float()[keep]) for a, b in zip(lists, other))


@pytest.mark.gpu
def test_python_function_and_torch_module_agree(cuda, monkeypatch):
    import trigrad_amd
    from trigrad_amd import _C
    results = []
    for route in (True, False):
        monkeypatch.setattr(_C, "ONE_CALL_OPERATORS", route)
        lists = make(cuda, [100, 5000, 33], 7, (torch.float32, torch.bfloat16))
        copies = [None, torch.zeros(5000, dtype=torch.bfloat16, device=cuda), None]
        trigrad_amd.adamw_step(*lists, 3, lr=torch.tensor([0.01], device=cuda), copies=copies, grad_scale=torch.tensor([0.5], device=cuda))
        eight, scales = make8(cuda, [100, 5000, 33], 7)
        for s in scales:
            s.fill_(1e-3)
        trigrad_amd.adamw_step(*eight, torch.tensor([3.0], device=cuda), scales=scales, seed=-5, maximize=True)
        results.append([t for l in (*lists, *eight, scales, [copies[1]]) for t in l])
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(*results))


@pytest.mark.gpu
def test_gradients_that_are_not_dense_in_memory(cuda):
    import trigrad_amd
    p, g, m, v = (t[0] for t in make(cuda, [(30, 40)], 8))
    turned = g.t().contiguous().t()
    before = [[t.clone()] for t in (p, g, m, v)]
    trigrad_amd.adamw_step([p], [turned], [m], [v], 2, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    assert_step(before, [[p], [g], [m], [v]], 2)
    one = torch.ones((1, 1), device=cuda).expand(30, 40)
    before = [[t.clone()] for t in (p, one, m, v)]
    trigrad_amd.adamw_step((p,), (one,), (m,), (v,), 2, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    assert_step(before, [[p], [one], [m], [v]], 2)


@pytest.mark.gpu
def test_double_precision(cuda):
    import trigrad_amd
    lists = [[t.double() for t in l] for l in make(cuda, [5, 300, 4097], 9)]
    before = [[t.clone() for t in l] for l in lists]
    trigrad_amd.adamw_step(*lists, 4, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, grad_scale=torch.tensor([0.5], dtype=torch.float64, device=cuda))
    for i, parts in enumerate(zip(*before)):
        for got, want in zip((lists[0][i], lists[2][i], lists[3][i]), expected(*parts, 4, grad_scale=0.5)):
            assert ((got - want).abs() <= 1e-14 * (want.abs() + 1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(cuda, bits):
    """Replays advance the count on the device: as eager steps do, bit by bit."""
    import trigrad_amd
    results = []
    for captured in (True, False):
        params = [t.requires_grad_() for t in make(cuda, [100, 7000], 10)[0]]
        grads = make(cuda, [100, 7000], 11)[1]
        for p, g in zip(params, grads):
            p.grad = g.clone()
        rate = torch.tensor([0.01], device=cuda)
        optimizer = trigrad_amd.AdamW(params, lr=rate, capturable=True, state_bits=bits)
        optimizer.step()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                optimizer.step()
        for turn in range(4):
            rate.mul_(0.5)
            for p in params:
                p.grad.mul_(1.5).add_(0.01)
            graph.replay() if captured else optimizer.step()
            torch.cuda.synchronize()
        results.append([t.detach().float() for p in params for t in (p, *(v for k, v in sorted(optimizer.state[p].items())))])
        assert optimizer.state[params[0]]["step"].item() == 5.0
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_replays_round_as_steps_do(cuda):
    """Averages in 8 bits are rounded with the step's number, also where the device counts: those of replays are those of eager steps without a
    count on the device, and small changes are not lost."""
    import trigrad_amd
    g = torch.linspace(0.5, 1.5, 1024, device=cuda)
    states = []
    for captured in (True, False):
        p = torch.zeros(1024, device=cuda, requires_grad=True)
        p.grad = g.clone()
        optimizer = trigrad_amd.AdamW([p], lr=0.0, state_bits=8, capturable=captured, seed=77)
        optimizer.step()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                optimizer.step()
        for _ in range(999):
            graph.replay() if captured else optimizer.step()
        torch.cuda.synchronize()
        s = optimizer.state[p]
        states.append((s["exp_avg"].float(), s["exp_avg_sq"].float(), s["scales"]))
    assert all(torch.equal(a, b) for a, b in zip(*states))
    root = states[0][1] * states[0][2][:, 1].repeat_interleave(256)
    # 1 - 0.999^1000 = 0.632 of the square, 0.795 of its root.  A root that goes up by steps of at most an eighth of itself, each by chance, has a
    # variance of at most its square / 16, and its square grows by half a step more: 0.05, beside 6 x 0.2 / 1024^(1/2) = 0.04
    assert abs((root / g).mean().item() - 0.795) <= 0.09


@pytest.mark.gpu
def test_optimizer_is_torchs(cuda):
    """Ten steps beside torch.optim.AdamW, with groups of their own numbers and a parameter whose gradients begin late."""
    import trigrad_amd
    mine, theirs = ([t.requires_grad_() for t in make(cuda, [300, (20, 30), 5], 12)[0]] for _ in range(2))
    groups = lambda p: [{"params": p[:1], "lr": 1e-2}, {"params": p[1:], "weight_decay": 0.1, "betas": (0.8, 0.99)}]  # noqa: E731
    a, b = trigrad_amd.AdamW(groups(mine), lr=1e-3), torch.optim.AdamW(groups(theirs), lr=1e-3, foreach=False)
    g = torch.Generator().manual_seed(0)
    for turn in range(10):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            if i != 2 or turn >= 4:
                p.grad = torch.randn(p.shape, generator=g).to(cuda)
                q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(mine, theirs):  # a change is at most ten rates, rounded like the param in each of ten steps, on either side
        assert ((p - q).abs() <= 2 * 10 * U * (4 * q.abs() + 16 * 0.1)).all()
    a.zero_grad()
    assert mine[0].grad is None
    assert a.step(lambda: torch.tensor(2.5)).item() == 2.5


@pytest.mark.gpu
def test_optimizer_of_parameters_in_16_bits(cuda):
    """They are what the ones in float32 are rounded to, which move by less than they could."""
    import trigrad_amd
    p = torch.ones(500, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    q = torch.ones(500, device=cuda, requires_grad=True)
    a, b = trigrad_amd.AdamW([p], lr=1e-4), trigrad_amd.AdamW([q], lr=1e-4)
    for _ in range(100):
        p.grad = torch.ones_like(p)
        q.grad = torch.ones_like(q)
        a.step()
        b.step()
    assert torch.equal(a.state[p]["master"], q) and torch.equal(p, q.to(torch.bfloat16)) and (p < 1.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kwargs", [{}, {"state_bits": 8}, {"capturable": True}])
def test_saved_and_loaded_state(cuda, kwargs):
    """An optimizer that goes on from a saved state does as the one that was saved."""
    import trigrad_amd
    results = []
    for saved in (False, True):
        params = [t.requires_grad_() for t in make(cuda, [300, 7], 13)[0]] + [torch.ones(64, device=cuda, dtype=torch.bfloat16, requires_grad=True)]
        optimizer = trigrad_amd.AdamW(params, lr=1e-2, **kwargs)
        for turn in range(6):
            if saved and turn == 3:
                room = io.BytesIO()
                torch.save(optimizer.state_dict(), room)
                room.seek(0)
                optimizer = trigrad_amd.AdamW(params, lr=5.0, **kwargs)
                optimizer.load_state_dict(torch.load(room, weights_only=True))
                if kwargs.get("state_bits") == 8:
                    assert optimizer.state[params[0]]["exp_avg"].dtype == torch.float8_e4m3fn
                assert optimizer.state[params[2]]["master"].dtype == torch.float32
            for i, p in enumerate(params):
                p.grad = torch.full_like(p, 0.1 * (turn + i + 1))
            optimizer.step()
        results.append([p.detach() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert copy.deepcopy(optimizer.state_dict())["param_groups"][0]["lr"] == 1e-2


@pytest.mark.gpu
def test_refusals(cuda):
    import trigrad_amd
    p, g, m, v = make(cuda, [100, 100], 14)
    step = trigrad_amd.adamw_step
    room = torch.zeros(150, device=cuda)
    for lists in (([p[0], p[0]], g, m, v), (p, g, m, [v[0], m[0]]), (p, [p[1], g[1]], m, v), ([room[:100], room[50:]], g, m, v), (p, g, [g[0], m[1]], v)):
        with pytest.raises(ValueError, match="overlap"):
            step(*lists, 1)
    for lists, error in (((p, g[:1], m, v), ValueError), (([p[0].t(), p[1][:50]], g, m, v), ValueError), (([p[0].half(), p[1]], g, m, v), TypeError),
                         ((p, [g[0].double(), g[1]], m, v), TypeError), ((p, g, [m[0].half(), m[1]], v), TypeError), ((p, [g[0].cpu(), g[1]], m, v), TypeError),
                         (([torch.zeros((20, 10), device=cuda)[:, :5].reshape(100), torch.zeros((100, 2), device=cuda)[:, 0]], g, m, v), ValueError)):
        with pytest.raises(error):
            step(*lists, 1)
    for kwargs in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            step(p, g, m, v, 1, **kwargs)
    with pytest.raises(ValueError):
        step(p, g, m, v, 0)
    with pytest.raises(TypeError):
        step(p, g, m, v, torch.tensor([1], device=cuda))
    with pytest.raises(TypeError):
        step(p, g, m, v, 1, grad_scale=torch.tensor([1.0, 2.0], device=cuda))
    with pytest.raises(TypeError):
        step(p, g, m, v, 1, scales=[trigrad_amd.adamw.scales_of(t) for t in p])  # averages that are not in 8 bits
    with pytest.raises(TypeError):
        step(p, g, m, v, 1, copies=[torch.zeros_like(t) for t in p])
    leaf = torch.zeros(100, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="leaves"):
        step([leaf * 2.0], g[:1], m[:1], v[:1], 1)
    before = leaf.detach().clone()
    step([leaf], g[:1], m[:1], v[:1], 1)  # a leaf needs no torch.no_grad
    assert not torch.equal(leaf, before) and leaf.requires_grad
    for kwargs in (dict(state_bits=16), dict(lr=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            trigrad_amd.AdamW([leaf], **kwargs)


def test_entry_points_without_a_gpu():
    import trigrad_amd
    t = [torch.zeros(4)]
    trigrad_amd.adamw_step([], [], [], [], 1)
    with pytest.raises(TypeError, match="must be on cuda"):
        trigrad_amd.adamw_step(t, t, t, t, 1)
    with pytest.raises(ValueError, match="must have 1 tensors"):
        trigrad_amd.adamw_step(t, [], t, t, 1)
    with pytest.raises(ValueError, match="betas"):
        trigrad_amd.adamw_step(t, t, t, t, 1, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="state_bits"):
        trigrad_amd.AdamW([torch.zeros(4, requires_grad=True)], state_bits=4)


@pytest.mark.parametrize("bits", [32, 64])
def test_library_refuses_on_the_host(bits):
    import ctypes as C
    from trigrad_amd import _lib
    lib = _lib.load(bits)
    room = (C.c_void_p * 1)(16)
    cast = lambda a: C.cast(a, C.c_void_p)  # noqa: E731
    kind = 0 if bits == 32 else 3
    good = dict(params=cast(room), grads=cast(room), averages=cast(room), squares=cast(room), sizes=cast((C.c_int64 * 1)(0)), grad_types=cast((C.c_int64 * 1)(kind)),
                count=1, bits=32, step=1.0, rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)

    def call(**changed):
        return lib.tg_adamw_step(C.byref(_lib.AdamW(**{**good, **changed})))
    assert call() == 0 and call(count=0) == 0  # an empty tensor, no tensor
    for changed in (dict(count=-1), dict(params=None), dict(sizes=None), dict(bits=16), dict(bits=8), dict(beta1=1.0), dict(beta2=-0.5), dict(eps=-1.0), dict(step=0.0),
                    dict(step=float("nan")), dict(sizes=cast((C.c_int64 * 1)(-1))), dict(copies=cast(room))):
        assert call(**changed) == -1, changed
    size = cast((C.c_int64 * 1)(5))
    assert call(sizes=size, params=cast((C.c_void_p * 1)(0))) == -1
    assert call(sizes=size, grad_types=cast((C.c_int64 * 1)(9))) == -1
    assert lib.tg_adamw_step(None) == -1
