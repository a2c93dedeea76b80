"""The gated linear recurrence and the channels-last group norm as timed cases.

A case is one pass through one operator:

  step    one step of the recurrence for a batch of sequences, as a program that answers token by token or frame by
          frame runs it: a 32-bit state for each sequence and channel, the new one written beside it
  scan    h_t = a_t h_{t-1} + b_t over whole sequences, (B, T, D), forward ("view") or forward and backward ("train")
  packed  the same over sequences of different lengths laid end to end, (T, D) with offsets; some are empty and some
          rows lie behind the last one
  layers  images that the renderer drew of a scene's depth slabs, composited back to front: a slab's remaining
          transmittance is the gate of its pixel's three colours, and only the last state, the finished image, is kept
  norm    group norm with an activation over (N, positions, C), positions in rows as an image of the renderer lies

The gates are values, logarithms or logits (`gate`); the input of a step is x itself or (1 - a) x (`mix`).
"""
import math

import torch

own = False

CASE = dict(kind="scan", task="train", batch=1, length=1, channels=64, gates=64, type="bfloat16", gate_type="same", gate="value",
            mix="plain", initial=False, reverse=False, pad=0, groups=8, activation="none", affine=True)


def _case(**kw):
    assert set(kw) <= set(CASE) | {"name"}
    return dict(CASE, **kw)


def listed():
    return [
        # one sequence answered token by token: nothing but a launch and host work
        _case(name="step_one", kind="step", task="view", batch=1, channels=1024, gates=1024, gate="logit", mix="complement"),
        # a full batch of sequences, a decay for each head of 128 channels
        _case(name="step_batch", kind="step", task="view", batch=512, channels=4096, gates=32, gate="log"),
        # a short odd sequence in 32 bits, what a test or a first try has
        _case(name="scan_short_train", batch=2, length=77, channels=96, gates=96, type="float32", initial=True),
        # reading one long prompt: few rows to split, the axis itself has to be
        _case(name="scan_prompt", task="view", length=32768, channels=2048, gates=2048, gate="logit", mix="complement", initial=True),
        # an ordinary training step, decays by head in logarithms
        _case(name="scan_heads_train", batch=4, length=4096, channels=2048, gates=16, gate="log", gate_type="float32"),
        # an ordinary training step, a gate for every channel
        _case(name="scan_channels_train", batch=2, length=8192, channels=1536, gates=1536, type="float16", gate="logit",
              mix="complement", initial=True),
        # documents of every length laid end to end, padded to the buffer's end
        _case(name="packed_train", kind="packed", batch=213, length=70001, channels=384, gates=384, type="bfloat16", initial=True, pad=57),
        # eight depth slabs of a full frame composited, the gradient going back to the slabs
        _case(name="layers_train", kind="layers", length=8, channels=3 * 1920 * 1080, gates=1920 * 1080, type="float32", reverse=True),
        # a thumbnail's features
        _case(name="norm_thumbnail", kind="norm", task="view", length=50 * 50, channels=32, type="float32", activation="silu"),
        # an odd batch of odd images whose groups end inside a vector
        _case(name="norm_ragged_train", kind="norm", batch=3, length=53 * 37, channels=120, groups=8, type="float16", activation="gelu"),
        # the states of a recurrence normalised by head, token by token
        _case(name="norm_heads_train", kind="norm", batch=16384, length=1, channels=2048, groups=16, activation="none"),
        # a frame's features in the network that shades it: one image, two million positions
        _case(name="norm_frame_train", kind="norm", length=1920 * 1080, channels=32, groups=8, activation="silu", gate_type="float32"),
    ]


def _log(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan", "packed", "layers", "norm", "norm", "norm"])
    case = dict(CASE, kind=kind, type=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), gate=rng.choice(["value", "log", "logit"]),
                mix=rng.choice(["plain", "complement"]), gate_type=rng.choice(["same", "same", "float32"]),
                task=rng.choice(["view", "train", "train"]), initial=rng.random() < 0.5, reverse=rng.random() < 0.25)
    if kind == "norm":
        channels = 0
        while not 4 <= channels <= 4096:
            case["groups"] = rng.choice([1, 2, 4, 5, 8, 16, 32])
            channels = case["groups"] * round(_log(rng, 1.0, 256.0))
        case.update(channels=channels, activation=rng.choice(["none", "relu", "silu", "gelu"]), affine=rng.random() < 0.85)
        rows = min(_log(rng, 64, 2_000_000), 120_000_000 / getattr(torch, case["type"]).itemsize / channels)
        case["batch"] = max(1, round(_log(rng, 1, rows))) if rng.random() < 0.5 else rng.randint(1, 4)
        case["length"] = max(1, int(rows // case["batch"]))
        return case
    shared = rng.choice([1, 1, 3, 4, 16, 64, 128])
    if kind == "step":
        case.update(task="view", batch=max(1, round(_log(rng, 1, 1024))), reverse=False, initial=False)
        case["gates"] = max(1, round(_log(rng, 64, 8192) / shared))
    elif kind == "layers":
        case.update(length=rng.randint(2, 24), gates=round(_log(rng, 2_500, 500_000)), gate="value", mix="plain", type="float32",
                    gate_type="same", initial=rng.random() < 0.3, reverse=True)
        shared = 3
    else:
        elements = _log(rng, 20_000, 56_000_000 / getattr(torch, case["type"]).itemsize)
        case["gates"] = max(1, round(min(_log(rng, 1, 4096), elements / 8) / shared))
        rows = max(1, round(elements / (case["gates"] * shared)))
        case["batch"] = max(1, round(_log(rng, 1, min(64, rows)))) if kind == "scan" else rng.randint(1, max(1, min(500, rows)))
        case["length"] = max(1, min(65_536, rows // case["batch"])) if kind == "scan" else min(400_000, rows)
        if kind == "packed":
            case["pad"] = rng.choice([0, 0, min(rng.randint(1, 200), case["length"] // 2)])
    case["channels"] = case["gates"] * shared
    return case


def _types(case):
    kind = getattr(torch, case["type"])
    return kind, torch.float32 if case["gate_type"] == "float32" else kind


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind, second = _types(case)
    B, T, D, G = case["batch"], case["length"], case["channels"], case["gates"]

    def normal(shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)

    s = dict(case, train=case["task"] == "train")
    if case["kind"] == "norm":
        # features have means and scales of their own in every channel
        mean, scale = normal((D,)), normal((D,), scale=0.5).exp()
        s["x"] = torch.randn((B, T, D), generator=g, device="cuda").mul_(scale).add_(mean).to(kind)
        s["weight"], s["bias"] = (normal((D,), second, 0.3, 1.0), normal((D,), second, 0.3)) if case["affine"] else (None, None)
        s["grad"] = normal((B, T, D), kind) if s["train"] else None
        return s
    rows = (B,) if case["kind"] == "step" else (T,) if case["kind"] == "packed" else (B, T)
    s["x"] = normal(rows + (D,), kind)
    if case["gate"] == "value":  # decays, or the transmittances that slabs leave: mostly between a half and one
        gates = torch.rand(rows + (G,), generator=g, device="cuda").sqrt_()
    elif case["gate"] == "log":  # rates from a tenth of a step to thousands of steps
        gates = -normal(rows + (G,), scale=1.5, mean=-3.5).exp()
    else:
        gates = normal(rows + (G,), scale=1.5, mean=2.0)
    s["gates_in"] = gates.to(second)
    s["offsets"] = None
    if case["kind"] == "packed":
        cuts = torch.randint(0, T - case["pad"] + 1, (B + 1,), generator=g, device="cuda").sort().values
        cuts[0], cuts[-1] = 0, T - case["pad"]
        if B > 2:
            cuts[B // 2] = cuts[B // 2 + 1]  # an empty sequence
        s["offsets"] = cuts.to(torch.int32)
    if case["kind"] == "step":
        s["state"], s["out"] = normal((B, D)), torch.empty((B, D), device="cuda")
        return s
    s["h0"] = normal((B, D)) if case["initial"] else None
    s["states"] = case["kind"] != "layers"
    s["grad_states"] = normal(rows + (D,), kind) if s["train"] and s["states"] else None
    s["grad_final"] = normal((B, D)) if s["train"] and (case["initial"] or not s["states"]) else None
    return s


def run(s):
    if s["kind"] == "norm":
        return _own_norm(s) if own else _plain_norm(s)
    if s["kind"] == "step":
        return _own_step(s) if own else _plain_step(s)
    return _own_scan(s) if own else _plain_scan(s)


# ---- the framework's calls -----------------------------------------------------------

def _leaf(t, train):
    return t.detach().requires_grad_() if train and t is not None else t


def _own_step(s):
    import trigrad_amd
    h, state = trigrad_amd.linear_recurrence_step(s["x"], s["gates_in"], s["state"], gate_form=s["gate"], input_form=s["mix"], out=s["out"])
    return [h, state]


def _own_scan(s):
    import trigrad_amd
    x, gates, h0 = (_leaf(s[k], s["train"]) for k in ("x", "gates_in", "h0"))
    h, final = trigrad_amd.linear_recurrence(x, gates, h0, s["offsets"], gate_form=s["gate"], input_form=s["mix"], reverse=s["reverse"],
                                             return_states=s["states"])
    if not s["train"]:
        return [h, final]
    ends = [(o, g) for o, g in ((h, s["grad_states"]), (final, s["grad_final"])) if g is not None]
    leaves = [t for t in (x, gates, h0) if t is not None]
    grads = torch.autograd.grad([o for o, _ in ends], leaves, [g for _, g in ends])
    return [None if h is None else h.detach(), final.detach(), *grads]


def _own_norm(s):
    import trigrad_amd
    x, weight, bias = (_leaf(s[k], s["train"]) for k in ("x", "weight", "bias"))
    y = trigrad_amd.group_norm(x, s["groups"], weight, bias, eps=1e-5, activation=s["activation"])
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, weight, bias) if t is not None], s["grad"])]


# ---- the plain forms -------------------------------------------------------------------

def _doubled(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0: after the step of width w, b_t holds the sum of the last 2 w terms."""
    width = 1
    while width < b.shape[1]:
        b = torch.cat([b[:, :width], torch.addcmul(b[:, width:], a[:, width:], b[:, :-width])], 1)
        a = torch.cat([a[:, :width], a[:, width:] * a[:, :-width]], 1)
        width *= 2
    return b


def _gate(s):
    """(a, 1 - a, da / dgate) in 32 bits."""
    g = s["gates_in"].float()
    if s["gate"] == "value":
        return g, 1.0 - g, torch.ones_like(g)
    if s["gate"] == "log":
        return g.exp(), -torch.expm1(g), g.exp()
    return torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(g) * torch.sigmoid(-g)


def _plain_step(s):
    a, rest, _ = (t.repeat_interleave(s["channels"] // s["gates"], -1) for t in _gate(s))
    x = s["x"].float()
    state = a * s["state"] + (x if s["mix"] == "plain" else rest * x)
    return [state.to(s["x"].dtype), state]


def _plain_scan(s):
    packed, R, D = s["kind"] == "packed", s["channels"] // s["gates"], s["channels"]
    x, h0 = s["x"].float(), s["h0"]
    ga, grest, gslope = _gate(s)
    a, rest = ga.repeat_interleave(R, -1), grest.repeat_interleave(R, -1)
    if packed:
        # end to end as one sequence, first of each, last of each and rows of none marked by place
        rows = torch.arange(s["length"], device="cuda")
        of = torch.searchsorted(s["offsets"][1:].long(), rows, right=True).clamp_max(s["batch"] - 1)
        begin, end = s["offsets"].long()[of], s["offsets"].long()[of + 1]
        inside = (rows < end)[None, :, None]
        first, last = (rows == begin)[None, :, None] & inside, (rows == end - 1)[None, :, None] & inside
        x, a, rest = x[None], a[None], rest[None]
        empty = (s["offsets"][1:] == s["offsets"][:-1])[:, None]
        ends = (s["offsets"][1:].long() - 1).clamp_min(0)
        starts = s["offsets"][:-1].long().clamp_max(s["length"] - 1)
        if s["reverse"]:
            first, last, ends, starts = last, first, starts, ends
        start_state = h0[of][None] if h0 is not None else torch.zeros((), device="cuda")
    else:
        place = torch.arange(s["length"], device="cuda")[None, :, None]
        first, last = place == 0, place == s["length"] - 1
        if s["reverse"]:
            first, last = last, first
        inside = torch.ones_like(first)
        start_state = h0[:, None] if h0 is not None else torch.zeros((), device="cuda")
    turn = (lambda t: t.flip(1)) if s["reverse"] else (lambda t: t)
    back = (lambda t: t) if s["reverse"] else (lambda t: t.flip(1))
    b = torch.where(inside, x if s["mix"] == "plain" else rest * x, 0.0)
    through = torch.where(first | ~inside, 0.0, a)  # what passes from the step before
    h = turn(_doubled(turn(through), turn(b + torch.where(first, a * start_state, 0.0))))
    h = torch.where(inside, h, 0.0)
    if packed:
        final = torch.where(empty, h0 if h0 is not None else torch.zeros((), device="cuda"), h[0, ends])
    else:
        final = h[:, 0] if s["reverse"] else h[:, -1]
    kind = s["x"].dtype
    out = [h.view(s["x"].shape).to(kind) if s["states"] else None, final]
    if not s["train"]:
        return out
    dh = s["grad_states"].float().view(x.shape) if s["grad_states"] is not None else torch.zeros_like(x)
    if s["grad_final"] is not None:
        df = s["grad_final"]
        dh = dh + torch.where(last, df[of][None] if packed else df[:, None], 0.0)
    # l_t = dh_t + a_{t+1} l_{t+1}: against the order, by the gate of the step after
    shift = -1 if not s["reverse"] else 1
    after = torch.where(last, 0.0, through.roll(shift, 1))
    lam = back(_doubled(back(after), back(torch.where(inside, dh, 0.0))))
    lam = torch.where(inside, lam, 0.0)
    before = torch.where(first, start_state, h.roll(-shift, 1))
    da = lam * before
    dx = lam
    if s["mix"] == "complement":
        da, dx = lam * (before - x), lam * rest
    dg = torch.where(inside, da, 0.0).view(*da.shape[:-1], s["gates"], R).sum(-1).view(s["gates_in"].shape) * gslope
    grads = [dx.view(s["x"].shape).to(kind), dg.to(s["gates_in"].dtype)]
    if h0 is not None:
        d0 = a * lam
        if packed:
            d0 = torch.where(empty, s["grad_final"], d0[0, starts])
        else:
            d0 = d0[:, -1] if s["reverse"] else d0[:, 0]
        grads.append(d0)
    return out + grads


def _plain_norm(s):
    N, S, D, G = s["batch"], s["length"], s["channels"], s["groups"]
    x = s["x"].float().view(N, S, G, D // G)
    centred = x - x.mean((1, 3), keepdim=True)
    rstd = (centred.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    hat = centred * rstd
    w = s["weight"].float().view(G, D // G) if s["affine"] else torch.ones((), device="cuda")
    z = hat * w + s["bias"].float().view(G, D // G) if s["affine"] else hat
    kind = s["activation"]
    if kind == "silu":
        sig = torch.sigmoid(z)
        y, slope = z * sig, sig * (1.0 + z * (1.0 - sig))
    elif kind == "gelu":
        phi = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        y, slope = z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    elif kind == "relu":
        y, slope = z.clamp_min(0.0), (z > 0.0).float()
    else:
        y, slope = z, torch.ones((), device="cuda")
    out = [y.view(N, S, D).to(s["x"].dtype)]
    if not s["train"]:
        return out
    dz = s["grad"].float().view(N, S, G, D // G) * slope
    dhat = dz * w
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    out.append(dx.view(N, S, D).to(s["x"].dtype))
    if s["affine"]:
        out += [(dz * hat).sum((0, 1)).view(D).to(s["weight"].dtype), dz.sum((0, 1)).view(D).to(s["bias"].dtype)]
    return out


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    kind, second = _types(case)
    wide, narrow = kind.itemsize, second.itemsize
    train = case["task"] == "train"
    D, G = case["channels"], case["gates"]
    if case["kind"] == "norm":
        n = case["batch"] * case["length"] * D
        return {"bytes": n * wide * (4 if train else 2) + (D * narrow * (4 if train else 2) if case["affine"] else 0), "flops": n * (40 if train else 15)}
    rows = case["batch"] if case["kind"] == "step" else case["length"] if case["kind"] == "packed" else case["batch"] * case["length"]
    n, gates, ends = rows * D, rows * G, case["batch"] * D * 4
    if case["kind"] == "step":
        return {"bytes": n * wide * 2 + gates * narrow + 2 * ends, "flops": 4 * n}
    states = case["kind"] != "layers"
    size = n * wide * (2 if states else 1) + gates * narrow + ends * (2 if case["initial"] else 1)
    if train:
        size += n * wide * (2 if states else 1) + gates * narrow + (ends if case["initial"] or not states else 0) + (ends if case["initial"] else 0)
    return {"bytes": size, "flops": n * (20 if train else 8)}


# ---- the definitions in 64 bits ----------------------------------------------------------

def exact(case, seed):
    if case["channels"] * case["length"] * case["batch"] > 400_000_000 and case["kind"] != "packed":
        return None
    s = prepare(case, seed)
    train = s["train"]
    leaf = lambda t: t.double().requires_grad_(train) if t is not None else None  # noqa: E731
    x = leaf(s["x"])
    if case["kind"] == "norm":
        w, b = leaf(s["weight"]), leaf(s["bias"])
        rows = x.reshape(case["batch"], case["length"], case["groups"], -1)
        var, mean = torch.var_mean(rows, (1, 3), unbiased=False, keepdim=True)
        z = ((rows - mean) / (var + 1e-5).sqrt()).reshape(x.shape)
        if case["affine"]:
            z = z * w + b
        act = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v / (1.0 + torch.exp(-v)),
               "gelu": lambda v: 0.5 * v * (1.0 + torch.erf(v / math.sqrt(2.0)))}
        y = act[case["activation"]](z)
        leaves = [t for t in (x, w, b) if t is not None]
        return [y.detach(), *(torch.autograd.grad(y, leaves, s["grad"].double()) if train else [])]
    gates = leaf(s["gates_in"])
    a = {"value": lambda v: v, "log": torch.exp, "logit": torch.sigmoid}[case["gate"]](gates)
    u = x.reshape(*gates.shape, -1)
    if case["mix"] == "complement":
        u = u * (1.0 - a)[..., None]
    if case["kind"] == "step":
        new = (a[..., None] * s["state"].double().reshape(u.shape) + u).reshape(x.shape)
        return [new, new]
    B, G, D = case["batch"], case["gates"], case["channels"]
    h0 = leaf(s["h0"])
    h = (h0 if h0 is not None else torch.zeros((B, D), dtype=torch.float64, device="cuda")).reshape(B, G, -1)
    if case["kind"] == "packed":
        cuts = s["offsets"].tolist()
        longest = max(q - p for p, q in zip(cuts, cuts[1:]))
        if B * longest * D > 400_000_000 or longest > 60_000:
            return None
        where = torch.tensor(cuts[:-1], device="cuda")[:, None] + torch.arange(longest, device="cuda")[None]
        there = where < torch.tensor(cuts[1:], device="cuda")[:, None]
        where = where.clamp_max(case["length"] - 1)
        a, u = a[where], u[where]
    else:
        longest = case["length"]
        there = None
    steps_a, steps_u, kept = a.unbind(1), u.unbind(1), [None] * longest
    for t in (reversed(range(longest)) if case["reverse"] else range(longest)):
        new = steps_a[t][..., None] * h + steps_u[t]
        h = new if there is None else torch.where(there[:, t, None, None], new, h)
        kept[t] = h
    final = h.reshape(B, D)
    states = None
    if s["states"]:
        states = torch.stack(kept, 1).reshape(B, longest, D)
        if there is not None:
            states = torch.zeros_like(x).index_put((where[there],), states[there])
    out = [None if states is None else states.detach(), final.detach()]
    if train:
        ends = [(o, g.double()) for o, g in ((states, s["grad_states"]), (final, s["grad_final"])) if g is not None]
        out += torch.autograd.grad([o for o, _ in ends], [t for t in (x, gates, h0) if t is not None], [g for _, g in ends])
    return out
