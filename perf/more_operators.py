"""Linear attention with decays, its single step, and the AdamW step over many tensors as timed cases.

A case is one pass through one operator:

  step       one step of linear attention for a batch of sequences, as a program that answers token by token or frame by frame runs it: a
             state of K x V in 32 bits for each sequence and head, the new one written beside it
  attention  S_t = a_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t over whole sequences, (B, T, heads, size), forward ("view") or forward and
             backward ("train"); the decay a is a head's own (`fixed`) or one for each step and head
  packed     the same over sequences of different lengths laid end to end, (T, heads, size) with offsets; one is empty and some rows lie behind
             the last one
  adamw      one step of AdamW over a list of tensors: a scene's vertices, colours and opacities, or a network's many weights; the averages in 32
             bits, or in 8 with two scales for every 256 values
"""
import math
import random

import torch

own = False

CASE = dict(kind="attention", task="train", batch=1, length=1, heads=1, key_heads=1, key_size=64, value_size=64, type="bfloat16",
            gate_type="float32", gate="log", fixed=False, initial=False, pad=0, tensors=1, elements=1, bits=32, copies=False, scene=False)


def _case(**kw):
    assert set(kw) <= set(CASE) | {"name"}
    return dict(CASE, **kw)


def listed():
    return [
        # one sequence answered token by token: nothing but a launch and host work
        _case(name="step_one", kind="step", task="view", batch=1, heads=16, key_heads=16),
        # a full batch of sequences: the states are all there is to move
        _case(name="step_batch", kind="step", task="view", batch=256, heads=32, key_heads=8, key_size=128, value_size=128, gate="logit",
              gate_type="same"),
        # reading one long prompt: few heads to split, the axis itself has to be
        _case(name="prompt", task="view", length=32768, heads=16, key_heads=16, key_size=128, value_size=128, initial=True),
        # a short odd sequence in 32 bits, what a test or a first try has
        _case(name="short_train", batch=2, length=77, heads=3, key_heads=3, key_size=24, value_size=40, type="float32", initial=True),
        # an ordinary training step, a decay for each step and head
        _case(name="heads_train", batch=4, length=4096, heads=16, key_heads=16, key_size=128, value_size=128),
        # smaller heads with a fixed decay each, which the gradient reaches too
        _case(name="fixed_train", batch=8, length=2048, heads=32, key_heads=32, key_size=64, value_size=64, fixed=True),
        # documents of every length laid end to end, queries and keys shared by four heads, padded to the buffer's end
        _case(name="packed_train", kind="packed", batch=37, length=30011, heads=16, key_heads=4, key_size=64, value_size=128, type="float16",
              gate="logit", gate_type="same", initial=True, pad=57),
        # a training step in 32 bits whose head sizes fill no tile
        _case(name="float_train", batch=2, length=3000, heads=8, key_heads=8, key_size=100, value_size=72, type="float32", gate="logit"),
        # a scene of a million triangles being fitted to images: vertices, colours, opacities
        _case(name="adamw_scene", kind="adamw", tensors=3, elements=8 * 1_500_000, type="float32", scene=True),
        # a small network's weights: hundreds of little tensors, where launches are what counts
        _case(name="adamw_small", kind="adamw", tensors=320, elements=900_000, type="float32"),
        # a large network's weights in mixed precision: gradients and copies in 16 bits
        _case(name="adamw_large", kind="adamw", tensors=96, elements=160_000_000, type="bfloat16", copies=True),
        # the same with the averages in 8 bits
        _case(name="adamw_large_8bit", kind="adamw", tensors=96, elements=160_000_000, type="bfloat16", copies=True, bits=8),
    ]


def _log(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    kind = rng.choice(["step", "attention", "attention", "attention", "packed", "adamw", "adamw"])
    case = dict(CASE, kind=kind, type=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), gate=rng.choice(["log", "logit"]),
                gate_type=rng.choice(["float32", "float32", "same"]), task=rng.choice(["view", "train", "train"]), fixed=rng.random() < 0.2,
                initial=rng.random() < 0.5)
    if kind == "adamw":
        case.update(tensors=rng.choice([1, 2, 3, 17, 60, 250]), elements=round(_log(rng, 20_000, 100_000_000)), bits=rng.choice([32, 32, 8]),
                    copies=case["type"] != "float32" and rng.random() < 0.7, task="train")
        return case
    case.update(key_size=rng.choice([16, 32, 48, 64, 64, 128, 128, rng.randint(5, 128)]), key_heads=rng.choice([1, 2, 4, 5, 8, 16]))
    case["value_size"] = case["key_size"] if rng.random() < 0.6 else rng.choice([16, 32, 64, 96, 128, rng.randint(5, 128)])
    case["heads"] = case["key_heads"] * rng.choice([1, 1, 1, 2, 4])
    if kind == "step":
        case.update(task="view", initial=False)
        case["batch"] = max(1, round(_log(rng, 1, 130_000_000 / (case["heads"] * case["key_size"] * case["value_size"]))))
        return case
    rows = max(1, round(_log(rng, 100, 2_000_000 / case["heads"] if case["task"] == "train" else 4_000_000 / case["heads"])))
    rows = max(1, min(rows, 60_000))
    if kind == "packed":
        case.update(batch=rng.randint(1, max(1, min(64, rows // 8))), length=rows, pad=rng.choice([0, 0, min(rng.randint(1, 200), rows // 2)]))
    else:
        case["batch"] = max(1, round(_log(rng, 1, min(64, rows))))
        case["length"] = max(1, min(16_384, rows // case["batch"]))
    return case


def _types(case):
    kind = getattr(torch, case["type"])
    return kind, torch.float32 if case["gate_type"] == "float32" else kind


BLOCK = 256  # values under one scale, and what a tensor's place in the flat buffers is a multiple of


def _sizes(case):
    """The numbers of elements of an adamw case's tensors: a scene's 4, 3 and 1 for a vertex, or a network's, odd ones among them."""
    n = case["elements"]
    if case["scene"]:
        return [n // 8 * 4, n // 8 * 3, n // 8]
    rng = random.Random(case["tensors"] * 1_000_003 + n)
    shares = [math.exp(rng.gauss(0.0, 1.3)) for _ in range(case["tensors"])]
    return [max(1, int(n * s / sum(shares))) for s in shares]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind, second = _types(case)

    def normal(shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean).to(dtype)

    s = dict(case, train=case["task"] == "train", scale=case["key_size"] ** -0.5)
    if case["kind"] == "adamw":
        sizes = _sizes(case)
        starts, total = [], 0
        for n in sizes:  # the tensors lie in one buffer each of weights, gradients and averages
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        for at, n in zip(starts, sizes):
            used[at:at + n] = True
        # gradients differ in size from place to place by orders of magnitude, and the averages belong to them
        size = torch.exp(normal((total,), scale=1.5, mean=-6.0)).mul_(used)
        s["p"] = normal((total,), scale=0.05).mul_(used)
        s["g"] = normal((total,)).mul_(size).to(kind)
        average, root = normal((total,), scale=0.3).mul_(size), size * (1.0 + 0.2 * torch.rand((total,), generator=g, device="cuda"))
        if case["bits"] == 8:
            s["m"], m_scale = _nearest8(average)
            s["v"], r_scale = _nearest8(root)
            s["scales"] = torch.stack([m_scale, r_scale], 1)
        else:
            s["m"], s["v"], s["scales"] = average, root * root, None
        s["copy"] = s["p"].to(kind) if case["copies"] else None
        parts = lambda t: None if t is None else [t[at:at + n] for at, n in zip(starts, sizes)]  # noqa: E731
        s["lists"] = {k: parts(s[k]) for k in ("p", "g", "m", "v", "copy")}
        s["lists"]["scales"] = None if s["scales"] is None else [s["scales"][at // BLOCK:-(-(at + n) // BLOCK)] for at, n in zip(starts, sizes)]
        s["grad_scale"] = torch.tensor([0.5], device="cuda")  # what clipping the gradients' norm left
        s.update(step=1000, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, decay=0.01, seed=seed & 0xFFFF)
        return s
    B, T, H, G, K, V = (case[k] for k in ("batch", "length", "heads", "key_heads", "key_size", "value_size"))
    rows = (B,) if case["kind"] == "step" else (T,) if case["kind"] == "packed" else (B, T)
    s["q"], s["k"], s["v"] = normal(rows + (G, K), kind), normal(rows + (G, K), kind), normal(rows + (H, V), kind)
    gates = (H,) if case["fixed"] else rows + (H,)
    if case["gate"] == "log":  # rates from a third of a step to thousands of steps
        s["gates_in"] = (-normal(gates, scale=1.5, mean=-3.5).exp()).to(second)
    else:
        s["gates_in"] = normal(gates, second, scale=1.5, mean=3.0)
    s["offsets"] = None
    if case["kind"] == "packed":  # lengths between nothing and twice the mean, one of them nothing
        share = torch.rand((B,), generator=g, device="cuda").double()
        if B > 2:
            share[B // 2] = 0.0
        cuts = torch.cat([share.new_zeros(1), (share.cumsum(0) / share.sum() * (T - case["pad"])).round()])
        s["offsets"] = cuts.to(torch.int32)
    if case["kind"] == "step":
        s["state"], s["out"] = normal((B, H, K, V)), torch.empty((B, H, K, V), device="cuda")
        return s
    s["h0"] = normal((B, H, K, V)) if case["initial"] else None
    s["grad_out"] = normal(rows + (H, V), kind) if s["train"] else None
    s["grad_final"] = normal((B, H, K, V)) if s["train"] and case["initial"] else None
    return s


def run(s):
    if s["kind"] == "adamw":
        return _own_adamw(s) if own else _plain_adamw(s)
    if s["kind"] == "step":
        return _own_step(s) if own else _plain_step(s)
    return _own_attention(s) if own else _plain_attention(s)


# ---- the framework's calls -----------------------------------------------------------

def _own_step(s):
    import trigrad_amd
    o, state = trigrad_amd.linear_attention_step(s["q"], s["k"], s["v"], s["gates_in"], s["state"], gate_form=s["gate"], out=s["out"])
    return [o, state]


def _own_attention(s):
    import trigrad_amd
    leaves = [s[k] for k in ("q", "k", "v", "gates_in", "h0")]
    if s["train"]:
        leaves = [None if t is None else t.detach().requires_grad_() for t in leaves]
    o, final = trigrad_amd.linear_attention(*leaves, s["offsets"], gate_form=s["gate"])
    if not s["train"]:
        return [o, final]
    ends = [(e, g) for e, g in ((o, s["grad_out"]), (final, s["grad_final"])) if g is not None]
    grads = torch.autograd.grad([e for e, _ in ends], [t for t in leaves if t is not None], [g for _, g in ends])
    return [o.detach(), final.detach(), *grads]


def _own_adamw(s):
    import trigrad_amd
    t = s["lists"]
    trigrad_amd.adamw_step(t["p"], t["g"], t["m"], t["v"], s["step"], lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["decay"],
                           copies=t["copy"], scales=t["scales"], grad_scale=s["grad_scale"], seed=s["seed"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "m", "v", "copy", "scales") if s[k] is not None}


# ---- the plain forms -------------------------------------------------------------------

def _plain_step(s):
    shared = s["heads"] // s["key_heads"]
    q, k = (s[n].float().repeat_interleave(shared, 1) for n in ("q", "k"))
    g = s["gates_in"].float()
    a = g.exp() if s["gate"] == "log" else torch.sigmoid(g)
    state = a[..., None, None] * s["state"] + k[..., :, None] * s["v"].float()[..., None, :]
    o = (state * q[..., :, None]).sum(-2) * s["scale"]
    return [o.to(s["q"].dtype), state]


CHUNK = 64


def _chunked(q, k, v, log_a, h0, scale):
    """(B, T, H, size) and decays' logarithms (B, T, H) in 64 bits -> outputs and final states, by chunks of 64 rows: within a chunk by products of all pairs,
    between chunks by their states, which are summed by doubling."""
    B, T, H, K = q.shape
    fill = -T % CHUNK

    def split(t):
        t = torch.cat([t, t.new_zeros((B, fill, *t.shape[2:]))], 1) if fill else t
        return t.reshape(B, -1, CHUNK, *t.shape[2:]).movedim(3, 1).contiguous()  # (B, H, chunks, 64, ...)
    q, k, v, reach = split(q), split(k), split(v), split(log_a).cumsum(-1)
    place = torch.arange(CHUNK, device=q.device)
    between = (reach[..., :, None] - reach[..., None, :]).float()
    pairs = torch.where(place[:, None] >= place, between, -math.inf).exp()
    inside = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * pairs, v)
    whole = reach[..., -1:]
    state = torch.matmul((k * (whole - reach).float().exp()[..., None]).transpose(-1, -2).contiguous(), v)
    a = whole.float().exp()[..., None]  # (B, H, chunks, 1, 1)
    if h0 is not None:
        state = torch.cat([state[:, :, :1] + a[:, :, :1] * h0[:, :, None], state[:, :, 1:]], 2)
    width = 1
    while width < state.shape[2]:
        state = torch.cat([state[:, :, :width], state[:, :, width:] + a[:, :, width:] * state[:, :, :-width]], 2)
        a = torch.cat([a[:, :, :width], a[:, :, width:] * a[:, :, :-width]], 2)
        width *= 2
    before = torch.cat([(h0 if h0 is not None else torch.zeros_like(state[:, :, 0]))[:, :, None], state[:, :, :-1]], 2)
    o = (inside + torch.matmul(q, before) * reach.float().exp()[..., None]) * scale
    return o.movedim(1, 3).reshape(B, T + fill, H, -1)[:, :T], state[:, :, -1]


def _plain_attention(s):
    packed = s["kind"] == "packed"
    names = ["q", "k", "v", "gates_in"] + (["h0"] if s["h0"] is not None else [])
    rows = {n: s[n].double() if n == "gates_in" else s[n].float() for n in names}
    if packed:
        # laid out side by side: what is behind a sequence's end has keys of zero and decays of one
        begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
        step = torch.arange(max(1, int((end - begin).max())), device="cuda")
        there = step < (end - begin)[:, None]
        at = (begin[:, None] + step).clamp_max(s["length"] - 1)
        lay = lambda t: torch.where(there.view(*there.shape, *(1,) * (t.dim() - 1)), t[at], torch.zeros((), dtype=t.dtype, device="cuda"))  # noqa: E731
        back = lambda t: t.new_zeros((s["length"], *t.shape[2:])).index_put_((at[there],), t[there])  # noqa: E731
        laid = ["q", "k", "v"] + ([] if s["fixed"] else ["gates_in"])
        rows.update({n: lay(rows[n]) for n in laid})
    leaves = [rows[n].detach().requires_grad_(s["train"]) for n in names]
    h0 = leaves[4] if s["h0"] is not None else None
    with torch.set_grad_enabled(s["train"]):
        shared = s["heads"] // s["key_heads"]
        q, k = (t.repeat_interleave(shared, -2) for t in leaves[:2])
        g = leaves[3]
        log_a = g if s["gate"] == "log" else -torch.log1p(torch.exp(-g))
        if s["fixed"]:
            log_a = log_a.expand(*q.shape[:-1])
        if packed:
            log_a = torch.where(there[..., None], log_a, 0.0)
        o, final = _chunked(q, k, leaves[2], log_a, h0, s["scale"])
    kind = s["q"].dtype
    out = [(back(o.detach()) if packed else o.detach()).to(kind), final.detach()]
    if not s["train"]:
        return out
    ends = [(o, lay(s["grad_out"].float()) if packed else s["grad_out"].float())] + ([(final, s["grad_final"])] if s["grad_final"] is not None else [])
    grads = torch.autograd.grad([e for e, _ in ends], leaves, [d for _, d in ends])
    return out + [(back(d) if packed and n in laid else d).to(s[n].dtype) for d, n in zip(grads, names)]


LARGEST8 = 448.0  # of an 8-bit value with 4 bits of exponent and 3 of fraction, whose smallest is 2^-9


def _blocks(t):
    return t.view(-1, BLOCK)


def _nearest8(x):
    """(values in 8 bits, scales): what an average is before the first step that is looked at."""
    scale = _blocks(x).abs().amax(1) / LARGEST8
    unit = torch.where(scale > 0.0, 1.0 / scale, 0.0)
    return (_blocks(x) * unit[:, None]).clamp(-LARGEST8, LARGEST8).to(torch.float8_e4m3fn).view(-1), scale


def _random16(count, seed):
    """Two random numbers of 16 bits for each place: a 32-bit integer of place and seed, mixed by products and shifts."""
    x = torch.arange(count, dtype=torch.int64, device="cuda") * 0x9E3779B1 + (seed * 0x85EBCA6B + 0xC2B2AE35 & 0xFFFFFFFF) & 0xFFFFFFFF
    x = (x ^ x >> 16) * 0x7FEB352D & 0xFFFFFFFF
    x = (x ^ x >> 15) * 0x846CA68B & 0xFFFFFFFF
    x = x ^ x >> 16
    return x & 0xFFFF, x >> 16


def _to8(x, noise, least):
    """Blocks of x in units of their largest / 448, rounded to one of the two neighbours in 8 bits by `noise`, up with the probability of what lies below;
    `least`: what is not zero does not become zero."""
    largest = _blocks(x).abs().amax(1)
    unit = torch.where(largest >= 2.0 ** -110, LARGEST8 / largest, 0.0)
    y = torch.clamp_max(_blocks(x).abs() * unit[:, None], LARGEST8).view(-1)
    normal = ((y.view(torch.int32) + (noise.to(torch.int32) << 4)) & -(1 << 20)).view(torch.float32)
    small = torch.floor(y * 512.0 + noise.float() * 2.0 ** -16)
    if least:
        small = torch.where(y > 0.0, small.clamp_min(1.0), small)
    y = torch.where(y >= 2.0 ** -6, normal, small * 2.0 ** -9)
    return torch.copysign(y, x).to(torch.float8_e4m3fn), torch.where(largest >= 2.0 ** -110, largest / LARGEST8, 0.0)


def _plain_adamw(s):
    b1, b2 = s["betas"]
    p, g = s["p"], s["g"].float() * s["grad_scale"]
    if s["bits"] == 8:
        m, root = ((_blocks(s[n].float()) * s["scales"][:, j, None]).view(-1) for j, n in enumerate(("m", "v")))
        v = root * root
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    root = v.sqrt()
    rate, unbias = s["lr"] / (1.0 - b1 ** s["step"]), 1.0 / math.sqrt(1.0 - b2 ** s["step"])
    p.copy_(p * (1.0 - s["lr"] * s["decay"]) - rate * (m / (root * unbias + s["eps"])))
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if s["bits"] == 8:
        low, high = _random16(p.numel(), s["seed"])
        m8, m_scale = _to8(m, low, False)
        r8, r_scale = _to8(root, high, True)
        s["m"].copy_(m8)
        s["v"].copy_(r8)
        s["scales"].copy_(torch.stack([m_scale, r_scale], 1))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    kind, second = _types(case)
    wide, narrow = kind.itemsize, second.itemsize
    train = case["task"] == "train"
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        one = 8 + wide + (4.0 + 16.0 / BLOCK if case["bits"] == 8 else 16) + (wide if case["copies"] else 0)
        return {"bytes": n * one, "flops": n * 15}
    B, H, G, K, V = (case[k] for k in ("batch", "heads", "key_heads", "key_size", "value_size"))
    rows = B if case["kind"] == "step" else case["length"] if case["kind"] == "packed" else B * case["length"]
    states, gates = B * H * K * V * 4, H * narrow * (1 if case["fixed"] else rows)
    keys, values = rows * G * K * wide, rows * H * V * wide
    if case["kind"] == "step":
        return {"bytes": 2 * keys + 2 * values + gates + 2 * states, "flops": 5 * rows * H * K * V}
    size = 2 * keys + 2 * values + gates + states * (2 if case["initial"] else 1)
    flops = rows * H * 4 * K * V
    if train:
        size += 2 * keys + 2 * values + gates + (2 * states if case["initial"] else 0)
        flops *= 4
    return {"bytes": size, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------

def _all_pairs(q, k, v, log_a, h0, scale, block):
    """One sequence of one head, (T, K), (T, K), (T, V), (T,), by the sum over all pairs, `block` rows of outputs at a time -> (T, V), (K, V)."""
    reach = log_a.cumsum(0)
    outs = []
    for at in range(0, q.shape[0], block):
        r = reach[at:at + block]
        upto = at + r.shape[0]
        w = r[:, None] - reach[None, :upto]
        w = torch.exp(w.masked_fill(torch.ones_like(w, dtype=torch.bool).triu(at + 1), -math.inf))
        o = ((q[at:upto] @ k[:upto].T) * w) @ v[:upto]
        outs.append((o if h0 is None else o + torch.exp(r)[:, None] * (q[at:upto] @ h0)) * scale)
    final = (k * torch.exp(reach[-1] - reach)[:, None]).T @ v
    return torch.cat(outs), final if h0 is None else final + torch.exp(reach[-1]) * h0


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adamw":
        p, g = s["p"].double(), s["g"].double() * s["grad_scale"].double()
        if case["bits"] == 8:
            spread = s["scales"].double().repeat_interleave(BLOCK, 0)
            m, v = s["m"].double() * spread[:, 0], (s["v"].double() * spread[:, 1]) ** 2
        else:
            m, v = s["m"].double(), s["v"].double()
        m, v = s["betas"][0] * m + (1 - s["betas"][0]) * g, s["betas"][1] * v + (1 - s["betas"][1]) * g ** 2
        corrected = [x / (1 - b ** s["step"]) for x, b in zip((m, v), s["betas"])]
        p = p - s["lr"] * s["decay"] * p - s["lr"] * corrected[0] / (corrected[1] ** 0.5 + s["eps"])
        scales = None
        if case["bits"] == 8:
            scales = torch.stack([m.view(-1, BLOCK).abs().max(1).values, v.view(-1, BLOCK).max(1).values ** 0.5], 1) / 448.0
        out = {"p": p, "m": m if case["bits"] == 32 else None, "v": v if case["bits"] == 32 else None, "copy": p, "scales": scales}
        return {k: out[k] for k in out if s[k] is not None}
    train, shared = s["train"], case["heads"] // case["key_heads"]
    gates = s["gates_in"].double()
    if case["kind"] == "step":
        a = torch.exp(gates) if case["gate"] == "log" else torch.sigmoid(gates)
        group = torch.arange(case["heads"], device="cuda") // shared
        q, k = s["q"].double()[:, group], s["k"].double()[:, group]
        state = s["state"].double().mul_(a[..., None, None])
        state += torch.einsum("bhk,bhv->bhkv", k, s["v"].double())
        return [torch.einsum("bhk,bhkv->bhv", q, state) * s["scale"], state]
    if case["kind"] == "packed":
        cuts = s["offsets"].tolist()
        spans = [(slice(p, q), n) for n, (p, q) in enumerate(zip(cuts, cuts[1:]))]
    else:
        spans = [((n, slice(None)), n) for n in range(case["batch"])]
    if len(spans) * case["heads"] > 1500:
        return None
    if train and max((s["q"][at].shape[0] for at, _ in spans), default=0) > 12_000:
        return None
    leaf = lambda t: None if t is None else t.double().requires_grad_(train)  # noqa: E731
    q, k, v, g, h0 = leaf(s["q"]), leaf(s["k"]), leaf(s["v"]), leaf(s["gates_in"]), leaf(s["h0"])
    leaves = [t for t in (q, k, v, g, h0) if t is not None]
    o = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    final = torch.zeros((case["batch"], case["heads"], case["key_size"], case["value_size"]), dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(t) for t in leaves] if train else []
    with torch.set_grad_enabled(train):
        for at, n in spans:
            for h in range(case["heads"]):
                rows = s["q"][at].shape[0]
                start = None if h0 is None else h0[n, h]
                if rows == 0:
                    if start is not None:
                        final[n, h] = start.detach()
                        if train:
                            grads[-1][n, h] += s["grad_final"][n, h]
                    continue
                log_a = (g[h].expand(rows) if case["fixed"] else g[at][:, h])
                if case["gate"] == "logit":
                    log_a = torch.nn.functional.logsigmoid(log_a)
                x, last = _all_pairs(q[at][:, h // shared], k[at][:, h // shared], v[at][:, h], log_a, start, s["scale"], rows if train else 2048)
                o[at][:, h], final[n, h] = x.detach(), last.detach()
                if train:
                    loss = (x * s["grad_out"][at][:, h].double()).sum()
                    if s["grad_final"] is not None:
                        loss = loss + (last * s["grad_final"][n, h].double()).sum()
                    for total, d in zip(grads, torch.autograd.grad(loss, leaves)):
                        total += d
    return [o, final, *grads]
