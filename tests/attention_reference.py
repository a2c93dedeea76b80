"""Linear attention in 64 bits by the sum over all pairs of rows, and how far a computation may be from it."""
import torch

U = 2.0 ** -24
TYPES = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of a rounding, relative


def _head(q, k, v, log_a, state, scale, weigh):
    """One sequence and head; weigh: pairs count (1 + |log of their decay|) times, as the error of a decay does."""
    reach = log_a.cumsum(0)
    between = (reach[:, None] - reach[None]).masked_fill(torch.ones(len(reach), len(reach), dtype=torch.bool, device=q.device).triu(1), -torch.inf)
    w, start, end = between.exp(), reach.exp(), (reach[-1] - reach).exp()
    if weigh:
        w, start, end = (d * (1.0 + l.clamp_min(-800.0).abs()) for d, l in ((w, between), (start, reach), (end, reach[-1] - reach)))
    o = ((q @ k.T) * w) @ v + start[:, None] * (q @ state)
    whole = reach[-1].exp() * (1.0 + reach[-1].abs() if weigh else 1.0)
    return o * scale, (k * end[:, None]).T @ v + whole * state


def reference(q, k, v, gates, initial, cuts, gate_form, scale=None, weigh=False):
    """(rows, G, K), (rows, H, V), gates (rows, H) or (H,) in float64 -> outputs, final states."""
    heads, shared = v.shape[1], v.shape[1] // k.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    log_a = (gates if gate_form == "log" else torch.nn.functional.logsigmoid(gates)).clamp_min(-1000.0)
    if log_a.dim() == 1:
        log_a = log_a.expand(q.shape[0], heads)
    outs, finals = torch.zeros_like(v), []
    for n, (a, b) in enumerate(zip(cuts, cuts[1:])):
        finals.append([])
        for h in range(heads):
            state = initial[n, h] if initial is not None else q.new_zeros((k.shape[-1], v.shape[-1]))
            if b > a:
                o, state = _head(q[a:b, h // shared], k[a:b, h // shared], v[a:b, h], log_a[a:b, h], state, scale, weigh)
                outs = outs.index_put((torch.arange(a, b, device=q.device), torch.tensor(h, device=q.device)), o)
            finals[-1].append(state)
    return outs, torch.stack([torch.stack(f) for f in finals])


def with_bounds(q, k, v, gates, initial, cuts, gate_form, grad_outputs, grad_final, scale=None):
    """-> [(value, magnitude)] of outputs, final states and the gradients of q, k, v, gates (and initial): a magnitude is the same sum over the
    terms' absolute values, for the gates' gradient over what it is computed from: k.dk and q.dq of all rows of its sequence and head."""
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v, gates)] + ([] if initial is None else [initial.detach().double().requires_grad_()])
    sizes = [t.detach().double().abs().requires_grad_() for t in (q, k, v)] + [gates.detach().double()] + (
        [] if initial is None else [initial.detach().double().abs().requires_grad_()])
    results = []
    for some, weigh in ((leaves, False), (sizes, True)):
        o, f = reference(*some[:4], some[4] if initial is not None else None, cuts, gate_form, scale, weigh)
        ends = [(e, g.double().abs() if weigh else g.double()) for e, g in ((o, grad_outputs), (f, grad_final)) if g is not None]
        wanted = [t for t in some if t.requires_grad]
        loss = sum((e * g).sum() for e, g in ends)
        grads = torch.autograd.grad(loss, wanted, allow_unused=True) if loss.requires_grad else [None] * len(wanted)
        grads = [torch.zeros_like(t) if g is None else g for g, t in zip(grads, wanted)]
        results.append([o.detach(), f.detach(), *grads])
    values, magnitudes = results
    dq, dk = magnitudes[2:4]
    shared = v.shape[1] // k.shape[1]
    rows = ((sizes[0] * dq + sizes[1] * dk).sum(-1)).detach().repeat_interleave(shared, 1)  # a key head's counts for each of its value heads
    change = torch.zeros((q.shape[0], v.shape[1]), dtype=torch.float64, device=q.device)
    for n, (a, b) in enumerate(zip(cuts, cuts[1:])):
        if b > a:
            change[a:b] = rows[a:b].sum(0)
            if initial is not None and len(magnitudes) > 5:
                change[a:b] += (sizes[4][n] * magnitudes[5][n]).sum((1, 2)).detach()
    magnitudes.insert(5, change if gates.dim() == 2 else change.sum(0))
    if gates.dim() == 1:
        magnitudes[5] = (change * torch.ones_like(change)).sum(0)
    return list(zip(values, magnitudes))


def assert_near(name, got, value, magnitude, rows, input_type):
    """What is computed from `rows` rows at most: sums of products in float32 (64 in a row and one for each chunk of 32 rows, the decays of two units
    of theirs), the pairs of a chunk rounded as the inputs are where the output has their type, and the output's own rounding."""
    half = TYPES[got.dtype]
    steps = 64 + rows / 32
    bound = steps * U * magnitude + (half * 1.01) * value.abs()
    if got.dtype == input_type and got.dtype != torch.float32:
        bound = bound + half * 1.01 * magnitude + 2.0 ** -16 * magnitude
    # decays below 2^-126 are zeros in float32, and what they would have scaled here is less than 2^26; a half has no steps below 2^-24
    bound = bound + 2.0 ** -100 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = (got.detach().double().reshape(value.shape) - value).abs()
    worst = (off / bound.clamp_min(1e-300)).nan_to_num(nan=0.0 if bool((off == 0).all()) else torch.inf)
    worst = torch.where(off == 0, torch.zeros_like(worst), worst)
    assert not got.isnan().any(), f"{name} has values that are none"
    assert worst.numel() == 0 or worst.max().item() <= 1.0, f"{name}: {worst.max().item():.3g} times the bound"
