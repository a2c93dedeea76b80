"""What linear attention in 16 bits rounds: outputs and gradients once, and everything in front of that far below it."""
import pytest
import torch

from attention_reference import TYPES, U, with_bounds
from test_attention import make

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("outputs", "final", "dq", "dk", "dv", "dgates", "dinitial")


def bound_of(name, got, value, magnitude, rows):
    """Sums of products in float32 (64 in a row and one for each chunk of 32 rows), the output's own rounding, and, in an output of bfloat16 that rows have,
    every term's: a pair, or a number of a state, is the sum of two parts there, which leave 2^-16 of it.  Two of float16 leave 2^-22, below the sums'."""
    bound = (64 + rows / 32) * U * magnitude + 1.01 * TYPES[got.dtype] * value.abs()
    if name in ("outputs", "dq", "dk", "dv") and got.dtype == BF16:
        bound = bound + 2.0 ** -16 * magnitude
    # decays below 2^-126 are zeros in float32; a half has no steps below 2^-24
    return bound + 2.0 ** -100 + (2.0 ** -25 if got.dtype == F16 else 0.0)


def assert_rounded_once(name, got, value, magnitude, rows):
    got = got.detach().reshape(value.shape)
    bound = bound_of(name, got, value, magnitude, rows)
    there = value.abs() + bound < torch.finfo(got.dtype).max  # a value beyond is infinite in the output's type
    assert got[there].isfinite().all(), name
    worst = ((got.double() - value).abs() / bound)[there]
    assert worst.numel() == 0 or worst.max().item() <= 1.0, f"{name}: {worst.max().item():.3g} times the bound"


def passes(cuda, parts, initial, batch, gate_form="log", scale=None, seed=0):
    """Outputs and gradients of `batch` sequences, and the same in 64 bits with the terms' magnitudes."""
    import trigrad_amd
    g = torch.Generator().manual_seed(seed)
    rows = parts[2].shape[0] // batch
    leaves = [t.view(batch, rows, *t.shape[1:]).detach().requires_grad_() if t.dim() > 1 else t.detach().requires_grad_() for t in parts]
    leaves += [] if initial is None else [initial.detach().requires_grad_()]
    out = trigrad_amd.linear_attention(*leaves[:4], *leaves[4:], gate_form=gate_form, scale=scale)
    grads = [torch.randn(t.shape, generator=g).to(cuda, t.dtype) for t in out]
    got = [*out, *torch.autograd.grad(out, leaves, grads)]
    wanted = with_bounds(*parts, initial, list(range(0, batch * rows + 1, rows)), gate_form, grads[0].reshape(parts[2].shape), grads[1], scale)
    return got, wanted


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(16, 24), (64, 64), (40, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_pairs_of_a_chunk(cuda, dtype, K, V):
    """Terms that cancel: an output near zero is off by what its terms leave of their parts, and not by half a step of the terms."""
    for rows, initial in ((64, False), (200, True)):
        parts, h0 = make(cuda, K + rows, 2 * rows, 2, 2, K, V, dtype, sequences=2 if initial else None)
        got, wanted = passes(cuda, parts, h0, 2)
        for name, t, (value, magnitude) in zip(NAMES, got, wanted):
            assert_rounded_once(name, t, value, magnitude, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [1e-6, 3.9, 4.0, 8.0, 1e4])
def test_chunks_of_zeros(cuda, dtype, scale):
    """Padding, or a projection that begins with zeros: a chunk's queries, keys, values or all of them are zero."""
    for zeros in ((0,), (1,), (2,), (0, 1, 2)):
        parts, h0 = make(cuda, 3, 192, 2, 1, 32, 32, dtype, sequences=1)
        for i in zeros:
            parts[i][64:128] = 0.0
        parts[2] *= 1.0 / max(scale, 1.0)  # outputs of 16 bits have a largest
        got, wanted = passes(cuda, parts, h0 / max(scale, 1.0), 1, scale=scale)
        for name, t, (value, magnitude) in zip(NAMES, got, wanted):
            assert_rounded_once(name, t, value, magnitude, 192)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_far_larger_than_others(cuda, dtype):
    """A row's query, or a later row's key, does not change how other rows' pairs are rounded."""
    for which, row in ((0, 20), (1, 50), (2, 50)):
        parts, _ = make(cuda, 7, 128, 1, 2, 32, 48, dtype, mean=-1.0)
        for t in parts[:2]:
            t *= 2.0 ** -12
        parts[which][row] *= 2.0 ** (25 if which < 2 else 12)
        got, wanted = passes(cuda, parts, None, 1, scale=2.0 ** 6)
        for name, t, (value, magnitude) in list(zip(NAMES, got, wanted))[:3 if which < 2 else 2]:
            assert_rounded_once(name, t, value, magnitude, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(32, 32), (128, 72), (24, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_pairs_of_a_query_that_is_not_finite(cuda, dtype, K, V, value):
    """A query is read by its own row: the others of its chunk keep all their terms, bit by bit."""
    import trigrad_amd
    parts, h0 = make(cuda, 5, 2 * 200, 2, 1, K, V, dtype, sequences=2)
    args = [t.view(2, 200, *t.shape[1:]) for t in parts] + [h0]
    want = trigrad_amd.linear_attention(*args)
    spoiled = args[0].clone()
    spoiled[1, 70, 0, 3] = value
    got = trigrad_amd.linear_attention(spoiled, *args[1:])
    assert torch.equal(got[1], want[1])
    assert not got[0][1, 70, 0].isfinite().any()
    keep = torch.ones_like(got[0], dtype=torch.bool)
    keep[1, 70, 0] = False
    assert torch.equal(got[0][keep], want[0][keep])


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(32, 32), (64, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_values_of_different_size(cuda, dtype, K, V):
    """Columns of a state far smaller than their neighbours have float32's accuracy too."""
    parts, _ = make(cuda, 9, 300, 2, 1, K, V, dtype)
    sizes = 2.0 ** torch.linspace(-9, 12, V, device=cuda).round()[torch.randperm(V, generator=torch.Generator().manual_seed(1)).to(cuda)]
    parts[2] *= sizes
    got, wanted = passes(cuda, parts, None, 1)
    for name, t, (value, magnitude) in list(zip(NAMES, got, wanted))[:2]:
        assert_rounded_once(name, t, value, magnitude, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(32, 32), (128, 72), (24, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_columns_that_are_not_finite(cuda, dtype, K, V, value):
    """A value, or an output's gradient, spoils its own column of states and outputs (in float32 its neighbour's too): the others keep all their terms, bit
    by bit."""
    import trigrad_amd
    parts, h0 = make(cuda, 5, 2 * 200, 2, 1, K, V, dtype, sequences=2)
    args = [t.view(2, 200, *t.shape[1:]) for t in parts] + [h0]
    g = torch.Generator().manual_seed(0)
    grads = [torch.randn(args[2].shape, generator=g).to(cuda, dtype), torch.randn(h0.shape, generator=g).to(cuda)]

    def results(args, grads):
        leaves = [t.detach().requires_grad_() for t in args]
        out = trigrad_amd.linear_attention(*leaves)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, grads)]
    want = results(args, grads)
    column = slice(4 if dtype == F32 else 5, 6)
    # a value's
    spoiled = [t.clone() for t in args]
    spoiled[2][1, 70, 0, 5] = value
    o, final = results(spoiled, grads)[:2]
    assert not o[1, 70:, 0, 5].isfinite().any() and not final[1, 0, :, 5].isfinite().any()
    for t, w, at in ((o, want[0], (1, slice(None), 0, column)), (final, want[1], (1, 0, slice(None), column))):
        keep = torch.ones_like(t, dtype=torch.bool)
        keep[at] = False
        assert torch.equal(t[keep], w[keep])
    # a gradient's: column 5 of D up to its row, the row's query, the keys up to it (and those of its chunk)
    spoiled = [t.clone() for t in grads]
    spoiled[0][1, 70, 0, 5] = value
    _, _, dq, dk, dv, dg, dh = results(args, spoiled)
    assert not dq[1, 70, 0].isfinite().any() and not dk[1, :71, 0].isfinite().any()
    assert not dv[1, :71, 0, 5].isfinite().any() and not dh[1, 0, :, 5].isfinite().any()
    for t, w, at in ((dq, want[2], (1, 70, 0)), (dk, want[3], (1, slice(0, 128), 0)), (dv, want[4], (1, slice(None), 0, column)), (dg, want[5], (1, slice(None), 0)),
                     (dh, want[6], (1, 0, slice(None), column))):
        keep = torch.ones_like(t, dtype=torch.bool)
        keep[at] = False
        assert torch.equal(t[keep], w[keep])
