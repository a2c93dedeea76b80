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
