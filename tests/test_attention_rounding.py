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
    assert got.isfinite().all(), name
    worst = ((got.double() - value).abs() / bound_of(name, got, value, magnitude, rows)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times the bound"


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
