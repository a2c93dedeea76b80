"""Linear attention over units of several chunks, as ordinary calls are split, against the definition in 64 bits: all types, widths and forms, and whole
sequences in one workgroup.  How a call is split is read from the memory that it asks for."""
import ctypes as C

import pytest
import torch

from attention_reference import with_bounds
from test_attention import make
from test_attention_rounding import NAMES, bound_of

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODES = {F32: 0, F16: 1, BF16: 2}
DENSE = [(K, V, shared, fixed) for K, V in ((24, 32), (64, 48), (128, 100)) for shared, fixed in ((4, False), (1, True))]
PACKED = [0, 0, 5, 700, 701, 2100, 2100, 2560, 2590]  # sequences of none, one and more rows, and rows behind the last
THROUGH = (64, 1100, 8)  # sequences, rows of each, heads: a workgroup goes through a whole sequence


def split_of(dtype, sequences, length, heads, key_heads, K, V, packed=False):
    """-> (units of all sequences at most, whether a workgroup has a whole sequence)"""
    from trigrad_amd import _lib
    sizes = (C.c_int64 * 4)()
    call = _lib.Attention(sequences=sequences, length=length, heads=heads, key_heads=key_heads, key_size=K, value_size=V, type=CODES[dtype], gate_type=0, gate_form=1,
                          scale=1.0, offsets=16 if packed else None)
    assert _lib.load(32).tg_linear_attention_sizes(C.byref(call), sizes) == 0
    return sizes[0] // (heads * K * V * 4) - sequences, sizes[1] == 0  # a state for each unit, and one for each sequence


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_calls_here_have_units_of_several_chunks(dtype):
    chunk = 32 if dtype == F32 else 64
    for K, V, shared, _ in DENSE:
        units, through = split_of(dtype, 1, 2573, 16, 16 // shared, K, V)
        assert 1 < units < 2573 / chunk / 2 and not through
    units, through = split_of(dtype, len(PACKED) - 1, 2600, 16, 4, 40, 64, True)
    assert len(PACKED) < units < 2600 / chunk / 2 + len(PACKED) and not through
    sequences, rows, heads = THROUGH
    units, through = split_of(dtype, sequences, rows, heads, heads, 16, 16)
    assert sequences < units < sequences * rows / chunk / 2 and through


def compare(got, wanted, rows, positive):
    for name, t, (value, magnitude) in zip(NAMES, got, wanted):
        t = t.detach().reshape(value.shape)
        bound = bound_of(name, t, value, magnitude, rows)
        assert t.isfinite().all(), name
        worst = ((t.double() - value).abs() / bound).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3g} times the bound"
        # of terms that do not cancel, what is missing or has the other sign is far beyond the bound
        assert not positive or bound.norm() <= 0.25 * value.norm(), name


def run(cuda, parts, initial, cuts, gate_form, dense, positive):
    import trigrad_amd
    g = torch.Generator().manual_seed(1)
    if positive:
        parts = [t.abs() for t in parts[:3]] + [parts[3]]
        initial = None if initial is None else initial.abs()
    leaves = [t.view(*dense, *t.shape[1:]).detach().requires_grad_() if dense and t.dim() > 1 else t.detach().requires_grad_() for t in parts]
    leaves += [] if initial is None else [initial.detach().requires_grad_()]
    offsets = None if dense else torch.tensor(cuts, dtype=torch.int32, device=cuda)
    out = trigrad_amd.linear_attention(*leaves[:4], leaves[4] if initial is not None else None, offsets, gate_form)
    grads = [torch.randn(t.shape, generator=g).to(cuda, t.dtype) for t in out]
    if positive:
        grads = [t.abs() for t in grads]
    got = [*out, *torch.autograd.grad(out, leaves, grads)]
    wanted = with_bounds(*parts, initial, cuts, gate_form, grads[0].reshape(parts[2].shape), grads[1])
    compare(got, wanted, max(b - a for a, b in zip(cuts, cuts[1:])), positive)


@pytest.mark.gpu
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("K,V,shared,fixed", DENSE)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_one_sequence(cuda, dtype, K, V, shared, fixed, positive):
    parts, initial = make(cuda, K + shared, 2573, 16 // shared, shared, K, V, dtype, "logit" if fixed else "log", BF16 if dtype == BF16 and fixed else F32, fixed, 1)
    if positive:  # sums that a half has room for
        parts[2] /= 16
    run(cuda, parts, initial, [0, 2573], "logit" if fixed else "log", (1, 2573), positive)


@pytest.mark.gpu
@pytest.mark.parametrize("gate_form", ["log", "logit"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gates_in_16_bits(cuda, dtype, gate_form):
    """Their gradients are made of float32 products and sums and rounded once."""
    parts, initial = make(cuda, 13, 2573, 16, 1, 64, 48, dtype, gate_form, dtype, False, 1)
    parts[2] /= 16
    run(cuda, parts, initial, [0, 2573], gate_form, (1, 2573), True)


@pytest.mark.gpu
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_packed_sequences(cuda, dtype, fixed, positive):
    parts, initial = make(cuda, 11, 2600, 4, 4, 40, 64, dtype, "logit", F32, fixed, len(PACKED) - 1)
    if positive:
        parts[2] /= 16
    run(cuda, parts, initial, PACKED, "logit", None, positive)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_whole_sequences_of_several_units(cuda, dtype):
    """The states between units are kept on the way, for the backward pass; without one the results are the same."""
    import trigrad_amd
    sequences, rows, heads = THROUGH
    parts, initial = make(cuda, 12, sequences * rows, heads, 1, 16, 16, dtype, sequences=sequences)
    run(cuda, parts, initial, list(range(0, sequences * rows + 1, rows)), "log", (sequences, rows), False)
    args = [t.view(sequences, rows, *t.shape[1:]) for t in parts] + [initial]
    trained = trigrad_amd.linear_attention(*args[:4], initial.detach().clone().requires_grad_())
    plain = trigrad_amd.linear_attention(*args)
    assert all(torch.equal(a, b) for a, b in zip(trained, plain))
