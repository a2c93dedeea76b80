"""Sizes that the operators' C calls ask for and refuse, without a GPU."""
import ctypes as C

import pytest

TYPES = {32: (0, 4), 64: (3, 8)}  # a type of each library, and its bytes


def norm_sizes(bits, **kw):
    from trigrad_amd import _lib
    kind = TYPES[bits][0]
    out = (C.c_int64 * 2)()
    n = _lib.Norm(**{**dict(type=kind, weight_type=kind, eps=1e-5), **kw})
    return _lib.load(bits).tg_group_norm_sizes(C.byref(n), out), list(out)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("positions,channels,groups", [(1024, 65536, 65536), (600, 262144, 262144), (600, 262143, 262143), (4000, 40000, 10000),
                                                       (2000, 100001, 1), (1920 * 1080, 32, 8), (3000, 2 ** 17, 2 ** 16)])
def test_group_norm_workspace_is_a_fraction_of_its_input(bits, positions, channels, groups):
    """What workgroups leave each other, two sums for a group or, backward, a channel that they have, is a small part of what they read, however many groups
    there are."""
    code, sizes = norm_sizes(bits, samples=1, positions=positions, channels=channels, groups=groups)
    assert code == 0 and max(sizes) <= positions * channels * TYPES[bits][1] // 4


def recurrence_sizes(bits, **kw):
    from trigrad_amd import _lib
    kind = TYPES[bits][0]
    out = (C.c_int64 * 3)()
    r = _lib.Recurrence(**{**dict(type=kind, gate_type=kind), **kw})
    return _lib.load(bits).tg_linear_recurrence_sizes(C.byref(r), out), list(out)


def test_linear_recurrence_beyond_a_grid():
    """A grid has fewer than 2^32 threads: of calls that one of the launches is too large for none is made."""
    most = (1 << 25) - 8  # channels of the starting states' launch, 1024 threads for eight
    assert recurrence_sizes(32, sequences=1, length=129, channels=most, gate_count=most)[0] == 0
    assert recurrence_sizes(32, sequences=1, length=129, channels=most + 1, gate_count=most + 1)[0] == -1
    assert recurrence_sizes(32, sequences=1, length=129, channels=1 << 25, gate_count=1, type=2)[0] == -1
    assert recurrence_sizes(32, sequences=1, length=128, channels=1 << 25, gate_count=1 << 25)[0] == 0  # a chunk: no such launch
    # a thread a sequence and channel
    most = (1 << 32) // 256 - 1
    assert recurrence_sizes(64, sequences=256, length=1, channels=most, gate_count=1)[0] == 0
    assert recurrence_sizes(64, sequences=256, length=1, channels=most + 1, gate_count=1)[0] == -1
    assert recurrence_sizes(64, sequences=1 << 20, length=3, channels=1 << 12, gate_count=1)[0] == -1
