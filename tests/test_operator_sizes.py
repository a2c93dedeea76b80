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
