"""Group norm of samples that are split over workgroups, where a group's first value is unlike all others: the statistics may not depend on it.

Tolerances, with u = 2^-24.  Let E^2 be the sum of squares of a thread's values (of one channel) about their mean; two of them are at most 1.5 E
apart.  A batch is at most eight rows, summed about its first: the squares about that are at most 8 times those about the batch's mean, their
sum is off by 11 u and the square of the sum of distances by 19 u of that, so a batch's squares by 245 u of themselves.  Its mean, from the
thread's first value, is off by 18 u E, and after at most 32 batches (256 rows, more than a thread has here) the mean so far by 48 u E more:
the distance of two means by 70 u E.  Merging adds w d^2 with weights w of at most 8 and distances d, sum w d^2 <= E^2, so
2 * 70 u E * sum w d <= 140 u E sqrt(32 * 8) E = 2240 u E^2.  Everything behind a thread is in 64 bits.  Hence the variance is off by 2500 u of
itself, rstd by half of that, and the mean by 70 u sqrt(256) = 1120 u standard deviations and, rounded once, u of itself.  Neither has the distance of
an outlier in it.  These go through the formulas to first order; beside that an output is rounded once."""
import pytest
import torch

import test_norm

U = 2.0 ** -24


def bounds(x, groups, eps=1e-5):
    """(y, its bound) in 64 bits, without weights and activation; on x's device."""
    N, C = x.shape[0], x.shape[-1]
    x64 = x.double().reshape(N, -1, groups, C // groups)
    mean = x64.mean((1, 3), keepdim=True)
    rstd = ((x64 - mean).square().mean((1, 3), keepdim=True) + eps) ** -0.5
    hat = (x64 - mean) * rstd
    d = hat.abs() * (1250 + 4) * U + 1120 * U + U * mean.abs() * rstd
    return hat.reshape(x.shape), d.reshape(x.shape)


def assert_near(name, got, want, bound):
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = ((got.double() - want).abs() / ((bound + want.abs()) * half + bound + tiny)).max().item()
    assert off <= 1.0, f"{name}: {off:.2f} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("distance", [30.0, 100.0, 300.0, 2000.0])
@pytest.mark.parametrize("shape,groups", [((1, 40000, 4), 1), ((1, 16384, 32), 1), ((2, 16384, 33), 3), ((1, 1080, 1920, 32), 8)])
def test_first_value_far_from_all_others(shape, groups, distance, dtype, cuda):
    import trigrad_amd
    rng = torch.Generator(cuda).manual_seed(int(distance))
    x = torch.randn(shape, generator=rng, device=cuda)
    if dtype == torch.float32:
        x += distance  # the others are far from zero, the first value is zero
    x = x.to(dtype)
    first = x.view(shape[0], -1, shape[-1])[:, 0, ::shape[-1] // groups]
    first.fill_(0.0 if dtype == torch.float32 else distance)
    y = trigrad_amd.group_norm(x, groups)
    assert_near("y", y, *bounds(x, groups))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 9, 64, 700])
def test_first_rows_far_from_all_others(rows, cuda):
    """A padded or background run in front, of part of a thread's rows, of all of some threads' and of whole workgroups'."""
    import trigrad_amd
    x = torch.randn((2, 40000, 24), generator=torch.Generator(cuda).manual_seed(rows), device=cuda) + 1000.0
    x[:, :rows] = 0.0
    assert_near("y", trigrad_amd.group_norm(x, 4), *bounds(x, 4))


@pytest.mark.gpu
def test_channels_with_means_of_their_own(cuda):
    """A group whose channels lie apart, all of them far from zero."""
    import trigrad_amd
    rng = torch.Generator(cuda).manual_seed(1)
    x = torch.randn((1, 30000, 64), generator=rng, device=cuda) + 3000.0 + 20.0 * torch.randn((64,), generator=rng, device=cuda)
    assert_near("y", trigrad_amd.group_norm(x, 2), *bounds(x, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("channels,groups,dtype", [(3000, 3000, torch.float32), (3000, 1500, torch.float32), (5000, 1000, torch.bfloat16), (4104, 27, torch.bfloat16),
                                                   (2999, 2999, torch.float16), (1025, 5, torch.float32)])
def test_groups_of_several_tiles(channels, groups, dtype, cuda):
    """Rows of several workgroups, each with some of the groups, the ends of which lie anywhere."""
    x, w, b, dy = test_norm.make(cuda, groups, (1, 1100, channels), dtype, torch.float32)
    test_norm.run_and_check(x, groups, w, b, dy, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups,ahead,lines", [((1024, 4096, 257), 1, None, 1), ((2 ** 21, 65), 1, 2048, 1), ((2 ** 25, 64), 8, 65536, 32)])
def test_long_chains_of_additions(shape, groups, ahead, lines, cuda):
    """A thread adds at most 256 values to each other, whatever there are: streamed rows, tokens, held samples.  The gradient of the bias where the first value of every
    chain is 2^24, to which a 1 is lost: 255 and, over the workgroup's threads of a channel, `lines` more additions, each off by u of the sum."""
    import trigrad_amd
    channels = shape[-1]
    x = torch.zeros(shape, dtype=torch.bfloat16, device=cuda)
    dy = torch.ones(shape, dtype=torch.bfloat16, device=cuda)
    (dy[:, 0] if ahead is None else dy[:ahead]).fill_(2.0 ** 24)
    bias = torch.zeros((channels,), device=cuda, requires_grad=True)
    (got,) = torch.autograd.grad(trigrad_amd.group_norm(x, groups, None, bias), bias, dy)
    first = shape[0] if ahead is None else ahead
    want = first * 2.0 ** 24 + (x.numel() // channels - first)
    assert ((got.double() - want).abs() <= (255 + lines + 8) * U * want).all(), ((got.double() - want).abs().max() / want / U).item()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((64, 512), 8), ((64, 8, 64), 4), ((64, 1024), 1), ((64, 1001), 1), ((1, 30000, 32), 8)])
def test_the_slope_of_relu_is_its_outputs(shape, groups, cuda):
    """At the border, where the rounding decides: an output above 0 passes its gradient on, to the bias, the weight and x alike, and one of 0 to none."""
    import trigrad_amd
    rng = torch.Generator(cuda).manual_seed(1)
    channels = shape[-1]
    x = torch.randn(shape, generator=rng, device=cuda)
    weight = torch.rand((channels,), generator=rng, device=cuda) + 0.5
    hat, _ = bounds(x, groups)
    at = (0,) * (len(shape) - 1)  # the position that z is put to the border for, in every channel
    bias = -(hat[at] * weight).float()
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    y = trigrad_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="relu")
    dy = torch.zeros_like(y)
    dy[at] = 1.0
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    passes = y.detach()[at] > 0
    assert 0.2 < passes.float().mean() < 0.8
    assert torch.equal(db, passes.float())
    assert torch.equal(dw != 0, passes)
