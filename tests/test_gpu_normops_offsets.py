"""Group normalisation where a group's mean is large against its deviation, in every form of the statistics.

Bounds, in units of u = 2^-24.  A thread sums differences from its own first value (exact: the values are neighbours) and
squares of them: n u of sums of n terms, at most 95 here.  Its mean is rounded to 32 bits, and so is a block's: each is off
by at most e = u |mean|.  e^2 enters the variance, and so does twice the products of these errors with the differences
between the means, a deviation over the root of n or less; signs are random, so that M values of a group leave 2 e std / M^0.5
a level: two levels, half of it in rstd, 8 deviations: 16 e / (std M^0.5).  Sums of x and x^2 in 32 bits (or sums around a
value far away) are off by u mean^2 / (std^2 M^0.5) of the variance instead, at 1e4 deviations 600 times that.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N = 95                        # most terms a thread sums: 480 x 640 in 102 blocks of 32 pixels a sweep
K = 1.5 * N + 32              # in a mean and, halved, in a sum of squares; coefficients and roundings


@pytest.fixture(scope="module")
def ops():
    import miseg_amd  # noqa: F401
    from miseg_amd import lib as L
    from miseg_amd import normops
    L.check(L.load().miseg_device_check())
    return normops


def close(got, want, tol):
    off = ((got.double() - want).abs() - tol).max().item()
    assert off <= 0, "off by %g more than allowed" % off


# one launch (at most 2048 pixels), two (partial sums that a block adds up), three (many pixels; slabs that cut groups; more
# images than a step takes)
SHAPES = [(2, 40, 50, 64, 8), (3, 61, 83, 40, 5), (1, 90, 80, 72, 9), (1, 960, 1280, 64, 16), (2, 75, 80, 1560, 3), (6, 480, 640, 64, 1)]


def check(x, groups, saved, extra, K=K):
    n, h, w, c = x.shape
    for i in range(n):                                         # an image at a time: the reference is in 64 bits
        v = x[i].double().reshape(h * w, groups, c // groups)
        mean = v.mean(2).mean(0)                               # a dimension at a time: torch's means over two of them
        std = (v - mean[:, None]).square().mean(2).mean(0).sqrt()    # differ from call to call where few values are long sums
        close(saved.mean[i], mean, 4 * U * mean.abs() + K * U * std)
        off = U * mean.abs() / std
        close(saved.rstd[i], 1 / std, (K * U + 4 * off * off + 16 * off / (h * w * c / groups) ** 0.5 + extra(std)) / std)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("offset,dt", [(1e3, torch.float32), (1e4, torch.float32), (-1e4, torch.float32), (30.0, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_mean_of_many_deviations(ops, shape, offset, dt, checkpoint):
    n, h, w, c, groups = shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn((n, h, w, c), generator=gen, device="cuda") + offset).to(dt)
    _, saved = ops.group_norm_act(x, None, None, groups, eps=0.0, checkpoint=checkpoint)
    check(x, groups, saved, lambda std: 0.0)


@pytest.mark.parametrize("offset,dt", [(1e4, torch.float32), (30.0, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_first_pixel_far_from_the_rest(ops, shape, offset, dt):
    """The threads that start at it sum n differences of the offset: their squares, and the square of their sum, are off by n u
    and 2 n u of n offset^2 at the worst, one thread a channel, of the channel's share of a group, pixels * std^2; half of it
    in rstd.  So is their mean: n u offset for n of the pixels."""
    n, h, w, c, groups = shape
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((n, h, w, c), generator=gen, device="cuda") + offset
    x[:, 0, 0] = 0
    x = x.to(dt)
    _, saved = ops.group_norm_act(x, None, None, groups, eps=0.0)
    check(x, groups, saved, lambda std: 1.5 * U * N * N * offset * offset / (h * w * std * std))


# more terms a thread than the 64 that a K of 160 covers at the worst: pixels of a block over pixels of a sweep
LONG = [((1, 1920, 1280, 48, 6), 115), ((2, 300, 400, 1032, 43), 142), ((1, 3, 700, 65536, 1), 132), ((5, 480, 640, 64, 16), 95)]


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("shape,terms", LONG, ids=str)
def test_sums_of_many_terms_a_thread(ops, shape, terms, checkpoint):
    """Statistics within 1.5 of their own number of terms (and 32 roundings) of u; the parameters' gradients within that number
    and the 8 roundings of a term (g, x - mean, their product, rstd; mean and rstd are the call's own) of their magnitudes."""
    n, h, w, c, groups = shape
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn((n, h, w, c), generator=gen, device="cuda") + 1).to(torch.bfloat16)
    dy = torch.randn((n, h, w, c), generator=gen, device="cuda").to(torch.bfloat16)
    _, saved = ops.group_norm_act(x, None, None, groups, eps=0.0, checkpoint=checkpoint)
    check(x, groups, saved, lambda std: 0.0, 1.5 * terms + 32)
    _, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    sums = torch.zeros((4, c), dtype=torch.float64, device="cuda")
    for i in range(n):
        g = dy[i].double()
        if checkpoint:
            ck = saved.checkpoint
            xhat = ck.codes[i].double() * ck.scales[i].double().repeat_interleave(32, 2)[..., :c]
        else:
            xhat = (x[i].double() - saved.mean[i].double().repeat_interleave(c // groups)) * \
                saved.rstd[i].double().repeat_interleave(c // groups)
        sums += torch.stack([t.sum((0, 1)) for t in (g * xhat, g, (g * xhat).abs(), g.abs())])
    close(dgamma, sums[0], (terms + 8) * U * sums[2])
    close(dbeta, sums[1], (terms + 8) * U * sums[3])
