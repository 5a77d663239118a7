"""Group normalisation with an activation and the 8-bit activation checkpoints against their definitions in 64 bits.

Tolerances.  A result is rounded once to its type: at most eps / 2 of its value.  Before that the kernels work in 32 bits
(u = 2^-24): a sum of n terms held per thread is off by at most n u times the sum of magnitudes, and no case here gives a
thread more than 64 terms; sums across threads are in 64 bits.  K = 160 covers, in units of u, the worst of 64 terms in a
mean and 64 in a sum of squares (half of which reaches rstd), and the roundings of the coefficients, of the fma and of the
activation's exponential and reciprocal (2 + |z| and 1).
"""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 160
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    import miseg_amd  # noqa: F401
    from miseg_amd import lib as L
    from miseg_amd import normops
    L.check(L.load().miseg_device_check())
    return normops


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps          # half a subnormal step, and a bit


def close(got, want, tol):
    got = got.double()
    off = (got - want).abs() - tol
    worst = off.max().item()
    assert not torch.isnan(got).any() and worst <= 0, "off by up to %g more than allowed" % worst


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def spread(t, c):
    return t.repeat_interleave(c // t.shape[1], 1)[:, None, None, :]


def stats64(x, gamma, beta, groups, eps):
    n, h, w, c = x.shape
    v = x.double().reshape(n, h * w, groups, c // groups)
    mean = v.mean((1, 3))
    rstd = 1 / ((v - mean[:, None, :, None]).square().mean((1, 3)) + eps).sqrt()
    g = torch.ones(c, device=x.device).double() if gamma is None else gamma.double()
    b = torch.zeros(c, device=x.device).double() if beta is None else beta.double()
    scale = g * rstd.repeat_interleave(c // groups, 1)
    return mean, rstd, scale, b - mean.repeat_interleave(c // groups, 1) * scale


def backward64(xhat, z, zmag, dy, scale, groups, act, dt):
    """dx, dgamma, dbeta and their tolerances."""
    n, h, w, c = dy.shape
    d = act64(z, act)[1]
    g = dy.double() * d
    gabs = g.abs() if act != "silu" else dy.double().abs() * (1 + zmag)     # the derivative moves with z
    m = h * w * (c // groups)

    def share(s):
        return spread((scale * s).reshape(n, groups, -1).sum(2) / m, c)
    s1, s2 = g.sum((1, 2)), (g * xhat).sum((1, 2))
    a = scale[:, None, None]
    dx = a * g - share(s1) - xhat * share(s2)
    t1, t2 = gabs.sum((1, 2)), (gabs * xhat.abs()).sum((1, 2))

    def mag(s):
        return spread((scale.abs() * s).reshape(n, groups, -1).sum(2) / m, c)
    tol = K * U * (a.abs() * gabs + mag(t1) + xhat.abs() * mag(t2)) + half_step(dt) * dx.abs() + tiny(dt)
    return dx, s2.sum(0), s1.sum(0), tol, K * U * t2.sum(0) + 1e-30, K * U * t1.sum(0) + 1e-30


def make(n, h, w, c, dt, seed=0, offset=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=gen, device="cuda")
    x = (r(n, h, w, c) * (r(c).abs() + 0.3) + offset * r(c)).to(dt)
    return x, (r(n, h, w, c) * 0.1).to(dt), r(c) * 0.5 + 1, r(c) * 0.3


def check_forward(x, y, saved, gamma, beta, groups, eps, act):
    mean, rstd, scale, shift = stats64(x, gamma, beta, groups, eps)
    c = x.shape[3]
    xmax = spread(x.double().abs().amax((1, 2)).reshape(x.shape[0], groups, -1).amax(2), c)[:, 0, 0]
    dev = xmax * K * U                                         # of a mean: of the largest magnitude it sums
    close(saved.mean, mean, dev.reshape(x.shape[0], groups, -1).amax(2))
    close(saved.rstd, rstd, K * U * rstd)
    close(saved.scale, scale, K * U * scale.abs())
    close(saved.shift, shift, K * U * shift.abs() + 2 * scale.abs() * dev + K * U * (scale * xmax).abs())
    z = x.double() * scale[:, None, None] + shift[:, None, None]
    want = act64(z, act)[0]
    mag = (scale[:, None, None] * x.double()).abs() + shift.abs()[:, None, None] + (scale.abs() * xmax)[:, None, None]
    close(y, want, half_step(y.dtype) * want.abs() + 2 * K * U * mag + tiny(y.dtype))


SHAPES = [
    # n, h, w, c, groups
    (1, 1, 1, 8, 1),             # one pixel, one group
    (1, 1, 1, 64, 64),           # one value a group: nothing is left of it
    (2, 1, 5, 8, 8),
    (1, 2, 3, 512, 32),          # the deepest map of a 64 x 96 image
    (3, 7, 9, 40, 5),            # a block of 32 channels that ends after 8
    (2, 13, 11, 72, 24),         # groups of 3 channels
    (2, 17, 19, 24, 1),          # one group
    (1, 33, 65, 96, 4),
    (5, 6, 7, 128, 32),
    (2, 60, 80, 256, 32),
    (1, 21, 23, 264, 11),        # more than 32 groups of 8 channels, odd
    (1, 9, 5, 1032, 3),          # three slabs of channels
    (2, 5, 4, 4096, 64),
    (4, 97, 131, 64, 16),
    (1, 480, 640, 32, 32),
]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(ops, shape, dt):
    n, h, w, c, groups = shape
    for act in ("none", "relu", "silu"):
        x, dy, gamma, beta = make(n, h, w, c, dt, seed=c + h)
        y, saved = ops.group_norm_act(x, gamma, beta, groups, act=act)
        check_forward(x, y, saved, gamma, beta, groups, 1e-3, act)
        dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
        xhat = (x.double() - spread(saved.mean.double(), c)) * spread(saved.rstd.double(), c)
        z = x.double() * saved.scale.double()[:, None, None] + saved.shift.double()[:, None, None]
        zmag = (x.double() * saved.scale.double()[:, None, None]).abs() + saved.shift.double().abs()[:, None, None]
        wdx, wg, wb, tx, tg, tb = backward64(xhat, z, zmag, dy, saved.scale.double(), groups, act, dt)
        close(dx, wdx, tx)
        close(dgamma, wg, tg)
        close(dbeta, wb, tb)


def values(ck):
    c = ck.shape[3]
    return ck.codes.double() * ck.scales.double().repeat_interleave(32, 3)[..., :c]


def blocks_amax(v):
    n, h, w, c = v.shape
    pad = torch.zeros(n, h, w, (-c) % 32, dtype=v.dtype, device=v.device)
    return torch.cat([v, pad], 3).reshape(n, h, w, -1, 32).abs().amax(4)


def check_checkpoint(ck, v, err):
    """ck holds v (fp64), which the kernel knew to `err`."""
    amax = blocks_amax(v)
    bmax = blocks_amax(err)
    s = ck.scales.double()
    assert ((s - amax / 127).abs() <= (amax / 127 + bmax / 127) * (half_step(torch.bfloat16) + 4 * U) + bmax / 127).all()
    per = s.repeat_interleave(32, 3)[..., :v.shape[3]]
    # half a step; the product with the rounded reciprocal of the scale is off by at most 127 * 2 u of a step
    close(values(ck), v, per * (0.5 + 256 * U) + err)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_checkpoint_of_the_forward_pass_and_backward_out_of_it(ops, shape, dt):
    n, h, w, c, groups = shape
    for act in ("relu", "silu"):
        x, dy, gamma, beta = make(n, h, w, c, dt, seed=3 * c + w)
        y, saved = ops.group_norm_act(x, gamma, beta, groups, act=act, checkpoint=True)
        check_forward(x, y, saved, gamma, beta, groups, 1e-3, act)
        assert saved.x is None
        mean, rstd, scale, _ = stats64(x, gamma, beta, groups, 1e-3)
        xhat = (x.double() - spread(mean, c)) * spread(rstd, c)
        xmax = spread(x.double().abs().amax((1, 2)).reshape(n, groups, -1).amax(2), c)
        check_checkpoint(saved.checkpoint, xhat, K * U * (xhat.abs() + 3 * xmax * spread(rstd, c)))
        dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
        v = values(saved.checkpoint)
        z = v * gamma.double() + beta.double()
        wdx, wg, wb, tx, tg, tb = backward64(v, z, (v * gamma.double()).abs() + beta.double().abs(), dy,
                                             saved.scale.double(), groups, act, dt)
        close(dx, wdx, tx)
        close(dgamma, wg, tg)
        close(dbeta, wb, tb)


# one image in a launch of its own, several; both tensors of the backward pass in the memory-side cache, one of them, none
@pytest.mark.parametrize("shape", [(5, 480, 640, 64, 16), (3, 960, 1280, 48, 12), (1, 1920, 1280, 48, 6), (2, 300, 400, 1032, 43)], ids=str)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_large_maps(ops, shape, checkpoint):
    n, h, w, c, groups = shape
    dt, act = torch.bfloat16, "relu"
    x, dy, gamma, beta = make(n, h, w, c, dt, seed=1)
    y, saved = ops.group_norm_act(x, gamma, beta, groups, act=act, checkpoint=checkpoint)
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    sums = torch.zeros(4, c, dtype=torch.float64, device="cuda")
    for i in range(n):                                          # an image at a time: the references are in 64 bits
        one = slice(i, i + 1)
        part = ops.Saved(None, None, saved.mean[one], saved.rstd[one], saved.scale[one], saved.shift[one], gamma, beta, groups, act)
        check_forward(x[one], y[one], part, gamma, beta, groups, 1e-3, act)
        if checkpoint:
            xhat = values(ops.Checkpoint8(saved.checkpoint.codes[one], saved.checkpoint.scales[one]))
            z = xhat * gamma.double() + beta.double()
        else:
            xhat = (x[one].double() - spread(part.mean.double(), c)) * spread(part.rstd.double(), c)
            z = x[one].double() * part.scale.double()[:, None, None] + part.shift.double()[:, None, None]
        wdx, wg, wb, tx, tg, tb = backward64(xhat, z, None, dy[one], part.scale.double(), groups, act, dt)
        close(dx[one], wdx, tx)
        sums += torch.stack([wg, wb, tg, tb])
    close(dgamma, sums[0], sums[2])
    close(dbeta, sums[1], sums[3])


# groups of so many channels that the chip rather than a block adds up their partial sums; slabs that cut a group at one end, at
# both ends, in the middle
@pytest.mark.parametrize("shape,dt", [((3, 190, 200, 464, 1), torch.float32), ((2, 200, 210, 448, 2), torch.float32),
                                      ((1, 75, 80, 1536, 1), torch.bfloat16), ((2, 75, 80, 1560, 3), torch.float16),
                                      ((2, 64, 70, 1536, 6), torch.bfloat16), ((1, 90, 90, 2056, 1), torch.float32),
                                      ((1, 90, 90, 4104, 27), torch.bfloat16)], ids=str)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_groups_of_many_channels(ops, shape, dt, checkpoint):
    n, h, w, c, groups = shape
    act = "silu"
    x, dy, gamma, beta = make(n, h, w, c, dt, seed=c + groups)
    y, saved = ops.group_norm_act(x, gamma, beta, groups, act=act, checkpoint=checkpoint)
    check_forward(x, y, saved, gamma, beta, groups, 1e-3, act)
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    if checkpoint:
        xhat = values(saved.checkpoint)
        z, zmag = xhat * gamma.double() + beta.double(), (xhat * gamma.double()).abs() + beta.double().abs()
    else:
        scale, shift = saved.scale.double()[:, None, None], saved.shift.double()[:, None, None]
        xhat = (x.double() - spread(saved.mean.double(), c)) * spread(saved.rstd.double(), c)
        z, zmag = x.double() * scale + shift, (x.double() * scale).abs() + shift.abs()
    wdx, wg, wb, tx, tg, tb = backward64(xhat, z, zmag, dy, saved.scale.double(), groups, act, dt)
    close(dx, wdx, tx)
    close(dgamma, wg, tg)
    close(dbeta, wb, tb)


def test_parameters_may_be_missing(ops):
    x, dy, gamma, beta = make(2, 9, 11, 48, torch.bfloat16)
    ones, zeros = torch.ones_like(gamma), torch.zeros_like(beta)
    for ck in (False, True):
        for g, b in ((None, beta), (gamma, None), (None, None)):
            y, s = ops.group_norm_act(x, g, b, 6, act="silu", checkpoint=ck)
            yw, sw = ops.group_norm_act(x, ones if g is None else g, zeros if b is None else b, 6, act="silu", checkpoint=ck)
            assert torch.equal(y, yw)
            for got, want in zip(ops.group_norm_act_backward(dy, s), ops.group_norm_act_backward(dy, sw)):
                assert torch.equal(got, want)


@pytest.mark.parametrize("offset,dt", [(1e3, torch.float32), (1e4, torch.float32), (30.0, torch.bfloat16)], ids=str)
def test_an_offset_that_is_large_against_the_spread(ops, offset, dt):
    """No cancellation in the variance: rstd keeps K u of its value next to the unavoidable error of the mean.  The first
    pixel lies far from all others, so a sum around it would lose the digits of an uncentred one."""
    n, h, w, c, groups = 2, 40, 50, 64, 8
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((n, h, w, c), generator=gen, device="cuda") + offset
    x[:, 0, 0] = 0
    x = x.to(dt)
    y, saved = ops.group_norm_act(x, None, None, groups, eps=0.0)
    mean, rstd, _, _ = stats64(x, None, None, groups, 0.0)
    close(saved.mean, mean, K * U * mean.abs())
    # the means of threads and blocks are held in 32 bits, u |mean| off each; their squares enter the variance, as does
    # twice their product with the differences between threads, at most the group's spread
    std = 1 / rstd
    close(saved.rstd, rstd, rstd * (K * U + 4 * (U * mean.abs() / std) ** 2 + 8 * U * mean.abs() / std))


def test_channel_slices_and_in_place(ops):
    """Reading and writing channel slices of wider tensors leaves the other channels alone; y over x and dx over dy."""
    for dt in TYPES:
        wide = torch.randn((2, 15, 17, 160), device="cuda").to(dt)
        x, gamma, beta = wide[..., 32:104], torch.randn(72, device="cuda"), torch.randn(72, device="cuda")
        want, sw = ops.group_norm_act(x.contiguous(), gamma, beta, 9, act="relu", checkpoint=True)
        before = wide.clone()
        dst = torch.full((2, 15, 17, 96), 7.0, device="cuda").to(dt)
        y, s = ops.group_norm_act(x, gamma, beta, 9, act="relu", out=dst[..., 16:88], checkpoint=True)
        assert torch.equal(y, want) and torch.equal(wide, before)
        assert (dst[..., :16] == 7).all() and (dst[..., 88:] == 7).all()
        assert torch.equal(s.checkpoint.codes, sw.checkpoint.codes) and torch.equal(s.checkpoint.scales, sw.checkpoint.scales)
        y, _ = ops.group_norm_act(x, gamma, beta, 9, act="relu", checkpoint=True, out=x)
        assert torch.equal(y, want) and torch.equal(wide[..., :32], before[..., :32]) and torch.equal(wide[..., 104:], before[..., 104:])
        # backward: slices, then over dy
        dyw = torch.randn((2, 15, 17, 80), device="cuda").to(dt)
        dy = dyw[..., 8:80]
        dx, dg, db = ops.group_norm_act_backward(dy.contiguous(), sw)
        keep = dyw.clone()
        dx2, dg2, db2 = ops.group_norm_act_backward(dy, sw, out=dy)
        assert torch.equal(dx, dx2) and torch.equal(dg, dg2) and torch.equal(db, db2) and torch.equal(dyw[..., :8], keep[..., :8])
        # into another channel range of the same buffer
        half = torch.randn((2, 15, 17, 64), device="cuda").to(dt)
        a, _ = ops.group_norm_act(half[..., :32], None, None, 4)
        b, _ = ops.group_norm_act(half[..., :32], None, None, 4, out=half[..., 32:])
        assert torch.equal(a, b)


def test_batch_normalisation_is_the_case_of_one_image_and_groups_of_one(ops):
    """(1, N * H, W, C) with C groups: the sums of miseg_bn_relu_bwd_reduce, and torch's batch statistics in 64 bits."""
    x, dy, gamma, beta = make(3, 20, 24, 64, torch.bfloat16, seed=9)
    flat, dflat = x.reshape(1, 60, 24, 64), dy.reshape(1, 60, 24, 64)
    y, saved = ops.group_norm_act(flat, gamma, beta, 64, act="relu")
    v = x.double().reshape(-1, 64)
    mean, var = v.mean(0), v.var(0, unbiased=False)
    z = (v - mean) / (var + 1e-3).sqrt() * gamma.double() + beta.double()
    close(y.reshape(-1, 64), z.clamp_min(0), half_step(x.dtype) * z.abs() + 2 * K * U * (8 + v.abs().amax(0)) * saved.scale[0].double().abs() + 8 * K * U)
    dx, dgamma, dbeta = ops.group_norm_act_backward(dflat, saved)
    from miseg_amd import lib as L
    lib = L.load()
    sums = torch.empty(128, dtype=torch.float64, device="cuda")
    mean32, var32 = saved.mean[0].contiguous(), (1 / saved.rstd[0].double().square() - 1e-3).float()
    st = torch.cuda.current_stream().cuda_stream
    L.check(lib.miseg_bn_relu_bwd_reduce(x.data_ptr(), dy.data_ptr(), 3 * 480, 64, 64, 64, saved.scale.data_ptr(),
                                         saved.shift.data_ptr(), mean32.data_ptr(), var32.data_ptr(), 1e-3, 1,
                                         sums.data_ptr(), st))
    g = dy.double().reshape(-1, 64) * (z > 0)
    close(dbeta, sums[:64], 4 * K * U * g.abs().sum(0) + 1e-30)
    close(dgamma, sums[64:], 4 * K * U * (g * (v - mean) * saved.rstd[0].double()).abs().sum(0) + 1e-30)
    out = torch.empty_like(x)
    L.check(lib.miseg_bn_relu_bwd_apply(x.data_ptr(), dy.data_ptr(), out.data_ptr(), 3 * 480, 64, 64, 64, 64,
                                        saved.scale.data_ptr(), saved.shift.data_ptr(), mean32.data_ptr(),
                                        var32.data_ptr(), 1e-3, 1, sums.data_ptr(), None, 0, st))
    big = (saved.scale[0].double().abs() * (g.abs().amax(0)))
    close(dx.reshape(-1, 64), out.double().reshape(-1, 64),
          2 * half_step(x.dtype) * out.double().reshape(-1, 64).abs() + 16 * K * U * big + 1e-30)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8), (3, 7, 9, 40), (2, 13, 11, 72), (1, 5, 6, 1032), (4, 30, 41, 64), (1, 3, 5, 32)], ids=str)
def test_checkpoint_write_is_bitwise_its_definition(ops, shape, dt):
    """Without coefficients every step is one rounded 32-bit operation, so codes and scales have one value."""
    n, h, w, c = shape
    x = make(n, h, w, c, dt, seed=c)[0]
    ck = ops.checkpoint8_write(x)
    amax = blocks_amax(x.float())
    scales = (amax / 127.0).to(torch.bfloat16)
    assert torch.equal(ck.scales, scales)
    inv = (1.0 / scales.float()).repeat_interleave(32, 3)[..., :c]
    assert torch.equal(ck.codes, torch.round(x.float() * inv).to(torch.int8))
    back = ops.checkpoint8_read(ck, dtype=dt)
    want = values(ck)
    close(back, want, half_step(dt) * want.abs() + tiny(dt))


@pytest.mark.parametrize("per_image", [False, True])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_checkpoint_with_coefficients_and_the_activated_result(ops, dt, per_image):
    n, h, w, c = 3, 17, 13, 104
    x = make(n, h, w, c, dt, seed=2)[0]
    shape = (n, c) if per_image else (c,)
    a, b, ya, yb = (torch.randn(shape, device="cuda") for _ in range(4))

    def full(t):
        return t.double().reshape(-1, 1, 1, c)
    for act in ("none", "relu", "silu"):
        ck, y = ops.checkpoint8_write(x, a, b, ya, yb, act=act)
        v = x.double() * full(a) + full(b)
        check_checkpoint(ck, v, 2 * U * v.abs())
        z = x.double() * full(ya) + full(yb)
        want = act64(z, act)[0]
        close(y, want, half_step(dt) * want.abs() + 16 * U * (1 + z.abs()) * want.abs() + 4 * U * z.abs() + tiny(dt))
        back = ops.checkpoint8_read(ck, ya, yb, act=act, dtype=dt)
        z = values(ck) * full(ya) + full(yb)
        want = act64(z, act)[0]
        close(back, want, half_step(dt) * want.abs() + 16 * U * (1 + z.abs()) * want.abs() + 4 * U * z.abs() + tiny(dt))
    only, y2 = ops.checkpoint8_write(x, None, None, ya, yb, act="relu", out=(buf := x.clone()))
    assert torch.equal(ops.checkpoint8_write(x).codes, only.codes) and y2 is buf
    inplace = x.clone()
    ck3, y3 = ops.checkpoint8_write(inplace, None, None, ya, yb, act="relu", out=inplace)
    assert torch.equal(y3, y2) and torch.equal(ck3.codes, only.codes)


def test_values_that_are_not_finite_and_values_that_vanish(ops):
    x = torch.randn((1, 4, 4, 64), device="cuda")
    x[0, 0, 0, 3], x[0, 1, 1, 40], x[0, 2, 2, 5] = float("nan"), float("inf"), float("-inf")
    x[0, 3, 3, :32] = 0
    x[0, 3, 2, 32:] = 1e-37                                    # under the smallest block that is kept (2^-119 = 1.5e-36)
    x[0, 3, 1, :32] = 2e-36
    x[0, 3, 0, 32:] = 3.0e38
    ck = ops.checkpoint8_write(x)
    back = ops.checkpoint8_read(ck, dtype=torch.float32)
    bad = torch.zeros((1, 4, 4, 2), dtype=torch.bool, device="cuda")
    bad[0, 0, 0, 0] = bad[0, 1, 1, 1] = bad[0, 2, 2, 0] = True
    assert torch.equal(torch.isnan(back), bad.repeat_interleave(32, 3))
    assert (ck.codes[bad.repeat_interleave(32, 3)] == 0).all()
    assert (back[0, 3, 3, :32] == 0).all() and (back[0, 3, 2, 32:] == 0).all()
    assert ((back[0, 3, 1, :32] / 2e-36 - 1).abs() <= 2.0 ** -8).all()
    assert ((back[0, 3, 0, 32:] / 3.0e38 - 1).abs() <= 2.0 ** -8).all()
    good = ~bad.repeat_interleave(32, 3)
    assert torch.isfinite(back[good]).all()
    # and a ReLU keeps a NaN, in both directions of the checkpoint
    one = torch.ones(64, device="cuda")
    _, y = ops.checkpoint8_write(x, None, None, one, 0 * one, act="relu")
    assert torch.isnan(y[0, 0, 0, 3]) and torch.isinf(y[0, 1, 1, 40]) and y[0, 2, 2, 5] == 0
    assert torch.isnan(ops.checkpoint8_read(ck, one, 0 * one, act="relu")).sum() == 96


def test_a_nan_stays_in_its_group(ops):
    x, dy, gamma, beta = make(2, 8, 9, 64, torch.bfloat16)
    x[1, 3, 4, 17] = float("nan")                               # image 1, group 2 of 8
    for ck in (False, True):
        y, saved = ops.group_norm_act(x, gamma, beta, 8, act="none", checkpoint=ck)
        nan = torch.isnan(y)
        want = torch.zeros_like(nan)
        want[1, ..., 16:24] = True
        assert torch.equal(nan, want)
        dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
        if not ck:
            assert torch.equal(torch.isnan(dx), want) and torch.isnan(dgamma[16:24]).all() and not torch.isnan(dgamma[24:]).any()
        else:                                                   # its block of 32 channels is lost, and with it their groups
            assert torch.isnan(dx[1, ..., :32]).all() and not torch.isnan(dx[0]).any() and not torch.isnan(dx[1, ..., 32:]).any()


def test_a_constant_image(ops):
    x = torch.full((2, 6, 7, 32), 3.0, device="cuda").to(torch.bfloat16)
    gamma, beta = torch.randn(32, device="cuda"), torch.randn(32, device="cuda")
    for ck in (False, True):
        y, saved = ops.group_norm_act(x, gamma, beta, 4, checkpoint=ck)
        close(y, beta.double().expand_as(y), half_step(x.dtype) * beta.double().abs() + K * U * 3 * saved.scale.double().abs()[:, None, None])
        dx, dgamma, _ = ops.group_norm_act_backward(torch.ones_like(x), saved)
        # dy is constant too: dx = a (1 - mean a / a) per channel, up to rounding, and xhat = 0
        a = saved.scale.double()
        want = a - a.reshape(2, 4, 8).mean(2).repeat_interleave(8, 1)
        close(dx, want[:, None, None].expand_as(dx), half_step(x.dtype) * want.abs()[:, None, None] + K * U * a.abs().amax())
        assert (dgamma.abs() <= K * U * 84 * 3 * saved.rstd.max()).all()


def test_gradient_against_differences(ops):
    """sum(y t) along a direction, central differences of the forward kernel in 32 bits: error h^2 / 6 of the third derivative
    along the direction plus the sum's rounding over h."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    n, h, w, c, groups = 2, 5, 6, 24, 4
    x = torch.randn((n, h, w, c), generator=gen, device="cuda")
    t = torch.randn((n, h, w, c), generator=gen, device="cuda")
    v = torch.randn((n, h, w, c), generator=gen, device="cuda")
    gamma, beta = torch.rand(c, generator=gen, device="cuda") + 0.5, torch.randn(c, generator=gen, device="cuda")
    vg, vb = torch.randn(c, generator=gen, device="cuda"), torch.randn(c, generator=gen, device="cuda")
    for act in ("none", "silu"):
        _, saved = ops.group_norm_act(x, gamma, beta, groups, act=act)
        dx, dgamma, dbeta = ops.group_norm_act_backward(t, saved)
        got = (dx.double() * v).sum() + (dgamma.double() * vg).sum() + (dbeta.double() * vb).sum()
        step, side = 1e-2, []
        for s in (-1, 1):
            y, _ = ops.group_norm_act(x + s * step * v, gamma + s * step * vg, beta + s * step * vb, groups, act=act)
            side.append((y.double() * t).sum())
        diff = (side[1] - side[0]) / (2 * step)
        # third derivatives along v of a normalised value are a few |v|^3 / std^3 per value, and 1440 values enter with
        # random signs: 50 sqrt(1440) h^2 / 6; rounding 8 u |y t| / h, random signs
        tol = 50 * 1440 ** 0.5 * step ** 2 / 6 + 8 * U * 1440 ** 0.5 * 10 / step
        assert abs(got - diff) <= tol, (act, got.item(), diff.item(), tol)


def test_equal_calls_give_equal_bits_and_calls_on_two_streams_do_not_meet(ops):
    x, dy, gamma, beta = make(4, 97, 131, 64, torch.bfloat16, seed=8)
    first = ops.group_norm_act(x, gamma, beta, 16, act="silu", checkpoint=True)
    fb = ops.group_norm_act_backward(dy, first[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            y, s = ops.group_norm_act(x, gamma, beta, 16, act="silu", checkpoint=True)
            results.append((y, s, ops.group_norm_act_backward(dy, s)))
    torch.cuda.synchronize()
    for y, s, b in results:
        assert torch.equal(y, first[0]) and torch.equal(s.checkpoint.codes, first[1].checkpoint.codes)
        assert torch.equal(s.rstd, first[1].rstd)
        assert all(torch.equal(p, q) for p, q in zip(b, fb))


def test_captured_and_replayed(ops):
    """Two graphs of the same calls, each replayed between eager work on the same leaves."""
    for shape in ((4, 97, 131, 64), (1, 6, 7, 64)):
        x, dy, gamma, beta = make(*shape, torch.bfloat16, seed=1)

        def step():
            y, s = ops.group_norm_act(x, gamma, beta, 16, act="relu", checkpoint=True)
            op = ops.checkpoint8_read(s.checkpoint, gamma, beta, act="relu")
            y2, s2 = ops.group_norm_act(x, gamma, beta, 16, act="relu")
            return (y, op, y2) + tuple(ops.group_norm_act_backward(dy, s)) + tuple(ops.group_norm_act_backward(dy, s2))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = step()
            graphs.append((g, out))
        for seed in (11, 12, 13):
            nx, ndy, _, _ = make(*shape, torch.bfloat16, seed=seed)
            x.copy_(nx)
            dy.copy_(ndy)
            want = step()
            for g, out in graphs:
                for t in out:
                    t.fill_(float("nan"))
                g.replay()
                torch.cuda.synchronize()
                step()
                assert all(torch.equal(p, q) for p, q in zip(out, want))


# the forms of three launches: steps of several images, groups that the chip adds up, slabs that cut groups
@pytest.mark.parametrize("shape,dt", [((5, 480, 640, 64, 16), torch.bfloat16), ((3, 190, 200, 464, 1), torch.float32),
                                      ((2, 75, 80, 1560, 3), torch.float16)], ids=str)
def test_large_forms_on_two_streams_and_replayed(ops, shape, dt):
    n, h, w, c, groups = shape
    x, dy, gamma, beta = make(n, h, w, c, dt, seed=5)

    def step():
        y, s = ops.group_norm_act(x, gamma, beta, groups, act="silu", checkpoint=True)
        y2, s2 = ops.group_norm_act(x, gamma, beta, groups, act="relu")
        return (y, y2) + tuple(ops.group_norm_act_backward(dy, s)) + tuple(ops.group_norm_act_backward(dy, s2))
    want = step()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            results.append(step())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(p, q) for p, q in zip(r, want))
    del results
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (6, 7):
        nx, ndy, _, _ = make(n, h, w, c, dt, seed=seed)
        x.copy_(nx)
        dy.copy_(ndy)
        want = step()
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        step()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_offsets_past_32_bits(ops):
    """Channel slices of a 9 GB tensor: the second image starts 2^32 bytes in, rows of it lie past 2^31 elements."""
    c, wide = 32, 2048
    buf = torch.empty((2, 1100, 1000, wide), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((2, 1100, 1000, c), generator=gen, device="cuda").to(torch.bfloat16)
    dy = torch.randn((2, 1100, 1000, c), generator=gen, device="cuda").to(torch.bfloat16)
    buf[..., 64:96] = x
    buf[..., 128:160] = dy
    gamma, beta = torch.randn(c, device="cuda"), torch.randn(c, device="cuda")
    want, ws = ops.group_norm_act(x, gamma, beta, 8, act="relu", checkpoint=True)
    y, s = ops.group_norm_act(buf[..., 64:96], gamma, beta, 8, act="relu", checkpoint=True, out=buf[..., 256:288])
    assert torch.equal(y, want) and torch.equal(s.checkpoint.codes, ws.checkpoint.codes)
    _, keep = ops.group_norm_act(x, gamma, beta, 8, act="relu")
    wb = ops.group_norm_act_backward(dy, keep)
    _, keep = ops.group_norm_act(buf[..., 64:96], gamma, beta, 8, act="relu")
    got = ops.group_norm_act_backward(buf[..., 128:160], keep, out=buf[..., 320:352])
    assert all(torch.equal(p, q) for p, q in zip(got, wb))
    wb = ops.group_norm_act_backward(dy, ws)
    got = ops.group_norm_act_backward(buf[..., 128:160], s, out=buf[..., 384:416])
    assert all(torch.equal(p, q) for p, q in zip(got, wb))
    back = ops.checkpoint8_read(s.checkpoint, gamma, beta, act="relu", out=buf[..., 448:480])
    assert torch.equal(back, ops.checkpoint8_read(ws.checkpoint, gamma, beta, act="relu"))


def test_many_images(ops):
    x, dy, gamma, beta = make(3000, 1, 3, 16, torch.float32, seed=6)
    y, saved = ops.group_norm_act(x, gamma, beta, 2, act="relu")
    check_forward(x, y, saved, gamma, beta, 2, 1e-3, "relu")
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    xhat = (x.double() - spread(saved.mean.double(), 16)) * spread(saved.rstd.double(), 16)
    z = x.double() * saved.scale.double()[:, None, None] + saved.shift.double()[:, None, None]
    wdx, wg, wb, tx, tg, tb = backward64(xhat, z, z.abs(), dy, saved.scale.double(), 2, "relu", torch.float32)
    close(dx, wdx, tx)
    close(dgamma, wg, tg)
    close(dbeta, wb, tb)


def test_a_layer_chain_of_convolution_and_normalisation(ops):
    """Forward: 1x1 convolution, group norm + ReLU with its checkpoint, 1x1 convolution.  Backward: the second
    convolution's data and weight gradients, the latter's operand out of the checkpoint, and the normalisation's backward
    pass out of it.  Each result against 64-bit arithmetic on the tensors that its kernel was given."""
    from miseg_amd import lib as L
    lib = L.load()
    n, h, w, ci, cm, co, groups = 2, 24, 32, 64, 64, 64, 8
    gen = torch.Generator(device="cuda").manual_seed(7)

    def r(*s):
        return torch.randn(s, generator=gen, device="cuda")
    bf = torch.bfloat16
    x, w1, w2 = r(n, h, w, ci).to(bf), (r(cm, ci) * 0.1).to(bf), (r(co, cm) * 0.1).to(bf)
    gamma, beta, dout = r(cm) * 0.3 + 1, r(cm) * 0.2, (r(n, h, w, co) * 0.05).to(bf)
    st = torch.cuda.current_stream().cuda_stream

    def conv(inp, wt):
        out = torch.empty((n, h, w, wt.shape[0]), dtype=bf, device="cuda")
        d = L.ConvDesc()
        d.inp, d.weight, d.out = inp.data_ptr(), wt.data_ptr(), out.data_ptr()
        d.N, d.H, d.W, d.Cin, d.Ho, d.Wo, d.Cout = n, h, w, inp.shape[3], h, w, wt.shape[0]
        d.KH = d.KW = d.stride_y = d.stride_x = 1
        d.in_pix_stride, d.in_row_stride, d.in_img_stride = inp.shape[3], inp.shape[3] * w, inp.shape[3] * w * h
        d.out_pix_stride, d.out_row_stride, d.out_img_stride = wt.shape[0], wt.shape[0] * w, wt.shape[0] * w * h
        d.temperature = 1.0
        L.check(lib.miseg_conv2d_fwd(C.byref(d), st))
        return out

    def rel(got, want):
        return ((got.double() - want).norm() / want.norm()).item()
    pre = conv(x, w1)
    y, saved = ops.group_norm_act(pre, gamma, beta, groups, act="relu", checkpoint=True)
    check_forward(pre, y, saved, gamma, beta, groups, 1e-3, "relu")
    out = conv(y, w2)
    want = (y.double().reshape(-1, cm) @ w2.double().t()).reshape(out.shape)
    assert rel(out, want) <= half_step(bf)
    # backward
    dy = conv(dout, w2.t().contiguous())
    operand = ops.checkpoint8_read(saved.checkpoint, gamma, beta, act="relu")
    dw = torch.zeros((co, cm), dtype=torch.float32, device="cuda")
    d = L.WgradDesc()
    d.x, d.dy, d.dw = operand.data_ptr(), dout.data_ptr(), dw.data_ptr()
    d.N, d.H, d.W, d.Cin, d.Ho, d.Wo, d.Cout, d.KH, d.KW, d.stride_y, d.stride_x = n, h, w, cm, h, w, co, 1, 1, 1, 1
    d.x_pix, d.x_row, d.x_img, d.dy_pix, d.dy_row, d.dy_img = cm, cm * w, cm * w * h, co, co * w, co * w * h
    L.check(lib.miseg_conv2d_wgrad(C.byref(d), st))
    wantw = dout.double().reshape(-1, co).t() @ operand.double().reshape(-1, cm)
    assert rel(dw, wantw) <= 1536 * U
    exactw = dout.double().reshape(-1, co).t() @ y.double().reshape(-1, cm)
    # 8 bits: a uniform error of a block's step (its largest value, under 4.5 deviations of 32 normal values, over 127) has
    # a deviation of step / sqrt(12) = 0.0102 of the values' own; dout is independent of it, so the products' errors add up
    # like the products themselves (random signs): 0.0102 of a gradient of a standard normal operand; after beta and the
    # ReLU at least half of the operand's square sum is left, and twice that covers the spread of a sample
    assert rel(dw, exactw) <= 2 * 0.0102 * 2 ** 0.5
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    v = values(saved.checkpoint)
    z = v * gamma.double() + beta.double()
    wdx, wg, wb, tx, tg, tb = backward64(v, z, z.abs(), dy, saved.scale.double(), groups, "relu", bf)
    close(dx, wdx, tx)
    close(dgamma, wg, tg)
    close(dbeta, wb, tb)


@pytest.mark.parametrize("shape", [(2, 9, 11, 72, 9), (2, 90, 80, 72, 9), (2, 500, 400, 72, 9), (1, 30, 31, 520, 5)], ids=str)
def test_parameters_from_a_flat_buffer(ops, shape):
    """Slices of one float32 buffer at odd offsets, as an optimiser's flat parameters are, give what aligned copies give."""
    n, h, w, c, groups = shape
    x, dy, gamma, beta = make(n, h, w, c, torch.bfloat16, seed=4)
    flat = torch.cat([torch.zeros(1, device="cuda"), gamma, torch.zeros(2, device="cuda"), beta])
    g, b = flat[1:1 + c], flat[3 + c:3 + 2 * c]
    assert g.data_ptr() % 16 and b.data_ptr() % 16
    for ck in (False, True):
        y, s = ops.group_norm_act(x, g, b, groups, act="relu", checkpoint=ck)
        yw, sw = ops.group_norm_act(x, gamma, beta, groups, act="relu", checkpoint=ck)
        assert torch.equal(y, yw) and torch.equal(s.shift, sw.shift)
        for got, want in zip(ops.group_norm_act_backward(dy, s), ops.group_norm_act_backward(dy, sw)):
            assert torch.equal(got, want)


def test_views_that_are_refused(ops):
    """Slices that start or step off 16 bytes, strides of other layouts, broadcasts, overlaps, types and sizes that differ."""
    from miseg_amd import lib as L
    wide = torch.zeros((2, 6, 7, 160), dtype=torch.bfloat16, device="cuda")
    x = wide[..., :64]
    odd = torch.zeros((2, 6, 7, 68), dtype=torch.bfloat16, device="cuda")[..., :64]
    bad = [wide[..., 4:68], odd, wide.permute(0, 3, 1, 2)[:, :6, :7, :7], wide[:, ::2, :, :64], wide[..., :60],
           wide[:1, ..., :64].expand(2, 6, 7, 64), wide[..., :128:2], wide[:0, ..., :64], x.to(torch.float64)]
    for t in bad:
        with pytest.raises(L.MisegError):
            ops.group_norm_act(t, None, None, 1)
        with pytest.raises(L.MisegError):
            ops.checkpoint8_write(t)
    y, s = ops.group_norm_act(x, None, None, 8)
    for t in bad[:6] + [x.float(), x[:1], wide[..., :56]]:
        with pytest.raises(L.MisegError):
            ops.group_norm_act_backward(t, s)
        with pytest.raises(L.MisegError):
            ops.group_norm_act(x, None, None, 8, out=t)
    for out in (x, wide[..., 32:96], wide[:, :, :, 8:72]):
        with pytest.raises(L.MisegError):
            ops.group_norm_act(x, None, None, 8, out=out)
    gamma = torch.zeros(64, device="cuda")
    for g in (gamma[:32], gamma.double(), gamma.cpu(), torch.zeros(128, device="cuda")[::2]):
        with pytest.raises(L.MisegError):
            ops.group_norm_act(x, g, None, 8)
    for groups in (0, 7, 128, 8.0, None):
        with pytest.raises(L.MisegError):
            ops.group_norm_act(x, None, None, groups)
    with pytest.raises(L.MisegError):
        ops.group_norm_act(x, None, None, 8, act="gelu")
    with pytest.raises(L.MisegError):
        ops.checkpoint8_write(x, gamma)
    with pytest.raises(L.MisegError):
        ops.checkpoint8_write(x, act="relu")
    ck = ops.checkpoint8_write(x)
    with pytest.raises(L.MisegError):
        ops.checkpoint8_read(ck, out=wide[..., 4:68])
    with pytest.raises(L.MisegError):
        ops.checkpoint8_read(ck, dtype=torch.int8)
    torch.cuda.synchronize()


@pytest.mark.parametrize("shape", [(2, 1, 3, 65536, 4096), (1, 3, 700, 65536, 1), (65535, 1, 1, 8, 2), (65535, 1, 2, 32, 32),
                                   (1, 2100, 1, 520, 4), (1, 1, 2100, 1024, 8), (3, 47, 50, 8, 1)], ids=str)
def test_extreme_extents(ops, shape):
    n, h, w, c, groups = shape
    dt, act = torch.bfloat16, "relu"
    x, dy, gamma, beta = make(n, h, w, c, dt, seed=c)
    for checkpoint in (False, True):
        y, saved = ops.group_norm_act(x, gamma, beta, groups, act=act, checkpoint=checkpoint)
        check_forward(x, y, saved, gamma, beta, groups, 1e-3, act)
        dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
        if checkpoint:
            xhat = values(saved.checkpoint)
            z = xhat * gamma.double() + beta.double()
        else:
            xhat = (x.double() - spread(saved.mean.double(), c)) * spread(saved.rstd.double(), c)
            z = x.double() * saved.scale.double()[:, None, None] + saved.shift.double()[:, None, None]
        wdx, wg, wb, tx, tg, tb = backward64(xhat, z, None, dy, saved.scale.double(), groups, act, dt)
        close(dx, wdx, tx)
        close(dgamma, wg, tg)
        close(dbeta, wb, tb)


def test_most_pixels(ops):
    """23170 x 23170 pixels, just under the 2^29 that are allowed: statistics against sums in 64 bits, results against the
    coefficients, a strip at a time."""
    side, c = 23170, 8
    x = torch.empty((1, side, side, c), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    strips = [slice(i, min(i + 2000, side)) for i in range(0, side, 2000)]
    for s in strips:
        x[:, s] = torch.randn((1, s.stop - s.start, side, c), generator=gen, device="cuda") + 0.5
    gamma, beta = torch.randn(c, generator=gen, device="cuda"), torch.randn(c, generator=gen, device="cuda")
    count = side * side * 4
    mean = sum(x[:, s].double().reshape(-1, 2, 4).sum((0, 2)) for s in strips) / count
    var = sum((x[:, s].double().reshape(-1, 2, 4) - mean[None, :, None]).square().sum((0, 2)) for s in strips) / count
    y, saved = ops.group_norm_act(x, gamma, beta, 2, act="relu", checkpoint=True)
    # 512 blocks of 256 rows of pixels: 4096 terms a thread instead of 64, their roundings of random sign: 64^0.5 = 8 times K
    close(saved.mean[0], mean, 8 * K * U * torch.ones_like(mean))
    close(saved.rstd[0], 1 / (var + 1e-3).sqrt(), 8 * K * U * torch.ones_like(mean))
    a, b = saved.scale[0].double(), saved.shift[0].double()
    for s in strips:
        z = x[:, s].double() * a + b
        close(y[:, s], z.clamp_min(0), half_step(y.dtype) * z.abs() + 4 * U * (z.abs() + b.abs()) + 1e-30)
    dx, dgamma, dbeta = ops.group_norm_act_backward(torch.ones_like(y), saved)
    s1 = torch.zeros(c, dtype=torch.float64, device="cuda")
    s2 = torch.zeros(c, dtype=torch.float64, device="cuda")
    for s in strips:
        v = saved.checkpoint.codes[:, s].double() * saved.checkpoint.scales[:, s].double()
        m = (v * gamma.double() + beta.double() > 0).double()
        s1 += m.sum((0, 1, 2))
        s2 += (m * v).sum((0, 1, 2))
    # a thread's 4096 terms are counted exactly (dbeta), or at most 6 each in a running sum below 4096 * 6 (dgamma): each addition
    # off by u times that; 131072 threads, random signs, 8 deviations
    assert ((dbeta.double() - s1).abs() <= U * s1 + 1).all()
    assert ((dgamma.double() - s2).abs() <= 8 * U * 4096 * 6 * (4096 * 131072.0) ** 0.5 + U * s2.abs()).all()
    k1 = (a * s1).reshape(2, 4).sum(1).repeat_interleave(4) / count
    k2 = (a * s2).reshape(2, 4).sum(1).repeat_interleave(4) / count
    for s in strips[::4]:
        v = saved.checkpoint.codes[:, s].double() * saved.checkpoint.scales[:, s].double()
        m = (v * gamma.double() + beta.double() > 0).double()
        want = a * m - k1 - v * k2
        # k1 and k2 are known to the bound of the sums over the count
        close(dx[:, s], want, half_step(dx.dtype) * want.abs() + 8 * U * a.abs().max() * (8 + v.abs()))


@pytest.mark.parametrize("shape,view", [((1, 1, 2, 2 ** 32 + 8), lambda t: t[..., :8]), ((1, 1, 1, 2 ** 32 + 8), lambda t: t),
                                        ((2 ** 16, 1, 1, 8), lambda t: t), ((1, 1, 1, 65544), lambda t: t)],
                         ids=["pixel stride", "channels cut", "images", "channels"])
def test_extents_past_those_of_a_descriptor_are_refused(ops, shape, view):
    from miseg_amd import lib as L
    x = view(torch.empty(shape, dtype=torch.bfloat16, device="cuda"))
    n, h, w, c = x.shape
    flat = torch.zeros(1, device="cuda")
    with pytest.raises(L.MisegError):
        ops.group_norm_act(x, None, None, 1, checkpoint=True, out=x)
    with pytest.raises(L.MisegError):
        ops.checkpoint8_write(x)
    with pytest.raises(L.MisegError):
        ops.group_norm_act_backward(x, ops.Saved(x, None, flat, flat, flat, flat, None, None, 1, "none"))
