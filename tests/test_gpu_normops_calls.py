"""Calls of the normalisation and checkpoint operators that their documentation allows, next to those of everyday use:
slices of maps of one pixel, parameters that change before the backward pass, coefficients inside a flat buffer, arguments
of other kinds, more blocks than one launch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    import miseg_amd  # noqa: F401
    from miseg_amd import lib as L
    from miseg_amd import normops
    L.check(L.load().miseg_device_check())
    return normops


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 4])
def test_slices_of_maps_of_one_pixel(ops, dt, n):
    """The pixel stride of a 1 x 1 map has no meaning: another channel range of the same buffer, reads and writes apart."""
    buf = normal(1, n, 1, 1, 64).to(dt)
    x, dst, gamma, beta = buf[..., :32], buf[..., 32:], normal(2, 32), normal(3, 32)
    dy = normal(4, n, 1, 1, 32).to(dt)
    keep = x.clone()
    for ck in (False, True):
        want, sw = ops.group_norm_act(keep, gamma, beta, 4, act="silu", checkpoint=ck)
        y, s = ops.group_norm_act(x, gamma, beta, 4, act="silu", checkpoint=ck, out=dst)
        assert torch.equal(y, want) and torch.equal(dst, want) and torch.equal(x, keep)
        grads = ops.group_norm_act_backward(dy, sw)
        dst.copy_(dy)
        got = ops.group_norm_act_backward(dst, s, out=dst)
        assert all(torch.equal(a, b) for a, b in zip(got, grads)) and torch.equal(x, keep)
        if not ck:                                             # dx into the other half of x's buffer
            got = ops.group_norm_act_backward(dy, s, out=dst)
            assert all(torch.equal(a, b) for a, b in zip(got, grads)) and torch.equal(x, keep)
    cw, yw = ops.checkpoint8_write(keep, None, None, gamma, beta, act="relu")
    c, y = ops.checkpoint8_write(x, None, None, gamma, beta, act="relu", out=dst)
    assert torch.equal(y, yw) and torch.equal(c.codes, cw.codes) and torch.equal(x, keep)


def test_overlaps_of_maps_of_one_pixel_are_refused(ops):
    from miseg_amd import lib as L
    buf = normal(1, 3, 1, 1, 64).to(torch.bfloat16)
    for out in (buf[..., 16:48], buf[..., 8:40]):
        with pytest.raises(L.MisegError):
            ops.group_norm_act(buf[..., :32], None, None, 4, out=out)
    flat = normal(2, 128).to(torch.bfloat16)
    with pytest.raises(L.MisegError):                          # the second image of x is the first of out
        ops.group_norm_act(flat[:64].view(2, 1, 1, 32), None, None, 4, out=flat[32:96].view(2, 1, 1, 32))


# the form of one launch, of two, of three; one image and several
@pytest.mark.parametrize("shape", [(1, 15, 20, 64, 8), (2, 9, 11, 72, 9), (2, 90, 80, 72, 9), (2, 30, 31, 520, 5), (9, 480, 640, 64, 16)], ids=str)
def test_parameters_that_change_before_the_backward_pass(ops, shape):
    """The backward pass is that of the forward call: what an optimiser does to gamma and beta in between is not seen."""
    n, h, w, c, groups = shape
    x, dy = normal(1, n, h, w, c).to(torch.bfloat16), normal(2, n, h, w, c).to(torch.bfloat16)
    for ck in (False, True):
        for which in ("both", "gamma", "beta"):
            gamma = None if which == "beta" else normal(3, c)
            beta = None if which == "gamma" else normal(4, c)
            _, saved = ops.group_norm_act(x, gamma, beta, groups, act="relu", checkpoint=ck)
            want = ops.group_norm_act_backward(dy, saved)
            first = [None if t is None else t.clone() for t in (gamma, beta)]
            for t in (gamma, beta):
                if t is not None:
                    t.neg_().add_(0.25)
            got = ops.group_norm_act_backward(dy, saved)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (ck, which)
            if ck:
                for have, t in zip((saved.gamma, saved.beta), first):
                    assert have is None and t is None or torch.equal(have, t)


def test_tensors_that_ask_for_a_gradient_are_refused(ops):
    """No autograd behind these calls: a result without a gradient in place of one that was asked for would go unseen."""
    from miseg_amd import lib as L
    x, dy, gamma, beta = normal(1, 2, 5, 6, 32), normal(2, 2, 5, 6, 32), normal(3, 32), normal(4, 32)
    y, saved = ops.group_norm_act(x, gamma, beta, 4, act="silu", checkpoint=True)
    ck = saved.checkpoint

    def calls(x, dy, gamma, beta):
        return {"forward": lambda: ops.group_norm_act(x, gamma, beta, 4, act="silu", checkpoint=True)[0],
                "backward": lambda: ops.group_norm_act_backward(dy, saved)[0],
                "write": lambda: ops.checkpoint8_write(x, gamma, beta, gamma, beta)[1],
                "read": lambda: ops.checkpoint8_read(ck, gamma, beta, dtype=torch.float32)}
    takes = {"x": ("forward", "write"), "dy": ("backward",), "gamma": ("forward", "write", "read"), "beta": ("forward", "write", "read")}
    plain = {k: f() for k, f in calls(x, dy, gamma, beta).items()}
    for name, users in takes.items():
        args = dict(x=x, dy=dy, gamma=gamma, beta=beta)
        args[name] = args[name].clone().requires_grad_()
        for user, f in calls(**args).items():
            if user in users:
                with pytest.raises(L.MisegError, match="gradient"):
                    f()
                with torch.no_grad():
                    assert torch.equal(f(), plain[user])
            else:
                assert torch.equal(f(), plain[user])
    with pytest.raises(L.MisegError, match="gradient"):
        ops.group_norm_act(x, gamma, beta, 4, out=torch.empty_like(x, requires_grad=True))


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("per_image", [False, True])
def test_coefficients_inside_a_flat_buffer(ops, dt, per_image):
    """Slices at odd offsets, as group_norm_act takes them, in the calls that go with it."""
    n, h, w, c = 2, 7, 9, 40
    x = normal(1, n, h, w, c).to(dt)
    count = n * c if per_image else c
    flat = normal(2, 4 * count + 8)
    odd = [flat[i * (count + 1) + 1:][:count] for i in range(4)]
    if per_image:
        odd = [t.view(n, c) for t in odd]
    assert any(t.data_ptr() % 16 for t in odd)
    even = [t.clone() for t in odd]
    ck, y = ops.checkpoint8_write(x, *odd, act="silu")
    cw, yw = ops.checkpoint8_write(x, *even, act="silu")
    assert torch.equal(y, yw) and torch.equal(ck.codes, cw.codes) and torch.equal(ck.scales, cw.scales)
    got = ops.checkpoint8_read(ck, odd[0], odd[1], act="relu", dtype=dt)
    assert torch.equal(got, ops.checkpoint8_read(ck, even[0], even[1], act="relu", dtype=dt))
    if not per_image:
        gamma, beta = odd[0], odd[1]
        _, saved = ops.group_norm_act(x, gamma, beta, 5, act="relu", checkpoint=True)
        got = ops.checkpoint8_read(saved.checkpoint, gamma, beta, act="relu", dtype=dt)
        assert torch.equal(got, ops.checkpoint8_read(saved.checkpoint, even[0], even[1], act="relu", dtype=dt))


def test_coefficients_inside_a_flat_buffer_captured(ops):
    x, flat = normal(1, 2, 7, 9, 40).to(torch.bfloat16), normal(2, 83)
    gamma, beta = flat[1:41], flat[42:82]

    def step():
        ck, y = ops.checkpoint8_write(x, gamma, beta, gamma, beta, act="relu")
        return y, ck.codes, ops.checkpoint8_read(ck, gamma, beta, act="relu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (3, 4, 5):
        x.copy_(normal(seed, 2, 7, 9, 40))
        flat.copy_(normal(seed + 10, 83))
        want = step()
        out[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_coefficients_of_one_image_in_either_shape(ops):
    x = normal(1, 1, 7, 9, 40).to(torch.bfloat16)
    a, b, ya, yb = (normal(i, 40) for i in range(2, 6))
    cw, yw = ops.checkpoint8_write(x, a, b, ya, yb, act="relu")
    for first in (False, True):
        one = [t.view(1, 40) if (i < 2) == first else t for i, t in enumerate((a, b, ya, yb))]
        ck, y = ops.checkpoint8_write(x, *one, act="relu")
        assert torch.equal(y, yw) and torch.equal(ck.codes, cw.codes)
    assert torch.equal(ops.checkpoint8_read(cw, a.view(1, 40), b.view(1, 40)), ops.checkpoint8_read(cw, a, b))


def test_arguments_of_other_kinds_are_refused(ops):
    from miseg_amd import lib as L
    x, g = normal(1, 2, 5, 6, 32), normal(2, 32)
    ck = ops.checkpoint8_write(x)
    for out in ("y", 1, [x]):
        for call in (lambda: ops.group_norm_act(x, g, g, 4, out=out), lambda: ops.checkpoint8_write(x, None, None, g, g, out=out),
                     lambda: ops.checkpoint8_read(ck, out=out)):
            with pytest.raises(L.MisegError):
                call()
    for bad in (1.0, "a", [1.0] * 32):
        for call in (lambda: ops.checkpoint8_write(x, bad, g), lambda: ops.checkpoint8_write(x, g, bad),
                     lambda: ops.checkpoint8_read(ck, bad, g), lambda: ops.checkpoint8_read(ck, g, bad),
                     lambda: ops.group_norm_act(x, bad, g, 4)):
            with pytest.raises(L.MisegError):
                call()
    for bad in (x, None, (ck.codes, ck.scales)):
        with pytest.raises(L.MisegError):
            ops.checkpoint8_read(bad)
        with pytest.raises(L.MisegError):
            ops.group_norm_act_backward(x, bad)
    with pytest.raises(L.MisegError):
        ops.group_norm_act_backward(x, ops.Saved(None, (ck.codes, ck.scales), g, g, g, g, g, g, 4, "none"))


@pytest.mark.parametrize("checkpoint", [False, True])
def test_more_small_blocks_than_a_launch_takes(ops, checkpoint):
    """65535 images of one pixel in 257 slabs of 40 channels: 16.8 million blocks of 256 threads, and a launch takes 2^32
    threads at most in a direction.  Images are apart, so the last ones give what a call of their own gives."""
    n, c, groups = 65535, 10280, 257
    x = torch.empty((n, 1, 1, c), dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 8192):
        m = min(8192, n - i)
        x[i:i + m] = normal(i, m, 1, 1, c)
    gamma, beta = normal(1, c), normal(2, c)
    dy = x.flip(0)
    y, saved = ops.group_norm_act(x, gamma, beta, groups, act="relu", checkpoint=checkpoint)
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, saved)
    sums = torch.zeros((2, c), dtype=torch.float64, device="cuda")
    size = torch.zeros((2, c), dtype=torch.float64, device="cuda")
    for i in range(0, n, 4096):
        part = slice(i, min(i + 4096, n))
        yw, sw = ops.group_norm_act(x[part], gamma, beta, groups, act="relu", checkpoint=checkpoint)
        dxw, _, _ = ops.group_norm_act_backward(dy[part], sw)
        assert torch.equal(y[part], yw) and torch.equal(dx[part], dxw), i
        assert torch.equal(saved.mean[part], sw.mean) and torch.equal(saved.shift[part], sw.shift)
        if checkpoint:
            assert torch.equal(saved.checkpoint.codes[part], sw.checkpoint.codes)
            xhat = sw.checkpoint.codes.double() * sw.checkpoint.scales.double().repeat_interleave(32, 3)[..., :c]
            z = xhat * gamma.double() + beta.double()
        else:
            xhat = (x[part].double() - sw.mean.double().repeat_interleave(40, 1)[:, None, None]) * \
                sw.rstd.double().repeat_interleave(40, 1)[:, None, None]
            z = x[part].double() * sw.scale.double()[:, None, None] + sw.shift.double()[:, None, None]
        g = dy[part].double() * (z > 0)
        for k, t in enumerate((g * xhat, g)):
            sums[k] += t.sum((0, 1, 2))
            size[k] += t.abs().sum((0, 1, 2))
    # an image's term a channel is one product of 32-bit numbers (x - mean, rstd, g: 4 roundings), images are added up in 64
    # bits and the sum is rounded once
    for k, got in enumerate((dgamma, dbeta)):
        assert ((got.double() - sums[k]).abs() <= 4 * U * size[k] + U * sums[k].abs()).all()
