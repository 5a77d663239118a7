"""What a trainer with 8-bit checkpoints keeps, against the tensors of its forward pass, and the backward operations that read
it: poolings and transpose convolutions next to those of every layer.

Bounds.  A value lies within half a step of what was kept (scale * (0.5 + 256 u): the product with the rounded reciprocal of
the scale).  The normalised input is fma(x, r, -mean r): r = 1 / sqrt(var + eps) is off by 2 u at most, the product and the
fma by u each, and the coefficients of the layer's own pass by as much: 8 u (|x| + |mean|) r covers either side.  Batch
statistics: sums of n <= 12288 stored values in 32 bits at the worst, n u of the magnitudes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = 2.0 ** -8
SUMS = 2.0 ** -10             # 32-bit sums of at most 2^13 terms, errors of random sign, as a share of a tensor's norm
NETS = [("resnet18", "U-Net"), ("resnet34", "Linknet"), ("densenet169", "U-Net"), ("resnet18", "FPN"), ("densenet121", "Linknet")]


def make(enc, dec, h=64, w=96, n=2, c=3, **kw):
    import miseg_amd  # noqa: F401
    from miseg_amd import netspec, trainer, weights as W
    g = netspec.build_graph(enc, dec, (h, w, 3), c, "softmax", None)
    tr = trainer.Trainer(g, W.init_weights(g, seed=3, randomize_bn=True), n, learning_rate=1e-3, **kw)
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.random((n, h, w, 3), dtype=np.float32)).cuda()
    lab = rng.integers(0, c, (n, h // 8, w // 8)).repeat(8, 1).repeat(8, 2)
    return tr, x, torch.from_numpy(np.eye(c, dtype=np.float32)[lab]).cuda()


def steps(ck):
    return ck.scales.double().repeat_interleave(32, 3)[..., :ck.shape[3]]


def values(ck):
    return ck.codes.double() * steps(ck)


def of(act):
    return act.t[..., act.c0:act.c0 + act.c].double()


def within(got, want, tol, name):
    off = ((got - want).abs() - tol).max().item()
    assert off <= 0, "%s: off by %g more than allowed" % (name, off)


def rel(a, b):
    return ((a.double() - b.double()).norm() / (b.double().norm() + 1e-30)).item()


@pytest.mark.parametrize("enc,dec", NETS)
def test_what_is_kept_is_what_the_forward_pass_had(enc, dec):
    tr, x, gt = make(enc, dec, checkpoint_8bit=True)
    tr._drop_read = lambda position: None                      # the activations stay
    tr.forward(x)
    torch.cuda.synchronize()
    g, kept_of = tr.g, {}
    seen = {"bn": 0, "own": 0, "readers": 0}
    for name, l in g.layers.items():
        if l.cls in ("Conv2D", "Conv2DTranspose", "MaxPooling2D") and name in tr.saved and l.config.get("kernel_size") != 7:
            kept = tr.saved[name] if l.cls == "MaxPooling2D" else tr.saved[name][0]
            src = tr._src(l.inbound[0])[0]
            assert kept is tr.kept[src], name
            kept_of[src] = kept
            seen["readers"] += 1
        if l.cls == "BatchNormalization" and g.layers[l.inbound[0]].cls != "InputLayer":
            s, v = tr.bn_state[name], of(tr.acts[l.inbound[0]])
            c, count = l.out.c, v[..., 0].numel()
            mean, var = s["mean"][:c].double(), s["var"][:c].double()
            within(mean, v.mean((0, 1, 2)), count * U * v.abs().mean((0, 1, 2)), name)
            square = v.square().mean((0, 1, 2))
            within(var, (v - v.mean((0, 1, 2))).square().mean((0, 1, 2)), 3 * count * U * square, name)
            r = 1 / (var + l.config["epsilon"]).sqrt()
            saved, n = tr.saved[name], v.shape[0]
            ck = saved.checkpoint
            codes = ck.codes.view(n, -1, ck.shape[2], c)
            step = ck.scales.view(n, -1, ck.shape[2], ck.scales.shape[3]).double().repeat_interleave(32, 3)[..., :c]
            known = 8 * U * (v.abs() + mean.abs()) * r
            within(codes.double() * step, (v - mean) * r, step * (0.5 + 256 * U) + known, name)
            seen["bn"] += 1
    for src, kept in tr.kept.items():
        want = of(tr.acts[src])
        step, v = steps(kept.checkpoint), values(kept.checkpoint)
        if kept.scale is None:
            within(v, want, step * (0.5 + 256 * U), src)
            seen["own"] += 1
            continue
        bn = g.layers[src].inbound[0]
        x_in, s = of(tr.acts[g.layers[bn].inbound[0]]), tr.bn_state[bn]
        c = x_in.shape[3]
        mean, gamma, beta = s["mean"][:c].double(), kept.scale.double(), kept.shift.double()
        r = 1 / (s["var"][:c].double() + g.layers[bn].config["epsilon"]).sqrt()
        z = v * gamma + beta
        assert kept.act == "relu"
        tol = gamma.abs() * (step * (0.5 + 256 * U) + 16 * U * (x_in.abs() + mean.abs()) * r) + 4 * U * beta.abs()
        within(z.clamp_min(0), want, tol + BF * want.abs(), src)
    assert seen["bn"] >= 10 and seen["own"] >= 1 and seen["readers"] >= 10, seen


def first_maximum_gradient(x, dy):
    """dx of ZeroPadding2D(1) + MaxPooling2D(3, 2) of (n, h, w, c): to the first maximum of a window in row-major order."""
    n, h, w, c = x.shape
    pad = torch.nn.functional.pad(x.permute(0, 3, 1, 2), (1, 1, 1, 1))
    win = pad.unfold(2, 3, 2).unfold(3, 3, 2)[:, :, :dy.shape[1], :dy.shape[2]].reshape(n, c, dy.shape[1], dy.shape[2], 9)
    most = win == win.amax(4, keepdim=True)
    first = most & (most.cumsum(4) == 1)
    grad = first.double() * dy.permute(0, 3, 1, 2)[..., None]
    out = torch.zeros_like(pad)
    for k in range(9):
        ky, kx = divmod(k, 3)
        out[:, :, ky:ky + 2 * dy.shape[1]:2, kx:kx + 2 * dy.shape[2]:2] += grad[..., k]
    return out[:, :, 1:-1, 1:-1].permute(0, 2, 3, 1)


@pytest.mark.parametrize("enc,dec,kind", [("resnet18", "U-Net", "pool"), ("densenet121", "FPN", "pool"),
                                          ("resnet18", "Linknet", "transpose"), ("resnet34", "U-Net", "transpose")])
def test_poolings_and_transpose_convolutions(enc, dec, kind):
    tr, x, gt = make(enc, dec, checkpoint_8bit=True)
    tr.keep_grads = True
    tr.forward(x)
    tr.loss_and_metrics(gt)
    tr.backward()
    torch.cuda.synchronize()
    seen = 0
    for name, l in tr.g.layers.items():
        if kind == "pool" and l.cls == "MaxPooling2D":
            assert l.config["pool_size"] == 3
            dy, dx = tr.grad_log[name]
            xin = of(tr._operand(tr.saved[name]))
            assert rel(of(dx), first_maximum_gradient(xin, of(dy))) <= BF + SUMS, name
            seen += 1
        if kind == "transpose" and l.cls == "Conv2DTranspose":
            xin, dy = of(tr._operand(tr.saved[name][0])), of(tr.accum_final[name])
            co, ci = l.out.c, xin.shape[3]
            got = tr.gview(name, "kernel")[..., :ci].double().cpu()
            xt = xin.permute(0, 3, 1, 2).cpu()
            for a in range(2):
                for b in range(2):                             # out[2y + a, 2x + b] = sum in[y + a - 1 + i, x + b - 1 + j] w[i][j]
                    wt = torch.zeros((co, ci, 2, 2), dtype=torch.float64, requires_grad=True)
                    y = torch.nn.functional.conv2d(torch.nn.functional.pad(xt, (1 - b, b, 1 - a, a)), wt)
                    y.backward(dy[:, a::2, b::2].permute(0, 3, 1, 2).cpu())
                    assert rel(got[a * 2 + b], wt.grad.permute(0, 2, 3, 1)) <= SUMS, (name, a, b)
            seen += 1
    assert seen >= (1 if kind == "pool" else 4), seen


def test_a_profiled_step_lists_the_normalisation_and_checkpoint_launches():
    """Trainer.profile_step times every launch: a checkpoint a BatchNormalization + ReLU and a kept tensor, a read an operand, a
    backward pass a BatchNormalization, with the bytes they move."""
    tr, x, gt = make("resnet18", "U-Net", checkpoint_8bit=True)
    tr.train_step(x, gt)
    before = tr.P.clone()
    prof = tr.profile_step(x, gt)
    assert not torch.equal(tr.P, before)
    g = tr.g
    bns = [n for n, l in g.layers.items() if l.cls == "BatchNormalization" and g.layers[l.inbound[0]].cls != "InputLayer"]
    convs = [n for n, l in g.layers.items() if l.cls in ("Conv2D", "Conv2DTranspose") and l.config["kernel_size"] != 7]
    pools = [n for n, l in g.layers.items() if l.cls == "MaxPooling2D"]
    want = {"miseg_checkpoint8_write": len(tr.kept), "miseg_checkpoint8_read": len(convs) + len(pools),
            "miseg_group_norm_act_bwd": len(bns)}
    got = {v["entry"]: v for v in prof.values() if v["entry"] in want}
    assert {k: v["launches"] for k, v in got.items()} == want
    assert all(v["ms"] > 0 for v in got.values())
    eight = sum(k.checkpoint.nbytes() for k in tr.kept.values())
    acts = [2 * k.checkpoint.codes.numel() for k in tr.kept.values()]
    both = [2 * k.checkpoint.codes.numel() for k in tr.kept.values() if k.scale is not None]
    assert got["miseg_checkpoint8_write"]["bytes"] == eight + sum(acts) + sum(both)
    norm = sum(tr.saved[n].checkpoint.nbytes() + 4 * tr.saved[n].checkpoint.codes.numel() for n in bns)
    assert got["miseg_group_norm_act_bwd"]["bytes"] == norm
    layers = {tag for tag, kernel, _, _, _ in tr.lib.calls() if "group_norm" in kernel}
    assert layers == {"bwd " + n for n in bns}
    tr.train_step(x, gt)                                       # and nothing is recorded afterwards
    assert len(tr.lib.records) == sum(v["launches"] for v in prof.values())


def test_the_choice_may_change_between_steps():
    """model.checkpoint_8bit counts when it is set: the next step keeps 8 bits, with the parameters and the optimiser's state of
    the steps before, and one that cannot is refused before anything changes."""
    from utils.model import make_model, CUSTOM_OBJECTS, METRICS
    rng = np.random.default_rng(0)
    x = rng.random((2, 64, 96, 3), dtype=np.float32)
    y = np.eye(3, dtype=np.float32)[rng.integers(0, 3, (2, 64, 96))]
    for dec in ("U-Net", "FPN"):
        model = make_model("resnet18", dec, (64, 96, 3), 3, 1e-3, CUSTOM_OBJECTS["categorical_crossentropy_plus_dice_loss"],
                           METRICS, False, "m")
        model.train_on_batch(x, y)
        tr = model._train_state
        assert not tr.checkpoint_8bit and not tr.drops
        for on in (True, False, True):
            model.checkpoint_8bit = on
            before = tr.P.clone()
            model.train_on_batch(x, y)
            assert model._train_state is tr and tr.checkpoint_8bit == on and bool(tr.kept) == on
            assert not torch.equal(tr.P, before)
        assert tr.step_count == 4
        # the folded forms of a network are those of a trainer that never kept 8 bits
        fresh, _, _ = make("resnet18", dec)
        tr.set_checkpoint_8bit(False)
        assert (tr.head_up, tr.fs, tr.p2, tr.place) == (fresh.head_up, fresh.fs, fresh.p2, fresh.place)
        fresh.load_state(tr.state())
        xt, gt = torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda()
        assert rel(tr.forward(xt), fresh.forward(xt)) <= 20 ** 0.5 * BF      # twenty layers' roundings of random sign
    tr, _, _ = make("vgg16", "U-Net")
    with pytest.raises(NotImplementedError):
        tr.set_checkpoint_8bit(True)
    assert not tr.checkpoint_8bit
