"""Training with activations kept in 8 bits (`Trainer(checkpoint_8bit=True)`): every backward operation against 64-bit
arithmetic on the tensors it was given, for a residual, a dense and a pyramid network; memory; refusals.

Tolerances: a data gradient is rounded once to bf16 (2^-8 of a value) after sums in 32 bits; norms over a tensor, so the
rounding enters with at most 2^-8, and every bound below is that plus 2^-10 for the 32-bit sums (at most 2^13 terms a
thread-level chain, errors of random sign)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8
SUMS = 2.0 ** -10


def rel(a, b):
    return ((a.double() - b.double()).norm() / (b.double().norm() + 1e-30)).item()


def make(enc, dec, h=64, w=96, n=2, c=3, **kw):
    import miseg_amd  # noqa: F401
    from miseg_amd import netspec, trainer, weights as W
    g = netspec.build_graph(enc, dec, (h, w, 3), c, "softmax", None)
    tr = trainer.Trainer(g, W.init_weights(g, seed=3, randomize_bn=True), n, learning_rate=1e-3, **kw)
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.random((n, h, w, 3), dtype=np.float32)).cuda()
    lab = rng.integers(0, c, (n, h // 8, w // 8)).repeat(8, 1).repeat(8, 2)
    return tr, x, torch.from_numpy(np.eye(c, dtype=np.float32)[lab]).cuda()


def values(ck):
    return ck.codes.double() * ck.scales.double().repeat_interleave(32, 3)[..., :ck.shape[3]]


@pytest.mark.parametrize("enc,dec", [("resnet18", "U-Net"), ("resnet34", "Linknet"), ("densenet169", "U-Net"),
                                     ("resnet18", "FPN")])
def test_every_backward_operation(enc, dec):
    from miseg_amd.trainer import Act, Kept
    tr, x, gt = make(enc, dec, checkpoint_8bit=True)
    tr.keep_grads = True
    probs = tr.forward(x)
    assert torch.isfinite(probs).all() and (probs.sum(-1) - 1).abs().max() <= 4 * 2.0 ** -23
    assert not tr.acts and not tr.concat_bufs, "16-bit activations outlive the forward pass: %s" % list(tr.acts)[:5]
    tr.loss_and_metrics(gt)
    tr.backward()
    torch.cuda.synchronize()
    g = tr.g
    seen = {"bn": 0, "conv": 0}
    for name, l in g.layers.items():
        if l.cls == "BatchNormalization" and name in tr.grad_log:
            dy, dx = tr.grad_log[name]
            saved, c = tr.saved[name], l.out.c
            xhat = values(saved.checkpoint)[0]
            d = dy.t[..., dy.c0:dy.c0 + c].double().reshape(xhat.shape)
            z = xhat * saved.gamma.double() + saved.beta.double()
            gz = d * (z > 0)
            m = xhat.shape[0] * xhat.shape[1]
            s1, s2 = gz.sum((0, 1)), (gz * xhat).sum((0, 1))
            a = saved.scale[0].double()
            want = a * (gz - s1 / m - xhat * s2 / m)
            assert rel(dx.t[..., :c].reshape(xhat.shape), want) <= BF + SUMS, name
            # the sums' terms cancel: against the norm of what they add up
            mag = gz.abs().sum((0, 1)).norm(), (gz * xhat).abs().sum((0, 1)).norm()
            assert (tr.gview(name, "beta").double() - s1).norm() <= 2.0 ** -20 * mag[0], name
            if l.config["scale"]:
                assert (tr.gview(name, "gamma").double() - s2).norm() <= 2.0 ** -20 * mag[1], name
            seen["bn"] += 1
        elif l.cls == "Conv2D" and l.config["kernel_size"] != 7 and name in tr.accum_final:
            kept, pad = tr.saved[name]
            assert isinstance(kept, Kept), name
            op = tr._operand(kept)
            v = values(kept.checkpoint)
            if kept.scale is not None:
                v = v * kept.scale.double() + kept.shift.double()
            if kept.act == "relu":
                v = v.clamp_min(0)
            assert rel(op.t[..., :op.c], v) <= BF, name
            dy = tr.accum_final[name]
            co, ci, k, s = l.out.c, op.c, l.config["kernel_size"], l.config["strides"]
            got = tr.gview(name, "kernel")[:co, :, :, :ci].double()
            xt = op.t[..., :ci].double().cpu().permute(0, 3, 1, 2)
            wt = torch.zeros((co, ci, k, k), dtype=torch.float64, requires_grad=True)
            y = torch.nn.functional.conv2d(xt, wt, stride=s, padding=pad)
            y.backward(dy.t[..., dy.c0:dy.c0 + co].double().cpu().permute(0, 3, 1, 2)[:, :, :y.shape[2], :y.shape[3]])
            assert rel(got.cpu(), wt.grad.permute(0, 2, 3, 1)) <= SUMS, name
            seen["conv"] += 1
    assert seen["bn"] >= 10 and seen["conv"] >= 10, seen
    del Act


def test_the_forward_pass_and_the_heads_gradient_against_16_bits():
    """The forward pass reads no checkpoint: what differs from a trainer without them is the order of the statistics' sums
    (64-bit atomics) and the layers that apply a BatchNormalization on the way in, each by at most a bf16 rounding of a
    value here and there.  The head's weight gradient differs by the 8 bits of its operand: 0.0102 of a standard normal
    operand's rounding (a step of the block's largest value, under 4.5 deviations, over 127 and sqrt(12)); at least half of
    the square sum is left behind the ReLU, and twice that covers a sample's spread.  Probabilities enter the gradient at
    the logits linearly, with the roundings of some twenty layers of random sign: 20^0.5 * 2^-8."""
    a, x, gt = make("resnet18", "U-Net")
    b, _, _ = make("resnet18", "U-Net", checkpoint_8bit=True)
    pa, pb = a.forward(x), b.forward(x)
    assert rel(pb, pa) <= 20 ** 0.5 * BF
    for t in (a, b):
        t.loss_and_metrics(gt)
        t.backward()
    torch.cuda.synchronize()
    head = a.g.logits_layer
    assert rel(b.gview(head, "kernel"), a.gview(head, "kernel")) <= 2 * 0.0102 * 2 ** 0.5 + 20 ** 0.5 * BF


def test_steps_run_and_memory_shrinks():
    """Two steps, with the optimiser; what is held between the passes is at most 0.62 of the 16-bit trainer's: per value of
    a convolution + BatchNormalization + ReLU 1.06 bytes instead of 4 (2 where the apply pass is not stored), next to
    tensors that both hold (image, prepared image, probabilities, parameters)."""
    held = []
    for ck in (False, True):
        tr, x, gt = make("resnet18", "U-Net", h=256, w=320, n=2, checkpoint_8bit=ck)
        before = torch.cuda.memory_allocated()
        for _ in range(2):
            tr.train_step(x, gt)
        tr.forward(x)
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated() - before)
        assert torch.isfinite(tr.P).all() and torch.isfinite(tr.G).all()
        del tr
        torch.cuda.empty_cache()
    assert held[1] <= 0.62 * held[0], held


def test_frozen_encoder_and_refusal():
    tr, x, gt = make("resnet18", "U-Net", checkpoint_8bit=True, freeze_encoder=True)
    before = tr.P.clone()
    tr.train_step(x, gt)
    torch.cuda.synchronize()
    assert torch.isfinite(tr.P).all() and not torch.equal(tr.P, before)
    name = next(n for n in tr.frozen if (n, "kernel") in tr.segs)
    s = tr.segs[(name, "kernel")]
    assert torch.equal(tr.P[s.off:s.off + s.count], before[s.off:s.off + s.count])
    with pytest.raises(NotImplementedError):
        make("vgg16", "U-Net", checkpoint_8bit=True)


def test_model_passes_the_choice_on():
    from utils.model import make_model, CUSTOM_OBJECTS, METRICS
    model = make_model("resnet18", "U-Net", (64, 96, 3), 3, 1e-3, CUSTOM_OBJECTS["categorical_crossentropy_plus_dice_loss"],
                       METRICS, False, "m")
    model.checkpoint_8bit = True
    rng = np.random.default_rng(0)
    x = rng.random((2, 64, 96, 3), dtype=np.float32)
    y = np.eye(3, dtype=np.float32)[rng.integers(0, 3, (2, 64, 96))]
    model.fit(x, y, batch_size=2, epochs=1, verbose=0)
    assert model._train_state.checkpoint_8bit and np.isfinite(model.get_weights()[0]).all()
