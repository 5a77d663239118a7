"""Group normalisation with an activation, and activation checkpoints in 8 bits, on channels-last torch tensors.

The layers beside `Trainer`'s BatchNormalization + ReLU (the reference's networks, utils/model.py:176-211, normalise by
batch statistics only): `group_norm_act` and `group_norm_act_backward` for batches too small for batch statistics, and
`checkpoint8_write` / `checkpoint8_read`, which keep an activation for the backward pass in 8.5 bits a value.

Tensors are (N, H, W, C) with C a multiple of 8, in bfloat16, float16 or float32, dense or a channel slice of a wider
dense tensor that starts at a multiple of 16 bytes.  Every function launches on the current stream of its tensors' device.
"""
import ctypes as C

import torch

from . import lib as L

ACTS = {"none": L.ACT_NONE, "relu": L.ACT_RELU, "silu": L.ACT_SILU}
_TYPES = {torch.bfloat16: (L.DT_BF16, L.FMT_BF16), torch.float16: (L.DT_BF16, L.FMT_F16),
          torch.float32: (L.DT_F32, L.FMT_BF16)}


class Checkpoint8:
    """An activation (N, H, W, C) in 8 bits: int8 `codes` of its shape and one bfloat16 of `scales` (N, H, W, ceil(C / 32))
    for 32 channels of a pixel.  A value is code * scale; a scale that is NaN marks a block that held no finite value."""

    def __init__(self, codes, scales):
        if codes.dim() != 4 or codes.dtype != torch.int8 or scales.dtype != torch.bfloat16 or \
                tuple(scales.shape) != tuple(codes.shape[:3]) + ((codes.shape[3] + 31) // 32,):
            raise L.MisegError("a checkpoint is int8 (N, H, W, C) and bfloat16 (N, H, W, ceil(C / 32)): got %s %s and %s %s"
                               % (codes.dtype, tuple(codes.shape), scales.dtype, tuple(scales.shape)))
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device:
            raise L.MisegError("the codes and scales of a checkpoint are dense and on one device")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + 2 * self.scales.numel()


class Saved:
    """What `group_norm_act_backward` takes of a forward call: x or its checkpoint, the statistics (N, groups), the
    coefficients of z = x * scale + shift (N, C), and the layer's parameters."""

    def __init__(self, x, checkpoint, mean, rstd, scale, shift, gamma, beta, groups, act):
        self.x, self.checkpoint = x, checkpoint
        self.mean, self.rstd, self.scale, self.shift = mean, rstd, scale, shift
        self.gamma, self.beta, self.groups, self.act = gamma, beta, groups, act


def _view(t, name, like=None):
    """(pixel stride, image stride) of a channels-last tensor or channel slice."""
    if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _TYPES:
        raise L.MisegError("%s has to be a (N, H, W, C) tensor in bfloat16, float16 or float32" % name)
    if t.device.type != "cuda":
        raise L.MisegError("%s is on %s: these operators run on the GPU" % (name, t.device))
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise L.MisegError("%s is %s on %s, not %s on %s" % (name, tuple(t.shape), t.device, tuple(like.shape), like.device))
    n, h, w, c = t.shape
    if t.numel() == 0:
        raise L.MisegError("%s is empty: %s" % (name, tuple(t.shape)))
    sn, sh, sw, sc = t.stride()
    pix = sw if w > 1 else sh if h > 1 else max(sw, c)
    if (c > 1 and sc != 1) or (w > 1 and h > 1 and sh != w * pix) or pix < c or (n > 1 and sn < (h * w - 1) * pix + c):
        raise L.MisegError("%s is not channels last: shape %s, strides %s" % (name, tuple(t.shape), t.stride()))
    per = 16 // t.element_size()
    if h == 1 and w == 1:
        pix = (c + per - 1) // per * per                     # one pixel: its stride is never used
    return pix, sn if n > 1 else h * w * pix


def _coef(t, name, shape, device, optional=True):
    if t is None and optional:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != tuple(shape) or \
            t.device != device or not t.is_contiguous():
        raise L.MisegError("%s has to be a dense float32 tensor %s on %s" % (name, tuple(shape), device))
    return t.data_ptr()


def _act(act):
    if act not in ACTS:
        raise L.MisegError("activation %r: one of %s" % (act, ", ".join(ACTS)))
    return ACTS[act]


def _workspace(lib, n, pixels, c, backward, device):
    size = lib.miseg_group_norm_workspace(n, pixels, c, backward)
    if size < 0:
        L.check(int(size))
    return torch.empty(size, dtype=torch.uint8, device=device)


def _new_checkpoint(shape, device):
    n, h, w, c = shape
    return Checkpoint8(torch.empty((n, h, w, c), dtype=torch.int8, device=device),
                       torch.empty((n, h, w, (c + 31) // 32), dtype=torch.bfloat16, device=device))


def group_norm_act(x, gamma, beta, groups, eps=1e-3, act="none", out=None, checkpoint=False):
    """y = act(gamma * (x - mean) / sqrt(var + eps) + beta), mean and biased variance over the pixels and the C / groups
    consecutive channels of a group of each image.  gamma, beta: float32 (C,) or None (1 and 0).  act: "none", "relu", "silu".
    out: where y goes, a view like x (x itself only with `checkpoint`).  checkpoint: keep the normalised x in 8 bits, not x.
    Returns y and the `Saved` that the backward pass takes."""
    lib = L.load()
    x_pix, x_img = _view(x, "x")
    n, h, w, c = x.shape
    device = x.device
    y = torch.empty((n, h, w, c), dtype=x.dtype, device=device) if out is None else out
    y_pix, y_img = _view(y, "out", x)
    if y.dtype != x.dtype:
        raise L.MisegError("out is %s, x %s" % (y.dtype, x.dtype))
    if y.data_ptr() == x.data_ptr() and not checkpoint:
        raise L.MisegError("out is x, which the backward pass needs: pass checkpoint=True or another tensor")
    if not isinstance(groups, int) or groups < 1 or c % groups:
        raise L.MisegError("%d channels in %r groups" % (c, groups))
    stats = torch.empty(2 * n * (groups + c) + 8, dtype=torch.float32, device=device)
    scale, shift = stats[:n * c].view(n, c), stats[n * c:2 * n * c].view(n, c)
    mean, rstd = stats[2 * n * c:2 * n * c + n * groups].view(n, groups), stats[2 * n * c + n * groups:2 * n * (c + groups)].view(n, groups)
    ck = _new_checkpoint(x.shape, device) if checkpoint else None
    d = L.GroupNormDesc()
    d.x, d.y, d.x_pix, d.x_img, d.y_pix, d.y_img = x.data_ptr(), y.data_ptr(), x_pix, x_img, y_pix, y_img
    d.gamma, d.beta = _coef(gamma, "gamma", (c,), device), _coef(beta, "beta", (c,), device)
    d.mean, d.rstd, d.scale, d.shift = mean.data_ptr(), rstd.data_ptr(), scale.data_ptr(), shift.data_ptr()
    if ck is not None:
        d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    d.N, d.C, d.groups, d.pixels, d.eps, d.act = n, c, groups, h * w, eps, _act(act)
    d.dtype, d.fmt = _TYPES[x.dtype]
    with torch.cuda.device(device):
        ws = _workspace(lib, n, h * w, c, 0, device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        L.check(lib.miseg_group_norm_act_fwd(C.byref(d), torch.cuda.current_stream(device).cuda_stream))
    return y, Saved(None if checkpoint else x, ck, mean, rstd, scale, shift, gamma, beta, groups, act)


def group_norm_act_backward(dy, saved, out=None):
    """dx, dgamma and dbeta (float32 (C,)) of `group_norm_act` from the gradient of its result and what it saved.  out: where
    dx goes, a view like dy (dy itself allowed)."""
    lib = L.load()
    dy_pix, dy_img = _view(dy, "dy")
    n, h, w, c = dy.shape
    device, groups = dy.device, saved.groups
    if (saved.x is None) == (saved.checkpoint is None):
        raise L.MisegError("the backward pass takes x or its checkpoint")
    dx = torch.empty((n, h, w, c), dtype=dy.dtype, device=device) if out is None else out
    d = L.GroupNormBwdDesc()
    d.dx_pix, d.dx_img = _view(dx, "out", dy)
    if saved.x is not None:
        d.x_pix, d.x_img = _view(saved.x, "x", dy)
        d.x = saved.x.data_ptr()
        if saved.x.dtype != dy.dtype:
            raise L.MisegError("dy is %s, x %s" % (dy.dtype, saved.x.dtype))
    else:
        ck = saved.checkpoint
        if ck.shape != dy.shape or ck.device != device:
            raise L.MisegError("the checkpoint is %s on %s, dy %s on %s" % (tuple(ck.shape), ck.device, tuple(dy.shape), device))
        d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    if dx.dtype != dy.dtype:
        raise L.MisegError("out is %s, dy %s" % (dx.dtype, dy.dtype))
    if not isinstance(groups, int) or groups < 1 or c % groups:
        raise L.MisegError("%d channels in %r groups" % (c, groups))
    d.mean = _coef(saved.mean, "mean", (n, groups), device, False)
    d.rstd = _coef(saved.rstd, "rstd", (n, groups), device, False)
    d.scale = _coef(saved.scale, "scale", (n, c), device, False)
    d.shift = _coef(saved.shift, "shift", (n, c), device, False)
    d.gamma, d.beta = _coef(saved.gamma, "gamma", (c,), device), _coef(saved.beta, "beta", (c,), device)
    grads = torch.empty((2, c), dtype=torch.float32, device=device)
    d.dgamma, d.dbeta = grads[0].data_ptr(), grads[1].data_ptr()
    d.dy, d.dx, d.dy_pix, d.dy_img = dy.data_ptr(), dx.data_ptr(), dy_pix, dy_img
    d.N, d.C, d.groups, d.pixels, d.act = n, c, groups, h * w, _act(saved.act)
    d.dtype, d.fmt = _TYPES[dy.dtype]
    with torch.cuda.device(device):
        ws = _workspace(lib, n, h * w, c, 1, device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        L.check(lib.miseg_group_norm_act_bwd(C.byref(d), torch.cuda.current_stream(device).cuda_stream))
    return dx, grads[0], grads[1]


def _pair(a, b, what, n, c, device):
    """Coefficients (C,) or (N, C) as (pointer, pointer, elements from one image's to the next's)."""
    if (a is None) != (b is None):
        raise L.MisegError("%s: a scale and a shift go together" % what)
    if a is None:
        return None, None, 0
    shape = (n, c) if a.dim() == 2 else (c,)
    return _coef(a, what + " scale", shape, device), _coef(b, what + " shift", shape, device), c if a.dim() == 2 else 0


def checkpoint8_write(x, scale=None, shift=None, y_scale=None, y_shift=None, act="none", out=None):
    """The 8-bit checkpoint of x, or of x * scale + shift with float32 coefficients (C,) or (N, C).  With y_scale and y_shift
    also y = act(x * y_scale + y_shift) of the same pass, into `out` if given (x itself allowed): returns (checkpoint, y)."""
    lib = L.load()
    x_pix, x_img = _view(x, "x")
    n, h, w, c = x.shape
    d = L.Checkpoint8Desc()
    d.x, d.x_pix, d.x_img = x.data_ptr(), x_pix, x_img
    d.code_a, d.code_b, img = _pair(scale, shift, "code", n, c, x.device)
    d.y_a, d.y_b, y_of = _pair(y_scale, y_shift, "y", n, c, x.device)
    if scale is not None and y_scale is not None and img != y_of:
        raise L.MisegError("the coefficients of the codes and of y are both (C,) or both (N, C)")
    d.coef_img = max(img, y_of)
    y = None
    if y_scale is not None:
        y = torch.empty((n, h, w, c), dtype=x.dtype, device=x.device) if out is None else out
        if y.dtype != x.dtype:
            raise L.MisegError("out is %s, x %s" % (y.dtype, x.dtype))
        d.y_pix, d.y_img = _view(y, "out", x)
        d.y = y.data_ptr()
    elif out is not None or act != "none":
        raise L.MisegError("an activation and out belong to y, which takes y_scale and y_shift")
    ck = _new_checkpoint(x.shape, x.device)
    d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    d.N, d.C, d.pixels, d.act = n, c, h * w, _act(act)
    d.dtype, d.fmt = _TYPES[x.dtype]
    with torch.cuda.device(x.device):
        L.check(lib.miseg_checkpoint8_write(C.byref(d), torch.cuda.current_stream(x.device).cuda_stream))
    return ck if y is None else (ck, y)


def checkpoint8_read(checkpoint, scale=None, shift=None, act="none", dtype=torch.bfloat16, out=None):
    """act(v * scale + shift) of a checkpoint's values v as a tensor of `dtype` (of out's type where it is given)."""
    lib = L.load()
    n, h, w, c = checkpoint.shape
    device = checkpoint.device
    if out is None:
        out = torch.empty((n, h, w, c), dtype=dtype, device=device)
    d = L.Checkpoint8Desc()
    d.y_pix, d.y_img = _view(out, "out", checkpoint)
    d.y, d.codes, d.code_scales = out.data_ptr(), checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr()
    d.y_a, d.y_b, d.coef_img = _pair(scale, shift, "y", n, c, device)
    d.N, d.C, d.pixels, d.act = n, c, h * w, _act(act)
    d.dtype, d.fmt = _TYPES[out.dtype]
    with torch.cuda.device(device):
        L.check(lib.miseg_checkpoint8_read(C.byref(d), torch.cuda.current_stream(device).cuda_stream))
    return out
