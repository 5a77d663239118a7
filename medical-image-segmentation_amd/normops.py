"""Group normalisation with an activation, and activation checkpoints in 8 bits, on channels-last torch tensors.

The layers beside `Trainer`'s BatchNormalization + ReLU (the reference's networks, utils/model.py:176-211, normalise by
batch statistics only): `group_norm_act` and `group_norm_act_backward` for batches too small for batch statistics, and
`checkpoint8_write` / `checkpoint8_read`, which keep an activation for the backward pass in 8.5 bits a value.

Tensors are (N, H, W, C) with C a multiple of 8, in bfloat16, float16 or float32, dense or a channel slice of a wider
dense tensor that starts at a multiple of 16 bytes; empty ones are refused.  Every function launches on the current stream of
its tensors' device, through `lib` where one is given (the proxy that times the launches of `Trainer.profile_step`).  There is
no autograd behind them: the caller runs the backward pass, as `Trainer` does.  Where autograd is recording, a tensor that
asks for a gradient is refused: take `.detach()` of it or call under `torch.no_grad()`.
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

    @classmethod
    def _like(cls, x):
        """An unwritten checkpoint for a tensor that `_view` has accepted."""
        self = cls.__new__(cls)
        n, h, w, c = x.shape
        self.codes = x.new_empty((n, h, w, c), dtype=torch.int8)
        self.scales = x.new_empty((n, h, w, (c + 31) // 32), dtype=torch.bfloat16)
        return self

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + 2 * self.scales.numel()


class Saved:
    """What `group_norm_act_backward` takes of a forward call: x or its checkpoint, the statistics `mean` and `rstd`
    (N, groups), the coefficients of z = x * scale + shift (N, C), and the layer's parameters `gamma` and `beta` (None
    where it has none), which only the backward pass from a checkpoint reads: a forward call that writes one keeps them as
    it read them, so that an update in between changes no gradient."""

    def __init__(self, x, checkpoint, mean, rstd, scale, shift, gamma, beta, groups, act):
        self.x, self.checkpoint = x, checkpoint
        self._four, self._flat = (mean, rstd, scale, shift), None
        self.gamma, self.beta, self.groups, self.act = gamma, beta, groups, act

    @classmethod
    def _of(cls, x, checkpoint, flat, n, c, gamma, beta, groups, act):
        """From the buffer of a forward call, scale, shift, mean, rstd and with a checkpoint gamma and beta between shift and
        mean, one behind the other: taken apart where somebody asks."""
        self = cls(x, checkpoint, None, None, None, None, gamma, beta, groups, act)
        self._four, self._flat, self._n, self._c, self._stats = None, flat, n, c, 2 * n * c
        if checkpoint is not None:
            self._stats += 2 * c
            if gamma is not None:
                del self.gamma                               # __getattr__ finds it in the buffer
            if beta is not None:
                del self.beta
        return self

    def __getattr__(self, name):
        if name not in ("gamma", "beta"):
            raise AttributeError(name)
        t = self._flat.as_strided((self._c,), (1,), (2 * self._n + (name == "beta")) * self._c)
        setattr(self, name, t)
        return t

    def _part(self, which, columns, start):
        return self._four[which] if self._four else self._flat.as_strided((self._n, columns), (columns, 1), start)

    @property
    def mean(self):
        return self._part(0, self.groups, 0 if self._four else self._stats)

    @property
    def rstd(self):
        return self._part(1, self.groups, 0 if self._four else self._stats + self._n * self.groups)

    @property
    def scale(self):
        return self._part(2, 0 if self._four else self._c, 0)

    @property
    def shift(self):
        return self._part(3, 0 if self._four else self._c, 0 if self._four else self._n * self._c)

    def _addresses(self, n, c, device):
        """Of mean, rstd, scale and shift, for an (n, ., ., c) tensor."""
        g = self.groups
        if self._flat is not None:
            if (self._n, self._c) != (n, c) or self._flat.device != device:
                raise L.MisegError("saved from %d images of %d channels on %s, not %d of %d on %s"
                                   % (self._n, self._c, self._flat.device, n, c, device))
            at = self._flat.data_ptr()
            stats = at + 4 * self._stats
            return stats, stats + 4 * n * g, at, at + 4 * n * c
        return tuple(_coef(t, name, shape, device, False) for t, name, shape in
                     zip(self._four, ("mean", "rstd", "scale", "shift"), ((n, g), (n, g), (n, c), (n, c))))

    def _parameters(self, n, c, device):
        """Addresses of gamma and beta, or None, for the pass from a checkpoint; after `_addresses`."""
        own = self.__dict__.get
        gamma, beta = own("gamma", self), own("beta", self)      # self: in the buffer
        at = self._flat.data_ptr() + 8 * n * c if gamma is self or beta is self else 0
        return at if gamma is self else _coef(gamma, "gamma", (c,), device), \
            at + 4 * c if beta is self else _coef(beta, "beta", (c,), device)


def _view(t, name, like=None):
    """(pixel stride, image stride) of a channels-last tensor or channel slice."""
    if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _TYPES:
        raise L.MisegError("%s has to be a (N, H, W, C) tensor in bfloat16, float16 or float32" % name)
    if not t.is_cuda:
        raise L.MisegError("%s is on %s: these operators run on the GPU" % (name, t.device))
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise L.MisegError("%s is %s on %s, not %s on %s" % (name, tuple(t.shape), t.device, tuple(like.shape), like.device))
    n, h, w, c = t.shape
    if not (n and h and w and c):
        raise L.MisegError("%s is empty: %s" % (name, tuple(t.shape)))
    if n > 65535 or c > 65536:                               # before the 32 bits of a descriptor cut them
        raise L.MisegError("%s: %d images of %d channels (at most 65535 of 65536)" % (name, n, c))
    if t.is_contiguous():
        return c, h * w * c
    sn, sh, sw, sc = t.stride()
    pix = sw if w > 1 else sh if h > 1 else max(sw, c)
    if (c > 1 and sc != 1) or (w > 1 and h > 1 and sh != w * pix) or not c <= pix < 1 << 31 or \
            (n > 1 and sn < (h * w - 1) * pix + c):
        raise L.MisegError("%s is not channels last: shape %s, strides %s" % (name, tuple(t.shape), t.stride()))
    if h == 1 and w == 1:
        per = 16 // t.element_size()
        pix = (c + per - 1) // per * per                     # one pixel: its stride is never used
    return pix, sn if n > 1 else h * w * pix


def _coef(t, name, shape, device, optional=True):
    if t is None and optional:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != shape or \
            t.device != device or not t.is_contiguous():
        raise L.MisegError("%s has to be a dense float32 tensor %s on %s" % (name, shape, device))
    return t.data_ptr()


def _plain(a, b=None, c=None):
    """Nothing that autograd would have to see."""
    if (a is not None and a.requires_grad or b is not None and b.requires_grad or c is not None and c.requires_grad) and \
            torch.is_grad_enabled():
        raise L.MisegError("a tensor asks for a gradient, and no autograd is behind this call: detach it or call under "
                           "torch.no_grad()")


def _act(act):
    if act not in ACTS:
        raise L.MisegError("activation %r: one of %s" % (act, ", ".join(ACTS)))
    return ACTS[act]


def _groups(groups, c):
    if not isinstance(groups, int) or groups < 1 or c % groups:
        raise L.MisegError("%d channels in %r groups" % (c, groups))


def _launch(fn, d, device):
    """fn on the current stream of `device`, whichever device is current."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(C.byref(d), stream)
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(d), stream)
    if rc:
        L.check(rc)


def _workspace(lib, d, n, pixels, c, groups, dtype, checkpoint, backward, x):
    size = lib.miseg_group_norm_workspace(n, pixels, c, groups, dtype, checkpoint, backward)
    if size < 0:
        L.check(int(size))
    if size == 0:
        return None
    ws = x.new_empty(size, dtype=torch.uint8)
    d.workspace, d.workspace_bytes = ws.data_ptr(), size
    return ws


def group_norm_act(x, gamma, beta, groups, eps=1e-3, act="none", out=None, checkpoint=False, lib=None):
    """y = act(gamma * (x - mean) / sqrt(var + eps) + beta), mean and biased variance over the pixels and the C / groups
    consecutive channels of a group of each image.  gamma, beta: float32 (C,) or None (1 and 0).  act: "none", "relu", "silu".
    out: where y goes, a view like x (x itself only with `checkpoint`).  checkpoint: keep the normalised x in 8 bits, not x.
    Returns y and the `Saved` that the backward pass takes."""
    lib = L.load() if lib is None else lib
    d = L.GroupNormDesc()
    d.x_pix, d.x_img = _view(x, "x")
    n, h, w, c = x.shape
    device, dtype = x.device, x.dtype
    _groups(groups, c)
    d.x = x.data_ptr()
    if out is None:
        y = x.new_empty((n, h, w, c))
        d.y_pix, d.y_img = c, h * w * c
    else:
        y = out
        d.y_pix, d.y_img = _view(y, "out", x)
        if y.dtype != dtype:
            raise L.MisegError("out is %s, x %s" % (y.dtype, dtype))
        if y.data_ptr() == d.x and not checkpoint:
            raise L.MisegError("out is x, which the backward pass needs: pass checkpoint=True or another tensor")
        _plain(y)
    d.y = y.data_ptr()
    d.gamma, d.beta = _coef(gamma, "gamma", (c,), device), _coef(beta, "beta", (c,), device)
    _plain(x, gamma, beta)
    flat = x.new_empty(2 * (n * (c + groups) + (c if checkpoint else 0)), dtype=torch.float32)
    d.scale = at = flat.data_ptr()
    d.shift, stats = at + 4 * n * c, at + 8 * n * c
    ck = None
    if checkpoint:
        if gamma is not None:
            d.gamma_kept = stats
        if beta is not None:
            d.beta_kept = stats + 4 * c
        stats += 8 * c
        ck = Checkpoint8._like(x)
        d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    d.mean, d.rstd = stats, stats + 4 * n * groups
    d.N, d.C, d.groups, d.pixels, d.eps, d.act = n, c, groups, h * w, eps, _act(act)
    d.dtype, d.fmt = kind = _TYPES[dtype]
    # the workspace lives until the launch is in its stream
    ws = _workspace(lib, d, n, h * w, c, groups, kind[0], 1 if checkpoint else 0, 0, x)      # noqa: F841
    _launch(lib.miseg_group_norm_act_fwd, d, device)
    return y, Saved._of(None if checkpoint else x, ck, flat, n, c, gamma, beta, groups, act)


def group_norm_act_backward(dy, saved, out=None, lib=None):
    """dx, dgamma and dbeta (float32 (C,)) of `group_norm_act` from the gradient of its result and what it saved.  out: where
    dx goes, a view like dy (dy itself allowed)."""
    lib = L.load() if lib is None else lib
    if not isinstance(saved, Saved) or not isinstance(saved.checkpoint, (Checkpoint8, type(None))):
        raise L.MisegError("the backward pass takes what group_norm_act saved")
    d = L.GroupNormBwdDesc()
    d.dy_pix, d.dy_img = _view(dy, "dy")
    n, h, w, c = dy.shape
    device, dtype, groups, ck = dy.device, dy.dtype, saved.groups, saved.checkpoint
    if (saved.x is None) == (ck is None):
        raise L.MisegError("the backward pass takes x or its checkpoint")
    _groups(groups, c)
    d.dy = dy.data_ptr()
    if ck is None:
        d.x_pix, d.x_img = _view(saved.x, "x", dy)
        d.x = saved.x.data_ptr()
        if saved.x.dtype != dtype:
            raise L.MisegError("dy is %s, x %s" % (dtype, saved.x.dtype))
    else:
        if ck.shape != dy.shape or ck.device != device:
            raise L.MisegError("the checkpoint is %s on %s, dy %s on %s" % (tuple(ck.shape), ck.device, tuple(dy.shape), device))
        d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    if out is None:
        dx = dy.new_empty((n, h, w, c))
        d.dx_pix, d.dx_img = c, h * w * c
    else:
        dx = out
        d.dx_pix, d.dx_img = _view(dx, "out", dy)
        if dx.dtype != dtype:
            raise L.MisegError("out is %s, dy %s" % (dx.dtype, dtype))
    _plain(dy, out)
    d.dx = dx.data_ptr()
    d.mean, d.rstd, d.scale, d.shift = saved._addresses(n, c, device)
    if ck is not None:
        d.gamma, d.beta = saved._parameters(n, c, device)
    grads = dy.new_empty((2, c), dtype=torch.float32)
    d.dgamma = at = grads.data_ptr()
    d.dbeta = at + 4 * c
    d.N, d.C, d.groups, d.pixels, d.act = n, c, groups, h * w, _act(saved.act)
    d.dtype, d.fmt = kind = _TYPES[dtype]
    ws = _workspace(lib, d, n, h * w, c, groups, kind[0], 0 if ck is None else 1, 1, dy)     # noqa: F841
    _launch(lib.miseg_group_norm_act_bwd, d, device)
    dgamma, dbeta = grads.unbind(0)
    return dx, dgamma, dbeta


def _pair(a, b, what, n, c, device):
    """Coefficients (C,) or (N, C) as (pointer, pointer, elements from one image's to the next's, what the caller holds until
    the launch is in its stream)."""
    if a is None and b is None:
        return None, None, 0, None
    if a is None or b is None:
        raise L.MisegError("%s: a scale and a shift go together" % what)
    shape = (n, c) if isinstance(a, torch.Tensor) and a.dim() == 2 else (c,)
    pa, pb = _coef(a, what + " scale", shape, device), _coef(b, what + " shift", shape, device)
    _plain(a, b)
    held = None
    if (pa | pb) & 15:                                       # slices of a flat buffer: copies start at a multiple of 16 bytes
        held = a.clone(), b.clone()
        pa, pb = held[0].data_ptr(), held[1].data_ptr()
    return pa, pb, c if n > 1 and len(shape) == 2 else 0, held               # of one image both shapes are the same


def checkpoint8_write(x, scale=None, shift=None, y_scale=None, y_shift=None, act="none", out=None, lib=None):
    """The 8-bit checkpoint of x, or of x * scale + shift with float32 coefficients (C,) or (N, C).  With y_scale and y_shift
    also y = act(x * y_scale + y_shift) of the same pass, into `out` if given (x itself allowed): returns (checkpoint, y)."""
    lib = L.load() if lib is None else lib
    d = L.Checkpoint8Desc()
    d.x_pix, d.x_img = _view(x, "x")
    n, h, w, c = x.shape
    device = x.device
    d.x = x.data_ptr()
    d.code_a, d.code_b, img, held = _pair(scale, shift, "code", n, c, device)                # noqa: F841
    d.y_a, d.y_b, y_of, y_held = _pair(y_scale, y_shift, "y", n, c, device)                  # noqa: F841
    if scale is not None and y_scale is not None and img != y_of:
        raise L.MisegError("the coefficients of the codes and of y are both (C,) or both (N, C)")
    d.coef_img = max(img, y_of)
    y = None
    if y_scale is not None:
        y = x.new_empty((n, h, w, c)) if out is None else out
        d.y_pix, d.y_img = _view(y, "out", x)
        if y.dtype != x.dtype:
            raise L.MisegError("out is %s, x %s" % (y.dtype, x.dtype))
        d.y = y.data_ptr()
    elif out is not None or act != "none":
        raise L.MisegError("an activation and out belong to y, which takes y_scale and y_shift")
    _plain(x, out)
    ck = Checkpoint8._like(x)
    d.codes, d.code_scales = ck.codes.data_ptr(), ck.scales.data_ptr()
    d.N, d.C, d.pixels, d.act = n, c, h * w, _act(act)
    d.dtype, d.fmt = _TYPES[x.dtype]
    _launch(lib.miseg_checkpoint8_write, d, device)
    return ck if y is None else (ck, y)


def checkpoint8_read(checkpoint, scale=None, shift=None, act="none", dtype=torch.bfloat16, out=None, lib=None):
    """act(v * scale + shift) of a checkpoint's values v as a tensor of `dtype` (of out's type where it is given)."""
    lib = L.load() if lib is None else lib
    if not isinstance(checkpoint, Checkpoint8):
        raise L.MisegError("checkpoint8_read takes a Checkpoint8, not %s" % type(checkpoint).__name__)
    codes = checkpoint.codes
    n, h, w, c = codes.shape
    device = codes.device
    if out is None:
        out = codes.new_empty((n, h, w, c), dtype=dtype)
    d = L.Checkpoint8Desc()
    d.y_pix, d.y_img = _view(out, "out", checkpoint)
    d.y, d.codes, d.code_scales = out.data_ptr(), codes.data_ptr(), checkpoint.scales.data_ptr()
    _plain(out)
    d.y_a, d.y_b, d.coef_img, held = _pair(scale, shift, "y", n, c, device)                  # noqa: F841
    d.N, d.C, d.pixels, d.act = n, c, h * w, _act(act)
    d.dtype, d.fmt = _TYPES[out.dtype]
    _launch(lib.miseg_checkpoint8_read, d, device)
    return out
