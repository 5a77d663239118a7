"""What the normalisation and checkpoint entry points refuse.  Every refusal is the host's: nothing is launched, so the
tests run without a GPU (addresses are made up and never read)."""
import ctypes as C

import pytest
import torch

from miseg_amd import lib as L
from miseg_amd import normops

A = 1 << 20                                       # an aligned address


def lib():
    try:
        return L.load()
    except L.MisegError:
        pytest.skip("libmiseg.so is not built")


def fwd(**kw):
    d = L.GroupNormDesc()
    for i, f in enumerate(("x", "y", "mean", "rstd", "scale", "shift", "workspace")):
        setattr(d, f, A + (i << 24))
    d.N, d.C, d.groups, d.pixels, d.x_pix, d.y_pix, d.x_img, d.y_img, d.eps = 2, 64, 8, 3000, 64, 64, 192000, 192000, 1e-3
    d.workspace_bytes = 1 << 20
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def bwd(**kw):
    d = L.GroupNormBwdDesc()
    for i, f in enumerate(("x", "dy", "dx", "mean", "rstd", "scale", "shift", "workspace")):
        setattr(d, f, A + (i << 24))
    d.N, d.C, d.groups, d.pixels = 2, 64, 8, 3000
    d.x_pix = d.dy_pix = d.dx_pix = 64
    d.x_img = d.dy_img = d.dx_img = 192000
    d.workspace_bytes = 1 << 20
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def ckpt(**kw):
    d = L.Checkpoint8Desc()
    d.x, d.codes, d.code_scales = A, A + (1 << 24), A + (2 << 24)
    d.N, d.C, d.pixels, d.x_pix, d.x_img = 2, 64, 100, 64, 6400
    for k, v in kw.items():
        setattr(d, k, v)
    return d


COMMON = [dict(dtype=2), dict(fmt=2), dict(act=L.ACT_SOFTMAX), dict(act=9), dict(N=0), dict(N=65536), dict(pixels=0),
          dict(pixels=1 << 29), dict(C=0), dict(C=60), dict(C=65544)]


@pytest.mark.parametrize("bad", COMMON + [
    dict(groups=0), dict(groups=7), dict(groups=-1), dict(x=None), dict(y=None), dict(x=A + 8), dict(y=A + 2), dict(x_pix=56),
    dict(x_pix=68), dict(y_pix=0), dict(x_img=191936), dict(x_img=192004), dict(y_img=0), dict(mean=None), dict(rstd=None),
    dict(scale=None), dict(shift=A + 4), dict(eps=-1.0), dict(eps=float("nan")), dict(codes=A), dict(code_scales=A),
    dict(codes=A + 4, code_scales=A), dict(codes=A, code_scales=A + 1), dict(workspace=None), dict(workspace=A + 8),
    dict(workspace_bytes=100), dict(y=A + 128), dict(y=A + 6400), dict(y=A, y_pix=72, y_img=216000),
], ids=str)
def test_group_norm_forward(bad):
    assert lib().miseg_group_norm_act_fwd(C.byref(fwd(**bad)), None) == L.E_INVALID_ARG
    assert L.load().miseg_last_error()


@pytest.mark.parametrize("bad", COMMON + [
    dict(groups=0), dict(groups=7), dict(x=None), dict(codes=A, code_scales=A), dict(x=None, codes=A),
    dict(x=None, codes=A + 4, code_scales=A), dict(x=None, codes=A, code_scales=A + 1), dict(dy=None), dict(dx=None),
    dict(dy=A + 8), dict(dy_pix=56), dict(dx_img=100), dict(dy_img=0), dict(mean=None), dict(rstd=None), dict(scale=None),
    dict(shift=None), dict(workspace=None), dict(workspace_bytes=64), dict(dx=A + 256), dict(dx=A + (1 << 24) + 256),
], ids=str)
def test_group_norm_backward(bad):
    assert lib().miseg_group_norm_act_bwd(C.byref(bwd(**bad)), None) == L.E_INVALID_ARG


@pytest.mark.parametrize("bad", COMMON + [
    dict(x=None), dict(x=A + 4), dict(x_pix=60), dict(codes=None), dict(code_scales=None), dict(codes=A + 4),
    dict(code_scales=A + 1), dict(code_a=A), dict(code_b=A), dict(code_a=A + 4, code_b=A), dict(y=A),
    dict(y_a=A, y_b=A), dict(y=A + (3 << 24), y_a=A, y_b=A, y_pix=8, y_img=6400),
    dict(y=A + (3 << 24), y_a=A, y_pix=64, y_img=6400), dict(act=L.ACT_RELU),
    dict(y=A + 64, y_a=A, y_b=A, y_pix=64, y_img=6400), dict(code_a=A, code_b=A, coef_img=2),
], ids=str)
def test_checkpoint_write(bad):
    assert lib().miseg_checkpoint8_write(C.byref(ckpt(**bad)), None) == L.E_INVALID_ARG


@pytest.mark.parametrize("bad", COMMON + [dict(y=None), dict(y=A + 8), dict(y_pix=32), dict(y_img=0), dict(codes=None),
                                          dict(code_scales=None), dict(y_a=A), dict(y_b=A), dict(y_a=A + 4, y_b=A),
                                          dict(y_a=A, y_b=A, coef_img=-4)], ids=str)
def test_checkpoint_read(bad):
    d = ckpt(**{**dict(y=A + (3 << 24), y_pix=64, y_img=6400), **bad})
    assert lib().miseg_checkpoint8_read(C.byref(d), None) == L.E_INVALID_ARG


def test_null_descriptors_and_workspace_sizes():
    l = lib()
    for f in (l.miseg_group_norm_act_fwd, l.miseg_group_norm_act_bwd, l.miseg_checkpoint8_write, l.miseg_checkpoint8_read):
        assert f(None, None) == L.E_INVALID_ARG
    for bad in ((0, 1, 8, 1, 0), (65536, 1, 8, 1, 0), (1, 0, 8, 1, 0), (1, 1 << 29, 8, 1, 0), (1, 1, 0, 1, 0),
                (1, 1, 12, 1, 0), (1, 1, 65544, 1, 0), (1, 1, 8, 0, 0), (1, 1, 8, 3, 0), (1, 1, 8, 1, 2)):
        assert l.miseg_group_norm_workspace(*bad, 0, 0) == L.E_INVALID_ARG
    assert l.miseg_group_norm_workspace(1, 1, 8, 1, 0, 0, 0) == 0
    big = [l.miseg_group_norm_workspace(4, 960 * 1280, 64, 16, 0, *k) for k in ((0, 0), (1, 0), (0, 1))]
    # of the order of the statistics, never of the tensor: 4 images at 960 x 1280 with 64 channels are 629 MB
    assert 0 < big[0] < big[1] < big[2] < 4 << 20


def test_python_refuses():
    x = torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16)
    for bad in (x, x.double(), x[0], x.to(torch.int8), None):            # on the CPU, another type, another rank
        with pytest.raises(L.MisegError):
            normops.group_norm_act(bad, None, None, 4)
        with pytest.raises(L.MisegError):
            normops.checkpoint8_write(bad)
    codes = torch.zeros(1, 2, 3, 40, dtype=torch.int8)
    scales = torch.zeros(1, 2, 3, 2, dtype=torch.bfloat16)
    ck = normops.Checkpoint8(codes, scales)
    assert ck.nbytes() == 240 + 24
    for c, s in ((codes[0], scales), (codes.float(), scales), (codes, scales[..., :1]), (codes, scales.float()),
                 (codes[..., ::2], scales[..., :1]), (codes.transpose(1, 2), scales.transpose(1, 2))):
        with pytest.raises(L.MisegError):
            normops.Checkpoint8(c, s)
    with pytest.raises(L.MisegError):
        normops.checkpoint8_read(ck)                                     # on the CPU
    saved = normops.Saved(None, ck, None, None, None, None, None, None, 4, "relu")
    with pytest.raises(L.MisegError):
        normops.group_norm_act_backward(torch.zeros(1, 2, 3, 40, dtype=torch.bfloat16), saved)


def test_structures_have_the_headers_layout(tmp_path):
    """Sizes and last fields of the ctypes mirrors against the compiler's."""
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"miseg_group_norm_desc": (L.GroupNormDesc, "eps"), "miseg_group_norm_bwd_desc": (L.GroupNormBwdDesc, "act"),
             "miseg_checkpoint8_desc": (L.Checkpoint8Desc, "act")}
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "miseg.h"\nint main(void) {\n' + "".join(
        'printf("%%zu %%zu\\n", sizeof(%s), offsetof(%s, %s));\n' % (n, n, f) for n, (_, f) in names.items()) + "return 0; }\n")
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    lines = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")
    for line, (cls, field) in zip(lines, names.values()):
        assert [int(v) for v in line.split()] == [C.sizeof(cls), getattr(cls, field).offset]
