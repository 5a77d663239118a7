"""Arguments of the normalisation entry points that the host refuses: nothing is launched, so the tests run without a GPU
(addresses are made up and never read)."""
import ctypes as C

import pytest

from miseg_amd import lib as L

A = 1 << 20                                       # an aligned address


def lib():
    try:
        return L.load()
    except L.MisegError:
        pytest.skip("libmiseg.so is not built")


@pytest.mark.parametrize("bad", [dict(gamma_kept=A + 4), dict(beta_kept=A + 8), dict(gamma_kept=A, beta_kept=A + 2)], ids=str)
def test_kept_parameters_are_aligned(bad):
    d = L.GroupNormDesc()
    for i, f in enumerate(("x", "y", "mean", "rstd", "scale", "shift", "workspace", "codes", "code_scales")):
        setattr(d, f, A + (i << 24))
    d.N, d.C, d.groups, d.pixels, d.x_pix, d.y_pix, d.x_img, d.y_img, d.eps = 2, 64, 8, 3000, 64, 64, 192000, 192000, 1e-3
    d.workspace_bytes = 1 << 20
    for k, v in bad.items():
        setattr(d, k, v)
    assert lib().miseg_group_norm_act_fwd(C.byref(d), None) == L.E_INVALID_ARG
    assert b"kept" in L.load().miseg_last_error()


def test_the_last_field_lies_where_the_header_says(tmp_path):
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "miseg.h"\nint main(void) {\n'
                   'printf("%zu %zu\\n", offsetof(miseg_group_norm_desc, gamma_kept), offsetof(miseg_group_norm_desc, beta_kept));\n'
                   'return 0; }\n')
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [L.GroupNormDesc.gamma_kept.offset, L.GroupNormDesc.beta_kept.offset]
