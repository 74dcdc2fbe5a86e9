"""Register and scratch budget of the kernel that joins the parts of many rows (CPU: compiles to gfx950
assembly with the library's own flags; no GPU)."""
import os
import shutil
import tempfile

import pytest

import test_kernel_resources as kr
from sager_amd import build_lib


@pytest.mark.skipif(not os.path.exists(build_lib.HIPCC) and shutil.which("hipcc") is None,
                    reason="hipcc not available")
def test_no_scratch_and_as_many_waves_as_planned():
    with tempfile.TemporaryDirectory() as d:
        _, asm = kr._asm("sg_slide.hip", d)
    ks = {n: v for n, v in kr._kernels(asm).items() if "slide_join_kernel" in n}
    assert len(ks) == 3, sorted(ks)  # a head dimension each
    for name, (scratch, vgpr) in ks.items():
        assert scratch == 0 and vgpr <= 128, f"{name}: {scratch} B of scratch, {vgpr} registers"
