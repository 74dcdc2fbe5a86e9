"""Register and scratch budget of the rotary, quantised cache and sliding attention kernels (CPU:
compiles to gfx950 assembly with the library's own flags; no GPU).  A spill in the attention's loops
waits for every load under way; the workgroups that share a CU follow from the registers."""
import concurrent.futures
import os
import re
import shutil
import tempfile

import pytest

import test_kernel_resources as kr
from sager_amd import build_lib

# (source, kernel-name pattern, max registers of a lane, vector and accumulation ones)
BUDGETS = [
    ("sg_rope.hip", r"rope_kernel", 128),
    ("sg_kvq8.hip", r"kv_(store|read)_q8_kernel", 128),
    ("sg_attn.hip", r"kv_commit_kernel", 128),
    ("sg_slide.hip", r"slide_few_kernelILi256E", 256),
    ("sg_slide.hip", r"slide_few_kernelILi128ELi2E", 168),
    ("sg_slide.hip", r"slide_few_kernelILi128ELi1E", 128),
    ("sg_slide.hip", r"slide_few_kernelILi64ELi2E", 128),
    ("sg_slide.hip", r"slide_few_kernelILi64ELi1E", 96),
    ("sg_slide.hip", r"slide_rows_kernel", 256),
    ("sg_slide.hip", r"slide_rows_kernelILi64E", 128),
    ("sg_slide.hip", r"attn_join_kernel", 128),
]


@pytest.mark.skipif(not os.path.exists(build_lib.HIPCC) and shutil.which("hipcc") is None,
                    reason="hipcc not available")
def test_no_scratch_and_as_many_waves_as_planned():
    srcs = sorted({s for s, *_ in BUDGETS})
    with tempfile.TemporaryDirectory() as d:
        with concurrent.futures.ThreadPoolExecutor(max_workers=len(srcs)) as ex:
            asm = dict(ex.map(lambda s: kr._asm(s, d), srcs))
    for src, pat, most in BUDGETS:
        ks = {n: v for n, v in kr._kernels(asm[src]).items() if re.search(pat, n)}
        assert ks, f"no kernel matches {pat} in {src}"
        for name, (scratch, vgpr) in ks.items():
            assert scratch == 0, f"{name}: {scratch} B of scratch per lane"
            assert vgpr <= most, f"{name}: {vgpr} registers (budget {most})"
