"""Register and scratch budgets of the verify window's kernels (CPU: compiles to gfx950 assembly
with the library's own flags; no GPU).  None may use scratch memory; the attention's vector registers
decide how many of its workgroups a CU holds, which the launch counts on (by head dimension one, two
or four of 256 threads, or one of 512)."""
import os
import re
import shutil

import pytest

import test_kernel_resources as res
from sager_amd import build_lib

# (source, kernel-name pattern, max VGPRs): 512 registers a SIMD lane, a wave on each of four SIMDs
# per 256 threads
BUDGETS = [
    ("sg_attn.hip", r"attn_few_kernelILi64ELi[12]E", 128),
    ("sg_attn.hip", r"attn_few_kernelILi128ELi[12]E", 256),
    ("sg_attn.hip", r"attn_few_kernelILi256ELi[12]E", 512),
    ("sg_attn.hip", r"attn_rows_kernelILi(64|128|256)E", 256),
    ("sg_attn.hip", r"attn_join_kernel", 128),
    ("sg_attn.hip", r"kv_commit_kernel", 128),
    ("sg_norm.hip", r"add_rmsnorm_kernel", 128),
    ("sg_verify.hip", r"verify_(rows|rest)_kernel", 128),
    ("sg_verify.hip", r"verify_walk_kernel", 128),  # 1024 threads
]


@pytest.mark.skipif(not os.path.exists(build_lib.HIPCC) and shutil.which("hipcc") is None,
                    reason="hipcc not available")
def test_window_kernels_within_register_budget(tmp_path):
    asm = dict(res._asm(s, str(tmp_path)) for s in sorted({s for s, *_ in BUDGETS}))
    for src, pat, most in BUDGETS:
        ks = {n: v for n, v in res._kernels(asm[src]).items() if re.search(pat, n)}
        assert ks, f"no kernel matches {pat} in {src}"
        for name, (scratch, vgpr) in ks.items():
            assert scratch == 0, f"{name}: {scratch} B of scratch per lane"
            assert vgpr <= most, f"{name}: {vgpr} VGPRs"
