"""What ties profiles/traffic_kernels.json to the kernels that were counted (no GPU)."""
import os
import re
import shutil

import bench

CSRC = os.path.join(bench.ROOT, "sager_amd", "csrc")


def test_the_hash_covers_the_counted_kernels_sources():
    text = {f: open(os.path.join(CSRC, f)).read() for f in bench.TRAFFIC_SOURCES}
    for kernel in bench.TRAFFIC_KERNELS:
        name = kernel.split("<")[0]
        assert any(re.search(r"\b%s\(" % name, t) for t in text.values()), name
    for t in text.values():
        for inc in re.findall(r'#include "(sg_\w+\.hpp)"', t):
            assert inc in text, inc


def test_another_operator_does_not_change_the_hash(tmp_path, monkeypatch):
    shutil.copytree(CSRC, tmp_path / "sager_amd" / "csrc")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    before = bench.source_hash()
    (tmp_path / "sager_amd" / "csrc" / "sg_other.hip").write_text("// another operator\n")
    assert bench.source_hash() == before
    with open(tmp_path / "sager_amd" / "csrc" / "sg_layer.hip", "a") as f:
        f.write("// another form of a counted kernel\n")
    assert bench.source_hash() != before
