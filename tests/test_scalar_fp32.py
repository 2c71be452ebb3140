"""Every HIP unit is compiled without packed fp32 instructions, and none writes them by hand."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "instascene_amd", "csrc")
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def test_every_unit_is_compiled_without_packed_fp32():
    plan = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout.replace("\\\n", " ")
    compiles = [re.sub(r"\s+", " ", line) for line in plan.splitlines() if " -c " in line]
    assert len(compiles) >= 6 and all(FLAG in line for line in compiles), compiles


def test_no_source_writes_packed_fp32():
    sources = [f for kind in ("*.hip", "*.hpp") for f in glob.glob(os.path.join(CSRC, kind))]
    assert len(sources) > 15
    for f in sources:
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", open(f).read()), f
