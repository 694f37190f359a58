"""The eviction kernels take all of their registers: compiled to assembly, none of them
may have gone to scratch memory (weights of 4096 tokens on 8192 keys 234 us where 16
bytes did, 214 without)."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def test_no_scratch_memory(tmp_path):
    if not Path(HIPCC).exists():
        pytest.skip("no hipcc")
    make = subprocess.run(["make", "-n", "-B", "_build/ops_k_evict.o"], cwd=ROOT / "cu-jev_amd",
                          capture_output=True, text=True, check=True)
    line = next(x for x in make.stdout.splitlines() if "evict.hip" in x)
    out = tmp_path / "evict.s"
    args = re.sub(r"\s-c\s", " --cuda-device-only -S ", re.sub(r"-o \S+", f"-o {out}", line)).split()
    subprocess.run(args, cwd=ROOT / "cu-jev_amd", check=True, capture_output=True)
    text = out.read_text()
    sizes = re.findall(r"ScratchSize: (\d+)", text)
    assert len(sizes) >= len(re.findall(r"^_Z\S*kernel\S*:\s*;\s*@", text, re.M)) >= 14
    assert set(sizes) == {"0"}
