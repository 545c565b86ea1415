"""Which decode units read adopted prompts shared: the rule against the measured cases, on the host."""
import os
import shutil
import subprocess

import pytest

from conftest import HIP_SO, ROOT


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not available")
def test_units_take_the_faster_attention(tmp_path):
    obj, exe = str(tmp_path / "check.o"), str(tmp_path / "shared_attention_rule_check")
    subprocess.run(["hipcc", "-O1", "-std=c++17", "-w", "--offload-arch=gfx950", "-c",
                    os.path.join(ROOT, "tests", "shared_attention_rule_check.cpp"), "-o", obj], check=True)
    libdir = os.path.dirname(HIP_SO)
    subprocess.run(["hipcc", obj, "-L" + libdir, "-lsslm_hip", "-Wl,-rpath," + libdir, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
