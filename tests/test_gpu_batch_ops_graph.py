"""The operators over a batch of different requests on streams and inside captured graphs."""
import os
import shutil
import subprocess

import pytest

from conftest import HIP_SO, ROOT

pytestmark = pytest.mark.gpu


def test_batch_ops_on_streams_and_in_graph_replays(tmp_path):
    """Two batches' attention, projection and pick at once, each with its own workspaces: on two streams, as two
    captured graphs, as the branches of one; four rounds of new inputs in the same buffers with eager work
    between (tests/batch_ops_graph_check.cpp, built here)."""
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not available")
    obj, exe = str(tmp_path / "check.o"), str(tmp_path / "batch_ops_graph_check")
    subprocess.run(["hipcc", "-O1", "-std=c++17", "-w", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-c", os.path.join(ROOT, "tests", "batch_ops_graph_check.cpp"), "-o", obj], check=True)
    libdir = os.path.dirname(HIP_SO)
    subprocess.run(["hipcc", obj, "-L" + libdir, "-lsslm_hip", "-Wl,-rpath," + libdir, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().splitlines()[-1].startswith("ok"), (r.returncode, r.stdout, r.stderr[-2000:])
