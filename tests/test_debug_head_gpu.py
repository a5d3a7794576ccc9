"""The head's operators and clipping in the debug build of the kernel library (selected with LLMC_DEBUG_CHECKS=1)."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_debug_library_reports_nothing():
    r = subprocess.run([sys.executable, os.path.join(HERE, "debug_head_worker.py")], env=dict(os.environ, LLMC_DEBUG_CHECKS="1"), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    out = json.loads(r.stdout.strip().splitlines()[-1])
    assert out["debug_lib"] == 1 and out["passes"] == 7 and not any(out["status"]), out
    assert out["losses"][-1] < out["losses"][0]
