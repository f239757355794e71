"""The tests of draws at borders, of clipping at the ends of the range and of several users at once, against the range-checking build of the library."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["test_gpu_draw_borders.py", "test_gpu_clip_more.py", "test_gpu_serve_uses.py"])
def test_operators_stay_in_bounds_in_the_checked_build(name):
    from albatross_b200 import build
    assert os.path.exists(build.LIB_CHECKED), "the range-checking build of the library is missing"
    cmd = [sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", os.path.join(ROOT, "tests", name)]
    res = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, AB_BOUNDS_CHECK="1"), capture_output=True, text=True, timeout=900)
    tail = (res.stdout + res.stderr)[-2000:]
    assert res.returncode == 0, tail
    assert "passed" in res.stdout and "AB_BOUNDS_CHECK: a kernel recorded" not in res.stdout, tail
