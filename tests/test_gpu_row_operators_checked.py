"""The row operators' suite once more on the bounds-checked build of the library (see test_gpu_bounds_checked.py): an access
of one of their kernels outside the live allocations fails the test that made it.  The longest rows are left out (every
access is a search), and what is captured into a graph, since a table cannot be installed during a capture."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_row_operators_on_the_bounds_checked_build(cuda):
    env = dict(os.environ, PXE_TEST_BOUNDS_CHECKED="1")
    cmd = [sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", "-k",
           "not graph and not captured and not served and not streams and not beyond and not many_large and not 70000 and not shape12 and not shape11",
           os.path.join("tests", "test_gpu_row_operators.py")]
    res = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=1500)
    tail = res.stdout[-3000:] + res.stderr[-2000:]
    assert res.returncode == 0, tail
    m = re.search(r"(\d+) passed", res.stdout)
    assert m and int(m.group(1)) >= 400, tail


@pytest.mark.gpu
def test_row_operators_edges_on_the_bounds_checked_build(cuda):
    """The same for the suite of values, states and places far from ordinary, without its longest rows and runs."""
    env = dict(os.environ, PXE_TEST_BOUNDS_CHECKED="1")
    cmd = [sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", "-k",
           "not 131072 and not 70000 and not 50003 and not many_rows and not long_run", os.path.join("tests", "test_gpu_row_operators_edges.py")]
    res = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    tail = res.stdout[-3000:] + res.stderr[-2000:]
    assert res.returncode == 0, tail
    m = re.search(r"(\d+) passed", res.stdout)
    assert m and int(m.group(1)) >= 75, tail
