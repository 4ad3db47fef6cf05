"""The sequence and cache operators on the checked debug build, whose kernels range-check the rows of weights, positions and
partial results that they compute (tests/test_gpu_checked_build.py has the deformable operator's): their tests once more
in a child process that loads it, the suite's fixture asking for a recorded index after every one."""
import os
import subprocess
import sys

import pytest

from test_gpu_checked_build import CHECKED, ROOT


@pytest.mark.gpu
def test_sequence_operators_on_the_checked_build():
    env = dict(os.environ, DSDPA_LIBRARY=str(CHECKED))
    res = subprocess.run([sys.executable, "-m", "pytest", "tests/test_gpu_cache.py", "tests/test_gpu_masked.py", "tests/test_gpu_sequence_edges.py",
                          "-m", "gpu", "-x", "-q", "-k", "not overflowed", "-p", "no:cacheprovider"], cwd=ROOT, env=env, capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[-4000:] + res.stderr[-2000:]
    assert " passed" in res.stdout
