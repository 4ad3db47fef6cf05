"""What can be held without a GPU about the sequence operators' sources, build and argument checks."""
import ctypes
import importlib
import math
import os
import re
from pathlib import Path


import pytest
import torch

import ops
from test_cpu_sequence import OK, cache_problem, evict_status, masked_problem, tree_status

be = ops.backend
cabi = be.cabi
PACKAGE = Path(be.__file__).resolve().parent
CSRC = PACKAGE / "csrc"


def test_overlapped_kernels_read_the_workspace_by_coherent_loads():
    """A kernel that is resident while the one before it still writes the workspace (st, sp: its parts) may not read it by the
    read-only path, whose data has to be constant for the whole kernel."""
    for name in ("dsdpa_masked_bwd.cuh", "dsdpa_share.cuh", "dsdpa_tree.cuh", "dsdpa_few.cuh", "dsdpa_few_f32.cuh", "dsdpa_cache_simt.cuh"):
        text = (CSRC / name).read_text()
        assert not re.search(r"(__ldg|ldg128_nc|ldg128_stream)\(\s*(\([^)]*\)\s*)?(st|sp)\.", text), name


def test_a_copied_tree_is_compiled_again(tmp_path, monkeypatch):
    """Dependency files hold absolute paths: in a copy of the tree they say nothing about the copy's headers."""
    build = importlib.import_module(be.__name__ + ".build")
    for name in ("here", "copy"):
        (tmp_path / name).mkdir()
        for f in ("a.cu", "a.cuh"):
            (tmp_path / name / f).write_text("")
            os.utime(tmp_path / name / f, (1000, 1000))
    dep = tmp_path / "a.d"
    dep.write_text(f"a.o : {tmp_path}/here/a.cu \\\n    /usr/include/stdio.h \\\n  {tmp_path}/here/a.cuh\n")
    monkeypatch.setattr(build, "HERE", tmp_path / "here" / "package")
    assert build._newest_source(tmp_path / "here" / "a.cu", dep) == 1000
    os.utime(tmp_path / "here" / "a.cuh", (2000, 2000))
    assert build._newest_source(tmp_path / "here" / "a.cu", dep) == 2000
    (tmp_path / "here" / "a.cuh").unlink()
    assert build._newest_source(tmp_path / "here" / "a.cu", dep) == float("inf")
    monkeypatch.setattr(build, "HERE", tmp_path / "copy" / "package")
    assert build._newest_source(tmp_path / "copy" / "a.cu", dep) == float("inf")
    assert build._newest_source(tmp_path / "copy" / "a.cu", tmp_path / "none.d") == float("inf")


@pytest.mark.parametrize("sm_scale,softcap", [(1e39, 0.0), (-math.inf, 0.0), (math.nan, 0.0), (0.125, math.nan), (0.125, -1.0), (0.125, math.inf),
                                              (0.125, 1e39), (0.125, 3e38), (0.125, 1e-46), (0.125, 1e-40), (1e-8, 1e37), (1e10, 1e-30)])
def test_numbers_that_fp32_cannot_carry_are_refused(sm_scale, softcap):
    """Neither a silent infinity, nor a cap that becomes none, nor one whose ratio to the scale is lost."""
    q = torch.zeros(1, 2, 4, 64)
    with pytest.raises(ValueError, match="sm_scale"):
        be.masked_sdpa(q, q, q, sm_scale, softcap=softcap)
    with pytest.raises(ValueError, match="tree_sdpa: sm_scale"):
        be.masked._check_numbers(sm_scale, softcap, "tree_sdpa")
    if softcap < 0:                       # the C ABI's sign for no cap
        return
    as_float = [ctypes.c_float(x).value for x in (sm_scale, softcap)]
    if softcap == 0.0 or as_float[1] != 0.0:
        for p, call in ((masked_problem(sm_scale=as_float[0], softcap=as_float[1]), "dsdpa_masked_backward_workspace_bytes"),
                        (cache_problem(sm_scale=as_float[0], softcap=as_float[1]), "dsdpa_tree_workspace_bytes")):
            assert getattr(cabi.lib(), call)(ctypes.byref(p)) == 0
    assert tree_status(cache_problem(sm_scale=as_float[0], softcap=as_float[1] or math.nan)) == cabi.ERR_BAD_SHAPE


@pytest.mark.parametrize("sm_scale,softcap", [(0.125, 0.0), (0.0, 5.0), (-2.0, 1e30), (0.125, 50.0), (1e20, 1.0), (1e-20, 1.0)])
def test_numbers_that_it_can_are_not(sm_scale, softcap):
    be.masked._check_numbers(sm_scale, softcap, "masked_sdpa")
    assert cabi.lib().dsdpa_masked_backward_workspace_bytes(ctypes.byref(masked_problem(sm_scale=sm_scale, softcap=softcap))) > 0


def test_an_eviction_does_not_write_over_the_lengths_it_reads():
    p = cache_problem()
    lens, other = ctypes.c_void_p(16384), ctypes.c_void_p(8192)
    ptrs = [OK, OK, OK, lens, OK, None]
    assert evict_status(p, ptrs=ptrs, more=(OK, lens, other, None)) == cabi.ERR_BAD_SHAPE
