"""What can be held without a GPU about the sequence operators' sources, build and argument checks."""
import importlib
import os
import re
from pathlib import Path


import ops

be = ops.backend
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
