"""What can be held without a GPU about the sequence operators' sources, build and argument checks."""
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
