"""CPU: what the dense kernels' sources must hold that no run can show."""

import re
from pathlib import Path

import easy_as_b200

CSRC = Path(easy_as_b200.__file__).parent / "csrc"


def test_warps_are_whole_before_aligned_instructions():
    """Lanes that a branch split come together first: barriers and TMEM loads do so in their own wrappers, mma.sync and
    the allocation at their places."""
    shared = (CSRC / "tcgen05_ptx.cuh").read_text()
    for name, first in (("tmem_ld32", "tcgen05.ld."), ("cluster_sync_all", "barrier.cluster.arrive")):
        body = shared[shared.index(f"void {name}("):]
        body = body[body.index("{") + 1:]
        assert body.index("__syncwarp();") < body.index(first), name
    for path in sorted(CSRC.glob("dense*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        assert "barrier.cluster." not in text and "tcgen05.ld." not in text, path.name   # only through the wrappers
    rows = re.sub(r"//[^\n]*", "", (CSRC / "dense_rows.cu").read_text())
    kernel = rows[rows.index("dense_rows_kernel(const"):]
    calls = [m.start() for m in re.finditer(r"mma_16816<", kernel)]
    assert calls and re.search(r"__syncwarp\(\);\s*$", kernel[:calls[0]])
    tiles = re.sub(r"//[^\n]*", "", (CSRC / "dense_mma.cu").read_text())
    # a warp whose first lane does something else before the allocation
    body = tiles[tiles.index("dense_tile_kernel("):]
    alloc = body.index("tcgen05.alloc.")
    assert "threadIdx.x == 32" in body[:alloc] and re.search(r"__syncwarp\(\);\s*asm volatile\(\"$", body[:alloc])
    settle = tiles[tiles.index("void settle()"):]
    assert settle.index("__syncwarp();") < settle.index("\n}\n")
