"""What can be said of the kernels by reading their sources, where a run cannot show it: instructions that all
lanes of a warp have to execute together."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aimet_b200", "csrc")


def sources():
    paths = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))
    assert paths
    return {os.path.basename(p): open(p, encoding="utf-8").read() for p in paths}


def test_aligned_cluster_barriers_are_reached_by_whole_warps():
    """One helper holds the aligned cluster barrier and brings the warp's lanes together first; nothing else issues one."""
    found = [(name, m.start()) for name, text in sources().items() for m in re.finditer(r"barrier\.cluster\.arrive", text)]
    assert [name for name, _ in found] == ["common.cuh"]
    text = sources()["common.cuh"]
    body = text[text.rindex("cluster_barrier()", 0, found[0][1]):found[0][1]]
    assert "__syncwarp();" in body


def test_conditional_stores_are_followed_by_a_warp_barrier_before_tensor_memory_is_read():
    """The epilogue of the 4-bit product stores for some lanes only and reads tensor memory, a whole warp's
    instruction, again after that."""
    text = sources()["int4_gemm.cu"]
    stores = [m.end() for m in re.finditer(r"if \(live && c[^;]*;", text)]
    assert len(stores) == 2
    for at in stores:
        assert text[at:].lstrip().startswith("__syncwarp();")
