"""What is handed from one warp or kernel to another under the products on matrices in 8-bit floating point, read from the sources: which
instruction orders it.  (No GPU.)"""

import re

from zephyr_b200.kernels.build import SOURCE_DIR


def _source(name):
    return re.sub(r"//[^\n]*", "", (SOURCE_DIR / name).read_text())


def _in_order(text, *pieces):
    """The pieces, each behind the one before."""
    at = 0
    for piece in pieces:
        at = text.index(piece, at) + len(piece)
    return True


def test_parts_of_a_sum_are_ordered_by_barriers_of_the_warp():
    """A warp's lanes store a part each, one of them sets the flag; a warp's lanes look at a flag each, all of them read all parts.  Both times lanes
    depend on what other lanes did: a barrier of the warp stands between, ahead of the fence where the flag is set, behind the vote where flags are seen."""
    body = _source("gemm_block8.cu")
    writing = body[body.index("float* part = part_of(pair)"):body.index("atomicExch(flag_of(pair, group), 1)")]
    assert _in_order(writing, "__stcg(", "__syncwarp();", "__threadfence();") and writing.count("__syncwarp();") == writing.count("__threadfence();") == 1
    reading = body[body.index("load_acquire(flag)"):body.index("__ldcg(")]
    assert _in_order(reading, "__all_sync(0xffffffffu, ok)", "break;", "__syncwarp();") and reading.count("__all_sync") == 1
    assert len(re.findall(r"load_acquire\(", body)) == 2                 # the function, and this one wait
