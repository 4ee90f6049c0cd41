"""What is handed from one warp or kernel to another under the products on matrices in 8-bit floating point, read from the sources: which
instruction orders it.  (No GPU.)"""

import inspect
import re

from zephyr_b200.kernels import ops
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


def test_a_matrix_is_visible_before_a_product_may_start():
    """The products for few rows ask for codes and scales ahead of their wait.  So the kernel that packs a matrix is followed by one that waits for it and
    only then lets dependents start, and codes that are copied are followed by another copy."""
    streamer = _source("gemm_block8_small.cu")
    body = streamer[streamer.index("gemm_block8_small_kernel("):]
    assert body.index("tiled_copy_2d_g2s(") < body.index("wait_for_prior_grids();")          # (else none of this would be needed)
    text = _source("block8.cu")
    ready = text[text.index("void matrix_ready_kernel()"):]
    assert _in_order(ready[:ready.index("}")], "wait_for_prior_grids();", "let_dependents_launch();")
    packing = text[text.index("zb_pack_matrix("):text.index("zb_matrix_values(")]
    assert packing.rindex("pack_matrix_kernel<<<") < packing.index("launch_dependent(matrix_ready_kernel")
    copying = inspect.getsource(ops.BlockMatrix.from_codes)
    assert _in_order(copying, "made.codes.copy_(", "made.scales.copy_(", "made.data[sum(made._total) :] = ")


def test_kernels_that_read_ahead_of_their_wait_follow_one_that_waited():
    """The kernel for many rows asks for its first blocks ahead of its wait too: rows are coded directly ahead of it, or ahead of the product in front of it."""
    calls = _source("block8_calls.cu")
    for name in ("static int product(", "static int feed_forward(", "static int experts("):
        body = calls[calls.index(name):]
        body = body[:body.index("\n}\n")]
        tail = body[body.index("block8_code_rows("):]
        assert "block8_product({" in tail and "block8_product({" not in body[:body.index("block8_code_rows(")]
    rows = _source("block8.cu")
    rows = rows[rows.index("code_rows_kernel(const CodeRowsArgs a)"):]
    assert _in_order(rows[:rows.index("\n}\n")], "wait_for_prior_grids();", "let_dependents_launch();")
