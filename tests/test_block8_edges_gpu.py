"""Matrices in 8-bit floating point where calls meet and where numbers end."""

import pytest
import torch

from test_block8_gpu import _random
from zephyr_b200.kernels import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 8, 16, 40])
@pytest.mark.parametrize("n,k", [(4096, 1024), (333, 1500), (16, 128)])
def test_a_product_directly_behind_packing(m, n, k):
    """Memory that held other codes and scales is packed into and read by the next kernel, eager and captured: the product is that of the new matrix."""
    x = _random((m, k), 1, dtype=torch.bfloat16)
    raw = [_random((n, k), 2 + i, 2.0 ** (4 * i), torch.bfloat16) for i in range(4)]
    want = []
    for w in raw:
        packed = ops.pack_matrix(w)
        torch.cuda.synchronize()
        want.append(ops.block_linear(x, packed))
        torch.cuda.synchronize()
        del packed
    for i in range(40):                       # (the allocator gives the freed matrix's memory to the next one)
        got = ops.block_linear(x, ops.pack_matrix(raw[i % 4]))
        assert torch.equal(got, want[i % 4])
    graph = torch.cuda.CUDAGraph()
    source = raw[0].clone()
    with ops.capture(graph):
        got = ops.block_linear(x, ops.pack_matrix(source))
    for i in range(8):
        source.copy_(raw[i % 4])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[i % 4])


def test_a_product_directly_behind_copied_codes():
    made = [ops.pack_matrix(_random((256, 512), 6 + i, 2.0 ** (4 * i))) for i in range(3)]
    codes = [m.codes.transpose(2, 3).flatten(3, 4).flatten(1, 2)[0].contiguous() for m in made]
    x = _random((4, 512), 9, dtype=torch.bfloat16)
    want = [ops.block_linear(x, m) for m in made]
    torch.cuda.synchronize()
    for i in range(12):
        assert torch.equal(ops.block_linear(x, ops.BlockMatrix.from_codes(codes[i % 3], made[i % 3].exponents())), want[i % 3])
