"""The 4-bit cache's entry points at the edges of what they are asked: no rows, prompts again and again."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from zephyr_b200.kernels import ops
    return ops


def i32(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("max_context", [1, 500, 20000, 1000000])
@pytest.mark.parametrize("plan", [None, (0, 4), (1, 148), (2, 296)])
def test_a_call_without_rows_leaves_everything_as_it_was(ops, cuda_device, max_context, plan):
    nh, nkv, hd = 8, 2, 64
    packed = torch.zeros(ops.packed_cache_shape(3, nkv, 16, hd), dtype=torch.uint8, device=cuda_device)
    q = torch.ones((3, nh * hd), dtype=torch.bfloat16, device=cuda_device)
    out, none, status = torch.full_like(q, 7.0), i32(cuda_device, []), ops.new_status(cuda_device)
    got = ops.paged_decode_packed(q, packed, i32(cuda_device, [[1]]), none, i32(cuda_device, [0]), i32(cuda_device, [0]), max_context, nh, nkv, hd, 0,
                                  0.1, status, out, plan=plan)
    ops.check_status(status)
    assert got is out and (out == 7.0).all()


@pytest.mark.parametrize("nh,nkv,new,cached", [(4, 2, 200, 5000), (32, 8, 1024, 3000), (16, 8, 130, 40), (18, 3, 900, 1000)])
def test_prompts_again_and_again(ops, cuda_device, nh, nkv, new, cached):
    """A head a CTA and pairs of heads, contexts of two to many tiles: every launch ends, with the same result."""
    hd, page, tile = 128, 16, ops.paged_prefill_tile_tokens()
    blocks = -(-(new + cached) // page)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    packed = torch.zeros(ops.packed_cache_shape(blocks + 1, nkv, page, hd), dtype=torch.uint8, device=cuda_device)
    table, status = torch.arange(1, blocks + 1, dtype=torch.int32, device=cuda_device).view(1, -1), ops.new_status(cuda_device)
    total = new + cached
    qkv = torch.randn((total, (1 + 2 * nkv) * hd), generator=g, device=cuda_device).to(torch.bfloat16)
    ops.qk_norm_rope_packed(qkv, 1, nkv, hd, None, None, 1e-6, None, None, torch.arange(total, dtype=torch.int32, device=cuda_device),
                            torch.zeros(total, dtype=torch.int32, device=cuda_device), packed, table, status)
    q = torch.randn((new, nh * hd), generator=g, device=cuda_device).to(torch.bfloat16)
    starts = list(range(0, new, tile))
    rest = (i32(cuda_device, [0] * len(starts)), i32(cuda_device, starts), i32(cuda_device, [0]), i32(cuda_device, [new]), i32(cuda_device, [cached]),
            nh, nkv, hd, 0, hd ** -0.5, status)
    first = ops.paged_prefill_packed(q, packed, table, *rest, torch.empty_like(q))
    outs = [torch.empty_like(q) for _ in range(4)]
    for _ in range(50):
        for out in outs:
            ops.paged_prefill_packed(q, packed, table, *rest, out)
    ops.check_status(status)
    assert torch.isfinite(first).all() and all(torch.equal(out, first) for out in outs)
