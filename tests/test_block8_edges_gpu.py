"""Matrices in 8-bit floating point where calls meet and where numbers end."""

import pytest
import torch

import plain_block8 as plain
from test_block8_gpu import F64, HALF_STEP, _close, _feed_forward, _random
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


# ------------------------------------------------------------------------------------------------- the ends of the range
def _coded_matrix(shape, exponents, seed):
    """A matrix of random codes with these bytes for its blocks, and what it stands for in 64 bits (which may be beyond float32)."""
    codes = _random(shape, seed, 100.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    blocks = exponents.repeat_interleave(128, -2)[..., : shape[-2], :].repeat_interleave(128, -1)[..., : shape[-1]]
    return ops.BlockMatrix.from_codes(codes, exponents), codes.to(F64) * torch.exp2(blocks.to(F64) - 127)


def _bytes(shape, value):
    return torch.full((*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128)), value, dtype=torch.uint8, device="cuda")


# Powers of two of a matrix's scales (2^w) and of the rows' values (2^x): at each end, the result an ordinary number, or one close to an end of float32.
ENDS = [(127, -126), (127, -120), (110, -110), (64, -60), (65, -60), (-126, 118), (-126, 60), (-110, 110), (60, 50), (-70, -40)]


@pytest.mark.parametrize("m", [1, 8, 16, 17, 300])
@pytest.mark.parametrize("n,k", [(200, 640), (48, 2300)])
def test_products_where_scales_are_at_the_ends(m, n, k):
    for i, (w_power, x_power) in enumerate(ENDS):
        matrix, values = _coded_matrix((n, k), _bytes((n, k), w_power + 127), 20 + i)
        x = (_random((m, k), 40 + i).double() * 2.0 ** x_power).float()
        want, magnitude = plain.product(x, values)
        assert bool((want.abs() < 2.0 ** 127).all())
        _close(ops.block_linear(x, matrix), want, plain.sum_error(k) * magnitude, torch.float32)
        zero = ops.block_linear(torch.zeros_like(x), matrix)
        assert bool((zero == 0).all())


@pytest.mark.parametrize("m", [2, 16, 40, 300])
def test_feed_forwards_and_experts_where_scales_are_at_the_ends(m):
    width, ff = 384, 264
    # Sums of 2^11 times the powers, hidden values of their square; also hidden values far from one, with matrices that bring them back.
    for i, (up_power, x_power, down_power) in enumerate([(127, -126, -10), (-126, 118, 3), (115, -120, 90), (-126, 102, 127), (127, -82, -126)]):
        shapes = (2 * ff, width), (width, ff)
        (up, up_values), (down, down_values) = (_coded_matrix(s, _bytes(s, p + 127), 60 + 2 * i + j) for j, (s, p) in enumerate(zip(shapes, (up_power, down_power))))
        x = (_random((m, width), 80 + i).double() * 2.0 ** x_power).float()
        want, error = _feed_forward(x, up_values, down_values, "relu")
        assert bool((want.abs() < 2.0 ** 127).all()) and bool((want != 0).any())
        _close(ops.block_feed_forward(x, up, down, act="relu"), want, error, torch.float32)
        experts = 3
        several = [ops.BlockMatrix.from_codes(w.codes.transpose(2, 3).flatten(3, 4).flatten(1, 2)[:, : w.N, : w.K].expand(experts, -1, -1),
                                              w.exponents().expand(experts, -1, -1).contiguous()) for w in (up, down)]
        ids = (torch.arange(m, device="cuda") % experts).int()[:, None].contiguous()
        got = ops.routed_experts(x, ids, torch.ones((m, 1), device="cuda"), several[0], None, several[1], act="relu")
        _close(got, want, error + HALF_STEP[torch.float32] * (want.abs() + error), torch.float32)


# ------------------------------------------------------------------------------------------------- long sums of one sign
def _positive(shape, seed):
    """Numbers that e4m3 holds beside one another in a block: eight fractions at nine sizes, none of them zero or negative."""
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    integers = lambda high: torch.randint(0, high, shape, generator=generator, device="cuda", dtype=torch.int32)
    return (1 + integers(8) / 8) * torch.exp2(-integers(9).float())


def _lost(got, want):
    """How much of itself a sum loses on average: the tensor cores cut what a sum of 24 bits does not hold, always towards zero."""
    return ((want - got.double()) / want).mean().item()


def test_long_sums_to_float32_are_taken_in_two_accumulators():
    """Of K > 8192 values: each half has lost what a sum of half as many terms loses, not twice that.  Sizes whose tiles go to one pair of SMs whole; 1.3
    leaves room for the draws."""
    k, n, m = 9216, 2304, 256
    x, w = _positive((m, k), 1), _positive((n, k), 2)
    half = _lost(ops.block_linear(x[:, : k // 2], ops.pack_matrix(w[:, : k // 2].contiguous()), torch.float32), x[:, : k // 2].double() @ w[:, : k // 2].double().t())
    assert half > 0
    assert _lost(ops.block_linear(x, ops.pack_matrix(w), torch.float32), x.double() @ w.double().t()) < 1.3 * half
    # A feed-forward and experts whose hidden values are exact: gates of a power of two (relu), ups that e4m3 holds.
    for tokens, width, experts in ((256, 2304, 1), (256, 2048, 2), (80, 4352, 2)):
        up, values, down = torch.zeros((experts, 2 * k, 128), device="cuda"), _positive((experts, k), 3), _positive((experts, width, k), 4)
        up.view(experts, -1, 2, 8, 128)[:, :, 0, :, 0] = 1
        up.view(experts, -1, 2, 8, 128)[:, :, 1, :, 0] = values.view(experts, -1, 8)
        x = torch.zeros((tokens, 128), device="cuda")
        x[:, 0] = torch.exp2((torch.arange(tokens, device="cuda") % 5).float())
        ids = torch.arange(tokens, device="cuda") % experts
        if experts == 1:
            got = ops.block_feed_forward(x, ops.pack_matrix(up[0]), ops.pack_matrix(down[0]), act="relu")
        else:           # (the experts' rows are as wide as their outputs)
            wide = torch.zeros((experts, 2 * k, width), device="cuda")
            wide[:, :, :128] = up
            x = torch.nn.functional.pad(x, (0, width - 128))
            got = ops.routed_experts(x, ids.int()[:, None].contiguous(), torch.ones((tokens, 1), device="cuda"), ops.pack_matrix(wide), None, ops.pack_matrix(down), act="relu")
        sums = torch.einsum("ewk,ek->ew", down.double(), values.double())
        assert _lost(got, x[:, :1].double() ** 2 * sums[ids]) < 1.3 * half


# ------------------------------------------------------------------------------------------------- choices that other tests do not make
@pytest.mark.parametrize("tokens,experts,top", [(5, 64, 40), (50, 64, 40), (3, 5, 3), (30, 5, 3)])
@pytest.mark.parametrize("chosen", ["any", "none", "one"])
def test_many_choices_a_token_and_tokens_without_an_expert(tokens, experts, top, chosen):
    """More choices than a warp has lanes; ids outside the experts on either side, which stand for the token itself; no expert at all; all on the last one."""
    width, ff = 136, 72
    x = _random((tokens, width), 70, dtype=torch.bfloat16)
    raw_up, raw_down = _random((experts, 2 * ff, width), 71, 0.1), _random((experts, width, ff), 72, 0.1)
    up, down = ops.pack_matrix(raw_up), ops.pack_matrix(raw_down)
    ids = torch.stack([torch.randperm(experts + 4, generator=torch.Generator().manual_seed(t))[:top] for t in range(tokens)]).cuda() - 2      # from -2 to experts + 1
    if chosen == "none":
        ids = torch.where(ids % 2 == 0, -1, experts + 7)
    elif chosen == "one":
        ids = torch.full_like(ids, experts - 1)
    ids, weights = ids.int().contiguous(), (_random((tokens, top), 73).abs() / top).contiguous()
    got = ops.routed_experts(x, ids, weights, up, None, down)
    want, error = torch.zeros((tokens, width), dtype=F64, device="cuda"), torch.zeros((tokens, width), dtype=F64, device="cuda")
    for e in ids.unique().tolist():
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        weight = weights[token, choice].double()[:, None]
        y, off = x[token].double(), torch.zeros((len(token), width), dtype=F64, device="cuda")
        if 0 <= e < experts:
            y, off = _feed_forward(x[token], plain.code_blocks(raw_up[e], 128)[0], plain.code_blocks(raw_down[e], 128)[0], "silu")
            off = off + HALF_STEP[torch.bfloat16] * (y.abs() + off)
        want.index_add_(0, token, weight * y)
        error.index_add_(0, token, weight * off + (top + 2) * 2.0 ** -24 * (weight * y).abs())
    _close(got, want, error * (1 + 2.0 ** -20) + top * 2.0 ** -24 * want.abs(), torch.bfloat16)
