"""The 4-bit cache over keys, queries and values of any size.  Sizes are powers of two, so results are compared after the power has been
taken out again: no bound here has a part that does not shrink with what it bounds."""

import math

import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from zephyr_b200.kernels import ops
    return ops


def i32(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


def held_cache(ops, device, keys, values, page=16):
    """A cache of one row that holds keys and values [positions, kv_heads, hd] (float32), its table, and what it holds as (codes, steps,
    offsets), [positions, kv_heads, hd] each in float64."""
    n, nkv, hd = keys.shape
    blocks = -(-n // page)
    packed = torch.zeros(ops.packed_cache_shape(blocks + 1, nkv, page, hd), dtype=torch.uint8, device=device)
    table, status = torch.arange(1, blocks + 1, dtype=torch.int32, device=device).view(1, -1), ops.new_status(device)
    qkv = torch.cat([torch.zeros((n, hd)), keys.flatten(1), values.flatten(1)], dim=1).to(device)
    ops.qk_norm_rope_packed(qkv, 1, nkv, hd, None, None, 1e-6, None, None, i32(device, list(range(n))), i32(device, [0] * n), packed, table, status)
    ops.check_status(status)
    held = plain.read(packed[1:].cpu())                                # [blocks, heads, page / 16, 16, hd]
    return packed, table, [[x.permute(0, 2, 3, 1, 4).reshape(-1, nkv, hd)[:n].double() for x in part] for part in held]


def times(part, power):
    codes, steps, offsets = part
    return codes, steps * 2.0 ** power, offsets * 2.0 ** power


def decode(ops, device, packed, table, q, n, nh, nkv, hd, scale, plan, **masks):
    status = ops.new_status(device)
    out = ops.paged_decode_packed(q.to(device), packed, table, i32(device, [0]), i32(device, [0]), i32(device, [n - 1]), n, nh, nkv, hd,
                                  masks.pop("window", 0), scale, status, torch.empty_like(q, device=device), plan=plan, **masks)
    ops.check_status(status)
    return out.cpu().double().view(1, nh, hd)


PLANS = [(0, 1), (0, 4), (1, 3), (2, 2)]


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("power", [-100, -70, -45, -25, 25, 50, 66, 100])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (8, 2, 128), (2, 1, 96), (3, 3, 32)])
def test_single_tokens_over_values_of_any_size(ops, cuda_device, nh, nkv, hd, power, plan):
    n, g = 700, torch.Generator().manual_seed(5)
    keys, values = torch.randn((n, nkv, hd), generator=g), torch.randn((n, nkv, hd), generator=g)
    packed, table, (k, v) = held_cache(ops, cuda_device, keys, values * 2.0 ** power)
    q = torch.randn((1, nh * hd), generator=g).to(torch.bfloat16)
    got = decode(ops, cuda_device, packed, table, q, n, nh, nkv, hd, hd ** -0.5, plan) * 2.0 ** -power
    expected, bound = plain.attention(q.double().view(1, nh, hd), k, times(v, -power), torch.tensor([n - 1]), hd ** -0.5)
    assert ((got - expected).abs() <= bound).all()


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("powers", [(0, 40), (40, 0), (-60, 0), (0, -60), (-90, -30, 20, 80), (80, -90), (None, -50, 10), (None, None, 60)])
def test_single_tokens_over_values_of_several_sizes(ops, cuda_device, powers, plan):
    """Runs of positions whose values differ in size (None: zeros), none of which begins where a tile does."""
    nh, nkv, hd, n, g = 6, 2, 64, 900, torch.Generator().manual_seed(7)
    keys, values = torch.randn((n, nkv, hd), generator=g), torch.randn((n, nkv, hd), generator=g)
    run = -(-n // len(powers)) + 5
    for i, power in enumerate(powers):
        values[i * run:(i + 1) * run] *= 0.0 if power is None else 2.0 ** power
    packed, table, (k, v) = held_cache(ops, cuda_device, keys, values)
    q = torch.randn((1, nh * hd), generator=g).to(torch.bfloat16)
    top = max(p for p in powers if p is not None)
    for length in (n, run, run + 1, n - 3):
        got = decode(ops, cuda_device, packed, table, q, length, nh, nkv, hd, hd ** -0.5, plan)
        seen = [p for i, p in enumerate(powers) if i * run < length and p is not None]
        by = max(seen) if seen else top
        expected, bound = plain.attention(q.double().view(1, nh, hd), [x[:length] for x in k], times([x[:length] for x in v], -by),
                                          torch.tensor([length - 1]), hd ** -0.5)
        assert ((got * 2.0 ** -by - expected).abs() <= bound).all(), length


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("power", [30, 100])
def test_single_tokens_do_not_hang_on_values_that_they_do_not_see(ops, cuda_device, power, plan):
    nh, nkv, hd, n, window, g = 4, 2, 64, 400, 77, torch.Generator().manual_seed(11)
    keys, values = torch.randn((n, nkv, hd), generator=g), torch.randn((n, nkv, hd), generator=g)
    loud = values.clone()
    loud[:n - window] *= 2.0 ** power
    q, outs = torch.randn((1, nh * hd), generator=g).to(torch.bfloat16), []
    for one in (values, loud):
        packed, table, _ = held_cache(ops, cuda_device, keys, one)
        outs.append(decode(ops, cuda_device, packed, table, q, n, nh, nkv, hd, hd ** -0.5, plan, window=window))
    assert torch.isfinite(outs[0]).all() and torch.equal(*outs)


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("power", [-90, -16, -12, 10, 40, 90])
def test_single_tokens_over_keys_of_any_size(ops, cuda_device, power, plan):
    """Keys times a power of two under queries divided by it: the same scores."""
    nh, nkv, hd, n, g = 8, 2, 128, 600, torch.Generator().manual_seed(13)
    keys, values = torch.randn((n, nkv, hd), generator=g), torch.randn((n, nkv, hd), generator=g)
    packed, table, (k, v) = held_cache(ops, cuda_device, keys * 2.0 ** power, values)
    q = (torch.randn((1, nh * hd), generator=g) * 2.0 ** -power).to(torch.bfloat16)
    got = decode(ops, cuda_device, packed, table, q, n, nh, nkv, hd, hd ** -0.5, plan)
    expected, bound = plain.attention(q.double().view(1, nh, hd) * 2.0 ** power, times(k, -power), v, torch.tensor([n - 1]), hd ** -0.5)
    assert ((got - expected).abs() <= bound).all()


# -------------------------------------------------------------------------------------------- prompts
def prompt(ops, device, packed, table, q, n, context, nh, nkv, hd, scale, tensor_memory=True, **masks):
    """The last n of ``context`` positions, queries [n, nh * hd]."""
    status, out, tile = ops.new_status(device), torch.empty_like(q, device=device), ops.paged_prefill_tile_tokens()
    starts = list(range(0, n, tile))
    ops.paged_prefill_packed(q.to(device), packed, table, i32(device, [0] * len(starts)), i32(device, starts), i32(device, [0]), i32(device, [n]),
                             i32(device, [context - n]), nh, nkv, hd, masks.pop("window", 0), scale, status, out, tensor_memory=tensor_memory, **masks)
    ops.check_status(status)
    return out.cpu().double().view(n, nh, hd)


KERNELS = [(64, False), (96, False), (128, False), (128, True)]


@pytest.mark.parametrize("nh", [4, 32])                 # (a head a CTA, pairs of heads)
@pytest.mark.parametrize("power", [30, 40, 90, -40])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_earlier_tokens_do_not_hang_on_later_ones_values(ops, cuda_device, hd, tensor_memory, power, nh):
    """From some position on values are of another size: what sees none of them is what it is without them, bit by bit."""
    nkv, n, context, first, g = 2, 300, 420, 333, torch.Generator().manual_seed(17)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    loud = values.clone()
    loud[first:] *= 2.0 ** power
    q, outs = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16), []
    for one in (values, loud):
        packed, table, held = held_cache(ops, cuda_device, keys, one)
        outs.append(prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory))
    before = first - (context - n)
    assert torch.equal(outs[0][:before], outs[1][:before])
    expected, bound = plain.attention(q.double().view(n, nh, hd), held[0], times(held[1], -max(power, 0)), context - n + torch.arange(n), hd ** -0.5, rounded=True)
    assert ((outs[1] * 2.0 ** -max(power, 0) - expected).abs() <= bound)[before:].all()


@pytest.mark.parametrize("power", [40, 90])
@pytest.mark.parametrize("masks", [dict(window=70), dict(chunk=64), dict(chunk=100, window=30)])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_tokens_do_not_hang_on_values_behind_their_window_or_chunk(ops, cuda_device, hd, tensor_memory, masks, power):
    nh, nkv, n, context, last, g = 4, 2, 300, 420, 200, torch.Generator().manual_seed(19)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    loud = values.clone()
    loud[:last] *= 2.0 ** power
    q, outs = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16), []
    for one in (values, loud):
        packed, table, _ = held_cache(ops, cuda_device, keys, one)
        outs.append(prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory, **masks))
    pos = context - n + torch.arange(n)
    seen = torch.zeros_like(pos)
    if masks.get("window"):
        seen = torch.maximum(seen, pos + 1 - masks["window"])
    if masks.get("chunk"):
        seen = torch.maximum(seen, pos // masks["chunk"] * masks["chunk"])
    apart = seen >= last
    assert apart.sum() > 100 and torch.isfinite(outs[1]).all() and torch.equal(outs[0][apart], outs[1][apart])


@pytest.mark.parametrize("power", [-100, -60, -30, 30, 60, 100])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_prompts_over_values_of_other_sizes(ops, cuda_device, hd, tensor_memory, power):
    nh, nkv, n, context, g = 4, 2, 200, 441, torch.Generator().manual_seed(23)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    packed, table, (k, v) = held_cache(ops, cuda_device, keys, values * 2.0 ** power)
    q = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16)
    got = prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory) * 2.0 ** -power
    expected, bound = plain.attention(q.double().view(n, nh, hd), k, times(v, -power), context - n + torch.arange(n), hd ** -0.5, rounded=True)
    assert ((got - expected).abs() <= bound).all()


@pytest.mark.parametrize("nh", [4, 32])
@pytest.mark.parametrize("power", [-90, -40, -16, -12, -5, 10, 12, 16, 24, 40, 90])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS + [(32, False)])
def test_prompts_over_keys_of_any_size(ops, cuda_device, hd, tensor_memory, power, nh):
    """Keys times a power of two under queries divided by it: the same scores."""
    nkv, n, context, g = 2, 140, 333, torch.Generator().manual_seed(29)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    packed, table, (k, v) = held_cache(ops, cuda_device, keys * 2.0 ** power, values)
    q = (torch.randn((n, nh * hd), generator=g) * 2.0 ** -power).to(torch.bfloat16)
    for masks in ({}, dict(window=90), dict(chunk=100, softcap=9.0)):
        got = prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory, **masks)
        expected, bound = plain.attention(q.double().view(n, nh, hd) * 2.0 ** power, times(k, -power), v, context - n + torch.arange(n), hd ** -0.5,
                                          rounded=True, **masks)
        assert ((got - expected).abs() <= bound).all(), masks


@pytest.mark.parametrize("scale", [0.125, -0.1])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_prompts_over_positions_and_rows_of_several_sizes(ops, cuda_device, hd, tensor_memory, scale):
    """Keys of one head far above one with queries far below, the other way round for the next; among the first's positions some whose
    keys are 2^-30 of the others', and some that are zero."""
    nh, nkv, n, context, g = 6, 3, 200, 300, torch.Generator().manual_seed(31)
    size = torch.tensor([2.0 ** 35, 1.0, 2.0 ** -28]).view(1, 3, 1)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    keys[5::7, 0] *= 2.0 ** -30
    keys[3::11] = 0.0
    packed, table, (k, v) = held_cache(ops, cuda_device, keys * size, values)
    q = (torch.randn((n, nkv, nh // nkv, hd), generator=g) / size.view(1, 3, 1, 1)).to(torch.bfloat16)
    got = prompt(ops, cuda_device, packed, table, q.view(n, -1), n, context, nh, nkv, hd, scale, tensor_memory)
    unit = (k[0], k[1] / size.double(), k[2] / size.double())
    expected, bound = plain.attention((q.double() * size.double().view(1, 3, 1, 1)).view(n, nh, hd), unit, v, context - n + torch.arange(n), scale, rounded=True)
    assert ((got - expected).abs() <= bound).all()


@pytest.mark.parametrize("nh", [4, 32])
@pytest.mark.parametrize("power", [-40, 13, 20, 50, 90])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_earlier_tokens_do_not_hang_on_later_ones_keys(ops, cuda_device, hd, tensor_memory, power, nh):
    nkv, n, context, first, g = 2, 300, 420, 333, torch.Generator().manual_seed(37)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    loud = keys.clone()
    loud[first:] *= 2.0 ** power
    q, outs = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16), []
    q[first - (context - n) + 5:] *= 2.0 ** power                     # (and rows of queries of that size)
    for one in (keys, loud):
        packed, table, _ = held_cache(ops, cuda_device, one, values)
        outs.append(prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory))
    before = first - (context - n)
    assert torch.isfinite(outs[0][:before]).all() and torch.equal(outs[0][:before], outs[1][:before])


@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_keys_that_are_not_finite_spoil_what_sees_them(ops, cuda_device, hd, tensor_memory):
    """... and keys far out of the usual range beside them do not hide it."""
    nh, nkv, n, context, first, g = 4, 2, 150, 200, 120, torch.Generator().manual_seed(41)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    keys[first - 3] *= 2.0 ** -40
    keys[first, 0, 7] = math.nan
    q = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16)
    packed, table, _ = held_cache(ops, cuda_device, keys, values)
    got = prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory)
    spoiled = torch.zeros((n, nh), dtype=torch.bool)
    spoiled[first - (context - n):, :2] = True
    assert torch.equal(torch.isnan(got).all(-1), spoiled) and torch.equal(torch.isfinite(got).all(-1), ~spoiled)


@pytest.mark.parametrize("powers", [(0, 40), (40, 0), (-60, 0, -20), (0, -60), (-90, -30, 20, 80), (80, -90, 0), (None, -50, 10), (None, None, 60)])
@pytest.mark.parametrize("masks", [{}, dict(window=120), dict(chunk=200, softcap=7.0, sinks=True), dict(sinks=True)])
@pytest.mark.parametrize("hd,tensor_memory", KERNELS)
def test_prompts_over_values_of_several_sizes(ops, cuda_device, hd, tensor_memory, masks, powers):
    """Runs of positions whose values differ in size (None: zeros), none of which begins where a tile does; keys of other sizes among them.
    Every row is held against the largest that it sees."""
    nh, nkv, n, context, g = 6, 2, 300, 420, torch.Generator().manual_seed(43)
    keys, values = torch.randn((context, nkv, hd), generator=g), torch.randn((context, nkv, hd), generator=g)
    keys[3::17] *= 2.0 ** -30
    run = -(-context // len(powers)) + 5
    size = torch.full((context,), -1000)
    for i, power in enumerate(powers):
        values[i * run:(i + 1) * run] *= 0.0 if power is None else 2.0 ** power
        size[i * run:(i + 1) * run] = -1000 if power is None else power
    masks = dict(masks)
    sinks = torch.randn(nh, generator=g) if masks.pop("sinks", False) else None
    packed, table, (k, v) = held_cache(ops, cuda_device, keys, values)
    q = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16)
    got = prompt(ops, cuda_device, packed, table, q, n, context, nh, nkv, hd, hd ** -0.5, tensor_memory, **masks,
                 sinks=None if sinks is None else sinks.to(cuda_device))
    pos = context - n + torch.arange(n)
    lowest = torch.zeros_like(pos)
    if masks.get("window"):
        lowest = torch.maximum(lowest, pos + 1 - masks["window"])
    if masks.get("chunk"):
        lowest = torch.maximum(lowest, pos // masks["chunk"] * masks["chunk"])
    most = torch.stack([size[lo:p + 1].max() for lo, p in zip(lowest.tolist(), pos.tolist())])
    for power in most.unique().tolist():
        rows, by = most == power, 0 if power == -1000 else power
        expected, bound = plain.attention(q[rows].double().view(-1, nh, hd), k, times(v, -by), pos[rows], hd ** -0.5, sinks=sinks, rounded=True, **masks)
        # (What no row of these sees may be far out of range on their scale.)
        assert ((got[rows] * 2.0 ** -by - expected).abs() <= bound).all(), power


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("power", [-90, 0, 90])
def test_single_tokens_over_values_some_of_which_are_not_finite(ops, cuda_device, power, plan):
    """A group that is not finite spoils its own channels; the others hold whatever their size is."""
    nh, nkv, hd, n, g = 4, 2, 64, 200, torch.Generator().manual_seed(47)
    keys, values = torch.randn((n, nkv, hd), generator=g), torch.randn((n, nkv, hd), generator=g) * 2.0 ** power
    values[0, 0, 3], values[77, 1, 40] = math.nan, math.inf
    packed, table, (k, v) = held_cache(ops, cuda_device, keys, values)
    q = torch.randn((1, nh * hd), generator=g).to(torch.bfloat16)
    got = decode(ops, cuda_device, packed, table, q, n, nh, nkv, hd, hd ** -0.5, plan) * 2.0 ** -power
    spoiled = torch.zeros((1, nh, hd), dtype=torch.bool)
    spoiled[:, :2, :32] = spoiled[:, 2:, 32:] = True
    assert torch.equal(torch.isnan(got), spoiled)
    finite = [torch.where(torch.isnan(x), torch.zeros_like(x), x) for x in times(v, -power)]
    expected, bound = plain.attention(q.double().view(1, nh, hd), k, finite, torch.tensor([n - 1]), hd ** -0.5)
    assert ((got - expected).abs() <= bound)[~spoiled].all()
