"""The 4-bit cache on the GPU: writing into it, reading it back, and attention over it, against the definition in float64."""

import math
import random

import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu
U = 2.0 ** -8          # the most that a rounding to bfloat16 moves a value, relative to it


@pytest.fixture(scope="module")
def ops():
    from zephyr_b200.kernels import ops
    return ops


def paged_case(device, nkv, hd, page, totals, seed, poison=True):
    """A 4-bit cache with ``totals[r]`` positions of row r, its table, and its keys and values (codes, steps, offsets), row by row.  Positions
    behind a row's last, and unused pages, hold parameters that are NaN."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in totals]
    pages = sum(blocks) + 3
    order = list(range(1, pages))
    random.Random(seed).shuffle(order)
    loud = 1 + 4 * (torch.rand((nkv, 1, 1, hd), generator=g) < 0.06)
    shape = (pages, nkv, page // 16, 16, hd)
    packed = plain.pack(torch.randn(shape, generator=g) * loud, torch.randn(shape, generator=g) * 0.7)
    table = torch.zeros((len(totals), max(1, *blocks) + 1), dtype=torch.int32)
    at = 0
    for r, n in enumerate(blocks):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    rows = []
    for r, n in enumerate(totals):
        own = packed[table[r, :blocks[r]].long()]
        rows.append([[x.permute(0, 2, 3, 1, 4).reshape(-1, nkv, hd)[:n] for x in part] for part in plain.read(own)])
    if poison:
        for r, n in enumerate(totals):
            for pos in range(n, blocks[r] * page):
                block = packed[table[r, pos // page], :, pos % page // 16]
                for _, _, step, offset in plain.places(hd):
                    for where in (step[pos % 16], offset[pos % 16]):
                        block[:, where] = 0xff
                        block[:, where + 1] = 0xff
        packed[0] = 0xff
        for unused in order[at:]:
            packed[unused] = 0xff
    return packed.to(device), table.to(device), rows


def i32(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------- writing
def write_case(device, nh, nkv, hd, page, lengths, cached, seed, dtype, dims, layout, norm, bias, stride=0):
    g = torch.Generator().manual_seed(seed)
    T, width = sum(lengths), (nh + 2 * nkv) * hd
    packed, table, _ = paged_case("cpu", nkv, hd, page, [c + n for n, c in zip(lengths, cached)], seed, poison=False)
    qkv = (torch.randn((T, width + stride), generator=g) * 1.5).to(dtype)
    case = dict(qkv=qkv.to(device)[:, :width], table=table.to(device), packed=packed.to(device), before=packed,
                positions=[c + i for n, c in zip(lengths, cached) for i in range(n)], token_row=[r for r, n in enumerate(lengths) for _ in range(n)])
    x = qkv[:, :width].double()
    case["bias"] = torch.randn(width, generator=g) * 0.3 if bias else None
    if bias:
        x = x + case["bias"].double()
    heads = x.view(T, -1, hd)
    q, k, v = heads[:, :nh], heads[:, nh:nh + nkv], heads[:, nh + nkv:]
    case["norms"] = [1 + 0.2 * torch.randn(hd, generator=g) for _ in range(2)] if norm else [None, None]
    if norm:
        q, k = (h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double() for h, w in zip((q, k), case["norms"]))
    case["cos"] = case["sin"] = None
    if dims:
        angles = torch.arange(max(case["positions"]) + 1)[:, None] * 10000.0 ** (-2.0 * torch.arange(dims // 2).double() / dims)
        case["cos"], case["sin"] = torch.cos(angles).float() * 1.1, torch.sin(angles).float() * 1.1
        at = torch.tensor(case["positions"])
        c, s = case["cos"][at].double()[:, None], case["sin"][at].double()[:, None]
        def turned(h):
            h = h.clone()
            first, second = (slice(0, dims // 2), slice(dims // 2, dims)) if layout == "halves" else (slice(0, dims, 2), slice(1, dims, 2))
            a, b = h[..., first].clone(), h[..., second].clone()
            h[..., first], h[..., second] = a * c - b * s, b * c + a * s
            return h
        q, k = turned(q), turned(k)
    case["expected"] = (q, k, v)
    return case


WRITES = [
    (8, 2, 128, 16, [1], [0], torch.bfloat16, 128, "halves", True, False, 0),
    (4, 4, 64, 32, [1, 1, 1], [15, 16, 31], torch.bfloat16, 64, "halves", True, False, 8),
    (6, 3, 32, 16, [17, 1], [5, 300], torch.bfloat16, 16, "halves", False, True, 0),
    (5, 1, 96, 64, [33], [40], torch.float32, 96, "halves", True, True, 4),
    (3, 3, 96, 16, [7, 2], [9, 0], torch.bfloat16, 40, "pairs", True, False, 0),
    (8, 2, 128, 16, [50], [3], torch.float32, 128, "pairs", True, True, 0),
    (2, 1, 64, 16, [16, 31], [0, 17], torch.float32, 10, "pairs", False, False, 0),
    (16, 8, 128, 32, [64, 1, 9], [31, 7, 4000], torch.bfloat16, 0, "halves", False, False, 0),
    (1, 1, 32, 16, [3], [14], torch.float32, 8, "halves", True, False, 0),
    (20, 2, 128, 16, [65], [0], torch.bfloat16, 64, "halves", True, True, 0),
]


def run_write(ops, device, case, nh, nkv, hd, layout, dtype):
    up = lambda x: None if x is None else x.to(device)
    status = ops.new_status(device)
    q = ops.qk_norm_rope_packed(case["qkv"], nh, nkv, hd, up(case["norms"][0]), up(case["norms"][1]), 1e-6, up(case["cos"]), up(case["sin"]),
                                i32(device, case["positions"]), i32(device, case["token_row"]), case["packed"], case["table"], status,
                                dtype, layout=layout, bias=up(case["bias"]))
    ops.check_status(status)
    return q


@pytest.mark.parametrize("nh,nkv,hd,page,lengths,cached,dtype,dims,layout,norm,bias,stride", WRITES)
def test_writing(ops, cuda_device, nh, nkv, hd, page, lengths, cached, dtype, dims, layout, norm, bias, stride):
    case = write_case(cuda_device, nh, nkv, hd, page, lengths, cached, 7, dtype, dims, layout, norm, bias, stride)
    got_q = run_write(ops, cuda_device, case, nh, nkv, hd, layout, torch.bfloat16).cpu().double().view(-1, nh, hd)
    q, k, v = case["expected"]
    # float32 arithmetic of a few dozen roundings on values of a head, then one rounding to bfloat16.
    slack = 2.0 ** -18 * torch.cat([q, k, v], 1).abs().amax(-1, keepdim=True)
    assert ((got_q - q).abs() <= U * q.abs() + slack[:, :nh]).all()
    after, expected = case["packed"].cpu(), case["before"].clone()
    T = len(case["positions"])
    for t in range(T):
        row, pos = case["token_row"][t], case["positions"][t]
        at = (case["table"][row, pos // page].item(), slice(None), pos % page // 16)
        for kind, new in enumerate((k, v)):
            codes, step, offset = (x[:, pos % 16] for x in plain.read(after[at])[kind])
            x = new[t]
            grouped = x.view(nkv, -1, 32)
            low = grouped.amin(-1, keepdim=True).expand_as(grouped).reshape(nkv, hd)
            high = grouped.amax(-1, keepdim=True).expand_as(grouped).reshape(nkv, hd)
            off = slack[t, nh + kind * nkv:nh + (kind + 1) * nkv]
            # The group's ends as the definition has them, but for float32's error; every value within half a step.
            assert ((offset + step * codes - x).abs() <= step / 2 + 2 * off).all()
            assert (offset <= low + off).all() and (offset >= low - 2 * U * low.abs() - off).all()
            assert (step <= (high - offset) / 15 * (1 + 2 * U) + off).all()
        # Nothing but this position's codes and parameters is written.
        for byte, shift, step_at, offset_at in plain.places(hd):
            p = pos % 16
            whole = torch.zeros(20 * hd, dtype=torch.int)
            whole.index_put_((byte[p],), torch.bitwise_left_shift(torch.tensor(15), shift[p]).int(), accumulate=True)
            for one in (step_at[p], offset_at[p]):
                whole[one] = whole[one + 1] = 255
            mine = whole.to(torch.uint8)
            expected[at] = (expected[at] & ~mine) | (after[at] & mine)
    assert torch.equal(after, expected)


def test_values_get_the_codes_of_the_definition(ops, cuda_device):
    """Values are stored as they come (no norm, no rotation): their codes, steps and offsets are the definition's, ties included."""
    nh, nkv, hd = 2, 4, 128
    case = write_case(cuda_device, nh, nkv, hd, 16, [160], [0], 11, torch.bfloat16, 0, "halves", False, False)
    run_write(ops, cuda_device, case, nh, nkv, hd, "halves", torch.bfloat16)
    for kind in (0, 1):
        got = [x.permute(0, 2, 3, 1, 4).reshape(-1, nkv, hd) for x in plain.read(case["packed"].cpu()[case["table"][0, :10].long().cpu()])[kind]]
        for a, b in zip(got, plain.quantise(case["expected"][1 + kind])):
            assert torch.equal(a.double(), b)


def test_groups_of_one_value_extremes_and_what_is_not_finite(ops, cuda_device):
    nh = nkv = 1
    hd, T = 64, 6
    case = write_case(cuda_device, nh, nkv, hd, 16, [T], [0], 13, torch.float32, 0, "halves", False, False)
    v = case["qkv"][:, 2 * hd:]
    v[0] = 0.0
    v[1, :32], v[1, 32:] = -3.5, 1e-30
    v[2, 5], v[3, 40], v[4, 0] = float("nan"), float("inf"), -float("inf")
    v[5] = torch.linspace(-1.5e38, 1.5e38, hd, device=cuda_device)
    before = v.cpu().double()
    run_write(ops, cuda_device, case, nh, nkv, hd, "halves", torch.float32)
    got = ops.unpack_pages(case["packed"], case["table"][0, :1].contiguous(), torch.float32).cpu().double()[0, 1, 0, :T]
    assert torch.equal(got[0], torch.zeros(hd, dtype=torch.float64)) and (got[1, :32] == -3.5).all()
    assert ((got[1, 32:] - 1e-30).abs() <= U * 1e-30).all()
    for t, bad in ((2, slice(0, 32)), (3, slice(32, 64)), (4, slice(0, 32))):
        good = slice(32, 64) if bad.start == 0 else slice(0, 32)
        assert torch.isnan(got[t, bad]).all() and torch.isfinite(got[t, good]).all()
    assert ((got[5] - before[5]).abs() <= 1.5e38 / 15 * 0.52).all()


def test_queries_alone_and_float32_queries(ops, cuda_device):
    nh, nkv, hd = 6, 2, 64
    case = write_case(cuda_device, nh, nkv, hd, 16, [21], [4], 17, torch.float32, 64, "halves", True, False)
    status = ops.new_status(cuda_device)
    q = ops.qk_norm_rope_packed(case["qkv"], nh, nkv, hd, *(w.to(cuda_device) for w in case["norms"]), 1e-6, case["cos"].to(cuda_device),
                                case["sin"].to(cuda_device), i32(cuda_device, case["positions"]), i32(cuda_device, case["token_row"]), None,
                                case["table"], status, torch.float32)
    ops.check_status(status)
    expected = case["expected"][0]
    assert ((q.cpu().double().view(-1, nh, hd) - expected).abs() <= 2.0 ** -18 * expected.abs().amax(-1, keepdim=True)).all()
    assert torch.equal(case["packed"].cpu(), case["before"])


@pytest.mark.parametrize("fault,code", [("page", 3), ("null page", 3), ("row", 4), ("block", 4), ("position", 2), ("negative", 2)])
def test_writes_outside_are_reported_and_not_made(ops, cuda_device, fault, code):
    nh, nkv, hd = 2, 1, 64
    case = write_case(cuda_device, nh, nkv, hd, 16, [1, 1], [3, 20], 19, torch.bfloat16, 64, "halves", True, False)
    if fault == "page":
        case["table"][1, 1] = 10 ** 6
    elif fault == "null page":
        case["table"][1, 1] = 0
    elif fault == "row":
        case["token_row"][1] = 7
    elif fault == "block":
        case["table"] = case["table"][:, :1].contiguous()
    else:
        case["positions"][1] = 21 if fault == "position" else -1
    with pytest.raises(ops.KernelError, match=ops.STATUS_TEXT[code].split("(")[0]):
        run_write(ops, cuda_device, case, nh, nkv, hd, "halves", torch.bfloat16)


@pytest.mark.parametrize("nkv,hd,page,dtype", [(2, 128, 16, torch.bfloat16), (3, 96, 32, torch.float32), (1, 64, 64, torch.bfloat16), (4, 32, 16, torch.float32)])
def test_pages_read_back(ops, cuda_device, nkv, hd, page, dtype):
    packed, table, _ = paged_case(cuda_device, nkv, hd, page, [page * 5], 23, poison=False)
    pages = i32(cuda_device, [4, 1, 1, 6])
    got = ops.unpack_pages(packed, pages, dtype).cpu()
    k, v = (x.flatten(2, 3) for x in plain.values(packed.cpu()[pages.long().cpu()]))
    expected = torch.stack([k, v], 1)
    assert ((got.double() - expected).abs() <= (U if dtype == torch.bfloat16 else 2.0 ** -24) * expected.abs()).all()
    status = ops.new_status(cuda_device)
    ops.unpack_pages(packed, i32(cuda_device, [1, 10 ** 6]), dtype, status)
    with pytest.raises(ops.KernelError):
        ops.check_status(status)


# ------------------------------------------------------------------------------------ single tokens
DECODES = [
    # nh, nkv, hd, page, contexts before the new token, masks
    (16, 8, 128, 16, [0], {}),
    (16, 8, 128, 16, [15, 16, 31, 32, 33, 300, 1, 63], {}),
    (32, 8, 128, 16, [511, 1000], {}),
    (8, 1, 128, 32, [700], dict(sinks=True)),
    (12, 4, 64, 16, [0, 250, 31, 1023], dict(window=100, sinks=True, softcap=20.0)),
    (5, 5, 96, 64, [129, 64, 3], dict(chunk=50)),
    (20, 2, 128, 16, [77, 400], dict(window=33)),
    (6, 3, 32, 16, [5, 600], dict(softcap=5.0)),
    (64, 4, 64, 32, [90], dict(window=1)),
    (4, 2, 128, 64, [2047], dict(chunk=2048, window=1500)),
]


@pytest.mark.parametrize("plan", [None, (0, 1), (0, 2), (0, 8), (1, 3), (1, 296), (2, 1), (2, 148)])
@pytest.mark.parametrize("nh,nkv,hd,page,ctx,masks", DECODES)
def test_single_tokens(ops, cuda_device, nh, nkv, hd, page, ctx, masks, plan):
    n = len(ctx)
    packed, table, rows = paged_case(cuda_device, nkv, hd, page, [c + 1 for c in ctx], 29)
    g = torch.Generator().manual_seed(31)
    q = (torch.randn((n, nh * hd), generator=g) * 1.5).to(torch.bfloat16)
    masks = dict(masks)
    sinks = torch.randn(nh, generator=g) if masks.pop("sinks", False) else None
    scale, status = 1 / math.sqrt(hd), ops.new_status(cuda_device)
    out = torch.full((n + 2, nh * hd), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    order = torch.randperm(n, generator=g)                     # rows of the step in another order than their tokens
    ops.paged_decode_packed(torch.cat([q, q[:2]] if n > 1 else [q, q, q])[:n + 2].to(cuda_device), packed, table, order.to(torch.int32).to(cuda_device),
                            i32(cuda_device, list(range(n))), i32(cuda_device, ctx), max(ctx) + 1, nh, nkv, hd, masks.get("window", 0), scale,
                            status, out, chunk=masks.get("chunk", 0), softcap=masks.get("softcap", 0.0),
                            sinks=None if sinks is None else sinks.to(cuda_device), plan=plan)
    ops.check_status(status)
    assert torch.isnan(out[n:]).all()                          # rows behind the last stay as they were
    for r in range(n):
        expected, bound = plain.attention(q[r].double().view(1, nh, hd), *rows[r], torch.tensor([ctx[r]]), scale, sinks=sinks, **masks)
        assert ((out[r].cpu().double().view(1, nh, hd) - expected).abs() <= bound).all(), r


def test_many_rows(ops, cuda_device):
    """Rows of one to a few hundred positions, more pairs than a launch has CTAs: shares that begin and end inside pairs."""
    nh, nkv, hd, n = 8, 4, 64, 90
    ctx = [(37 * r * r) % 331 for r in range(n)]
    packed, table, rows = paged_case(cuda_device, nkv, hd, 16, [c + 1 for c in ctx], 37)
    q = (torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(41)) * 1.5).to(torch.bfloat16)
    outs = []
    for plan in (None, (0, 1), (1, 17), (2, 17)):
        status = ops.new_status(cuda_device)
        outs.append(ops.paged_decode_packed(q.to(cuda_device), packed, table, torch.arange(n, dtype=torch.int32, device=cuda_device), i32(cuda_device, list(range(n))),
                                            i32(cuda_device, ctx), max(ctx) + 1, nh, nkv, hd, 0, 0.125, status,
                                            torch.empty((n, nh * hd), dtype=torch.bfloat16, device=cuda_device), plan=plan))
        ops.check_status(status)
    for r in range(n):
        expected, bound = plain.attention(q[r].double().view(1, nh, hd), *rows[r], torch.tensor([ctx[r]]), 0.125)
        for out in outs:
            assert ((out[r].cpu().double().view(1, nh, hd) - expected).abs() <= bound).all(), r


@pytest.mark.parametrize("plan", [(0, 1), (0, 4), (1, 5), (2, 5)])
def test_bad_rows_and_pages_are_reported(ops, cuda_device, plan):
    nh, nkv, hd, ctx = 4, 2, 64, [40, 90]
    packed, table, rows = paged_case(cuda_device, nkv, hd, 16, [c + 1 for c in ctx], 43)
    q = torch.randn((2, nh * hd), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    def call(table, rows, status):
        return ops.paged_decode_packed(q, packed, table, i32(cuda_device, rows), i32(cuda_device, [0, 1]), i32(cuda_device, ctx), 91, nh, nkv, hd, 0, 0.125,
                                       status, torch.zeros_like(q), plan=plan)
    good = call(table, [0, 1], ops.new_status(cuda_device))
    for bad_table, bad_rows, code in ((None, [0, 2], 4), (None, [0, -1], 4), (10 ** 6, [0, 1], 3), (0, [0, 1], 3)):
        status, bad = ops.new_status(cuda_device), table.clone()
        if bad_table is not None:
            bad[1, 2] = bad_table
        got = call(bad, bad_rows, status)
        with pytest.raises(ops.KernelError, match=ops.STATUS_TEXT[code].split("(")[0]):
            ops.check_status(status)
        assert torch.equal(got[0], good[0])


# -------------------------------------------------------------------------------------------- prompts
PROMPTS = [
    # nh, nkv, hd, page, new tokens, cached, masks
    (16, 8, 128, 16, [2], [0], {}),
    (8, 2, 128, 16, [129, 1, 128, 63], [0, 5, 127, 700], {}),
    (8, 4, 128, 32, [300], [1000], {}),
    (6, 2, 128, 64, [200, 17], [64, 0], dict(window=90, sinks=True, softcap=15.0)),
    (4, 4, 128, 16, [260, 50], [33, 250], dict(chunk=100)),
    (4, 2, 128, 16, [200], [5000], {}),                        # a head a CTA, many tiles
    (32, 8, 128, 16, [600, 65], [2000, 3], {}),                # pairs of heads
    (18, 3, 128, 32, [900, 150], [100, 777], dict(window=300, sinks=True, softcap=20.0)),
    (3, 3, 128, 16, [40], [129], dict(window=1)),
    (20, 2, 128, 16, [140], [0], dict(sinks=True)),
    (12, 4, 64, 16, [333, 90, 2], [100, 0, 61], {}),
    (5, 5, 96, 32, [70, 130], [31, 0], dict(chunk=64, sinks=True)),
    (6, 3, 32, 64, [65, 64], [0, 300], dict(window=100, softcap=10.0)),
    (2, 1, 64, 16, [16], [15], dict(window=17)),
]


@pytest.mark.parametrize("tensor_memory", [True, False])
@pytest.mark.parametrize("nh,nkv,hd,page,new,cached,masks", PROMPTS)
def test_prompts(ops, cuda_device, nh, nkv, hd, page, new, cached, masks, tensor_memory):
    if hd != 128 and tensor_memory:
        pytest.skip("this head size has one kernel")
    packed, table, rows = paged_case(cuda_device, nkv, hd, page, [c + n for n, c in zip(new, cached)], 59)
    g = torch.Generator().manual_seed(61)
    T, starts = sum(new), [sum(new[:r]) for r in range(len(new))]
    q = (torch.randn((T, nh * hd), generator=g) * 1.5).to(torch.bfloat16)
    masks = dict(masks)
    sinks = torch.randn(nh, generator=g) if masks.pop("sinks", False) else None
    scale, status = 1 / math.sqrt(hd), ops.new_status(cuda_device)
    tile = ops.paged_prefill_tile_tokens()
    tiles = sorted((cached[r] + q0, r, q0) for r, n in enumerate(new) for q0 in range(0, n, tile))
    out = torch.full((T, nh * hd), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    ops.paged_prefill_packed(q.to(cuda_device), packed, table, i32(cuda_device, [t[1] for t in tiles]), i32(cuda_device, [t[2] for t in tiles]),
                             i32(cuda_device, starts), i32(cuda_device, new), i32(cuda_device, cached), nh, nkv, hd, masks.get("window", 0), scale,
                             status, out, chunk=masks.get("chunk", 0), softcap=masks.get("softcap", 0.0),
                             sinks=None if sinks is None else sinks.to(cuda_device), tensor_memory=tensor_memory)
    ops.check_status(status)
    for r, n in enumerate(new):
        mine = slice(starts[r], starts[r] + n)
        expected, bound = plain.attention(q[mine].double().view(n, nh, hd), *rows[r], cached[r] + torch.arange(n), scale, sinks=sinks, rounded=True, **masks)
        assert ((out[mine].cpu().double().view(n, nh, hd) - expected).abs() <= bound).all(), r


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_that_are_not_positive(ops, cuda_device, hd, scale):
    packed, table, rows = paged_case(cuda_device, 2, hd, 16, [150], 79)
    q = torch.randn((130, 4 * hd), generator=torch.Generator().manual_seed(83)).to(torch.bfloat16)
    status, out, one = ops.new_status(cuda_device), torch.zeros_like(q, device=cuda_device), torch.zeros_like(q, device=cuda_device)
    tile = ops.paged_prefill_tile_tokens()
    starts = list(range(0, 130, tile))
    ops.paged_prefill_packed(q.to(cuda_device), packed, table, i32(cuda_device, [0] * len(starts)), i32(cuda_device, starts), i32(cuda_device, [0]),
                             i32(cuda_device, [130]), i32(cuda_device, [20]), 4, 2, hd, 0, scale, status, out)
    ops.paged_decode_packed(q.to(cuda_device), packed, table, i32(cuda_device, [0]), i32(cuda_device, [129]), i32(cuda_device, [149]), 150, 4, 2,
                            hd, 0, scale, status, one)
    ops.check_status(status)
    for got, some, rounded in ((out, slice(0, 130), True), (one, slice(129, 130), False)):
        n = some.stop - some.start
        expected, bound = plain.attention(q[some].double().view(n, 4, hd), *rows[0], 20 + torch.arange(some.start, some.stop), scale, rounded=rounded)
        assert ((got[some].cpu().double().view(n, 4, hd) - expected).abs() <= bound).all()


@pytest.mark.parametrize("power", [-90, -40, 0, 40, 100])
@pytest.mark.parametrize("hd,tensor_memory", [(64, False), (128, False), (128, True)])
def test_prompts_over_values_of_any_size(ops, cuda_device, hd, tensor_memory, power):
    """Values times a power of two give results times it, but for roundings; keys stay.  Behind the end of the row a position holds what
    would be far out of range."""
    g, nkv, nh, n, context = torch.Generator().manual_seed(73), 2, 4, 200, 441
    keys, values = torch.randn((context + 1, nkv, hd), generator=g), torch.randn((context + 1, nkv, hd), generator=g)
    values[context] = 2.0 ** 20
    qkv = torch.cat([torch.zeros((context + 1, hd)), keys.flatten(1), values.flatten(1) * 2.0 ** power], dim=1).to(cuda_device)
    table, status = torch.arange(1, 29, dtype=torch.int32, device=cuda_device).view(1, -1), ops.new_status(cuda_device)
    packed = torch.zeros(ops.packed_cache_shape(30, nkv, 16, hd), dtype=torch.uint8, device=cuda_device)
    ops.qk_norm_rope_packed(qkv, 1, nkv, hd, None, None, 1e-6, None, None, i32(cuda_device, list(range(context + 1))),
                            torch.zeros(context + 1, dtype=torch.int32, device=cuda_device), packed, table, status)
    held = plain.read(packed[1:29].squeeze(2).cpu())                  # (codes, steps, offsets) [pages, heads, page, hd], of keys and of values
    k, v = ([x.transpose(1, 2).reshape(-1, nkv, hd)[:context] for x in part] for part in held)
    q = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16)
    out, tile = torch.empty_like(q, device=cuda_device), ops.paged_prefill_tile_tokens()
    starts = list(range(0, n, tile))
    ops.paged_prefill_packed(q.to(cuda_device), packed, table, i32(cuda_device, [0] * len(starts)), i32(cuda_device, starts), i32(cuda_device, [0]),
                             i32(cuda_device, [n]), i32(cuda_device, [context - n]), nh, nkv, hd, 0, hd ** -0.5, status, out, tensor_memory=tensor_memory)
    ops.check_status(status)
    expected, bound = plain.attention(q.double().view(n, nh, hd), k, v, context - n + torch.arange(n), hd ** -0.5, rounded=True)
    assert ((out.cpu().double().view(n, nh, hd) - expected).abs() <= bound).all()


@pytest.mark.parametrize("hd,tensor_memory", [(64, False), (128, False), (128, True)])
def test_a_query_that_is_not_finite_spoils_its_own_result_only(ops, cuda_device, hd, tensor_memory):
    packed, table, _ = paged_case(cuda_device, 2, hd, 16, [150, 70], 67)
    q = torch.randn((70, 4 * hd), generator=torch.Generator().manual_seed(71)).to(torch.bfloat16).to(cuda_device)
    status, outs, tile = ops.new_status(cuda_device), [], ops.paged_prefill_tile_tokens()
    assert tile >= 70
    for value in (0.5, float("inf"), float("nan")):
        q[69, hd + 5] = value
        out = torch.zeros_like(q)
        ops.paged_prefill_packed(q, packed, table, i32(cuda_device, [0]), i32(cuda_device, [0]), i32(cuda_device, [0, 0]), i32(cuda_device, [70, 0]),
                                 i32(cuda_device, [80, 0]), 4, 2, hd, 0, hd ** -0.5, status, out, tensor_memory=tensor_memory)
        one = torch.zeros_like(q)
        ops.paged_decode_packed(q, packed, table, i32(cuda_device, [0]), i32(cuda_device, [69, 0]), i32(cuda_device, [149, 69]), 150, 4, 2, hd, 0,
                                hd ** -0.5, status, one)
        outs.append(torch.stack([out, one]).view(2, 70, 4, hd))
    ops.check_status(status)
    for bad in outs[1:]:
        assert not torch.isfinite(bad[:, 69, 1]).any()
        bad[:, 69, 1] = outs[0][:, 69, 1]
        assert torch.equal(bad, outs[0])


@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_report_bad_pages_and_rows(ops, cuda_device, hd):
    nh, nkv, new, cached = 4, 2, [150, 140], [40, 20]
    packed, table, _ = paged_case(cuda_device, nkv, hd, 16, [c + n for n, c in zip(new, cached)], 67)
    q = torch.randn((290, nh * hd), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    def call(table, tile_row, status):
        return ops.paged_prefill_packed(q, packed, table, i32(cuda_device, tile_row), i32(cuda_device, [0, 0, 128, 128]), i32(cuda_device, [0, 150]),
                                        i32(cuda_device, new), i32(cuda_device, cached), nh, nkv, hd, 0, 0.1, status, torch.zeros_like(q))
    good = call(table, [0, 1, 0, 1], ops.new_status(cuda_device))
    for page, tile_row, code in ((10 ** 6, [0, 1, 0, 1], 3), (0, [0, 1, 0, 1], 3), (-5, [0, 1, 0, 1], 3), (None, [0, 1, 0, 9], 4)):
        status, bad = ops.new_status(cuda_device), table.clone()
        if page is not None:
            bad[1, 3] = page
        got = call(bad, tile_row, status)
        with pytest.raises(ops.KernelError, match=ops.STATUS_TEXT[code].split("(")[0]):
            ops.check_status(status)
        assert torch.equal(got[:150], good[:150])


# --------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("plan", [(0, 2), (1, 296), (2, 148)])
def test_captured_and_on_a_side_stream(ops, cuda_device, plan):
    """Two captured graphs, replayed at the same time on two streams, with contexts that change between replays."""
    nh, nkv, hd, n = 16, 8, 128, 40
    ctx = [(53 * r) % 700 for r in range(n)]
    packed, table, _ = paged_case(cuda_device, nkv, hd, 16, [c + 1 for c in ctx], 47)
    status, rows = ops.new_status(cuda_device), torch.arange(n, dtype=torch.int32, device=cuda_device)
    contexts, starts = i32(cuda_device, [0] * n), i32(cuda_device, list(range(n)))
    g = torch.Generator().manual_seed(53)
    qs = [(torch.randn((n, nh * hd), generator=g) * 1.5).to(torch.bfloat16).to(cuda_device) for _ in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    def call(i, out):
        return ops.paged_decode_packed(qs[i], packed, table, rows, starts, contexts, 701, nh, nkv, hd, 0, 0.09, status, out, plan=plan)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with ops.capture(graph):
            call(i, outs[i])
        graphs.append(graph)
    contexts.copy_(i32(cuda_device, ctx))
    want = [call(i, torch.zeros_like(qs[i])) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for stream, graph in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    ops.check_status(status)
