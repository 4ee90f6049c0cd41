"""The 4-bit cache without a GPU: its layout, its codes' error bound, and what its entry points refuse."""

import math

import pytest
import torch

import plain_packed as plain
from zephyr_b200.config.errors import InvalidArgumentError
from zephyr_b200.kernels import ops
from zephyr_b200.kernels.ops import KernelError


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_every_byte_of_a_block_has_one_meaning(hd):
    seen = torch.zeros(20 * hd, 8, dtype=torch.int)
    for byte, shift, step, offset in plain.places(hd):
        for bit in range(4):
            seen.index_put_((byte.reshape(-1), shift.reshape(-1) + bit), torch.ones(16 * hd, dtype=torch.int), accumulate=True)
        for at in (step, offset):
            first = torch.unique(at)
            assert first.numel() == 16 * hd // 32
            seen[first] += 1
            seen[first + 1] += 1
    assert torch.equal(seen, torch.ones_like(seen))
    assert ops.packed_block_bytes(hd) == 20 * hd
    assert ops.packed_cache_shape(7, 3, 32, hd) == (7, 3, 2, 20 * hd)


def test_codes_are_within_half_a_step():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((50, 16, 64), generator=g) * torch.logspace(-6, 6, 50).view(50, 1, 1)
    x[3, 4] = 0.0
    x[4, 5] = -7.25
    k, v = plain.values(plain.pack(x, 2 * x))
    codes, step, offset = plain.quantise(x)
    assert ((k - x.double()).abs() <= step / 2).all()
    assert torch.equal(v, 2 * k)
    assert (offset <= x.double()).all() and (x.double() <= offset + 15 * step).all()
    assert torch.equal(k[3, 4], torch.zeros(64, dtype=torch.float64)) and (k[4, 5] == -7.25).all()


def decode_args(**change):
    nh, nkv, hd = 8, 2, 64
    a = dict(q=torch.zeros((2, nh * hd), dtype=torch.bfloat16), packed=torch.zeros(ops.packed_cache_shape(5, nkv, 16, hd), dtype=torch.uint8),
             block_table=torch.ones((2, 3), dtype=torch.int32), rows=torch.arange(2, dtype=torch.int32),
             row_q_start=torch.arange(2, dtype=torch.int32), row_ctx=torch.zeros(2, dtype=torch.int32), max_context=1, nh=nh, nkv=nkv, hd=hd,
             window=0, scale=0.125, status=torch.zeros(4, dtype=torch.int32), out=torch.zeros((2, nh * hd), dtype=torch.bfloat16))
    a.update(change)
    return a


DECODE_REFUSALS = {
    "heads": dict(nh=7), "head size": dict(hd=80), "cache type": dict(packed=torch.zeros((5, 2, 1, 1280), dtype=torch.int8)),
    "cache shape": dict(packed=torch.zeros((5, 2, 1, 1281), dtype=torch.uint8)), "cache heads": dict(packed=torch.zeros((5, 3, 1, 1280), dtype=torch.uint8)),
    "page size": dict(packed=torch.zeros((5, 2, 3, 1280), dtype=torch.uint8)), "queries' type": dict(q=torch.zeros((2, 512)), out=torch.zeros((2, 512))),
    "queries' width": dict(q=torch.zeros((2, 520), dtype=torch.bfloat16)), "result": dict(out=torch.zeros((2, 512))),
    "table's type": dict(block_table=torch.ones((2, 3), dtype=torch.int64)), "table's shape": dict(block_table=torch.ones(6, dtype=torch.int32)),
    "window": dict(window=-1), "chunk": dict(chunk=-1), "softcap": dict(softcap=-1.0), "sinks": dict(sinks=torch.zeros(7)),
    "status": dict(status=torch.zeros(4)), "strided queries": dict(q=torch.zeros((2, 1024), dtype=torch.bfloat16)[:, ::2]),
    "contexts": dict(row_ctx=torch.zeros(1, dtype=torch.int32)),
}


@pytest.mark.parametrize("what", DECODE_REFUSALS)
def test_decode_refuses(what):
    with pytest.raises(InvalidArgumentError):
        ops.paged_decode_packed(**decode_args(**DECODE_REFUSALS[what]))


def prompt_args(**change):
    a = decode_args()
    for name in ("rows", "max_context"):
        del a[name]
    a.update(tile_row=torch.arange(2, dtype=torch.int32), tile_q0=torch.zeros(2, dtype=torch.int32), row_q_len=torch.ones(2, dtype=torch.int32))
    a.update(change)
    return a


PROMPT_REFUSALS = {**{k: v for k, v in DECODE_REFUSALS.items()}, "tiles": dict(tile_q0=torch.zeros(3, dtype=torch.int32)),
                   "lengths": dict(row_q_len=torch.ones(1, dtype=torch.int32)), "lengths' type": dict(row_q_len=torch.ones(2))}


@pytest.mark.parametrize("what", PROMPT_REFUSALS)
def test_prompts_refuse(what):
    with pytest.raises(InvalidArgumentError):
        ops.paged_prefill_packed(**prompt_args(**PROMPT_REFUSALS[what]))


def write_args(**change):
    nh, nkv, hd = 8, 2, 64
    a = dict(qkv=torch.zeros((2, (nh + 2 * nkv) * hd), dtype=torch.bfloat16), nh=nh, nkv=nkv, hd=hd, q_norm_w=torch.ones(hd), k_norm_w=torch.ones(hd),
             eps=1e-6, cos=torch.zeros((9, 32)), sin=torch.zeros((9, 32)), positions=torch.zeros(2, dtype=torch.int32),
             token_row=torch.arange(2, dtype=torch.int32), packed=torch.zeros(ops.packed_cache_shape(5, nkv, 16, hd), dtype=torch.uint8),
             block_table=torch.ones((2, 3), dtype=torch.int32), status=torch.zeros(4, dtype=torch.int32))
    a.update(change)
    return a


WRITE_REFUSALS = {
    "width": dict(qkv=torch.zeros((2, 700), dtype=torch.bfloat16)), "type": dict(qkv=torch.zeros((2, 768), dtype=torch.float16)),
    "stride": dict(qkv=torch.zeros((768, 2), dtype=torch.bfloat16).T), "overlap": dict(qkv=torch.zeros(2000, dtype=torch.bfloat16).as_strided((2, 768), (8, 1))),
    "boundary": dict(qkv=torch.zeros(2000, dtype=torch.bfloat16)[1:1537].view(2, 768)), "float32 queries of bfloat16": dict(dtype=torch.float32),
    "one scale": dict(k_norm_w=None), "scale's size": dict(q_norm_w=torch.ones(63)), "layout": dict(layout="thirds"),
    "one table": dict(sin=None), "tables' sizes": dict(sin=torch.zeros((9, 16))), "too many turned": dict(cos=torch.zeros((9, 33)), sin=torch.zeros((9, 33)), layout="pairs"),
    "halves of 6": dict(cos=torch.zeros((9, 3)), sin=torch.zeros((9, 3))), "bias": dict(bias=torch.zeros(767)),
    "positions": dict(positions=torch.zeros(3, dtype=torch.int32)), "rows": dict(token_row=torch.zeros(2, dtype=torch.int64)),
    "cache": dict(packed=torch.zeros((5, 2, 1, 640), dtype=torch.uint8)), "head size": dict(hd=48),
}


@pytest.mark.parametrize("what", WRITE_REFUSALS)
def test_write_refuses(what):
    with pytest.raises(InvalidArgumentError):
        ops.qk_norm_rope_packed(**write_args(**WRITE_REFUSALS[what]))


def test_unpack_refuses():
    packed, pages = torch.zeros((5, 2, 1, 1280), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(pages=pages.long()), dict(dtype=torch.float16), dict(packed=packed[:, :, 0]), dict(packed=packed.int())):
        with pytest.raises(InvalidArgumentError):
            ops.unpack_pages(**{**dict(packed=packed, pages=pages, dtype=torch.bfloat16), **bad})


def test_sizes_are_refused():
    with pytest.raises(InvalidArgumentError):
        ops.packed_cache_shape(4, 2, 8, 64)
    with pytest.raises(InvalidArgumentError):
        ops.packed_cache_shape(4, 2, 48, 64)
    with pytest.raises(InvalidArgumentError):
        ops.packed_block_bytes(256)


def test_there_is_no_cpu_path():
    with pytest.raises(KernelError):
        ops.paged_decode_packed(**decode_args())
    with pytest.raises(KernelError):
        ops.paged_prefill_packed(**prompt_args())
    with pytest.raises(KernelError):
        ops.qk_norm_rope_packed(**write_args())
    with pytest.raises(KernelError):
        ops.unpack_pages(torch.zeros((5, 2, 1, 1280), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32), torch.bfloat16)
