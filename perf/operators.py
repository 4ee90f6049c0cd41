"""A paged cache whose keys and values are held in 4 bits: writing a step's new tokens into it (per-head norm and position
rotation on the way), and the attention that reads it, for single tokens and for prompts.

``run`` makes the calls that a program makes of ``zephyr_b200.kernels.ops`` (``own``), or computes the same in elementary torch
operations in 32 bits; ``exact`` is the definition in 64 bits.

The cache is a uint8 tensor [pages, kv_heads, page_size / 16, 20 * head_dim].  A block of 16 positions of one head holds, with
NG = head_dim / 32 groups of 32 channels:

* 8 head_dim bytes, keys: a position's row is words (t, j), t < 4, j < NG; nibble i of the word is channel 32 j + 8 t + i;
* 2 head_dim bytes: a position's NG steps and NG offsets of its key, bfloat16;
* 8 head_dim bytes, values: words (h, g, t, m), h < 2, g < 8, t < 4, m < NG; nibble e of the word's half u is channel
  32 m + 4 g + e of position 8 h + 2 t + u;
* 2 head_dim bytes: for a pair of positions NG pairs of steps, then NG pairs of offsets of their values.

A value stands for offset + step * code.  Of a group of 32 values the offset is the least one rounded down to bfloat16, the step is
(largest - offset) / 15 rounded up to bfloat16, the code is the quotient (value - offset) / step rounded to the nearest whole
number, ties to even, between 0 and 15 (0 where the step is 0).
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
TILE_TOKENS = 128           # new tokens of one request per entry of a prompt's tile list
EPS = 1e-6


# ------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # Single tokens.  One user's chat turn on the small model (16 / 8 heads): latency counts.
        dict(name="decode one", what="decode", rows=1, context=300, uneven=0, nh=16, nkv=8, hd=128, page=16),
        # The benchmark's batch at the 8B heads: eight requests of 4096 positions.
        dict(name="decode eight", what="decode", rows=8, context=4096, uneven=0, nh=32, nkv=8, hd=128, page=16),
        # A full server: 48 requests of unequal lengths at the 32B heads, larger pages.
        dict(name="decode uneven", what="decode", rows=48, context=6001, uneven=1, nh=64, nkv=8, hd=128, page=32),
        # One document of 120 thousand positions.
        dict(name="decode long", what="decode", rows=1, context=120001, uneven=0, nh=32, nkv=8, hd=128, page=16),
        # A windowed layer with sinks and a bound on its scores, heads of 64, few requests.
        dict(name="decode window", what="decode", rows=5, context=5000, uneven=1, nh=12, nkv=4, hd=64, page=16, window=1024, sinks=1,
             softcap=30.0),
        # Prompts.  Three requests' new prompts of odd lengths in one step.
        dict(name="prompt ragged", what="prompt", lengths="1531,500,17", cached="0,0,0", nh=32, nkv=8, hd=128, page=16),
        # The last portion of a long prompt.
        dict(name="prompt portion", what="prompt", lengths="1024", cached="7000", nh=32, nkv=8, hd=128, page=16),
        # A chunked mask with sinks on heads of 64, a question behind a cached context and a fresh one.
        dict(name="prompt chunked", what="prompt", lengths="333,90", cached="1200,0", nh=12, nkv=4, hd=64, page=32, chunk=512, sinks=1),
        # New tokens into the cache.  One token each of eight requests at the 8B heads.
        dict(name="append step", what="append", lengths="1*8", cached="4095,4080,300,17,0,1000,2047,3333", nh=32, nkv=8, hd=128, page=16,
             layout="halves", dims=128, norm=1, bias=0, qkv="bfloat16"),
        # A prompt step of 2048 tokens from three requests.
        dict(name="append prompt", what="append", lengths="1531,500,17", cached="0,37,900", nh=32, nkv=8, hd=128, page=16,
             layout="halves", dims=128, norm=1, bias=0, qkv="bfloat16"),
        # Rotation of adjacent pairs on part of a head, scaled for a long context, biases, a projection in 32 bits.
        dict(name="append pairs", what="append", lengths="650,1,49", cached="3,20000,11", nh=12, nkv=4, hd=64, page=32,
             layout="pairs", dims=32, norm=1, bias=1, qkv="float32"),
    ]


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((16, 8), (32, 8), (64, 8), (12, 4), (8, 1), (6, 3), (20, 2), (5, 5))


def draw(rng) -> dict:
    nh, nkv = rng.choice(HEADS)
    hd = rng.choice((128, 128, 128, 64, 96, 32))
    case = dict(nh=nh, nkv=nkv, hd=hd, page=rng.choice((16, 16, 32, 64)))
    kind = rng.random()
    if kind < 0.45:
        case.update(what="decode", rows=_spread(rng, 1, 64), uneven=rng.randint(0, 1))
        case["context"] = _spread(rng, 1, max(2, min(100000, 140000 // case["rows"])))
    elif kind < 0.75:
        rows = rng.randint(1, 4)
        lengths = [_spread(rng, 2, 1000 // rows) for _ in range(rows)]
        cached = [rng.choice((0, 0, _spread(rng, 1, 3000 // rows))) for _ in range(rows)]
        case.update(what="prompt", lengths=",".join(map(str, lengths)), cached=",".join(map(str, cached)))
    else:
        rows = rng.randint(1, 5)
        lengths = [rng.choice((1, _spread(rng, 2, 2000 // rows))) for _ in range(rows)]
        case.update(what="append", lengths=",".join(map(str, lengths)),
                    cached=",".join(str(rng.choice((0, _spread(rng, 1, 30000)))) for _ in range(rows)),
                    layout=rng.choice(("halves", "pairs")), norm=rng.randint(0, 1), bias=rng.randint(0, 1),
                    qkv=rng.choice(("bfloat16", "float32")))
        case["dims"] = hd if rng.random() < 0.6 else 8 * rng.randint(1, hd // 8)
        return case
    mask = rng.random()
    if mask < 0.2:
        case["window"] = _spread(rng, 1, 4096)
    elif mask < 0.35:
        case["chunk"] = _spread(rng, 16, 8192)
    if rng.random() < 0.3:
        case["sinks"] = 1
    if rng.random() < 0.2:
        case["softcap"] = 30.0
    return case


def _numbers(text: str) -> list[int]:
    out = []
    for part in text.split(","):
        one, _, times = part.partition("*")
        out += [int(one)] * int(times or 1)
    return out


def lengths_of(case: dict) -> tuple[list[int], list[int]]:
    """New tokens of every row, and the positions cached before them."""
    if case["what"] != "decode":
        return _numbers(case["lengths"]), _numbers(case["cached"])
    rows, most = case["rows"], case["context"]
    total = [max(1, int(most * ((0.3 + 0.6180339887498949 * r) % 1.0))) if case["uneven"] and r else most for r in range(rows)]
    return [1] * rows, [n - 1 for n in total]


def _first_seen(case: dict, pos: int) -> int:
    first = max(0, pos + 1 - case["window"]) if case.get("window") else 0
    return max(first, pos // case["chunk"] * case["chunk"]) if case.get("chunk") else first


def work(case: dict) -> dict:
    lengths, cached = lengths_of(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    position = nkv * hd * 2 * 5 // 8                  # 4 bits a value and 32 bits for 32 values, keys and values
    tokens = sum(lengths)
    if case["what"] == "append":
        width = (nh + 2 * nkv) * hd
        return {"bytes": tokens * (width * (4 if case["qkv"] == "float32" else 2) + nh * hd * 2 + position), "flops": 8 * tokens * width}
    if case["what"] == "decode":
        seen = sum(c + 1 - _first_seen(case, c) for c in cached)
        read = seen
    else:
        read = sum(c + n - _first_seen(case, c) for n, c in zip(lengths, cached))
        seen = sum(p + 1 - _first_seen(case, p) for n, c in zip(lengths, cached) for p in range(c, c + n))
    return {"bytes": read * position + 4 * tokens * nh * hd, "flops": 4 * seen * nh * hd}


# ------------------------------------------------------------------------------- the cache in elementary operations
def _bf16_down(x: torch.Tensor) -> torch.Tensor:
    """float32 values rounded down to bfloat16 ones."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    more = (bits != cut) & (bits < 0)
    return (cut + more.int() * 65536).view(torch.float32)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes, steps and offsets (float32) of the groups of 32 along the last dimension."""
    x = x.to(F32).unflatten(-1, (-1, 32))
    offset = _bf16_down(x.amin(-1).contiguous()).unsqueeze(-1)
    # (A division by a number would be a product with its rounded reciprocal, which is not on the border where the quotient is.)
    step = -_bf16_down(-((x.amax(-1, keepdim=True) - offset) / torch.full_like(offset, 15.0)))
    codes = torch.where(step > 0, torch.round((x - offset) / step), 0).clamp(0, 15)
    return codes, step.squeeze(-1), offset.squeeze(-1)


def _nibbles(codes: torch.Tensor) -> torch.Tensor:
    codes = codes.to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).flatten(1)


def _pack(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Keys and values [blocks, 16, head_dim] as blocks [blocks, 20 * head_dim]."""
    n, hd = k.shape[0], k.shape[2]
    ng = hd // 32
    kc, ks, ko = _quantise(k)
    vc, vs, vo = _quantise(v)
    k_words = kc.view(n, 16, ng, 4, 8).transpose(2, 3)
    v_words = vc.view(n, 2, 4, 2, ng, 8, 4).permute(0, 1, 5, 2, 4, 3, 6)
    k_params = torch.cat([ks, ko], dim=-1)
    v_params = torch.cat([p.view(n, 8, 2, ng).transpose(2, 3) for p in (vs, vo)], dim=2)
    as_bytes = [p.to(torch.bfloat16).contiguous().view(torch.uint8).view(n, -1) for p in (k_params, v_params)]
    return torch.cat([_nibbles(k_words), as_bytes[0], _nibbles(v_words), as_bytes[1]], dim=1)


def _codes(data: torch.Tensor) -> torch.Tensor:
    return torch.stack([data & 15, data >> 4], dim=-1).flatten(-2).to(F32)


def _unpack(blocks: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Blocks [n, 20 * head_dim] as float32 keys and values [n, 16, head_dim]."""
    n, hd = blocks.shape[0], blocks.shape[1] // 20
    ng = hd // 32
    k_words, k_params, v_words, v_params = blocks.split([8 * hd, 2 * hd, 8 * hd, 2 * hd], dim=1)
    kc = _codes(k_words).view(n, 16, 4, ng, 8).transpose(2, 3).reshape(n, 16, ng, 32)
    vc = _codes(v_words).view(n, 2, 8, 4, ng, 2, 4).permute(0, 1, 3, 5, 4, 2, 6).reshape(n, 16, ng, 32)
    k_params = k_params.contiguous().view(torch.bfloat16).to(F32).view(n, 16, 2, ng, 1)
    v_params = v_params.contiguous().view(torch.bfloat16).to(F32).view(n, 8, 2, ng, 2).permute(0, 1, 4, 2, 3).reshape(n, 16, 2, ng, 1)
    return (torch.addcmul(k_params[:, :, 1], kc, k_params[:, :, 0]).view(n, 16, hd),
            torch.addcmul(v_params[:, :, 1], vc, v_params[:, :, 0]).view(n, 16, hd))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(case: dict, seed: int):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + sum(map(ord, repr(sorted(case.items())))))


def _int(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case: dict, g) -> tuple[torch.Tensor, int]:
    """Every request's pages, scattered over the pool as they are after some serving, and the pool's size."""
    lengths, cached = lengths_of(case)
    need = [-(-(c + n) // case["page"]) for n, c in zip(lengths, cached)]
    first = [0] + torch.tensor(need).cumsum(0).tolist()
    order = 1 + torch.randperm(first[-1] + 3, generator=g, device="cuda")
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    for r, blocks in enumerate(need):
        table[r, :blocks] = order[first[r]:first[r] + blocks]
    return table, first[-1] + 4


def _pool(case: dict, pages: int, g) -> torch.Tensor:
    """A cache in use: some channels of the keys are much larger than the others, as trained models have them."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    loud = 1 + 4 * (torch.rand((nkv, 1, 1, hd), generator=g, device="cuda") < 0.05)
    parts = []
    for at in range(0, pages, 1024):
        shape = (min(1024, pages - at), nkv, page // 16, 16, hd)
        k = torch.randn(shape, generator=g, device="cuda") * loud
        v = torch.randn(shape, generator=g, device="cuda") * 0.7
        parts.append(_pack(k.view(-1, 16, hd), v.view(-1, 16, hd)).view(*shape[:3], 20 * hd))
    return torch.cat(parts)


def _angles(case: dict, positions: int) -> torch.Tensor:
    """Angles of a rotation whose slow frequencies are stretched four times over, float64 [positions, dims / 2]."""
    index = torch.arange(case["dims"] // 2, dtype=F64, device="cuda")
    freqs = 500000.0 ** (-2.0 * index / case["dims"])
    freqs = torch.where(freqs < 2 * math.pi / 8192, freqs / 4, freqs)
    return torch.arange(positions, dtype=F64, device="cuda")[:, None] * freqs


def prepare(case: dict, seed: int) -> dict:
    g = _gen(case, seed)
    lengths, cached = lengths_of(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    tokens = sum(lengths)
    table, pages = _table(case, g)
    starts = [0] + torch.tensor(lengths).cumsum(0).tolist()
    state = dict(case=case, table=table, packed=_pool(case, pages, g), row_q_start=_int(starts[:-1]), row_q_len=_int(lengths),
                 row_ctx=_int(cached), scale=1.0 / math.sqrt(hd), max_context=max(c + n for n, c in zip(lengths, cached)))
    state["positions"] = _int([c + i for n, c in zip(lengths, cached) for i in range(n)])
    state["token_row"] = _int([r for r, n in enumerate(lengths) for _ in range(n)])
    if case["what"] == "append":
        width = (nh + 2 * nkv) * hd
        state["qkv"] = torch.randn((tokens, width), generator=g, device="cuda").mul_(1.5).to(TYPES[case["qkv"]])
        if case["norm"]:
            state["norms"] = [1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
        if case["bias"]:
            state["bias"] = 0.3 * torch.randn(width, generator=g, device="cuda")
        angles = _angles(case, state["max_context"])
        state["cos"], state["sin"] = torch.cos(angles).to(F32), torch.sin(angles).to(F32)
        # The pages that get new tokens, and where in them every token goes.
        at = [(r, p // case["page"]) for r, (n, c) in enumerate(zip(lengths, cached)) for p in range(c, c + n)]
        written = list(dict.fromkeys(at))
        state["pages"] = torch.stack([table[r, b] for r, b in written])
        number = {one: i for i, one in enumerate(written)}
        state["page_of_token"] = torch.tensor([number[one] for one in at], device="cuda")
        return state
    state["q"] = torch.randn((tokens, nh * hd), generator=g, device="cuda").mul_(1.5).to(torch.bfloat16)
    state["sinks"] = torch.randn(nh, generator=g, device="cuda") if case.get("sinks") else None
    state["out"] = torch.empty_like(state["q"])
    state["rows"] = _int(list(range(len(lengths))))
    # A prompt's tiles, those with the fewest visible keys first.
    tiles = sorted((cached[r] + q0, r, q0) for r, n in enumerate(lengths) for q0 in range(0, n, TILE_TOKENS))
    state["tile_row"], state["tile_q0"] = _int([t[1] for t in tiles]), _int([t[2] for t in tiles])
    # Every row's tokens in a rectangle, and back.
    most = max(lengths)
    place = torch.arange(most, device="cuda")
    state["token_at"] = (state["row_q_start"][:, None] + place.clamp(max=most - 1)).clamp(max=tokens - 1).long()
    state["place_of_token"] = (state["positions"] - state["row_ctx"][state["token_row"].long()]).long()
    return state


# ------------------------------------------------------------------------------------------- one pass
def run(state: dict):
    what = state["case"]["what"]
    if own:
        return {"decode": _own_decode, "prompt": _own_prompt, "append": _own_append}[what](state)
    return _plain_append(state) if what == "append" else _plain_attention(state)


def _own_decode(s: dict):
    from zephyr_b200.kernels import ops

    case = s["case"]
    return ops.paged_decode_packed(s["q"], s["packed"], s["table"], s["rows"], s["row_q_start"], s["row_ctx"], s["max_context"],
                                   case["nh"], case["nkv"], case["hd"], case.get("window", 0), s["scale"],
                                   ops.device_status(s["q"].device), s["out"], chunk=case.get("chunk", 0), sinks=s["sinks"],
                                   softcap=case.get("softcap", 0.0))


def _own_prompt(s: dict):
    from zephyr_b200.kernels import ops

    case = s["case"]
    return ops.paged_prefill_packed(s["q"], s["packed"], s["table"], s["tile_row"], s["tile_q0"], s["row_q_start"], s["row_q_len"],
                                    s["row_ctx"], case["nh"], case["nkv"], case["hd"], case.get("window", 0), s["scale"],
                                    ops.device_status(s["q"].device), s["out"], chunk=case.get("chunk", 0), sinks=s["sinks"],
                                    softcap=case.get("softcap", 0.0))


def _own_append(s: dict):
    from zephyr_b200.kernels import ops

    case = s["case"]
    q_norm, k_norm = s.get("norms", (None, None))
    q = ops.qk_norm_rope_packed(s["qkv"], case["nh"], case["nkv"], case["hd"], q_norm, k_norm, EPS, s["cos"], s["sin"], s["positions"],
                                s["token_row"], s["packed"], s["table"], ops.device_status(s["qkv"].device), torch.bfloat16,
                                layout=case["layout"], bias=s.get("bias"))
    # What the written pages now stand for: [pages, keys and values, kv_heads, page_size, head_dim].
    return q, ops.unpack_pages(s["packed"], s["pages"], torch.bfloat16)


def _plain_attention(s: dict):
    case = s["case"]
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    rows, most = s["token_at"].shape
    # Every row's keys and values behind one another: [rows, kv_heads, positions, head_dim].
    blocks = s["packed"][s["table"].long()].transpose(1, 2)
    k, v = (x.view(rows, nkv, -1, hd) for x in _unpack(blocks.reshape(-1, 20 * hd)))
    q = s["q"].to(F32)[s["token_at"]].view(rows, most, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(rows, nkv, -1, hd)
    scores = (q @ k.transpose(-1, -2) * s["scale"]).view(rows, nh, most, -1)
    if case.get("softcap"):
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    pos = (s["row_ctx"][:, None] + torch.arange(most, device="cuda"))[:, None, :, None]
    key = torch.arange(scores.shape[-1], device="cuda")
    seen = key <= pos
    if case.get("window"):
        seen = seen & (key > pos - case["window"])
    if case.get("chunk"):
        seen = seen & (key // case["chunk"] == pos // case["chunk"])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].view(1, nh, 1, 1))
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].view(1, nh, 1, 1) - top)
    out = ((weights / total).view(rows, nkv, -1, scores.shape[-1]) @ v).view(rows, nh, most, hd).transpose(1, 2)
    return out[s["token_row"].long(), s["place_of_token"]].reshape(-1, nh * hd).to(torch.bfloat16)


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layout: str) -> torch.Tensor:
    """x [T, heads, head_dim], the first 2 * cos.shape[1] channels turned."""
    half = cos.shape[1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., :half], turned[..., half:]) if layout == "halves" else (turned[..., 0::2], turned[..., 1::2])
    a, b = a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]
    turned = torch.cat([a, b], dim=-1) if layout == "halves" else torch.stack([a, b], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _plain_append(s: dict):
    case = s["case"]
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    x = s["qkv"].to(F32)
    if "bias" in s:
        x = x + s["bias"]
    q, k, v = x.view(x.shape[0], -1, hd).split([nh, nkv, nkv], dim=1)
    if "norms" in s:
        q, k = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w for h, w in zip((q, k), s["norms"]))
    at = s["positions"].long()
    q, k = (_rotated(h, s["cos"][at], s["sin"][at], case["layout"]) for h in (q, k))
    stored = []
    for new in (k, v):
        codes, step, offset = _quantise(new)
        stored.append(torch.addcmul(offset.unsqueeze(-1), codes, step.unsqueeze(-1)).flatten(-2))
    old = _unpack(s["packed"][s["pages"].long()].view(-1, 20 * hd))
    pages = torch.stack([x.reshape(-1, nkv, page, hd) for x in old], dim=1)
    pages[s["page_of_token"], :, :, at % page] = torch.stack(stored, dim=1)
    return q.reshape(-1, nh * hd).to(torch.bfloat16), pages.to(torch.bfloat16)


# ------------------------------------------------------------------------------------- the definition in 64 bits
def _places(hd: int) -> list[torch.Tensor]:
    """For keys and for values [16, hd]: a code's byte, its shift, and the bytes of its step and offset."""
    ng = hd // 32
    p, d = torch.meshgrid(torch.arange(16, device="cuda"), torch.arange(hd, device="cuda"), indexing="ij")
    j, c = d // 32, d % 32
    k_nibble = p * hd + 8 * ((c // 8) * ng + j) + c % 8
    k_step = 8 * hd + p * 4 * ng + 2 * j
    h, t, u = p // 8, p % 8 // 2, p % 2
    v_nibble = 8 * (((h * 8 + c // 4) * 4 + t) * ng + j) + 4 * u + c % 4
    v_step = 18 * hd + (p // 2) * 8 * ng + 4 * j + 2 * u
    return [(k_nibble // 2, 4 * (k_nibble % 2), k_step, k_step + 2 * ng),
            (10 * hd + v_nibble // 2, 4 * (v_nibble % 2), v_step, v_step + 4 * ng)]


def _stand_for(blocks: torch.Tensor) -> list[torch.Tensor]:
    """Blocks [..., 20 * hd] as keys and values [..., 16, hd] in float64."""
    out = []
    for byte, shift, step, offset in _places(blocks.shape[-1] // 20):
        code = (blocks[..., byte] >> shift.to(torch.uint8)) & 15
        s, o = (((blocks[..., at].int() << 16) | (blocks[..., at + 1].int() << 24)).view(torch.float32) for at in (step, offset))
        out.append(code.to(F64) * s.to(F64) + o.to(F64))
    return out


def _nearest_values(x: torch.Tensor) -> torch.Tensor:
    """What is stored for x [..., hd] (float64), group by group."""
    groups = x.reshape(-1, 32)
    low = groups.min(dim=1).values

    def bf16(value, up):
        near = value.to(F32).to(torch.bfloat16)
        wrong = near.to(F64) < value if up else near.to(F64) > value
        toward = torch.full_like(near, math.inf if up else -math.inf)
        return torch.where(wrong, torch.nextafter(near, toward), near).to(F64)

    offset = bf16(low, False)
    step = bf16((groups.max(dim=1).values - offset) / 15, True)
    codes = torch.round((groups - offset[:, None]) / torch.where(step > 0, step, torch.ones_like(step))[:, None])
    return (offset[:, None] + step[:, None] * codes.clamp(0, 15)).view(x.shape)


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    lengths, cached = lengths_of(case)
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    if case["what"] == "append":
        x = s["qkv"].to(F64)
        if case["bias"]:
            x = x + s["bias"].to(F64)
        heads = x.view(x.shape[0], -1, hd)
        turned = heads[:, :nh + nkv]
        if case["norm"]:
            scales = torch.cat([s["norms"][0].expand(nh, hd), s["norms"][1].expand(nkv, hd)]).to(F64)
            turned = turned / torch.sqrt(turned.square().mean(-1, keepdim=True) + EPS) * scales
        else:
            turned = turned.clone()
        at, half = s["positions"].long(), case["dims"] // 2
        turn = torch.complex(s["cos"][at].to(F64), s["sin"][at].to(F64))[:, None]
        first = slice(0, half) if case["layout"] == "halves" else slice(0, 2 * half, 2)
        second = slice(half, 2 * half) if case["layout"] == "halves" else slice(1, 2 * half, 2)
        both = torch.complex(turned[..., first].contiguous(), turned[..., second].contiguous()) * turn
        turned[..., first], turned[..., second] = both.real, both.imag
        pages = torch.stack([x.flatten(2, 3) for x in _stand_for(s["packed"][s["pages"].long()])], dim=1)
        pages[s["page_of_token"], 0, :, at % page] = _nearest_values(turned[:, nh:])
        pages[s["page_of_token"], 1, :, at % page] = _nearest_values(heads[:, nh + nkv:])
        return turned[:, :nh].reshape(-1, nh * hd), pages
    q = s["q"].to(F64).view(-1, nh, hd)
    out = torch.empty_like(q)
    start = 0
    for r, (n, c) in enumerate(zip(lengths, cached)):
        blocks = s["packed"][s["table"][r, :-(-(c + n) // page)].long()]
        for kvh in range(nkv):
            k, v = (x.reshape(-1, hd)[:c + n] for x in _stand_for(blocks[:, kvh]))
            heads = slice(kvh * (nh // nkv), (kvh + 1) * (nh // nkv))
            scores = torch.einsum("thd,kd->htk", q[start:start + n, heads], k) / math.sqrt(hd)
            if case.get("softcap"):
                scores = case["softcap"] * torch.tanh(scores / case["softcap"])
            i, j = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
            hidden = j > i
            if case.get("window"):
                hidden |= j <= i - case["window"]
            if case.get("chunk"):
                hidden |= j < i // case["chunk"] * case["chunk"]
            scores = scores.masked_fill(hidden, -math.inf)
            if s["sinks"] is not None:
                sink = s["sinks"][heads].to(F64).view(-1, 1, 1).expand(-1, n, 1)
                weights = torch.softmax(torch.cat([scores, sink], dim=-1), dim=-1)[..., :-1]
            else:
                weights = torch.softmax(scores, dim=-1)
            out[start:start + n, heads] = torch.einsum("htk,kd->thd", weights, v)
        start += n
    return out.view(-1, nh * hd)
