"""Matrices held in 8-bit floating point with a scale for each block of 128: making them, products with them, a gated feed-forward
and a layer of routed experts on them.

``run`` makes the calls that a program makes of ``zephyr_b200.kernels.ops`` (``own``), or computes the same in elementary torch
operations in 32 bits; ``exact`` is the definition in 64 bits.

A matrix [N, K] is cut into blocks of 128 x 128 (the last ones of a row or column may be smaller), a row of activations into blocks of
128 values.  A block's scale is the least power of two 2^s, s >= -126, for which its largest finite magnitude is at most 448 * 2^s; it is
kept as the byte s + 127.  A value's code is value / 2^s rounded to the nearest e4m3 number, ties to even (a value that is not finite: NaN);
it stands for code * 2^s.

* product: y = sum over k of (what x's codes stand for) * (what the matrix's codes stand for), rounded once to the output's type;
* gated feed-forward: G and U are the products of x with the gate and the up matrix, h = act(G) * U is coded in blocks of 128 as a row of
  activations is, and y is the product of that with the down matrix;
* routed experts: y[t] = sum over j of weights[t, j] * (the feed-forward of expert ids[t, j])(x[t]), an expert's output rounded
  to x's type first; an id past the experts stands for x[t] itself.

Gate and up rows lie in one matrix, in blocks of 8 gate rows and their 8 up rows.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 128
LIMIT, ALPHA, SHIFT = 7.0, 1.702, 1.0          # of the bounded gate


# ------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # Loading a model: the q/k/v projection of the 8B shape, and the down matrices of a routed layer.
        dict(name="pack projection", what="pack", experts=1, n=6144, k=4096, stored="bfloat16"),
        dict(name="pack experts", what="pack", experts=16, n=2048, k=1536, stored="bfloat16"),
        # Odd sizes, stored in 32 bits.
        dict(name="pack odd", what="pack", experts=1, n=1001, k=777, stored="float32"),
        # One user's token through the q/k/v projection of the 0.6B shape: latency counts.
        dict(name="product token", what="product", m=1, n=4096, k=1024, x="bfloat16", y="bfloat16"),
        # Eight requests' tokens through the down projection of the 8B shape.
        dict(name="product step", what="product", m=8, n=4096, k=12288, x="bfloat16", y="bfloat16"),
        # A full server's step through the q/k/v projection of the 32B shape.
        dict(name="product batch", what="product", m=64, n=10240, k=5120, x="bfloat16", y="bfloat16"),
        # A prompt's portion of odd length, sizes that end inside blocks, unrounded sums out.
        dict(name="product ragged", what="product", m=333, n=2050, k=1000, x="bfloat16", y="float32"),
        # Eight requests' tokens, and a prompt's, through whole feed-forwards (8B and 32B shapes).
        dict(name="feed-forward step", what="ffn", m=8, width=4096, ff=12288, act="silu", x="bfloat16"),
        dict(name="feed-forward prompt", what="ffn", m=2048, width=5120, ff=25600, act="silu", x="bfloat16"),
        # A routed layer: a step of eight tokens, a prompt, and a prompt whose tokens crowd on some of many narrow experts.
        dict(name="experts step", what="experts", m=8, width=2048, ff=1536, experts=16, identity=0, top=4, act="silu", skew=0.5),
        dict(name="experts prompt", what="experts", m=2048, width=2048, ff=1536, experts=16, identity=2, top=4, act="relu", skew=0.5),
        dict(name="experts crowded", what="experts", m=777, width=1200, ff=712, experts=64, identity=0, top=6, act="bounded", skew=2.0),
    ]


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low: int, high: int) -> int:
    """A size out of a range: mostly a multiple of 64, else of 8, else any."""
    n = _spread(rng, low, high)
    step = rng.choice((64, 64, 64, 8, 1))
    return max(step, n // step * step)


def draw(rng) -> dict:
    kind = rng.random()
    if kind < 0.15:
        experts = rng.choice((1, 1, 4, 16))
        return dict(what="pack", experts=experts, n=_size(rng, 64, 24576 // experts), k=_size(rng, 64, 8192),
                    stored=rng.choice(("bfloat16", "bfloat16", "float32")))
    if kind < 0.55:
        n, k = _size(rng, 64, 28672), _size(rng, 64, 14336)
        return dict(what="product", m=_spread(rng, 1, min(4096, 8 * 10 ** 11 // (n * k))), n=n, k=k,
                    x=rng.choice(("bfloat16", "bfloat16", "float32")), y=rng.choice(("bfloat16", "bfloat16", "float32")))
    if kind < 0.75:
        return dict(what="ffn", m=_spread(rng, 1, 2048), width=_size(rng, 64, 5120), ff=max(8, _spread(rng, 64, 16384) // 8 * 8),
                    act=rng.choice(("silu", "silu", "relu", "bounded")), x="bfloat16")
    experts = rng.choice((4, 8, 16, 60, 128))
    ff = max(8, _spread(rng, 64, 4096 if experts <= 16 else 1024) // 8 * 8)
    width, top = _size(rng, 64, 4096 if experts <= 16 else 2048), rng.randint(1, 4 if experts < 8 else 8)
    return dict(what="experts", m=_spread(rng, 1, min(2048, 26 * 10 ** 10 // (top * width * ff))), width=width, ff=ff, experts=experts,
                identity=rng.choice((0, 0, 2)), top=top, act=rng.choice(("silu", "relu", "bounded")), skew=rng.choice((0.0, 0.5, 2.0)))


def work(case: dict) -> dict:
    what = case["what"]
    if what == "pack":
        values = case["experts"] * case["n"] * case["k"]
        return {"bytes": values * (TYPES[case["stored"]].itemsize + 2), "flops": 2 * values}
    if what == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + m * k * TYPES[case["x"]].itemsize + m * n * TYPES[case["y"]].itemsize, "flops": 2 * m * n * k}
    m, width, ff = case["m"], case["width"], case["ff"]
    if what == "ffn":
        return {"bytes": 3 * width * ff + m * width * 4, "flops": 6 * m * width * ff}
    routed = case["top"] * case["experts"] / (case["experts"] + case["identity"])       # of a token, on average
    touched = case["experts"] * (1.0 - (1.0 - routed / case["experts"]) ** m)
    return {"bytes": int(3 * touched * width * ff + m * width * 4), "flops": int(6 * m * routed * width * ff)}


# --------------------------------------------------------------------------------- blocks in elementary operations
def _pad(n: int) -> int:
    return -n % BLOCK


def _exponent_bytes(largest: torch.Tensor) -> torch.Tensor:
    """s + 127 for blocks' largest finite magnitudes (float32): 448 is 1.75 * 2^8."""
    bits = largest.contiguous().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)


def _power(byte: torch.Tensor) -> torch.Tensor:
    return (byte.int() << 23).view(F32)


def _coded(x: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """x / 2^s as e4m3 numbers (float32 in; the quotient by a power of two is exact)."""
    x = torch.where(x.isfinite(), x, math.nan)
    return (x * _power(254 - byte)).to(torch.float8_e4m3fn)


def _magnitudes(x: torch.Tensor) -> torch.Tensor:
    return torch.where(x.isfinite(), x.abs(), 0.0)


def _matrix(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A matrix [..., N, K] as e4m3 codes of its shape and bytes [..., blocks, blocks]."""
    n, k = w.shape[-2:]
    padded = torch.nn.functional.pad(w.to(F32), (0, _pad(k), 0, _pad(n)))
    blocks = padded.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))                 # [..., nb, 128, kb, 128]
    byte = _exponent_bytes(_magnitudes(blocks).amax(dim=(-3, -1)))                       # [..., nb, kb]
    codes = _coded(blocks, byte[..., :, None, :, None])
    return codes.flatten(-4, -3).flatten(-2, -1)[..., :n, :k].contiguous(), byte.to(torch.uint8)


def _matrix_values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape[-2:]
    scale = _power(byte).repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return codes.to(F32) * scale


def _rows(x: torch.Tensor) -> torch.Tensor:
    """What the codes of rows [M, K] stand for, float32."""
    blocks = torch.nn.functional.pad(x.to(F32), (0, _pad(x.shape[1]))).unflatten(1, (-1, BLOCK))
    byte = _exponent_bytes(_magnitudes(blocks).amax(-1, keepdim=True))
    return (_coded(blocks, byte).to(F32) * _power(byte)).flatten(1)[:, : x.shape[1]]


def _gated(sums: torch.Tensor, act: str) -> torch.Tensor:
    gate, up = (part.flatten(1) for part in sums.unflatten(1, (-1, 2, 8)).unbind(2))
    if act == "silu":
        return gate / (1.0 + torch.exp(-gate)) * up
    if act == "relu":
        return gate.clamp(min=0.0) * up
    gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    return gate / (1.0 + torch.exp(-ALPHA * gate)) * (up + SHIFT)


# ------------------------------------------------------------------------------------------------- inputs
def _random(shape, generator, scale=1.0) -> torch.Tensor:
    return torch.randn(shape, generator=generator, device="cuda", dtype=F32) * scale


def _activations(m: int, k: int, dtype, generator) -> torch.Tensor:
    """Rows as a norm leaves them: some channels are larger than others, a few much larger."""
    channel = torch.exp(0.5 * _random((k,), generator))
    return (_random((m, k), generator) * channel).to(dtype)


def _weights(shape, generator) -> torch.Tensor:
    return _random(shape, generator, 0.02).to(torch.bfloat16)


def _routes(case: dict, generator) -> tuple[torch.Tensor, torch.Tensor]:
    outputs = case["experts"] + case["identity"]
    logits = _random((case["m"], outputs), generator) + case["skew"] * _random((outputs,), generator)
    weights, ids = torch.softmax(logits, dim=1).topk(case["top"], dim=1)
    return ids.to(torch.int32).contiguous(), weights.contiguous()


def _inputs(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    what = case["what"]
    if what == "pack":
        shape = (case["n"], case["k"]) if case["experts"] == 1 else (case["experts"], case["n"], case["k"])
        return {"w": _weights(shape, generator).to(TYPES[case["stored"]]) * (1.0 if case["stored"] == "bfloat16" else 1.0 / 3.0)}
    if what == "product":
        return {"x": _activations(case["m"], case["k"], TYPES[case["x"]], generator),
                "matrices": [_matrix(_weights((case["n"], case["k"]), generator))]}
    width, ff = case["width"], case["ff"]
    lead = () if what == "ffn" else (case["experts"],)
    state = {"x": _activations(case["m"], width, torch.bfloat16, generator),
             "matrices": [_matrix(_weights((*lead, 2 * ff, width), generator)), _matrix(_weights((*lead, width, ff), generator))]}
    if what == "experts":
        state["ids"], state["weights"] = _routes(case, generator)
    return state


def prepare(case: dict, seed: int):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        from zephyr_b200.kernels import ops
        state["ops"] = ops
        state["held"] = [ops.BlockMatrix.from_codes(codes, byte) for codes, byte in state.pop("matrices", ())]
        state["bounded"] = ops.BoundedGate(None, LIMIT, ALPHA, SHIFT) if case.get("act") == "bounded" else None
    return state


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    what = case["what"]
    if own:
        ops = state["ops"]
        if what == "pack":
            matrix = ops.pack_matrix(state["w"])
            return matrix.values(torch.bfloat16), matrix.exponents()
        if what == "product":
            return ops.linear(state["x"], state["held"][0], out_dtype=TYPES[case["y"]])
        act = "silu" if case["act"] == "bounded" else case["act"]
        if what == "ffn":
            return ops.block_feed_forward(state["x"], *state["held"], act=act, bounded=state["bounded"])
        return ops.routed_experts(state["x"], state["ids"], state["weights"], state["held"][0], None, state["held"][1], act=act,
                                  bounded=state["bounded"])
    if what == "pack":
        codes, byte = _matrix(state["w"])
        return _matrix_values(codes, byte).to(torch.bfloat16), byte
    x, values = state["x"], [_matrix_values(*m) for m in state["matrices"]]
    if what == "product":
        return (_rows(x) @ values[0].t()).to(TYPES[case["y"]])
    if what == "ffn":
        hidden = _gated(_rows(x) @ values[0].t(), case["act"])
        return (_rows(hidden) @ values[1].t()).to(x.dtype)
    ids, weights, coded = state["ids"], state["weights"], _rows(x)
    out = torch.zeros(x.shape, dtype=F32, device=x.device)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        hidden = _gated(coded[token] @ values[0][e].t(), case["act"])
        y = (_rows(hidden) @ values[1][e].t()).to(x.dtype).to(F32)
        out.index_add_(0, token, y * weights[token, choice, None])
    same = torch.where(ids >= case["experts"], weights, 0.0).sum(1, keepdim=True)
    return (out + same * x.to(F32)).to(x.dtype)


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_blocks(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What the codes of x [R, C] stand for in blocks of rows x 128, and the blocks' powers s."""
    r, c = x.shape
    full = torch.zeros((-(-r // rows) * rows, -(-c // BLOCK) * BLOCK), dtype=F64, device=x.device)
    full[:r, :c] = x
    grid = full.view(full.shape[0] // rows, rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(grid.abs().amax(dim=(1, 3)))                          # mantissa in [0.5, 1): 448 = 0.875 * 2^9
    s = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126)
    s = torch.where(mantissa == 0, -126, s)
    unit = torch.exp2(s.to(F64))[:, None, :, None]
    scaled = grid / unit
    _, own_exponent = torch.frexp(scaled)
    step = torch.exp2((own_exponent - 1).clamp(min=-6).to(F64) - 3)                        # three fraction bits, the least step 2^-9
    return (torch.round(scaled / step) * step * unit).view(full.shape)[:r, :c], s


def _exact_values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    row = torch.arange(n, device=codes.device) // BLOCK
    column = torch.arange(k, device=codes.device) // BLOCK
    return codes.to(F64) * torch.exp2(byte.to(F64) - 127.0)[row][:, column]


def _exact_gated(sums: torch.Tensor, act: str) -> torch.Tensor:
    index = torch.arange(sums.shape[1] // 2, device=sums.device)
    at = index // 8 * 16 + index % 8
    g, u = sums[:, at], sums[:, at + 8]
    if act == "relu":
        return torch.where(g > 0, g, 0.0) * u
    if act == "silu":
        return g * torch.sigmoid(g) * u
    g, u = torch.minimum(g, torch.full_like(g, LIMIT)), u.clamp(-LIMIT, LIMIT)
    return g * torch.sigmoid(ALPHA * g) * (u + SHIFT)


def exact(case: dict, seed: int):
    state = _inputs(case, seed)
    what = case["what"]
    if what == "pack":
        w = state["w"]
        parts = [_exact_blocks(m.to(F64), BLOCK) for m in (w if w.dim() == 3 else (w,))]
        values, bytes_ = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]) + 127
        return values.reshape(w.shape), bytes_.reshape(*w.shape[:-2], *bytes_.shape[-2:])
    x = state["x"]
    coded = _exact_blocks(x.to(F64), 1)[0]
    if what == "product":
        return coded @ _exact_values(*state["matrices"][0]).t()
    (up_codes, up_byte), (down_codes, down_byte) = state["matrices"]

    def feed_forward(rows, up, down):
        hidden = _exact_gated(rows @ _exact_values(*up).t(), case["act"])
        return _exact_blocks(hidden, 1)[0] @ _exact_values(*down).t()

    if what == "ffn":
        return feed_forward(coded, (up_codes, up_byte), (down_codes, down_byte))
    out = torch.zeros(x.shape, dtype=F64, device=x.device)
    for j in range(case["top"]):
        expert, weight = state["ids"][:, j], state["weights"][:, j].to(F64)[:, None]
        for e in expert.unique().tolist():
            rows = torch.nonzero(expert == e)[:, 0]
            y = x[rows].to(F64) if e >= case["experts"] else feed_forward(coded[rows], (up_codes[e], up_byte[e]), (down_codes[e], down_byte[e]))
            out[rows] += weight[rows] * y
    return out
