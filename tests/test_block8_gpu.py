"""Matrices in 8-bit floating point with a scale for each block of 128: packing, products, gated feed-forwards and routed experts against 64 bits."""

import pytest
import torch

import plain_block8 as plain
from zephyr_b200.kernels import ops

pytestmark = pytest.mark.gpu
F64 = torch.float64
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LIMITS = (7.0, 1.702, 1.0)


def _random(shape, seed, scale=1.0, dtype=torch.float32):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return (torch.randn(shape, generator=generator, device="cuda") * scale).to(dtype)


def _matrix(shape, seed, scale=0.02):
    w = _random(shape, seed, scale, torch.bfloat16)
    packed = ops.pack_matrix(w)
    parts = [plain.code_blocks(m, 128)[0] for m in (w if w.dim() == 3 else (w,))]
    return packed, torch.stack(parts) if w.dim() == 3 else parts[0]


def _close(got, want, error, dtype):
    """Within ``error`` of ``want`` ahead of a rounding to ``dtype`` (bfloat16's least normal number is 2^-126)."""
    assert got.dtype == dtype and got.shape == want.shape
    bound = error + HALF_STEP[dtype] * (want.abs() + error) + 2.0 ** -133
    off = (got.to(F64) - want).abs()
    assert bool((off <= bound).all()), f"worst {(off / bound).max().item():.3g} of the bound"


# ------------------------------------------------------------------------------------------------- packing
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (16, 16), (7, 2049), (300, 515), (1000, 640), (3, 130, 200), (2, 128, 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packing(shape, dtype):
    w = _random(shape, 1, 1.0, dtype) * torch.exp(4 * _random(shape[-1:], 2)).to(dtype)
    packed = ops.pack_matrix(w)
    for m, got, byte in zip(w.view(-1, *shape[-2:]), packed.values(torch.float32).view(-1, *shape[-2:]),
                            packed.exponents().view(-1, *packed.exponents().shape[-2:])):
        want, s = plain.code_blocks(m, 128)
        assert torch.equal(got.to(F64), want) and torch.equal(byte.int(), s.int() + 127)
    assert torch.equal(packed.values(torch.bfloat16).float(), packed.values(torch.float32))
    rows = packed.codes.transpose(2, 3).flatten(3, 4).flatten(1, 2)                     # [matrices, N up to 128, K up to 128]
    assert packed.shape == tuple(shape) and not bool(rows[:, shape[-2]:].any()) and not bool(rows[:, :, shape[-1]:].any())


def test_packing_borders_ties_and_what_is_not_finite():
    # Largest magnitudes on and beside 448 * 2^s, ties between codes, numbers under the least code, blocks of zeros, the ends of float32.
    w = torch.zeros((9 * 128, 128), device="cuda")
    for b, top in enumerate((448.0, 448.0000305, 447.99997, 1.75 * 2.0 ** -130, 3.0e38, 1.0e-45, 0.0, 1.0, 480.0)):
        w[128 * b] = torch.linspace(-1, 1, 128, device="cuda").double().mul(top).float()
        w[128 * b + 1, 0] = top
    w[128 * 7 + 2, :16] = torch.arange(16, device="cuda") * 2.0 ** -4 + 1.0 + 2.0 ** -5
    packed = ops.pack_matrix(w)
    want, s = plain.code_blocks(w, 128)
    assert torch.equal(packed.values(torch.float32).double(), want) and torch.equal(packed.exponents().int(), s.int() + 127)
    w[5, 7], w[200, 3], w[300, 100] = float("inf"), float("nan"), -float("inf")
    got, (want, _) = ops.pack_matrix(w).values(torch.float32).double(), plain.code_blocks(w, 128)
    assert torch.equal(got.isnan(), ~w.isfinite()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def test_packing_rows_that_are_not_side_by_side_and_from_codes():
    wide = _random((300, 700), 3, dtype=torch.bfloat16)
    for w in (wide[:, 5:300], wide[::2, :256], wide[:, 8:520]):
        packed = ops.pack_matrix(w)
        assert torch.equal(packed.values(torch.float32).double(), plain.code_blocks(w, 128)[0])
        codes = packed.codes.transpose(2, 3).flatten(3, 4).flatten(1, 2)[0, : w.shape[0], : w.shape[1]]
        again = ops.BlockMatrix.from_codes(codes.contiguous().view(torch.float8_e4m3fn), packed.exponents())
        assert torch.equal(again.codes, packed.codes) and torch.equal(again.scales, packed.scales)
    several = ops.pack_matrix(_random((3, 140, 600), 4))
    again = ops.BlockMatrix.from_codes(several.codes.transpose(2, 3).flatten(3, 4).flatten(1, 2)[:, :140, :600], several.exponents())
    assert torch.equal(again.scales, several.scales) and torch.equal(again.values(), several.values())


# ------------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 64, 65, 128, 129, 256, 257, 700])
@pytest.mark.parametrize("n,k", [(256, 512), (1, 1), (130, 129), (2050, 1000), (48, 2050), (4096, 1024)])
@pytest.mark.parametrize("x_dtype,y_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_products(m, n, k, x_dtype, y_dtype):
    x = _random((m, k), 5, dtype=x_dtype) * torch.exp(_random((k,), 6)).to(x_dtype)
    packed, w = _matrix((n, k), 7)
    want, magnitude = plain.product(x, w)
    _close(ops.linear(x, packed, y_dtype), want, plain.sum_error(k) * magnitude, y_dtype)


# Few rows of long matrices; then rows and columns for runs of 64, 128 and 256 rows, tiles of whole and shared K, result rows that are and are not
# multiples of 16 bytes.
@pytest.mark.parametrize("m,n,k", [(3, 5120, 25600), (16, 512, 25600), (12, 4096, 12288), (8, 30000, 256), (100, 640, 9000),
                                   (130, 2500, 14336), (100, 6400, 14336), (1000, 4864, 10240), (1500, 3840, 11520), (300, 8200, 640), (600, 4105, 260), (1030, 4110, 384), (333, 1030, 9100)])
def test_products_of_long_rows_and_of_many(m, n, k):
    x = _random((m, k), 8, dtype=torch.bfloat16)
    packed, w = _matrix((n, k), 9)
    want, magnitude = plain.product(x, w)
    for y in (torch.float32, torch.bfloat16):
        _close(ops.linear(x, packed, y), want, plain.sum_error(k) * magnitude, y)


@pytest.mark.parametrize("m", [5, 40, 300])
def test_product_types_strides_and_scales_of_any_size(m):
    wide = _random((m, 900), 10)
    packed, w = _matrix((200, 389), 11)
    for x in (wide[:, 3:392], wide[:, 4:393].bfloat16()[:, :389], wide.bfloat16()[:, 8:397]):
        want, magnitude = plain.product(x, w)
        for y in (torch.bfloat16, torch.float32):
            _close(ops.block_linear(x, packed, y), want, plain.sum_error(389) * magnitude, y)
    # Every block its own size, from 2^-60 to 2^60: the powers of two meet in the product.
    powers = torch.exp2(torch.randint(-60, 61, (m, 5), generator=torch.Generator().manual_seed(1)).float()).cuda()
    x = _random((m, 640), 12) * powers.repeat_interleave(128, 1)
    sizes = torch.exp2(torch.randint(-50, 51, (3, 5), generator=torch.Generator().manual_seed(2)).float()).cuda()
    raw = _random((300, 640), 13) * sizes.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)
    want, magnitude = plain.product(x, plain.code_blocks(raw, 128)[0])
    _close(ops.block_linear(x, ops.pack_matrix(raw), torch.float32), want, plain.sum_error(640) * magnitude, torch.float32)


@pytest.mark.parametrize("m", [2, 33, 290])
def test_what_is_not_finite_stays_in_its_row_or_column(m):
    x, raw = _random((m, 300), 14), _random((140, 300), 15)
    clean = ops.block_linear(x, ops.pack_matrix(raw))
    bad_x, bad_w = x.clone(), raw.clone()
    bad_x[1, 7], bad_x[0, 290] = float("inf"), float("nan")
    got = ops.block_linear(bad_x, ops.pack_matrix(raw))
    assert bool(got[:2].isnan().all()) and torch.equal(got[2:], clean[2:])
    bad_w[3, 100], bad_w[139, 0] = float("nan"), -float("inf")
    got = ops.block_linear(x, ops.pack_matrix(bad_w))
    assert bool(got[:, [3, 139]].isnan().all()) and not bool(got[:, :3].isnan().any()) and not bool(got[:, 4:139].isnan().any())
    zero = ops.block_linear(torch.zeros_like(x), ops.pack_matrix(raw))
    assert bool((zero == 0).all()) and ops.block_linear(x[:0], ops.pack_matrix(raw)).shape == (0, 140)


@pytest.mark.parametrize("m", [4, 20, 270])
@pytest.mark.parametrize("form", ["silu", "relu", "bounded", "bounded bias", "gelu_tanh", "relu_squared"])
def test_activations_of_the_sums(m, form):
    k, n = 500, 272
    x = _random((m, k), 16, dtype=torch.bfloat16)
    packed, w = _matrix((n, k), 17, 0.1)
    sums, magnitude = plain.product(x, w)
    error = plain.sum_error(k) * magnitude
    if form in ("gelu_tanh", "relu_squared"):
        got = ops.block_linear(x, packed, torch.float32, product_act=form)
        if form == "relu_squared":
            want, bound = sums.clamp(min=0) ** 2, (2 * sums.abs() + error) * error + 2.0 ** -22 * sums ** 2
        else:
            u = (2 / torch.pi) ** 0.5 * (sums + 0.044715 * sums ** 3)
            want = 0.5 * sums * (1 + torch.tanh(u))
            bound = 1.2 * error + 2.0 ** -18 * sums.abs()        # |d/dz| <= 1.13; float32's arithmetic and exponent
    else:
        bias = _random((n,), 18) if form == "bounded bias" else None
        act = form.split()[0]
        bounded = ops.BoundedGate(bias, *LIMITS) if act == "bounded" else None
        got = ops.block_linear(x, packed, torch.float32, swiglu=True, act="silu" if bounded else act, bounded=bounded)
        want, bound = plain.gated(sums, act, LIMITS, bias), plain.gated_error(sums, error, act, LIMITS, bias)
    _close(got, want, bound, torch.float32)


# ------------------------------------------------------------------------------------------------- feed-forwards and experts
def _feed_forward(x, up, down, act, limits=LIMITS, bias=None):
    """The value in 64 bits and a bound on its error ahead of the last rounding."""
    sums, magnitude = plain.product(x, up)
    hidden = plain.gated(sums, act, limits, bias)
    off = plain.gated_error(sums, plain.sum_error(up.shape[1]) * magnitude, act, limits, bias)
    want, size = plain.product(hidden, down)
    return want, plain.code_spread(hidden, off) @ down.abs().t() * (1 + 1e-4) + plain.sum_error(down.shape[1]) * size * 1.01


@pytest.mark.parametrize("m,width,ff,act", [(1, 256, 128, "silu"), (16, 1024, 904, "relu"), (17, 130, 8, "silu"), (64, 300, 1000, "bounded"),
                                            (200, 1024, 512, "silu"), (600, 640, 1544, "bounded"), (600, 4100, 4104, "silu"),
                                            (40, 12288, 640, "silu"), (40, 1000, 9000, "relu"), (100, 14336, 3200, "silu"), (1024, 10240, 2432, "bounded"), (1500, 11520, 1920, "relu")])
def test_feed_forwards(m, width, ff, act):
    x = _random((m, width), 20, dtype=torch.bfloat16)
    (up, up_values), (down, down_values) = _matrix((2 * ff, width), 21, 0.1), _matrix((width, ff), 22, 0.1)
    want, error = _feed_forward(x, up_values, down_values, act)
    bounded = ops.BoundedGate(None, *LIMITS) if act == "bounded" else None
    for y in (torch.bfloat16, torch.float32):
        _close(ops.block_feed_forward(x, up, down, act="silu" if bounded else act, bounded=bounded, out_dtype=y), want, error, y)


@pytest.mark.parametrize("tokens,width,ff,experts,identity,top,act,skew", [
    (1, 256, 128, 4, 0, 2, "silu", 0.0), (8, 512, 136, 16, 2, 4, "relu", 0.5), (100, 136, 72, 5, 0, 5, "bounded", 0.0),
    (300, 300, 200, 8, 3, 3, "silu", 4.0), (777, 256, 264, 60, 0, 6, "bounded", 2.0), (1500, 128, 128, 4, 0, 2, "silu", 6.0),
    (40, 129, 16, 3, 1, 2, "silu", 0.0), (20, 8192, 256, 4, 0, 2, "silu", 0.0), (30, 256, 6144, 3, 0, 2, "relu", 0.0), (300, 8192, 200, 4, 0, 1, "silu", 0.0),
    (500, 128, 16, 400, 0, 2, "silu", 0.0), (900, 128, 16, 3, 0, 1, "silu", 3.0), (60, 200, 72, 64, 2, 4, "bounded", 4.0), (170, 1024, 264, 160, 0, 3, "silu", 1.0),
    (50, 130, 200, 40, 0, 3, "relu", 5.0), (2, 300, 4200, 3, 0, 2, "silu", 0.0), (1, 9000, 16, 8, 0, 3, "silu", 0.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_routed_experts(tokens, width, ff, experts, identity, top, act, skew, dtype):
    x = _random((tokens, width), 30, dtype=dtype)
    (up, up_values), (down, down_values) = _matrix((experts, 2 * ff, width), 31, 0.1), _matrix((experts, width, ff), 32, 0.1)
    logits = _random((tokens, experts + identity), 33) + skew * _random((experts + identity,), 34)
    weights, ids = logits.softmax(1).topk(top, 1)
    ids, weights = ids.int().contiguous(), weights.contiguous()
    bounded = ops.BoundedGate(None, *LIMITS) if act == "bounded" else None
    got = ops.routed_experts(x, ids, weights, up, None, down, act="silu" if bounded else act, bounded=bounded)
    want, error = torch.zeros((tokens, width), dtype=F64, device="cuda"), torch.zeros((tokens, width), dtype=F64, device="cuda")
    for e in range(experts + identity):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        weight = weights[token, choice].double()[:, None]
        y, off = (x[token].double(), torch.zeros_like(x[token], dtype=F64)) if e >= experts else _feed_forward(x[token], up_values[e], down_values[e], act)
        off = off + (HALF_STEP[dtype] * (y.abs() + off) if e < experts else 0)            # an expert's output in x's type
        want[token] += weight * y
        error[token] += weight * off + 2.0 ** -22 * (weight * y).abs()
    _close(got, want, error, dtype)
    if bounded is None and identity == 0:
        # Weights on the inputs: one expert's choices, each with its weight on both sums.
        got = ops.routed_experts(x, ids, weights, up, None, down, act=act, weigh_inputs=True)
        want.zero_(), error.zero_()
        for e in range(experts):
            token, choice = torch.nonzero(ids == e, as_tuple=True)
            if token.numel() == 0:
                continue
            weight = weights[token, choice].double()[:, None]
            sums, magnitude = plain.product(x[token], up_values[e])
            sums, off = sums * weight, (plain.sum_error(width) + 2.0 ** -23) * magnitude * weight
            hidden, off = plain.gated(sums, act), plain.gated_error(sums, off, act)
            y, size = plain.product(hidden, down_values[e])
            off = plain.code_spread(hidden, off) @ down_values[e].abs().t() * (1 + 1e-4) + plain.sum_error(ff) * size * 1.01
            want[token] += y
            error[token] += off + HALF_STEP[dtype] * (y.abs() + off) + 2.0 ** -22 * y.abs()
        _close(got, want, error, dtype)


@pytest.mark.parametrize("tokens,experts", [(3, 4), (30, 16), (30, 4)])
def test_one_token_chooses_an_expert_twice(tokens, experts):
    width, ff = 256, 72
    x = _random((tokens, width), 70, dtype=torch.bfloat16)
    (up, up_values), (down, down_values) = _matrix((experts, 2 * ff, width), 71, 0.1), _matrix((experts, width, ff), 72, 0.1)
    ids = torch.arange(tokens, device="cuda")[:, None].expand(tokens, 2).remainder(experts).int().contiguous()
    weights = _random((tokens, 2), 73).abs().contiguous()
    got = ops.routed_experts(x, ids, weights, up, None, down)
    want = torch.empty((tokens, width), dtype=F64, device="cuda")
    error = torch.empty_like(want)
    for e in range(min(tokens, experts)):
        token = torch.arange(e, tokens, experts, device="cuda")
        y, off = _feed_forward(x[token], up_values[e], down_values[e], "silu")
        off = off + HALF_STEP[torch.bfloat16] * (y.abs() + off)
        weight = weights[token].double().sum(1, keepdim=True)
        want[token], error[token] = weight * y, weight * off + 2.0 ** -21 * (weight * y).abs()
    _close(got, want, error, torch.bfloat16)


# ------------------------------------------------------------------------------------------------- calls side by side
def test_calls_on_two_streams_at_once():
    """Calls that share a matrix, on two streams with no order between them, give what the same calls give one after the other, bit for bit."""
    (up, _), (down, _) = _matrix((2 * 1024, 640), 40, 0.1), _matrix((640, 1024), 41, 0.1)
    (ups, _), (downs, _) = _matrix((8, 512, 640), 42, 0.1), _matrix((8, 640, 256), 43, 0.1)
    long, _ = _matrix((640, 12800), 44)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [[_random((m, 640), 45 + 10 * s + m, dtype=torch.bfloat16) for m in (3, 40, 300)] for s in range(2)]
    wide = [_random((40, 12800), 90 + s, dtype=torch.bfloat16) for s in range(2)]
    chosen = [_random((300, 8), 50 + s).softmax(1).topk(2, 1) for s in range(2)]

    def calls(s):
        out = []
        for x in inputs[s]:
            out += [ops.linear(x, up), ops.block_feed_forward(x, up, down)]
        out.append(ops.linear(wide[s], long))
        out.append(ops.routed_experts(inputs[s][2], chosen[s][1].int().contiguous(), chosen[s][0].contiguous(), ups, None, downs))
        return out

    want = [calls(0), calls(1)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s in (0, 1):
            with torch.cuda.stream(streams[s]):
                got[s].append(calls(s))
    torch.cuda.synchronize()
    for s in (0, 1):
        for run in got[s]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[s]))


def test_the_same_layer_on_bfloat16_matrices_captured(cuda_device):
    """Every kernel of a routed layer in the model's type is on the caller's stream: a capture holds them all."""
    x = _random((8, 256), 60, dtype=torch.bfloat16)
    ups, downs = _random((5, 2 * 72, 256), 61, 0.1, torch.bfloat16), _random((5, 256, 72), 62, 0.1, torch.bfloat16)
    weights, ids = _random((8, 5), 63).softmax(1).topk(2, 1)
    ids, weights = ids.int().contiguous(), weights.contiguous()
    want = ops.routed_experts(x, ids, weights, ups, None, downs)
    graph = torch.cuda.CUDAGraph()
    with ops.capture(graph):
        got = ops.routed_experts(x, ids, weights, ups, None, downs)
    got.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
