"""What is not finite behind the activations of gates and products: a NaN sum stays NaN, whichever kernel applies the activation, and takes no other
row, column or token with it."""

import pytest
import torch

import plain_block8 as plain
from test_block8_gpu import F64, LIMITS, _random
from zephyr_b200.kernels import ops

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
FORMS = ["silu", "relu", "bounded", "bounded bias", "gelu_tanh", "relu_squared"]


def _blocked(n):
    """Of n columns in blocks of 8 gates and their 8 ups: which are gates."""
    return torch.arange(n, device="cuda") % 16 < 8


def _bounded(form, n):
    return ops.BoundedGate(_random((n,), 18) if form == "bounded bias" else None, *LIMITS) if form.startswith("bounded") else None


def _plain(sums, form, bias=None):
    if form == "gelu_tanh":
        return 0.5 * sums * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (sums + 0.044715 * sums ** 3)))
    if form == "relu_squared":
        return sums.clamp(min=0) ** 2
    return plain.gated(sums, form.split()[0], LIMITS, bias)


def _same_and_nan(got, clean, want):
    """NaN where the 64-bit form has it, elsewhere what the clean call gave."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~want.isnan()], clean[~want.isnan()])


# ------------------------------------------------------------------------------------------------- matrices in 8 bits
@pytest.mark.parametrize("m", [4, 16, 20, 270])
@pytest.mark.parametrize("form", FORMS)
def test_products_on_8_bits(m, form):
    k, n = 500, 272
    x, raw = _random((m, k), 16), _random((n, k), 17, 0.1)
    bounded = _bounded(form, n)
    bias = bounded.bias if bounded is not None else None

    def call(x, w):
        w = ops.pack_matrix(w)
        if form in ops.PRODUCT_ACTS:
            return ops.block_linear(x, w, product_act=form)
        return ops.block_linear(x, w, swiglu=True, act=form if bounded is None else "silu", bounded=bounded)

    clean = call(x, raw)
    bad_x, bad_w = x.clone(), raw.clone()
    bad_x[1, 7], bad_x[0, 490], bad_x[3, 130] = INF, NAN, -INF
    bad_w[3, 100], bad_w[8 + 5, 0], bad_w[270, 499] = NAN, -INF, NAN             # a gate's row, two ups'
    for a, b in ((bad_x, raw), (x, bad_w), (bad_x, bad_w)):
        sums = plain.rows(a) @ plain.code_blocks(b, 128)[0].t()
        _same_and_nan(call(a, b), clean, _plain(sums, form, bias))


@pytest.mark.parametrize("m", [4, 17, 300])
@pytest.mark.parametrize("act", ["silu", "relu", "bounded"])
def test_feed_forwards_and_experts_on_8_bits(m, act):
    width, ff, experts = 256, 136, 4
    x = _random((m, width), 30)
    up, down = _random((experts, 2 * ff, width), 31, 0.1), _random((experts, width, ff), 32, 0.1)
    bounded = _bounded(act, 2 * ff)
    options = dict(act="silu" if bounded else act, bounded=bounded)
    ids = torch.stack([torch.arange(m), torch.arange(m) + 1], 1).remainder(experts).int().cuda()
    weights = _random((m, 2), 33).abs().contiguous()
    one, many = (lambda x, u, d: ops.block_feed_forward(x, ops.pack_matrix(u[0]), ops.pack_matrix(d[0]), **options),
                 lambda x, u, d: ops.routed_experts(x, ids, weights, ops.pack_matrix(u), None, ops.pack_matrix(d), **options))
    clean = [one(x, up, down), many(x, up, down)]
    assert all(bool(c.isfinite().all()) for c in clean)
    # A token that is not finite: its row alone.
    bad = x.clone()
    bad[1, 3], bad[2, 255] = NAN, -INF
    rows = torch.zeros(m, dtype=torch.bool, device="cuda")
    rows[1:3] = True
    for call, want in zip((one, many), clean):
        got = call(bad, up, down)
        assert bool(got[rows].isnan().all()) and torch.equal(got[~rows], want[~rows])
    # A gate's or an up's row of one expert: the whole feed-forward, the tokens that chose the expert.  (NaN times a gate of zero is NaN too.)
    for row in (5, 8 + 5):
        bad = up.clone()
        bad[0, row, 9] = NAN
        assert bool(one(x, bad, down).isnan().all())
        got, chose = many(x, bad, down), (ids == 0).any(1)
        assert bool(got[chose].isnan().all()) and torch.equal(got[~chose], clean[1][~chose])
    if bounded is None:                                  # weights on the inputs: the same tokens
        got = ops.routed_experts(x, ids, weights, ops.pack_matrix(bad), None, ops.pack_matrix(down), act=act, weigh_inputs=True)
        assert torch.equal(got.isnan().all(1), chose) and bool(got[~chose].isfinite().all())


# ------------------------------------------------------------------------------------------------- the model's type
def _sums(shape, seed):
    sums = _random(shape, seed, 4.0)
    sums[1, 2], sums[2, 11], sums[0, 0], sums[3, 8] = NAN, NAN, NAN, INF
    return sums


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_activations_of_rows(dtype):
    sums = _sums((6, 48), 40).to(dtype)
    plain_sums = sums.to(F64)
    gate, up = plain_sums[:, _blocked(48)], plain_sums[:, ~_blocked(48)]
    for act, want in (("silu", gate * torch.sigmoid(gate) * up), ("relu", gate.clamp(min=0) * up)):
        assert torch.equal(ops.silu_mul(sums, blocked=True, act=act).isnan(), want.isnan())
        halves = torch.cat([sums[:, _blocked(48)], sums[:, ~_blocked(48)]], 1).contiguous()
        assert torch.equal(ops.silu_mul(halves, act=act).isnan(), want.isnan())
    for form in ("gelu_tanh", "relu_squared"):
        got = ops.act_rows(sums, form)
        assert bool(got[0, 0].isnan() & got[1, 2].isnan() & got[2, 11].isnan()) and int(got.isnan().sum()) == 3
    limit, alpha, shift = LIMITS
    for size in (48, 36):                                # eight values at a time, and one by one
        part = sums[:, :size].contiguous()
        g, u = part.to(F64)[:, : size // 2].clamp(max=limit), part.to(F64)[:, size // 2 :].clamp(-limit, limit)
        want = g * torch.sigmoid(alpha * g) * (u + shift)
        assert torch.equal(ops.clamped_gate(part, None, limit, alpha, shift, dtype).isnan(), want.isnan()) and int(want.isnan().sum()) >= 3
    got = ops.clamped_gate(sums, None, limit, alpha, shift, dtype, blocked=True)
    want = plain.gated(plain_sums, "bounded", LIMITS)
    assert torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("form", FORMS)
def test_products_in_bfloat16(m, form):
    k, n = 256, 272
    x, w = _random((m, k), 50, dtype=torch.bfloat16), _random((n, k), 51, 0.1, torch.bfloat16)
    bounded = _bounded(form, n)
    options = dict(product_act=form) if form in ops.PRODUCT_ACTS else dict(swiglu=True, act=form if bounded is None else "silu", bounded=bounded)
    product = ops.gemm_small if m <= ops.SMALL_GEMM_MAX_ROWS else ops.gemm_tc
    clean = product(x, w, **options)
    bad_x, bad_w = x.clone(), w.clone()
    bad_x[1, 7], bad_x[0, 200] = NAN, NAN
    bad_w[3, 100], bad_w[8 + 5, 0], bad_w[270, 255] = NAN, NAN, NAN
    for a, b in ((bad_x, w), (x, bad_w)):
        _same_and_nan(product(a, b, **options), clean, _plain(a.to(F64) @ b.to(F64).t(), form, bounded.bias if bounded is not None else None))


@pytest.mark.parametrize("dtype,grouped", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, False)])
@pytest.mark.parametrize("act", ["silu", "relu", "bounded"])
def test_experts_in_the_models_type(monkeypatch, dtype, grouped, act):
    monkeypatch.setattr(ops, "USE_GROUPED_TCGEN05", grouped)
    m, width, ff, experts = 40, 128, 72, 4
    x = _random((m, width), 60, dtype=dtype)
    up, down = _random((experts, 2 * ff, width), 61, 0.1, dtype), _random((experts, width, ff), 62, 0.1, dtype)
    ids = torch.stack([torch.arange(m), torch.arange(m) + 1], 1).remainder(experts).int().cuda()
    weights = _random((m, 2), 63).abs().contiguous()
    bounded = _bounded(act, 2 * ff)
    call = lambda x, up, **options: ops.routed_experts(x, ids, weights, up, None, down, act="silu" if bounded else act, bounded=bounded, **options)
    clean = call(x, up)
    bad = x.clone()
    bad[1, 3], bad[2, 100] = NAN, NAN
    got = call(bad, up)
    assert bool(got[1:3].isnan().all()) and torch.equal(got[3:], clean[3:]) and torch.equal(got[0], clean[0])
    for row in (5, 8 + 5):
        bad = up.clone()
        bad[0, row, 9] = NAN
        got, chose = call(x, bad), (ids == 0).any(1)
        assert bool(got[chose].isnan().all()) and torch.equal(got[~chose], clean[~chose])
    if bounded is None:
        got = call(x, bad, weigh_inputs=True)
        assert torch.equal(got.isnan().all(1), chose) and bool(got[~chose].isfinite().all())
