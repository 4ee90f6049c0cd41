"""Layers with a gate per head over a 4-bit cache, head counts that are no multiple of four among them: the gate's product comes along
with the projections, whose rows the writing kernel reads."""

import numpy as np
import pytest
import torch

import plain_tedulorn
from replay_util import BF16_UNITS, random_tokens, tolerance, trace_mixed, trace_portions, trace_tail, trace_whole
from tedulorn_models import attention, dense, model, read_model, rot, write_model
from test_packed_engine_gpu import attend_over, replay
from zephyr_b200.config.spec import MixerSpec, PositionSpec
from zephyr_b200.parts import Attention

# Groups of one, two and three heads, halves of part of a head and of all of it, windows; heads of 64, 32 and 96.
CONFIG = model(83, 72, 1e-5, 0, [
    attention(3, 3, 64, 64, 50, 0, rot(300.0, 16), 0.125, False, dense(100)),
    attention(6, 3, 32, 32, 19, 0, rot(10000.0, 32), 0.2, False, None),
    attention(5, 5, 96, 96, 400, 0, rot(1000.0, 40), 0.1, False, dense(60)),
    attention(9, 3, 128, 128, 33, 0, rot(50.0, 128), 0.09, False, None)])


@pytest.mark.parametrize("nh,nkv", [(1, 1), (3, 3), (6, 2), (5, 5), (18, 3), (8, 2)])
def test_rows_of_the_product_start_on_boundaries_of_four_values(monkeypatch, nh, nkv):
    from zephyr_b200.kernels import ops

    for name in ("paged_decode_supported", "paged_prefill_supported", "paged_attention_f32_supported"):      # (they ask the device)
        monkeypatch.setattr(ops, name, lambda *a: False)
    monkeypatch.setattr(ops, "heads_attention_tile_tokens", lambda *a: 0)
    hd, hidden = 32, 48
    weights = {"q": torch.randn(nh * hd, hidden), "k": torch.randn(nkv * hd, hidden), "v": torch.randn(nkv * hd, hidden),
               "o": torch.randn(hidden, nh * hd), "g": torch.randn(nh, hidden)}
    weights = {name: w.to(torch.bfloat16) for name, w in weights.items()}
    made = {}
    for bits in (0, 4):
        spec = MixerSpec("attention", dict(hidden_size=hidden, num_heads=nh, num_kv_heads=nkv, head_dim=hd, cache_bits=bits, q_proj="q", k_proj="k",
                                           v_proj="v", o_proj="o", head_gate="g"),
                         PositionSpec("rope_halves", head_dim=hd, max_positions=256, params={"base": 100.0, "dims": 16}))
        made[bits] = Attention(spec, weights, torch.bfloat16, "cpu")
    at = (nh + 2 * nkv) * hd
    assert made[4].w_qkv.shape[0] % 4 == 0 and made[0].w_qkv.shape[0] == at + nh
    assert torch.equal(made[4].w_qkv[:at + nh], made[0].w_qkv) and not made[4].w_qkv[at + nh:].any()
    assert torch.equal(made[4].w_q, weights["q"])


TRACES = {"whole": trace_whole, "tail": trace_tail, "portions": trace_portions, "mixed": trace_mixed}


@pytest.mark.gpu
@pytest.mark.parametrize("trace", list(TRACES))
def test_gated_models(tmp_path, cuda_device, monkeypatch, trace):
    folder = write_model(tmp_path, CONFIG, seed=31, dtype=torch.bfloat16)
    config, weights = read_model(folder)
    lengths = [100, 41, 129, 5]
    requests = {f"r{i}": random_tokens(83, n, seed=700 + n) for i, n in enumerate(lengths)}
    rows, stored = replay(folder, TRACES[trace](requests), 16, sum(-(-n // 16) for n in lengths) + 1, 4)
    raw_scores, weigh_values = plain_tedulorn.raw_scores, plain_tedulorn.weigh_values
    worst = 0.0
    for rid, tokens in requests.items():
        # The plain attention over what the cache held: keys where scores are formed, values where they are weighed.
        keys, layers = [], iter(stored[rid])
        checked = attend_over(stored[rid], BF16_UNITS, lambda q, k, v: (k, v))

        def scores(q, k, scale):
            keys.append(k)
            return raw_scores(q, next(layers)[0], scale)

        def weigh(p, v):
            return weigh_values(p, checked(None, keys.pop(), v)[1])

        with monkeypatch.context() as patch:
            patch.setattr(plain_tedulorn, "raw_scores", scores)
            patch.setattr(plain_tedulorn, "weigh_values", weigh)
            expected = plain_tedulorn.forward(config, weights, tokens).numpy()
        for (owner, position), got in rows.items():
            if owner == rid:
                assert np.isfinite(got).all()
                worst = max(worst, float(np.abs(got.astype(np.float64) - expected[position]).max()) / tolerance("bfloat16", expected[position]))
    print(f"worst error {worst:.2f} of its bound over {len(rows)} rows")
    assert worst <= 1.0
