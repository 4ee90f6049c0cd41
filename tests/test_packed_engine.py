"""The 4-bit cache in the engine's host code: what its pages cost, how groups form, what is refused, and the tables of rotations."""

import pytest
import torch

from legelix_models import CONFIGS
from tiny_configs import tiny_config
from zephyr_b200.cache import CacheManager, CacheStorage, PagedCacheSpec, bytes_per_page
from zephyr_b200.config import ConfigError, InvalidArgumentError, LegelixConfig
from zephyr_b200.config.spec import MixerSpec, PositionSpec
from zephyr_b200.parts import Attention, cache_specs, with_cache_bits
from zephyr_b200.parts.position import rotation_tables


def test_pages_of_four_bits():
    spec = PagedCacheSpec(2, 64, bits=4)
    plain = PagedCacheSpec(2, 64)
    assert spec.group_key != plain.group_key
    # 64 channels of a key and a value: 64 bytes of codes, 2 groups of 2 bfloat16 parameters each for both
    assert bytes_per_page([spec], 32, torch.bfloat16) == 32 * 2 * (64 + 16)
    assert bytes_per_page([spec, plain], 32, torch.bfloat16) == 32 * 2 * (64 + 16) + 32 * 2 * 2 * 64 * 2
    manager = CacheManager([spec, plain], 32, 5, 2)
    storage = CacheStorage(manager, torch.bfloat16, "cpu")
    assert storage[0].shape == (5, 2, 2, 20 * 64) and storage[0].dtype == torch.uint8 and storage[1].shape == (5, 2, 2, 32, 64)
    for view in (storage.keys, storage.values):
        assert view(1).shape == (5, 2, 32, 64)
        with pytest.raises(InvalidArgumentError, match="4-bit"):
            view(0)
    group = manager.group_of_cache[0]
    storage.poison_pages(manager, group, [0, 3])
    assert (storage[0][3] == 255).all() and not storage[0][[0, 1, 2, 4]].any()
    assert storage[0][3].view(torch.bfloat16).isnan().all()      # (steps and offsets among them)


@pytest.mark.parametrize("kwargs", [dict(bits=8), dict(bits=4, value_dim=32), dict(bits=4, keys_only=True), dict(bits=4, every=4)])
def test_specs_that_are_refused(kwargs):
    with pytest.raises(InvalidArgumentError):
        PagedCacheSpec(2, 64, **kwargs)


@pytest.mark.parametrize("page,hd", [(8, 64), (16, 48)])
def test_storage_that_is_refused(page, hd):
    with pytest.raises(ConfigError, match="4-bit"):
        CacheStorage(CacheManager([PagedCacheSpec(2, hd, bits=4)], page, 5, 2), torch.bfloat16, "cpu")


def test_a_models_caches():
    spec = tiny_config("D").to_model_spec()
    packed = with_cache_bits(spec, 4)
    assert [s.bits for s in cache_specs(spec)] == [0, 0] and [s.bits for s in cache_specs(packed)] == [4, 4]
    legelix = with_cache_bits(LegelixConfig.from_dict(CONFIGS["S"]).to_model_spec(), 4, 100)
    assert [getattr(s, "bits", None) for s in cache_specs(legelix) if isinstance(s, PagedCacheSpec)] == [4, 4]
    with pytest.raises(ConfigError, match="4 bits"):
        with_cache_bits(spec, 8)
    with pytest.raises(ConfigError, match="width"):            # a head size without kernels, and two widths
        cache_specs(with_cache_bits(tiny_config("A").to_model_spec(), 4))
    with pytest.raises(ConfigError, match="width"):
        cache_specs(with_cache_bits(LegelixConfig.from_dict(CONFIGS["P"]).to_model_spec(), 4))


def attention_part(params=None, position=("rope_neox", {}), dtype=torch.bfloat16, hd=64):
    names = dict(q_proj="q", k_proj="k", v_proj="v", o_proj="o")
    weights = {"q": torch.randn(4 * hd, 96), "k": torch.randn(2 * hd, 96), "v": torch.randn(2 * hd, 96), "o": torch.randn(96, 4 * hd),
               "m": torch.randn(4, 4), "r1": torch.randn(4), "r2": torch.randn(4), "g": torch.randn(4 * hd, 96)}
    spec = MixerSpec("attention", {"hidden_size": 96, "num_heads": 4, "num_kv_heads": 2, "head_dim": hd, "cache_bits": 4, **names, **(params or {})},
                     PositionSpec(position[0], head_dim=hd, max_positions=256, params=position[1]) if position else None)
    return Attention(spec, {k: w.to(dtype) for k, w in weights.items()}, dtype, "cpu")


@pytest.mark.parametrize("params,position,dtype", [
    (dict(values_from_keys=True), None, torch.bfloat16), (dict(unit_qk_norm=True, qk_norm_eps=1e-6), None, torch.bfloat16),
    (dict(q_temp={"coef": 0.1, "every": 8}), None, torch.bfloat16), (dict(value_unit_norm=True, qk_norm_eps=1e-6), None, torch.bfloat16),
    (dict(window=16, keep_first=2), None, torch.bfloat16), (dict(window=16, pool=4), None, torch.bfloat16), (dict(head_mix="m"), None, torch.bfloat16),
    (dict(score_mix="m"), None, torch.bfloat16), (dict(distance_bias=("r1", "r2")), None, torch.bfloat16),
    (dict(), ("rope_halves", {"dims": 12}), torch.bfloat16), (dict(), ("rope_neox", {}), torch.float32), (dict(cache_bits=8), ("rope_neox", {}), torch.bfloat16)])
def test_attention_that_is_refused(monkeypatch, params, position, dtype):
    from zephyr_b200.kernels import ops
    for name in ("paged_decode_supported", "paged_prefill_supported", "paged_attention_f32_supported"):      # (they ask the device)
        monkeypatch.setattr(ops, name, lambda *a: False)
    monkeypatch.setattr(ops, "heads_attention_tile_tokens", lambda *a: 0)
    with pytest.raises(ConfigError, match="bits"):
        attention_part(params, position, dtype)


def test_rotation_tables_are_shared_and_right():
    freqs = torch.tensor([1.0, 0.25, 0.01])
    one, two = rotation_tables(freqs, 1.5, 40), rotation_tables(freqs.clone(), 1.5, 40)
    assert one is two and rotation_tables(freqs, 1.0, 40) is not one and one.cos.shape == (40, 3)
    angles = torch.arange(40, dtype=torch.float64)[:, None] * freqs.double()
    # an angle is rounded once (2^-24 of it), the function to a few units of 2^-24, the multiplier once
    bound = 1.5 * 2.0 ** -24 * (angles + 6)
    assert ((one.cos - 1.5 * angles.cos()).abs() <= bound).all() and ((one.sin - 1.5 * angles.sin()).abs() <= bound).all()


def test_command_line_and_options():
    from zephyr_b200.cli import build_parser
    from zephyr_b200.engine import KvCacheOptions

    parse = build_parser().parse_args
    assert parse(["generate", "m", "--prompt-ids", "1"]).kv_bits is None and KvCacheOptions().bits is None
    assert parse(["generate", "m", "--prompt-ids", "1", "--kv-bits", "4"]).kv_bits == 4
    with pytest.raises(SystemExit):
        parse(["generate", "m", "--prompt-ids", "1", "--kv-bits", "3"])
