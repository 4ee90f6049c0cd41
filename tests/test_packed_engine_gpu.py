"""Whole models over the 4-bit cache: every way of cutting requests into steps (prompts, portions, single tokens, mixed batches, captured
steps, two lanes), with given-back pages filled with NaN.

Codes are discontinuous in what they encode, so the plain model is not asked to give the same ones: the keys and values that the cache
holds are read back as each step has written them, each is checked against the plain model's own (half a step of its group, and the
bound on bfloat16 activations), and the plain model then attends over those that were read."""

import math

import numpy as np
import pytest
import torch

import plain_legelix
import plain_qwen3
from legelix_models import CONFIGS, DECAY_RANK, read_model, write_model
from plain_qwen3 import load_model_folder
from replay_util import BF16_UNITS, random_tokens, tolerance, trace_batched_tail, trace_mixed, trace_portions, trace_tail, trace_whole

pytestmark = pytest.mark.gpu


def make_runner(folder, page_size, num_pages, max_requests, graphs=True):
    from zephyr_b200.config import load_model_spec
    from zephyr_b200.engine.runner import ModelRunner
    from zephyr_b200.parts import Model, with_cache_bits
    from zephyr_b200.weights import Checkpoint

    spec = with_cache_bits(load_model_spec(folder), 4)
    model = Model.load(spec, Checkpoint(folder), torch.bfloat16, torch.device("cuda", 0))
    runner = ModelRunner(model, page_size, num_pages, max_requests, max_seq_len=min(spec.max_seq_len, num_pages * page_size))
    runner.use_cuda_graphs = graphs
    runner.poison_freed_pages = True
    return runner


def replay(folder, steps, page_size, num_pages, max_requests, graphs=True):
    """(logits by (request, position), keys and values by request: per paged cache [2, positions, kv_heads, head_dim])."""
    from zephyr_b200.cache import PagedCacheSpec
    from zephyr_b200.engine.runner import StepEntry
    from zephyr_b200.kernels import ops

    runner = make_runner(folder, page_size, num_pages, max_requests, graphs)
    manager = runner.manager
    caches = [c for c, spec in enumerate(manager.cache_specs) if isinstance(spec, PagedCacheSpec)]
    assert all(runner.storage[c].dtype == torch.uint8 for c in caches)
    stored, rows, commit = {}, {}, manager.commit

    def reading_commit(request_id, computed):
        before = manager.computed(request_id)
        for index, cache in enumerate(caches):
            table = manager.block_table(request_id, manager.group_of_cache[cache])
            first = before // page_size
            pages = torch.tensor(list(table)[first:-(-computed // page_size)], dtype=torch.int32, device=runner.device)
            values = ops.unpack_pages(runner.storage[cache], pages, torch.float32).cpu().double()      # [pages, 2, heads, page, hd]
            flat = values.permute(1, 0, 3, 2, 4).reshape(2, -1, values.shape[2], values.shape[4])
            stored.setdefault(request_id, [[] for _ in caches])[index].append(flat[:, before - first * page_size:computed - first * page_size])
        commit(request_id, computed)

    manager.commit = reading_commit
    for step in steps:
        entries = []
        for item in step["entries"]:
            if item["id"] not in manager:
                assert runner.add_request(item["id"])
            entries.append(StepEntry(item["id"], item["tokens"], item["want"]))
        at = {e.request_id: manager.computed(e.request_id) for e in entries}
        logits = iter(runner.step(entries).cpu().numpy())
        runner.check()
        for e in entries:
            for place in e.want:
                rows[e.request_id, at[e.request_id] + place] = next(logits)
        for request_id in step["end"]:
            runner.free_request(request_id)
        manager.check_invariants()
    return rows, {rid: [torch.cat(parts, dim=1) for parts in per] for rid, per in stored.items()}


def attend_over(stored, units, core):
    """The plain attention ``core(q, k, v, ...)`` over what the cache held, layer after layer; its own keys and values are compared."""
    layers = iter(stored)

    def attend(q, k, v, *rest):
        held = next(layers)
        for own, got in ((k, held[0]), (v, held[1])):
            groups = own.reshape(own.shape[0], own.shape[1], -1, 32)
            close = units * 2.0 ** -8 * own.abs().max()
            spread = groups.amax(-1) - groups.amin(-1) + 2 * close
            # Half a step: the spread, and what the offset was rounded down by, over 15, the step rounded up.
            step = (spread + 2.0 ** -7 * groups.abs().amax(-1)) / 15 * (1 + 2.0 ** -6)
            off = (got - own).abs().reshape(groups.shape)
            assert torch.isfinite(got).all() and (off <= (step / 2 + close + 2.0 ** -7 * groups.abs().amax(-1))[..., None]).all()
        return core(q, held[0], held[1], *rest)

    return attend


TRACES = {"whole": trace_whole, "tail": trace_tail, "portions": trace_portions, "mixed": trace_mixed, "batched": trace_batched_tail}
# name -> page size, lengths: head sizes 32, 64 with windows, 128
QWEN = {"B": (16, [33, 70, 9, 120]), "W": (16, [90, 130, 17, 64]), "D": (32, [150, 41, 260, 5])}


def check_qwen(folder, requests, rows, stored, monkeypatch):
    config, weights = load_model_folder(folder)
    core, worst = plain_qwen3.plain_attention, 0.0
    for rid, tokens in requests.items():
        with monkeypatch.context() as patch:
            patch.setattr(plain_qwen3, "plain_attention", attend_over(stored[rid], BF16_UNITS, core))
            expected = plain_qwen3.plain_forward(config, weights, tokens).numpy()
        for (owner, position), got in rows.items():
            if owner == rid:
                error = float(np.abs(got.astype(np.float64) - expected[position]).max()) / tolerance("bfloat16", expected[position])
                worst = max(worst, error)
                assert error <= 1.0, (rid, position, error)
    print(f"worst error {worst:.2f} of its bound over {len(rows)} rows")


@pytest.mark.parametrize("trace", list(TRACES))
@pytest.mark.parametrize("name", list(QWEN))
def test_qwen3_over_four_bits(model_folders, cuda_device, monkeypatch, name, trace):
    page, lengths = QWEN[name]
    folder = model_folders(name, "bfloat16")
    vocab = load_model_folder(folder)[0]["vocab_size"]
    requests = {f"r{i}": random_tokens(vocab, n, seed=300 + n) for i, n in enumerate(lengths)}
    steps = TRACES[trace](requests)
    rows, stored = replay(folder, steps, page, sum(-(-n // page) for n in lengths) + 1, 4)
    check_qwen(folder, requests, rows, stored, monkeypatch)


@pytest.mark.parametrize("graphs", [False, True])
def test_many_requests_decode_together(model_folders, cuda_device, monkeypatch, graphs):
    """Fourteen requests a step: enough for two lanes; captured and not."""
    folder = model_folders("D", "bfloat16")
    requests = {f"r{i}": random_tokens(503, 12 + 5 * i, seed=400 + i) for i in range(14)}
    rows, stored = replay(folder, trace_batched_tail(requests, max_live=14, tail=7), 16, 120, 14, graphs)
    check_qwen(folder, requests, rows, stored, monkeypatch)


@pytest.mark.parametrize("trace", ["whole", "tail", "portions", "mixed"])
def test_legelix_over_four_bits(tmp_path, cuda_device, monkeypatch, trace):
    """Biases, norms without a window, adjacent pairs (all of a head and a part of it, scaled frequencies), chunks and sinks."""
    folder = write_model(tmp_path, CONFIGS["S"], DECAY_RANK["S"], seed=17 + ord("S"), dtype=torch.bfloat16)
    config, weights = read_model(folder)
    lengths = [100, 41, 129, 5]
    requests = {f"r{i}": random_tokens(80, n, seed=500 + n) for i, n in enumerate(lengths)}
    rows, stored = replay(folder, TRACES[trace](requests), 16, sum(-(-n // 16) for n in lengths) + 1, 4)
    core, ratios = plain_legelix.plain_attention_core, []
    for rid, tokens in requests.items():
        with monkeypatch.context() as patch:
            # (a layer norm behind a part's output magnifies its rounding at single positions: up to six bounds, as without this cache)
            patch.setattr(plain_legelix, "plain_attention_core", attend_over(stored[rid], 6 * BF16_UNITS, core))
            expected = plain_legelix.plain_legelix(config, weights, tokens)[0].numpy()
        ratios += [float(np.abs(got.astype(np.float64) - expected[position]).max()) / tolerance("bfloat16", expected[position])
                   for (owner, position), got in rows.items() if owner == rid]
    assert all(math.isfinite(r) for r in ratios)
    assert max(ratios) <= 6.0 and sum(r > 1.0 for r in ratios) <= max(1, len(ratios) // 25), (max(ratios), len(ratios))


def test_generation_with_four_bits(model_folders, cuda_device):
    """Through the engine: sized by bytes, a pool so small that it preempts, the same tokens at every run launch by launch.  (A captured
    step cuts contexts for the range of lengths that it serves, so its sums may round otherwise than the same step's launched alone.)"""
    from zephyr_b200 import Engine
    from zephyr_b200.engine import KvCacheOptions, PagedSchedulerConfig

    folder = model_folders("D", "bfloat16")
    prompts = [random_tokens(503, n, seed=600 + n) for n in (40, 25, 61)]

    def engine(**options):
        return Engine(folder, scheduler=PagedSchedulerConfig(max_num_seqs=3, max_num_batched_tokens=64, max_prefill_chunk_tokens=64),
                      kv_cache=KvCacheOptions(block_size=16, bits=4, **options))

    tight = engine(num_blocks=11)          # 176 positions for sequences that grow to 64, 49 and 85
    tight.runner.poison_freed_pages = True
    runs = []
    for graphs in (True, True, False, False):
        tight.runner.use_cuda_graphs = graphs
        runs.append([list(o.token_ids) for o in tight.generate(prompts, max_tokens=24, temperature=0.0, ignore_eos=True)])
    assert tight.stats.preemptions > 0 and all(len(tokens) == 24 for run in runs for tokens in run)
    assert runs[2] == runs[3]
    tight.runner.manager.check_invariants()
    # 2 layers of 2 key/value heads: 160 bytes a position, head and layer, where bfloat16 takes 512
    sized = engine(memory_bytes=200 * 16 * 2 * 2 * 160)
    assert sized.runner.manager.num_free_pages() == 192 and sized.runner.cache_bytes_per_token() == 640
    assert [list(o.token_ids) for o in sized.generate(prompts[:1], max_tokens=24, temperature=0.0, ignore_eos=True)][0]


def test_the_timing_program_times_it(cuda_device, capsys):
    import json

    from zephyr_b200.kernels import timing

    assert timing.main(["packed_cache", "--warmup", "1", "--iters", "2", "--batch", "2", "--context", "300", "--tokens", "70", "--head-dim", "64"]) == 0
    line = json.loads(capsys.readouterr().out)
    assert set(line["us"]) == {"decode", "decode_bfloat16", "prompt", "prompt_bfloat16", "write", "write_bfloat16", "read_back"}
