"""Which models are held in 8-bit matrices and which are refused, by name; that every part of those takes part; what experts with weights on their inputs
give; captured steps beside steps launch by launch."""

import pytest
import torch

import legelix_models
import plain_block8 as plain
from replay_util import random_tokens, trace_mixed
from test_block8_engine_gpu import MODELS, Checked, _replay, _runner
from test_block8_gpu import HALF_STEP
from zephyr_b200.config import ConfigError
from zephyr_b200.kernels import ops

pytestmark = pytest.mark.gpu
F64 = torch.float64

# Inner sizes of 50, 36, 36, 50, 27, 27 and 13: gate and up rows that cannot be laid out in blocks of 8.
REFUSED = [("gefovik", "B"), ("fekotar", "B"), ("rizovik", "A"), ("rizovik", "B"), ("legilix", "B"), ("tedulorn", "A"), ("tedulorn", "B")]
ALL = [(f, n) for f, m in MODELS.items() for n in m.CONFIGS] + [("legelix", n) for n in legelix_models.CONFIGS]
HELD = [c for c in ALL if c not in REFUSED]
# Attention whose captured steps cut these contexts otherwise than steps launch by launch, so that sums round otherwise and codes flip.
CUT_OTHERWISE = [("tedulorn", "C")]
LENGTHS = (40, 90, 7)
# What stays in the model's type among matrices: products head by head, routers, convolutions, low ranks, mixes of heads.
KEPT = {"w_q_to_latent", "w_latent_to_v", "w_router", "conv_w", "w_a2", "head_mix", "score_mix"}


def _made(tmp_path, family, name, graphs=False):
    module = legelix_models if family == "legelix" else MODELS[family]
    config, page = module.CONFIGS[name], module.PAGE_SIZE[name]
    extra = (module.DECAY_RANK[name],) if family == "legelix" else ()
    tmp_path.mkdir(exist_ok=True)
    folder = module.write_model(tmp_path, config, *extra, seed=3, dtype=torch.bfloat16)
    return _runner(folder, page, sum(-(-n // page) for n in LENGTHS) + 1, 3, graphs)


def _trace():
    return trace_mixed({f"r{i}": random_tokens(40, n, seed=800 + n) for i, n in enumerate(LENGTHS)})


class CheckedWeights(Checked):
    """Experts with weights on their inputs are compared too."""

    def routed(self, x, ids, weights, gate_up, down, act, weigh_inputs, bounded):
        got = super().routed(x, ids, weights, gate_up, down, act, weigh_inputs, bounded)
        if weigh_inputs:
            self._count("weighed experts", x)
            up, out = gate_up.values(torch.float32).to(F64), down.values(torch.float32).to(F64)
            want, error = torch.zeros(x.shape, dtype=F64, device=x.device), torch.zeros(x.shape, dtype=F64, device=x.device)
            for e in ids.unique().tolist():
                token, choice = torch.nonzero(ids == e, as_tuple=True)
                weight = weights[token, choice].to(F64)[:, None]
                sums, magnitude = plain.product(x[token], up[e])
                sums, off = sums * weight, (plain.sum_error(gate_up.K) + 2.0 ** -23) * magnitude * weight.abs()
                hidden, off = plain.gated(sums, act), plain.gated_error(sums, off, act)
                y, size = plain.product(hidden, out[e])
                off = plain.code_spread(hidden, off) @ out[e].abs().t() * (1 + 1e-4) + plain.sum_error(down.K) * size * 1.01
                want[token] += y
                error[token] += off + HALF_STEP[x.dtype] * (y.abs() + off) + 2.0 ** -22 * y.abs()
            self._compare(got, want, error)
        return got


@pytest.mark.parametrize("family,name", REFUSED)
def test_models_that_are_refused(tmp_path, cuda_device, family, name):
    with pytest.raises(ConfigError, match="multiple of 8"):
        _made(tmp_path, family, name)


@pytest.mark.parametrize("family,name", HELD)
def test_every_part_takes_part(tmp_path, cuda_device, monkeypatch, family, name):
    runner = _made(tmp_path, family, name)
    kinds = []
    for block in runner.model.layers:
        parts = [block.mixer, *getattr(block.mixer, "branches", ()), block.feed_forward, getattr(block.feed_forward, "shared", None)]
        kinds += [type(part).__name__ for part in parts[-2:] if part is not None]
        for part in parts:
            for attribute, value in (vars(part).items() if part is not None else ()):
                if attribute in part.block_matrices:
                    assert value is None or isinstance(value, ops.BlockMatrix), attribute
                elif isinstance(value, torch.Tensor) and value.dtype == torch.bfloat16 and value.dim() >= 2 and value.numel() > 0:
                    assert attribute in KEPT, attribute
    checked = CheckedWeights(monkeypatch)
    steps = list(_trace())
    _replay(runner, steps)
    gated, routed, plain_ones = (kinds.count(kind) for kind in ("SwiGLU", "RoutedFeedForward", "UngatedFeedForward"))
    assert checked.calls.get("feed-forward", 0) == gated * len(steps) and checked.calls.get("experts", 0) == routed * len(steps)
    assert checked.calls["linear"] >= (len(runner.model.layers) + 2 * plain_ones) * len(steps)
    weighed = [block.feed_forward for block in runner.model.layers if getattr(block.feed_forward, "weigh", "outputs") == "inputs"]
    assert checked.calls.get("weighed experts", 0) == len(weighed) * len(steps) and (weighed or family != "legilix")


@pytest.mark.parametrize("family,name", [c for c in HELD if c not in CUT_OTHERWISE])
def test_captured_steps_give_what_steps_launch_by_launch_give(tmp_path, cuda_device, family, name):
    results = []
    for graphs in (False, True):
        runner = _made(tmp_path / str(graphs), family, name, graphs)
        logits, step = [], runner.step
        runner.step = lambda entries: logits.append(step(entries).clone()) or logits[-1]
        for _ in range(3):                        # (a shape is captured when it comes again)
            _replay(runner, _trace())
        results.append(logits)
        assert not graphs or any(record["graph"] is not None for record in runner._graphs.values())
    assert len(results[0]) == len(results[1]) and all(torch.equal(a, b) for a, b in zip(*results))


def test_generation_with_captured_steps_repeats_itself(model_folders, cuda_device):
    """Once a step's shape is captured the same requests give the same tokens."""
    from zephyr_b200 import Engine
    from zephyr_b200.engine import KvCacheOptions, PagedSchedulerConfig

    prompts = [random_tokens(503, n, seed=900 + n) for n in (40, 25, 61)]
    for bits in (None, 4):
        engine = Engine(model_folders("D", "bfloat16"), scheduler=PagedSchedulerConfig(max_num_seqs=3, max_num_batched_tokens=64, max_prefill_chunk_tokens=64),
                        kv_cache=KvCacheOptions(block_size=16, num_blocks=60, bits=bits), weight_bits=8)
        engine.runner.use_cuda_graphs = True
        runs = [[list(o.token_ids) for o in engine.generate(prompts, max_tokens=24, temperature=0.0, ignore_eos=True)] for _ in range(4)]
        assert runs[2] == runs[3]
