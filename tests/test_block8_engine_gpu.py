"""Whole models whose matrices are held in 8-bit floating point.  Codes are discontinuous in what they encode, so no model is asked to follow another
one through its layers: every product that a step asks for is checked against 64 bits at the inputs it was given, in prompts, portions, mixed
batches and single tokens, and the engine runs them captured and not."""

import pytest
import torch

import fekotar_models
import gefovik_models
import legelix_models
import legilix_models
import plain_block8 as plain
import rizovik_models
import tedulorn_models
from replay_util import random_tokens, trace_batched_tail, trace_mixed
from test_block8_gpu import HALF_STEP, _feed_forward
from zephyr_b200.config import ConfigError
from zephyr_b200.kernels import ops

pytestmark = pytest.mark.gpu
F64 = torch.float64


def _runner(folder, page_size, pages, requests, graphs):
    from zephyr_b200.config import load_model_spec
    from zephyr_b200.engine.runner import ModelRunner
    from zephyr_b200.parts import Model, with_weight_bits
    from zephyr_b200.weights import Checkpoint

    spec = with_weight_bits(load_model_spec(folder), 8)
    model = Model.load(spec, Checkpoint(folder), torch.bfloat16, torch.device("cuda", 0))
    runner = ModelRunner(model, page_size, pages, requests, max_seq_len=min(spec.max_seq_len, pages * page_size))
    runner.use_cuda_graphs, runner.poison_freed_pages = graphs, True
    return runner


def _replay(runner, steps):
    from zephyr_b200.engine.runner import StepEntry

    for step in steps:
        entries = []
        for item in step["entries"]:
            if item["id"] not in runner.manager:
                assert runner.add_request(item["id"])
            entries.append(StepEntry(item["id"], item["tokens"], item["want"]))
        logits = runner.step(entries)
        runner.check()
        assert bool(logits.isfinite().all())
        for request_id in step["end"]:
            runner.free_request(request_id)


class Checked:
    """The calls that take a ``BlockMatrix``, each checked when it is made."""

    def __init__(self, monkeypatch):
        self.calls, self.rows = {}, set()
        self.real = {name: getattr(ops, name) for name in ("block_linear", "block_feed_forward", "_routed_blocks")}
        monkeypatch.setattr(ops, "block_linear", self.linear)
        monkeypatch.setattr(ops, "block_feed_forward", self.feed_forward)
        monkeypatch.setattr(ops, "_routed_blocks", self.routed)
        self.inside = False

    def _count(self, name, x):
        self.calls[name] = self.calls.get(name, 0) + 1
        self.rows.add(x.shape[0])

    def _compare(self, got, want, error):
        bound = error + HALF_STEP[got.dtype] * (want.abs() + error) + 2.0 ** -133
        assert bool(((got.to(F64) - want).abs() <= bound).all())

    def linear(self, x, w, out_dtype=None, **options):
        got = self.real["block_linear"](x, w, out_dtype, **options)
        if not self.inside:
            self._count("linear", x)
            want, magnitude = plain.product(x, w.values(torch.float32).to(F64))
            error = plain.sum_error(w.K) * magnitude
            if options:
                assert options == dict(product_act="relu_squared") or options == dict(product_act="gelu_tanh")
                if options["product_act"] == "relu_squared":
                    error, want = (2 * want.abs() + error) * error + 2.0 ** -22 * want ** 2, want.clamp(min=0) ** 2
                else:
                    error = 1.2 * error + 2.0 ** -18 * want.abs()
                    want = 0.5 * want * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (want + 0.044715 * want ** 3)))
            self._compare(got, want, error)
        return got

    def feed_forward(self, x, gate_up, down, act="silu", bounded=None, out_dtype=None):
        self.inside = True
        got = self.real["block_feed_forward"](x, gate_up, down, act=act, bounded=bounded, out_dtype=out_dtype)
        self.inside = False
        self._count("feed-forward", x)
        limits = (bounded.limit, bounded.alpha, bounded.shift) if bounded is not None else None
        bias = bounded.bias if bounded is not None else None
        self._compare(got, *_feed_forward(x, gate_up.values(torch.float32).to(F64), down.values(torch.float32).to(F64),
                                          "bounded" if bounded is not None else act, limits, bias))
        return got

    def routed(self, x, ids, weights, gate_up, down, act, weigh_inputs, bounded):
        got = self.real["_routed_blocks"](x, ids, weights, gate_up, down, act, weigh_inputs, bounded)
        self._count("experts", x)
        assert not weigh_inputs or bounded is None
        if not weigh_inputs:
            limits = (bounded.limit, bounded.alpha, bounded.shift) if bounded is not None else None
            up, out = gate_up.values(torch.float32).to(F64), down.values(torch.float32).to(F64)
            want, error = torch.zeros(x.shape, dtype=F64, device=x.device), torch.zeros(x.shape, dtype=F64, device=x.device)
            for e in ids.unique().tolist():
                token, choice = torch.nonzero(ids == e, as_tuple=True)
                weight = weights[token, choice].to(F64)[:, None]
                y, off = x[token].to(F64), 0.0
                if e < gate_up.matrices:
                    y, off = _feed_forward(x[token], up[e], out[e], "bounded" if bounded is not None else act, limits)
                    off = off + HALF_STEP[x.dtype] * (y.abs() + off)
                want[token] += weight * y
                error[token] += weight.abs() * off + 2.0 ** -22 * (weight * y).abs()
            self._compare(got, want, error)
        return got


@pytest.mark.parametrize("name", ["B", "D"])
def test_qwen3_in_8_bits(model_folders, cuda_device, monkeypatch, name):
    runner = _runner(model_folders(name, "bfloat16"), 16, 60, 4, False)
    assert runner.model.chains is None and all(isinstance(b.mixer.w_qkv, ops.BlockMatrix) for b in runner.model.layers)
    checked = Checked(monkeypatch)
    requests = {f"r{i}": random_tokens(300, n, seed=700 + n) for i, n in enumerate((33, 140, 9, 5))}
    _replay(runner, trace_mixed(requests))
    assert checked.calls["linear"] > 20 and checked.calls["feed-forward"] > 10 and min(checked.rows) <= 4 and max(checked.rows) > 16


MODELS = {"gefovik": gefovik_models, "fekotar": fekotar_models, "rizovik": rizovik_models, "legilix": legilix_models, "tedulorn": tedulorn_models}


@pytest.mark.parametrize("family,name", [(f, n) for f, m in MODELS.items() for n in m.CONFIGS] + [("legelix", n) for n in legelix_models.CONFIGS])
def test_other_models_in_8_bits(tmp_path, cuda_device, monkeypatch, family, name):
    if family == "legelix":
        config, page = legelix_models.CONFIGS[name], legelix_models.PAGE_SIZE[name]
        folder = legelix_models.write_model(tmp_path, config, legelix_models.DECAY_RANK[name], seed=3, dtype=torch.bfloat16)
    else:
        module = MODELS[family]
        config, page = module.CONFIGS[name], module.PAGE_SIZE[name]
        folder = module.write_model(tmp_path, config, seed=3, dtype=torch.bfloat16)
    lengths = (40, 90, 7)
    try:
        runner = _runner(folder, page, sum(-(-n // page) for n in lengths) + 1, 3, False)
    except ConfigError as refusal:
        assert "multiple of 8" in str(refusal)          # a feed-forward whose gate and up rows cannot be laid out in blocks of 8
        return
    checked = Checked(monkeypatch)
    _replay(runner, trace_mixed({f"r{i}": random_tokens(40, n, seed=800 + n) for i, n in enumerate(lengths)}))
    assert checked.calls["linear"] > 0 and runner.model.weight_bytes_read_per_step() > 0


def test_generation_in_8_bits(model_folders, cuda_device):
    """Through the engine, captured and not, beside a cache in 4 bits as well; the matrices take half the bytes.  (The same tokens at every run launch
    by launch: a captured step cuts contexts for the range of lengths that it serves, so its attention's sums may round otherwise.)"""
    from zephyr_b200 import Engine
    from zephyr_b200.engine import KvCacheOptions, PagedSchedulerConfig

    folder = model_folders("D", "bfloat16")
    prompts = [random_tokens(503, n, seed=900 + n) for n in (40, 25, 61)]
    read = {}
    for weight_bits, cache_bits in ((None, None), (8, None), (8, 4)):
        engine = Engine(folder, scheduler=PagedSchedulerConfig(max_num_seqs=3, max_num_batched_tokens=64, max_prefill_chunk_tokens=64),
                        kv_cache=KvCacheOptions(block_size=16, num_blocks=60, bits=cache_bits), weight_bits=weight_bits)
        runs = []
        for graphs in (True, True, False, False):
            engine.runner.use_cuda_graphs = graphs
            runs.append([list(o.token_ids) for o in engine.generate(prompts, max_tokens=24, temperature=0.0, ignore_eos=True)])
        assert all(len(tokens) == 24 for run in runs for tokens in run) and runs[2] == runs[3]
        read[weight_bits] = engine.model.weight_bytes_read_per_step()
    # Layers in bfloat16: 2 x (1024 x 256 + 256 x 512 + 3 x 520 x 256) matrices' values; codes are padded to blocks of 128 along K, and scales come on top.
    layers = 2 * (1024 * 256 + 256 * 512 + 3 * 520 * 256)
    assert read[None] - read[8] > 0.8 * layers


def test_a_captured_run_of_products(cuda_device):
    """A layer's products one behind the other, captured and replayed on new inputs, on a stream of its own, beside another captured run."""
    generator = torch.Generator(device="cuda")
    generator.manual_seed(5)
    random = lambda *shape: torch.randn(shape, generator=generator, device="cuda")
    qkv, gate_up, down = (ops.pack_matrix(random(*shape) * 0.05) for shape in ((640, 384), (2 * 264, 640), (384, 264)))
    experts = ops.pack_matrix(random(5, 2 * 72, 384) * 0.05), ops.pack_matrix(random(5, 384, 72) * 0.05)
    for m in (3, 30, 300):
        x, ids, weights = random(m, 384).bfloat16(), torch.randint(0, 5, (m, 2), generator=torch.Generator().manual_seed(m)).int().cuda(), random(m, 2).abs()

        def layer():
            y = ops.block_feed_forward(ops.linear(x, qkv), gate_up, down)
            return y, ops.routed_experts(y, ids, weights, experts[0], None, experts[1])

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            layer()
        torch.cuda.current_stream().wait_stream(stream)
        graphs, results = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with ops.capture(graph):
                results.append(layer())
            graphs.append(graph)
        for _ in range(3):
            x.copy_(random(m, 384))
            ids.copy_(torch.randint(0, 5, (m, 2)).int())
            for graph in graphs:
                graph.replay()
            with torch.cuda.stream(stream):
                stream.wait_stream(torch.cuda.current_stream())
                eager = layer()
            torch.cuda.synchronize()
            for got in results:
                assert all(torch.equal(a, b) for a, b in zip(got, eager))
    ops.check_status(ops.device_status("cuda"))


def test_the_timing_program_times_it(cuda_device, capsys):
    import json

    from zephyr_b200.kernels import timing

    for tokens in ("3", "70"):
        assert timing.main(["block_matrix", "--warmup", "1", "--iters", "2", "--tokens", tokens, "--hidden", "256", "--ffn", "384", "--experts", "4", "--top", "2"]) == 0
        line = json.loads(capsys.readouterr().out)
        assert {"product", "feed_forward", "experts", "pack", "read_back", "product_bfloat16"} <= set(line["us"])
