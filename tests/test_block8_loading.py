"""Bringing a model into 8-bit matrices: a layer at a time, so that a model that fits on the device in 8 bits only can be loaded."""

import dataclasses

import pytest
import torch

import plain_block8 as plain
from test_block8_gpu import _close
from tiny_configs import tiny_config
from zephyr_b200.config import WeightError
from zephyr_b200.kernels import ops
from zephyr_b200.parts import Model, expected_weights, with_weight_bits
from zephyr_b200.weights import RandomWeights, WeightDecl, load_weights
from zephyr_b200.weights.loader import WeightsOnDemand


class Counted(RandomWeights):
    def __init__(self, *args, **options):
        super().__init__(*args, **options)
        self.reads = []

    def read(self, name):
        self.reads.append(name)
        return super().read(name)


def test_weights_on_demand():
    decls = {"a": WeightDecl((3, 4)), "b": WeightDecl((5,)), "c": WeightDecl((2, 2))}
    store = Counted(decls, 1, torch.float32)
    weights = WeightsOnDemand(store, decls, torch.bfloat16, "cpu")
    assert store.reads == [] and list(weights) == ["a", "b", "c"] and len(weights) == 3 and "b" in weights and "d" not in weights
    a = weights["a"]
    assert a is weights["a"] and a.dtype == torch.bfloat16 and weights["b"].dtype == torch.float32 and store.reads == ["a", "b"]
    weights.let_go(["a", "c"])
    assert torch.equal(weights["a"], a) and weights["a"] is not a and store.reads == ["a", "b", "a"]
    with pytest.raises(KeyError):
        weights["d"]
    everything = load_weights(store, decls, torch.bfloat16, "cpu")
    assert list(everything) == list(decls) and all(torch.equal(everything[n], weights[n]) for n in decls)
    for wrong in ({**decls, "d": WeightDecl((1,))}, {"a": decls["a"]}, {**decls, "a": WeightDecl((4, 3))}):
        with pytest.raises(WeightError):
            WeightsOnDemand(store, wrong, torch.bfloat16, "cpu")
    with pytest.raises(WeightError):
        WeightsOnDemand(store, decls, torch.float16, "cpu")


@pytest.mark.gpu
def test_a_model_in_8_bits_is_loaded_a_layer_at_a_time(cuda_device):
    layers = 12
    spec = with_weight_bits(dataclasses.replace(tiny_config("E"), num_hidden_layers=layers).to_model_spec(), 8)
    expected = expected_weights(spec)
    store = Counted(expected, 5, device=cuda_device)
    in_bfloat16 = sum(2 * torch.Size(decl.shape).numel() for decl in expected.values())
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    model = Model.load(spec, store, torch.bfloat16, cuda_device)
    torch.cuda.synchronize()
    peak, kept = torch.cuda.max_memory_allocated() - before, torch.cuda.memory_allocated() - before
    # Codes take half, scales 512 bytes for 64 KB of them; every layer has tables of a rotation (float32, cosines and sines of 64 channels at 1024 positions); the
    # allocator gives a tensor up to 1 MB more than it asks for where it hands out what was freed: four matrices a layer and the table of embeddings.
    matrices = 2 * layers * (4096 * 1024 + 1024 * 2048 + 3 * 3072 * 1024)
    most = matrices * (0.5 + 1 / 256) + (in_bfloat16 - matrices) + layers * 2 * 1024 * 64 * 4 + (4 * layers + 1) * 2 ** 20
    # Beside that, of one layer of twelve its tensors, their fused copies and its codes: three layers at most.
    assert kept < most and peak < most + 3 * matrices / layers and most + 3 * matrices / layers < in_bfloat16
    assert sorted(store.reads) == sorted(expected)
    # The same model as from tensors that all lie there.
    other = Model(spec, load_weights(store, expected, torch.bfloat16, cuda_device), torch.bfloat16, cuda_device)
    for mine, theirs in zip(model.layers, other.layers):
        for part, name in (("mixer", "w_qkv"), ("mixer", "w_o"), ("feed_forward", "w_gate_up"), ("feed_forward", "w_down")):
            a, b = getattr(getattr(mine, part), name), getattr(getattr(theirs, part), name)
            assert isinstance(a, ops.BlockMatrix) and a.shape == b.shape and torch.equal(a.data, b.data)
    assert torch.equal(model.output.weights_read()[0], other.output.weights_read()[0])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_the_queries_rows_take_no_memory_of_their_own(cuda_device, name):
    """64, 192 and 512 rows of queries: within a block of 128, with a part of one, whole blocks."""
    spec = with_weight_bits(tiny_config(name).to_model_spec(), 8)
    model = Model.load(spec, RandomWeights(expected_weights(spec), 5, device=cuda_device), torch.bfloat16, cuda_device)
    for layer in model.layers:
        mixer = layer.mixer
        queries = mixer.nh * mixer.hd
        assert mixer.w_q.data is mixer.w_qkv.data and mixer.w_q.shape == (queries, mixer.hidden)
        assert torch.equal(mixer.w_q.values(), mixer.w_qkv.values()[:queries])
        values = mixer.w_q.values(torch.float32).double()
        for m in (1, 12, 50, 300):
            x = torch.randn((m, mixer.hidden), device=cuda_device, generator=torch.Generator(device="cuda").manual_seed(m))
            want, magnitude = plain.product(x, values)
            _close(ops.block_linear(x, mixer.w_q), want, plain.sum_error(mixer.hidden) * magnitude, torch.float32)
