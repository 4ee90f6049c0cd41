"""Matrices in 8-bit floating point on the host: layouts, what is refused, options.  (No GPU.)"""

import dataclasses

import pytest
import torch

import plain_block8 as plain
from tiny_configs import tiny_config
from zephyr_b200.cli import build_parser
from zephyr_b200.config import ConfigError, InvalidArgumentError
from zephyr_b200.kernels import ops
from zephyr_b200.parts import with_weight_bits
from zephyr_b200.parts.base import Part


def _matrix(*shape):
    return ops.BlockMatrix._empty(shape, "cpu")


def test_layout():
    m = _matrix(300, 1100)
    assert m.codes.shape == (1, 3, 9, 128, 128) and m.scales.shape == (1, 3, 3, 512) and m.shape == (300, 1100) and m.matrices == 1
    several = _matrix(4, 129, 16)
    assert several.codes.shape == (4, 2, 1, 128, 128) and several.scales.shape == (4, 2, 1, 512) and several.matrices == 4
    assert m.exponents().shape == (3, 9) and several.exponents().shape == (4, 2, 1)
    m.exponents().copy_(torch.arange(27, dtype=torch.uint8).view(3, 9))
    parts = [t.data_ptr() for t in (m.codes, m.scales, m.exponents())]
    assert parts == [m.data.data_ptr(), m.data.data_ptr() + 27 * 128 * 128, m.data.data_ptr() + 27 * 128 * 128 + 9 * 512]
    assert parts[:2] == [m.codes_at, m.scales_at] and m.data.numel() == 27 * 128 * 128 + 9 * 512 + 27
    first = m.first_rows(256)
    assert first.shape == (256, 1100) and first.codes.data_ptr() == m.codes.data_ptr() and first.scales.shape == (1, 2, 3, 512)
    assert torch.equal(first.exponents(), m.exponents()[:2]) and m.first_rows(300).shape == m.shape
    for rows in (0, 100, 301, 384):
        with pytest.raises(InvalidArgumentError):
            m.first_rows(rows)
    with pytest.raises(InvalidArgumentError):
        several.first_rows(128)


@pytest.mark.parametrize("shape", [(3,), (0, 4), (4, 0), (2, 0, 4), (1, 2, 3, 4)])
def test_matrices_that_are_refused(shape):
    with pytest.raises(InvalidArgumentError):
        ops.pack_matrix(torch.zeros(shape))
    with pytest.raises(InvalidArgumentError):
        ops.BlockMatrix._empty(shape, "cpu")


def test_what_a_call_refuses(monkeypatch):
    from zephyr_b200.kernels.ops import KernelError
    gate_up, down, x = _matrix(64, 48), _matrix(48, 32), torch.zeros(5, 48)
    with pytest.raises(KernelError):                                   # no CPU path
        ops.pack_matrix(torch.zeros(4, 4))
    with pytest.raises(KernelError):
        ops.block_linear(x, gate_up)
    with pytest.raises(KernelError):
        ops.BlockMatrix.from_codes(torch.zeros((4, 4), dtype=torch.uint8), torch.ones((1, 1), dtype=torch.uint8))
    for w in (torch.zeros(4, 4, dtype=torch.float16), torch.zeros(8, 8).t()[:, :4]):
        with pytest.raises(InvalidArgumentError):
            ops.pack_matrix(w)
    for bad in (torch.zeros(5, 47), torch.zeros(48), torch.zeros(5, 48, dtype=torch.float16), torch.zeros(48, 5).t(), torch.zeros(1, 48).expand(5, 48)):
        with pytest.raises(InvalidArgumentError):
            ops.block_linear(bad, gate_up)
    bounded = ops.BoundedGate(None, 7.0, 1.0, 0.0)
    for w, options in ((_matrix(2, 64, 48), {}), (gate_up, dict(out_dtype=torch.float16)), (gate_up, dict(swiglu=True, act="gelu")), (_matrix(24, 48), dict(swiglu=True)),
                       (gate_up, dict(bounded=bounded)), (gate_up, dict(product_act="silu")), (gate_up, dict(swiglu=True, product_act="gelu_tanh")),
                       (gate_up, dict(swiglu=True, bounded=dataclasses.replace(bounded, limit=0.0))),
                       (gate_up, dict(swiglu=True, bounded=dataclasses.replace(bounded, bias=torch.zeros(3))))):
        with pytest.raises(InvalidArgumentError):
            ops.block_linear(x, w, **options)
    for pair in ((gate_up, _matrix(48, 31)), (_matrix(1, 64, 48), _matrix(1, 48, 32)), (_matrix(2, 64, 48), down)):
        if pair[0].matrices != 1 or pair[1].K != 32:
            with pytest.raises(InvalidArgumentError):
                ops.block_feed_forward(x, *pair)
    ids, weights = torch.zeros((5, 2), dtype=torch.int32), torch.ones((5, 2))
    up, out = _matrix(3, 64, 48), _matrix(3, 48, 32)
    for args in ((x, ids.long(), weights, up, None, out), (x, ids, weights.double(), up, None, out), (x, ids[:4], weights[:4], up, None, out),
                 (x, ids, weights, up, up, out), (x, ids, weights, up, None, torch.zeros(3, 48, 32)), (x, ids, weights, up, None, _matrix(2, 48, 32)),
                 (x, ids, weights, gate_up, None, down), (x, ids, weights, _matrix(3, 24, 48), None, _matrix(3, 48, 12)), (x[:, :47], ids, weights, up, None, out)):
        with pytest.raises(InvalidArgumentError):
            ops.routed_experts(*args)
    for options in (dict(act="gelu"), dict(bounded=dataclasses.replace(bounded, limit=-1.0)), dict(bounded=dataclasses.replace(bounded, bias=torch.zeros(64))),
                    dict(bounded=bounded, weigh_inputs=True)):
        with pytest.raises(InvalidArgumentError):
            ops.routed_experts(x, ids, weights, up, None, out, **options)


def test_options():
    spec = tiny_config("D").to_model_spec()
    assert spec.weight_bits == 0 and with_weight_bits(spec, 8).weight_bits == 8
    for bits in (4, 0, 16):
        with pytest.raises(ConfigError):
            with_weight_bits(spec, bits)
    parser = build_parser()
    assert parser.parse_args(["generate", "m", "--prompt-ids", "1"]).weight_bits is None
    assert parser.parse_args(["generate", "m", "--prompt-ids", "1", "--weight-bits", "8"]).weight_bits == 8
    with pytest.raises(SystemExit):
        parser.parse_args(["generate", "m", "--prompt-ids", "1", "--weight-bits", "4"])
    assert not Part().hold_in_8_bits()


def test_the_plain_codes():
    """Every e4m3 number stands for itself, what lies between goes to the nearer, ties to the even code."""
    numbers = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    finite = numbers[numbers.isfinite()]
    assert torch.equal(plain.e4m3(finite), finite)
    ordered = finite.unique()
    middle = (ordered[1:] + ordered[:-1]) / 2
    assert torch.equal(plain.e4m3(middle), middle.float().to(torch.float8_e4m3fn).double())
    assert torch.equal(plain.e4m3(middle - middle.abs() * 1e-9), ordered[:-1]) and torch.equal(plain.e4m3(middle + middle.abs() * 1e-9), ordered[1:])
    tops = torch.tensor([448.0, 448.1, 1.0, 1.75, 1.7500001, 0.0, 1e-300], dtype=torch.float64)
    assert plain.block_power(tops).tolist() == [0, 1, -8, -8, -7, -126, -126]
