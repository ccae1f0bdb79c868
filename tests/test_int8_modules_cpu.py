"""Host logic of the 8-bit modules that needs no GPU: buffer layout, the
quantize_model walk, shards, refusals."""

import pytest
import torch
import torch.nn as nn

import nanosglang_b200
from nanosglang_b200 import quantization as Q
from nanosglang_b200 import tensor_parallel as TP
from nanosglang_b200.kv_cache import QuantizedKVCache


def test_int8_buffers_and_state_dict():
    m = Q.Int8Linear(96, 40, bias=True)
    assert m.weight_int8.shape == (40, 96) and m.weight_int8.dtype == torch.int8
    assert m.weight_scale.shape == (40,) and m.weight_scale.dtype == torch.float32
    assert sorted(m.state_dict()) == ["bias", "weight_int8", "weight_scale"]
    assert Q.Int8Linear(96, 40).bias is None and nanosglang_b200.Int8Linear is Q.Int8Linear
    m.weight_int8.copy_(torch.randint(-127, 128, (40, 96), dtype=torch.int8))
    m.weight_scale.copy_(torch.rand(40))
    other = Q.Int8Linear(96, 40, bias=True)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.weight_int8, m.weight_int8)
    assert torch.equal(m.dequantize(torch.float32), m.weight_int8.float() * m.weight_scale[:, None])


def test_cpu_fails_loudly():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Q.Int8Linear(64, 16)(torch.randn(2, 64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Q.Int8Linear.from_linear(nn.Linear(64, 16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Q.quantize_model(nn.ModuleDict({"layer": nn.ModuleDict({"q_proj": nn.Linear(64, 64)})}), "int8")
    with pytest.raises(ValueError, match="Unknown quantization method"):
        Q.quantize_model(nn.ModuleDict({"layer": nn.ModuleDict({"q_proj": nn.Linear(64, 64)})}), "int4")


@pytest.mark.parametrize("ws", [2, 4])
def test_int8_shards_are_slices(ws):
    m = Q.Int8Linear(256, 64, bias=True)
    m.weight_int8.copy_(torch.randint(-127, 128, (64, 256), dtype=torch.int8))
    m.weight_scale.copy_(torch.rand(64) + 0.1)
    m.bias.data.copy_(torch.randn(64))
    for r in range(ws):
        col = TP.shard_linear_rows(m, ws, r)
        n = 64 // ws
        assert torch.equal(col.weight_int8, m.weight_int8[n * r:n * (r + 1)]) and col.weight_int8.is_contiguous()
        assert torch.equal(col.weight_scale, m.weight_scale[n * r:n * (r + 1)])
        assert torch.equal(col.bias, m.bias[n * r:n * (r + 1)]) and (col.in_features, col.out_features) == (256, n)
        row = TP.shard_linear_cols(m, ws, r, keep_bias=r == 0)
        k = 256 // ws
        assert torch.equal(row.weight_int8, m.weight_int8[:, k * r:k * (r + 1)]) and row.weight_int8.is_contiguous()
        assert torch.equal(row.weight_scale, m.weight_scale) and (row.bias is not None) == (r == 0)
        assert row.in_features == k
    with pytest.raises(ValueError, match="not divisible"):
        TP.shard_linear_rows(m, 3, 0)


def test_cache_shapes_and_refusals():
    c = QuantizedKVCache(5, 16, 3, 64, "fp8", "cpu")
    assert c.k.shape == c.v.shape == (5, 16, 3, 64) and c.k.dtype == torch.float8_e4m3fn
    assert c.k_scale.shape == c.v_scale.shape == (5, 16, 3) and c.k_scale.dtype == torch.float32
    assert c.k[0, :, 0].is_contiguous() and c.k.data_ptr() != c.v.data_ptr()  # head-major
    assert QuantizedKVCache(5, 16, 3, 64, device="cpu").k.dtype == torch.int8
    with pytest.raises(ValueError):
        QuantizedKVCache(5, 16, 3, 64, "int4", "cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache(5, 16, 3, 72, "int8", "cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        c.write(torch.zeros(1, 3, 64).half(), torch.zeros(1, 3, 64).half(), torch.zeros(1, dtype=torch.int64))
