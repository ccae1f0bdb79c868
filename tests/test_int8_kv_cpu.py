"""Host-side checks of the int8 linear and the 8-bit key/value cache that need
no GPU: every refusal comes before any device access."""

import pytest
import torch

from nanosglang_b200 import _lib, ops

FAKE = 0x100000  # never dereferenced: validation fails before any device access


def _int8(x=FAKE, xd=1, m=4, k=64, n=48, w=FAKE, ws=FAKE, b=None, bd=-1, y=FAKE, work=FAKE, nbytes=1 << 20):
    return _lib.load().nsq_int8_linear(x, xd, m, k, n, w, ws, b, bd, y, work, nbytes, None)


def test_int8_linear_refusals():
    assert _int8(xd=2) == _lib.EINVAL  # fp32 activations
    assert _int8(m=-1) == _lib.EINVAL
    assert _int8(n=0) == _lib.EINVAL
    assert _int8(k=72) == _lib.ENOTSUP  # rows of 16 bytes
    assert _int8(k=131088) == _lib.ENOTSUP  # int32 sums
    assert _int8(b=FAKE) == _lib.EINVAL  # a bias without its type
    assert _int8(x=None) == _lib.EINVAL
    assert _int8(w=FAKE + 8) == _lib.EALIGN
    assert _int8(m=0) == _lib.OK  # nothing to do, needs no device
    lib = _lib.load()
    size = lib.nsq_int8_linear_workspace_size
    assert size(9, 48, 16) == 9 * 48 + 9 * 4
    assert size(8, 528, 16) == 8 * 528 + 8 * 4
    assert size(8, 512, 16) == size(8, 512, 4096) == 0  # one launch
    assert size(8, 512, 4112) == 8 * 512 + 8 * 4
    assert size(0, 48, 16) == size(4, 48, 0) == 0
    assert lib.nsq_int8_quantize(FAKE, 7, 1, 8, FAKE, FAKE, None) == _lib.EINVAL
    assert lib.nsq_int8_quantize(FAKE, 1, 1, 0, FAKE, FAKE, None) == _lib.EINVAL
    assert lib.nsq_int8_quantize(FAKE, 1, 0, 8, FAKE, FAKE, None) == _lib.OK
    assert lib.nsq_int8_linear_quantized(None, FAKE, 2, 64, 8, FAKE, FAKE, None, -1, FAKE, 1, None) == _lib.EINVAL


def _desc(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, num_pages=8, page_size=16, kv_heads=2, head_dim=64,
             k_stride=(2048, 128, 64), v_stride=(2048, 128, 64), k_scale_stride=(32, 2, 1),
             v_scale_stride=(32, 2, 1), codes=0)
    d.update(kw)
    flat = [x for v in d.values() for x in (v if isinstance(v, tuple) else (v,))]
    return _lib.KV_CACHE.pack(*flat)


@pytest.mark.parametrize("change,expect", [
    ({"codes": 2}, _lib.EINVAL), ({"k": 0}, _lib.EINVAL), ({"num_pages": 0}, _lib.EINVAL),
    ({"head_dim": 72}, _lib.ENOTSUP), ({"head_dim": 272}, _lib.ENOTSUP), ({"num_pages": 1 << 28}, _lib.ENOTSUP),
    ({"v": FAKE + 8}, _lib.EALIGN), ({"k_stride": (2048, 136, 64)}, _lib.EALIGN),
    ({"k_stride": (1 << 32, 128, 64)}, _lib.ENOTSUP), ({"v_scale_stride": (-1, 1, 1)}, _lib.EINVAL)])
def test_cache_descriptor_refusals(change, expect):
    lib = _lib.load()
    d = _desc(**change)
    assert lib.nsq_kv_cache_write(d, FAKE, FAKE, 1, 128, 64, 128, 64, 4, FAKE, None) == expect
    assert lib.nsq_kv_cache_read(d, FAKE, 4, FAKE, FAKE, 1, None) == expect
    assert lib.nsq_kv_attention_decode(d, FAKE, 1, 128, 64, 2, 4, FAKE, 4, 4, FAKE, 0.125, FAKE, None, FAKE, 1 << 30,
                                       None) == expect


def test_cache_call_refusals():
    lib = _lib.load()
    d = _desc()
    write = lambda k=FAKE, xd=1, st=128, t=4, sl=FAKE: lib.nsq_kv_cache_write(  # noqa: E731
        d, k, FAKE, xd, st, 64, 128, 64, t, sl, None)
    assert write(xd=2) == _lib.EINVAL
    assert write(k=FAKE + 2) == _lib.EALIGN
    assert write(st=132) == _lib.EALIGN
    assert write(st=-128) == _lib.EINVAL
    assert write(t=-1) == _lib.EINVAL
    assert write(sl=None) == _lib.EINVAL
    assert write(t=1 << 31) == _lib.ENOTSUP
    assert write(t=0) == _lib.OK
    att = lambda q=FAKE, b=2, h=4, w=4, sc=0.125, ws=FAKE, nb=1 << 30: lib.nsq_kv_attention_decode(  # noqa: E731
        d, q, 1, 128, 64, b, h, FAKE, w, w, FAKE, sc, FAKE, None, ws, nb, None)
    assert att(h=3) == _lib.EINVAL  # not a multiple of kv_heads
    assert att(sc=float("nan")) == _lib.EINVAL
    assert att(sc=float("inf")) == _lib.EINVAL
    assert att(q=FAKE + 2) == _lib.EALIGN
    assert att(w=1 << 30) == _lib.ENOTSUP
    assert att(b=1 << 28) == _lib.ENOTSUP
    assert att(b=0) == _lib.OK


def test_attention_workspace_size():
    size = _lib.load().nsq_kv_attention_workspace_size
    assert size(4, 8, 2, 64, 16, 8) == 0  # 128 tokens at most: no item is cut
    assert size(4, 8, 2, 64, 16, 9) > 0
    assert size(0, 8, 2, 64, 16, 5) == 0
    # bounded by the machine, not by the batch or the length
    assert size(4096, 64, 8, 128, 16, 8192) <= 2400 * 2 * (8 * 132 * 4 + 16)
    assert size(1, 12, 1, 128, 16, 65536) <= 2400 * 2 * (16 * 132 * 4 + 16)


def test_ops_refuse_cpu_tensors():
    x = torch.randn(2, 64, dtype=torch.bfloat16)
    w, ws = torch.zeros(16, 64, dtype=torch.int8), torch.ones(16)
    cache, scale = torch.zeros(4, 16, 2, 64, dtype=torch.int8), torch.zeros(4, 16, 2)
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    slots = torch.arange(2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.int8_quantize(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.int8_linear(x, w, ws)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.int8_linear_quantized(w, ws, w, ws)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.kv_cache_write(rows, rows, cache, cache, scale, scale, slots)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.kv_cache_read(cache, cache, scale, scale, slots, torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.kv_attention_decode(rows, cache, cache, scale, scale, torch.zeros(2, 4, dtype=torch.int32),
                                torch.zeros(2, dtype=torch.int32))
