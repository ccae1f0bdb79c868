"""Host-side checks of the 8-bit operators that need no GPU."""

import pytest

from test_int8_kv_cpu import FAKE, _desc

from nanosglang_b200 import _lib


@pytest.mark.parametrize("what", ["k_stride", "v_stride", "k_scale_stride", "v_scale_stride"])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_write_refuses_places_that_share_memory(what, dim):
    """A stride of 0 in a dimension of more than one: rows would overwrite one
    another. Of a dimension of one it is not looked at."""
    lib = _lib.load()
    strides = [2048, 128, 64] if "scale" not in what else [32, 2, 1]
    strides[dim] = 0
    write = lambda d: lib.nsq_kv_cache_write(d, FAKE, FAKE, 1, 128, 64, 128, 64, 0, FAKE, None)  # noqa: E731
    assert write(_desc(**{what: tuple(strides)})) == _lib.EINVAL
    one = {("num_pages", "page_size", "kv_heads")[dim]: 1}
    assert write(_desc(**{what: tuple(strides)}, **one)) == _lib.OK


@pytest.mark.parametrize("much", [2 ** 31 - 1, 2 ** 31 - 1023])
def test_int8_refuses_rows_that_tiles_would_take_past_32_bits(much):
    lib = _lib.load()
    linear = lambda m, n: lib.nsq_int8_linear(FAKE, 1, m, 16, n, FAKE, FAKE, None, -1, FAKE, FAKE, 1 << 40, None)  # noqa: E731
    assert linear(1, much) == linear(much, 1) == _lib.ENOTSUP
    assert lib.nsq_int8_linear_quantized(FAKE, FAKE, 1, 16, much, FAKE, FAKE, None, -1, FAKE, 1, None) == _lib.ENOTSUP
    assert lib.nsq_int8_quantize(FAKE, 1, much, 8, FAKE, FAKE, None) == _lib.ENOTSUP
