"""Torch-level wrappers of libnsq: device memory, dtypes and streams come from
PyTorch, all arithmetic runs in the library's sm_100a kernels.

Every function launches on ``torch.cuda.current_stream()`` (the capture stream
while a CUDA graph is being recorded), allocates its outputs through the torch
caching allocator and never synchronises the host, so the linears can live
inside the reference's CUDA-graph decode loop. Tensors on any other device
raise: there is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

_ACT_CODES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_BIAS_CODES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


try:  # the raw handle of the current stream without building a Stream object (hot path)
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # pragma: no cover - older torch
    _raw_stream = None


def _stream(t: torch.Tensor) -> int:
    if _raw_stream is not None:
        return _raw_stream(t.device.index)
    return torch.cuda.current_stream(t.device).cuda_stream


def _require_cuda(*ts, what: str) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                f"{what}: nanosglang_b200 runs on CUDA (sm_100a) only; got a tensor on {t.device}. "
                "There is no CPU fallback.")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, 16-byte aligned view (copies only when needed)."""
    if not t.is_contiguous():
        t = t.contiguous()
    if t.data_ptr() % 16 != 0:
        t = t.clone()
    return t


def _settled(c: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    """c, which is t or a copy of it just made. With programmatic launch on, the
    linears read weights, scales and biases before they wait for the kernel
    right ahead, which must not be that copy: another launch, which starts when
    the copy is complete, lies between."""
    if c.data_ptr() != t.data_ptr():
        torch.zeros(1, device=t.device)
    return c


def _weight(t: torch.Tensor) -> torch.Tensor:
    """A weight contiguous and 16-byte aligned, as the linears take it."""
    return _settled(_aligned(t), t)


def _dense(t: torch.Tensor) -> torch.Tensor:
    """The scales, zero points or bias of a linear, contiguous."""
    return t if t.is_contiguous() else _settled(t.contiguous(), t)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _bias_arg(bias: Optional[torch.Tensor]):
    if bias is None:
        return None, _lib.DTYPE_NONE
    if bias.dtype not in _BIAS_CODES:
        raise TypeError(f"bias dtype {bias.dtype} not supported")
    bias = _dense(bias)
    return bias, _BIAS_CODES[bias.dtype]


# ---------------------------------------------------------------------------
# AWQ
# ---------------------------------------------------------------------------


def awq_dequant(qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor, in_features: int,
                group_size: int) -> torch.Tensor:
    """Bit-exact ``AWQLinear._dequantize`` (quantization.py:126-148) -> fp16 [N, K]."""
    _require_cuda(qweight, scales, zeros, what="awq_dequant")
    n = qweight.shape[0]
    if in_features % 8 != 0 or qweight.shape[1] * 8 != in_features:
        raise RuntimeError("AWQ dequantisation needs in_features == 8 * qweight.shape[1] "
                           "(the reference raises in this case as well)")
    qweight = _aligned(qweight)
    scales = scales.contiguous()
    zeros = zeros.contiguous()
    if scales.dtype != torch.float16 or zeros.dtype != torch.float16:
        raise TypeError("scales and zeros must be float16 (reference layout)")
    out = torch.empty(n, in_features, dtype=torch.float16, device=qweight.device)
    rc = _lib.load().nsq_awq_dequant(_ptr(qweight), _ptr(scales), _ptr(zeros), _ptr(out), n, in_features,
                                     group_size, _stream(qweight))
    _lib.check(rc, "nsq_awq_dequant")
    return out


def _decode_workspace(lib, quant: int, m: int, k: int, n: int, group_size: int, device):
    """(tensor, bytes) of a workspace for the decode batch sizes whose kernel
    runs faster with one (x converted once per call, ahead of the linear),
    else (None, 0). The tensor comes from the caching allocator on the
    current stream, so its reuse is stream-ordered after the launches that
    read it (also under CUDA-graph capture)."""
    if m > 64:
        return None, 0
    nbytes = lib.nsq_linear_workspace_size(quant, m, k, n, group_size)
    if not nbytes:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def awq_linear(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor,
               group_size: int, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``AWQLinear.forward`` (quantization.py:150-152) on the tensor cores.

    x: [..., K] fp16 or bf16 (the reference only accepts fp16); returns
    [..., N] in x's dtype.
    """
    if not (x.is_cuda and qweight.is_cuda and scales.is_cuda and zeros.is_cuda) or (
            bias is not None and not bias.is_cuda):
        _require_cuda(x, qweight, scales, zeros, bias, what="awq_linear")
    code = _ACT_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"activation dtype {x.dtype} not supported (float16 / bfloat16)")
    n, k8 = qweight.shape
    k = k8 * 8
    if x.shape[-1] != k:
        raise RuntimeError(f"x has {x.shape[-1]} features, the layer expects {k}")
    if not qweight.is_contiguous() or qweight.data_ptr() & 15:
        qweight = _weight(qweight)
    scales, zeros = _dense(scales), _dense(zeros)
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    if not x2.is_contiguous() or x2.data_ptr() & 15:
        x2 = _aligned(x2)
    m = x2.shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if bias is None:
        bptr, bcode = None, _lib.DTYPE_NONE
    else:
        b, bcode = _bias_arg(bias)
        bptr = b.data_ptr()
    lib = _lib.load()
    ws, wsb = _decode_workspace(lib, 0, m, k, n, group_size, x.device)
    rc = lib.nsq_awq_linear(x2.data_ptr(), code, m, k, n, qweight.data_ptr(), scales.data_ptr(),
                            zeros.data_ptr(), group_size, bptr, bcode, y.data_ptr(),
                            None if ws is None else ws.data_ptr(), wsb, _stream(x))
    if rc:
        _lib.check(rc, "nsq_awq_linear")
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], n)


def awq_quantize(weight: torch.Tensor, group_size: int = 128):
    """``AWQLinear.from_linear`` arithmetic (quantization.py:154-194) on the GPU.

    Returns (qweight int32 [N, K//8], scales fp16 [N, G], zeros fp16 [N, G]).
    """
    _require_cuda(weight, what="awq_quantize")
    if weight.dtype not in _BIAS_CODES:
        raise TypeError(f"weight dtype {weight.dtype} not supported")
    weight = weight.contiguous()
    n, k = weight.shape
    g = (k + group_size - 1) // group_size
    qweight = torch.empty(n, k // 8, dtype=torch.int32, device=weight.device)
    scales = torch.empty(n, g, dtype=torch.float16, device=weight.device)
    zeros = torch.empty(n, g, dtype=torch.float16, device=weight.device)
    rc = _lib.load().nsq_awq_quantize(_ptr(weight), _BIAS_CODES[weight.dtype], n, k, group_size, _ptr(qweight),
                                      _ptr(scales), _ptr(zeros), _stream(weight))
    _lib.check(rc, "nsq_awq_quantize")
    return qweight, scales, zeros


def awq_from_autoawq(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor, group_size: int):
    """Repack one AutoAWQ (GEMM-format) layer into the reference layout, bit-exact.

    qweight int32 [K, N/8], qzeros int32 [K/group_size, N/8], scales fp16
    [K/group_size, N] -> (qweight int32 [N, K/8], scales fp16 [N, G], zeros
    fp16 [N, G]), the AWQLinear buffers of quantization.py:107-119.
    """
    _require_cuda(qweight, qzeros, scales, what="awq_from_autoawq")
    if qweight.dtype != torch.int32 or qzeros.dtype != torch.int32 or scales.dtype != torch.float16:
        raise TypeError("AutoAWQ layers hold int32 qweight/qzeros and float16 scales")
    k, n8 = qweight.shape
    n = n8 * 8
    g = k // group_size
    if qzeros.shape != (g, n8) or scales.shape != (g, n):
        raise ValueError(f"AutoAWQ shapes disagree: qweight {tuple(qweight.shape)}, qzeros {tuple(qzeros.shape)}, "
                         f"scales {tuple(scales.shape)}, group_size {group_size}")
    qweight, qzeros, scales = qweight.contiguous(), qzeros.contiguous(), scales.contiguous()
    out_q = torch.empty(n, k // 8, dtype=torch.int32, device=qweight.device)
    out_s = torch.empty(n, g, dtype=torch.float16, device=qweight.device)
    out_z = torch.empty(n, g, dtype=torch.float16, device=qweight.device)
    rc = _lib.load().nsq_awq_from_autoawq(_ptr(qweight), _ptr(qzeros), _ptr(scales), k, n, group_size, _ptr(out_q),
                                          _ptr(out_s), _ptr(out_z), _stream(qweight))
    _lib.check(rc, "nsq_awq_from_autoawq")
    return out_q, out_s, out_z


# ---------------------------------------------------------------------------
# FP8
# ---------------------------------------------------------------------------


def _u8(w: torch.Tensor) -> torch.Tensor:
    if w.dtype == torch.float8_e4m3fn:
        return w.view(torch.uint8)
    if w.dtype == torch.uint8:
        return w
    raise TypeError(f"fp8 weight must be float8_e4m3fn, got {w.dtype}")


def _scale_arg(weight_scale: torch.Tensor) -> torch.Tensor:
    if weight_scale.numel() != 1:
        raise RuntimeError("weight_scale must hold exactly one value (per-tensor scale)")
    return _settled(weight_scale.float().contiguous(), weight_scale)


_FP8_TYPES = (torch.float8_e4m3fn, torch.uint8)


def fp8_linear(x: torch.Tensor, weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``FP8Linear.forward`` (quantization.py:49-52): W8A16, the scale is read on
    the device (no host sync). Every check is a cheap attribute test on this
    path (eager prefill pays it per linear); anything unusual takes the
    general route (copies, errors)."""
    if not (x.is_cuda and weight_fp8.is_cuda and weight_scale.is_cuda) or (bias is not None and not bias.is_cuda):
        _require_cuda(x, weight_fp8, weight_scale, bias, what="fp8_linear")
    code = _ACT_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"activation dtype {x.dtype} not supported (float16 / bfloat16)")
    if weight_fp8.dtype not in _FP8_TYPES:
        raise TypeError(f"fp8 weight must be float8_e4m3fn, got {weight_fp8.dtype}")
    w = weight_fp8
    if not w.is_contiguous() or w.data_ptr() & 15:
        w = _weight(w)
    n, k = w.shape
    if x.shape[-1] != k:
        raise RuntimeError(f"x has {x.shape[-1]} features, the layer expects {k}")
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    if not x2.is_contiguous() or x2.data_ptr() & 15:
        x2 = _aligned(x2)
    m = x2.shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if bias is None:
        bptr, bcode = None, _lib.DTYPE_NONE
    else:
        b, bcode = _bias_arg(bias)
        bptr = b.data_ptr()
    s = weight_scale
    if s.dtype != torch.float32 or s.numel() != 1 or not s.is_contiguous():
        s = _scale_arg(s)
    lib = _lib.load()
    ws, wsb = _decode_workspace(lib, 1, m, k, n, 0, x.device)
    rc = lib.nsq_fp8_linear(x2.data_ptr(), code, m, k, n, w.data_ptr(), s.data_ptr(), bptr, bcode,
                            y.data_ptr(), None if ws is None else ws.data_ptr(), wsb, _stream(x))
    if rc:
        _lib.check(rc, "nsq_fp8_linear")
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], n)


def fp8_dequant(weight_fp8: torch.Tensor, weight_scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Bit-exact ``weight_fp8.to(dtype) * weight_scale`` (quantization.py:51)."""
    _require_cuda(weight_fp8, weight_scale, what="fp8_dequant")
    if dtype not in _ACT_CODES:
        raise TypeError(f"dtype {dtype} not supported")
    w = _aligned(_u8(weight_fp8))
    n, k = w.shape
    out = torch.empty(n, k, dtype=dtype, device=w.device)
    s = _scale_arg(weight_scale)
    rc = _lib.load().nsq_fp8_dequant(_ptr(w), _ptr(s), _ptr(out), _ACT_CODES[dtype], n, k, _stream(w))
    _lib.check(rc, "nsq_fp8_dequant")
    return out


def fp8_quantize(weight: torch.Tensor):
    """``FP8Linear.from_linear`` arithmetic (quantization.py:54-75) on the GPU.

    Returns (weight_fp8 float8_e4m3fn [N, K], scale fp32 0-dim, absmax_is_zero
    as a 0-dim bool tensor on the device)."""
    _require_cuda(weight, what="fp8_quantize")
    if weight.dtype not in _BIAS_CODES:
        raise TypeError(f"weight dtype {weight.dtype} not supported")
    weight = weight.contiguous()
    n, k = weight.shape
    lib = _lib.load()
    ws_bytes = lib.nsq_fp8_quantize_workspace_size(n, k)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=weight.device)
    codes = torch.empty(n, k, dtype=torch.uint8, device=weight.device)
    scale = torch.empty((), dtype=torch.float32, device=weight.device)
    rc = lib.nsq_fp8_quantize(_ptr(weight), _BIAS_CODES[weight.dtype], n, k, _ptr(codes), _ptr(scale), _ptr(ws),
                              ws_bytes, _stream(weight))
    _lib.check(rc, "nsq_fp8_quantize")
    absmax_zero = ws[:4].view(torch.int32)[0] == 0
    return codes.view(torch.float8_e4m3fn), scale, absmax_zero


# ---------------------------------------------------------------------------
# int8 linear (W8A8: int8 codes with one scale per token and output channel)
# ---------------------------------------------------------------------------

try:  # the current device without torch.cuda's initialisation checks (hot path)
    _current_device = torch._C._cuda_getDevice
except AttributeError:  # pragma: no cover - builds of torch without CUDA
    _current_device = torch.cuda.current_device


def _device_of(what: str, *ts) -> int:
    """The index of the one CUDA device that holds every tensor; raises otherwise."""
    dev = ts[0].get_device()
    for t in ts:
        if t.get_device() != dev or dev < 0:
            _require_cuda(*ts, what=what)
            raise RuntimeError(f"{what}: tensors on {ts[0].device} and {t.device}")
    return dev


def _call(dev: int, name: str, *args) -> None:
    """Runs an entry point on device ``dev`` (made current where it is not)."""
    fn = getattr(_lib.load(), name)
    if dev == _current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args)
    if rc:
        _lib.check(rc, name)


def _stream_on(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def int8_quantize(x: torch.Tensor):
    """Rows of x to int8 codes and one scale each (weights per output channel,
    activations per token): scale = max|row| / 127 (1 if that is 0), codes =
    rint(row / scale). x: [..., K] float16, bfloat16 or float32. Returns
    (codes int8 [..., K], scale float32 [...])."""
    dev = _device_of("int8_quantize", x)
    code = _BIAS_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"dtype {x.dtype} not supported (float16 / bfloat16 / float32)")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"int8_quantize needs rows of at least one element, got shape {tuple(shape)}")
    x = x.contiguous()
    k = shape[-1]
    codes = x.new_empty(shape, dtype=torch.int8)
    scale = x.new_empty(shape[:-1], dtype=torch.float32)
    _call(dev, "nsq_int8_quantize", x.data_ptr(), code, x.numel() // k, k, codes.data_ptr(), scale.data_ptr(),
          _stream_on(dev))
    return codes, scale


def _int8_operands(weight_int8: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor]):
    """Checks an int8 layer: (weight, weight_scale, N, K, bias or None, its dtype code)."""
    if weight_int8.dtype != torch.int8 or weight_int8.dim() != 2:
        raise TypeError(f"int8 weight must be int8 [N, K], got {weight_int8.dtype} {tuple(weight_int8.shape)}")
    n, k = weight_int8.shape
    if weight_scale.dtype != torch.float32 or weight_scale.numel() != n:
        raise TypeError(f"weight_scale must be float32 with one value per output channel ({n}), "
                        f"got {weight_scale.dtype} {tuple(weight_scale.shape)}")
    if not weight_int8.is_contiguous() or weight_int8.data_ptr() & 15:
        weight_int8 = _weight(weight_int8)
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is None:
        return weight_int8, weight_scale, n, k, None, _lib.DTYPE_NONE
    if bias.numel() != n:
        raise ValueError(f"bias has {bias.numel()} elements, the layer has {n} outputs")
    bias, code = _bias_arg(bias)
    return weight_int8, weight_scale, n, k, bias, code


def int8_linear(x: torch.Tensor, weight_int8: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """W8A8 linear: x is quantised per token (``int8_quantize``), the codes are
    multiplied in int32 (exact) and the sums scaled in float32:
    ``y = (codes @ weight_int8^T) * scale * weight_scale + bias``, in that order
    and rounded once to y's type.

    x: [..., K] float16 or bfloat16; weight_int8 int8 [N, K], weight_scale
    float32 [N]; returns [..., N] in x's dtype. K must be a multiple of 16, at
    most 131072.
    """
    if bias is None:
        dev = _device_of("int8_linear", x, weight_int8, weight_scale)
    else:
        dev = _device_of("int8_linear", x, weight_int8, weight_scale, bias)
    code = _ACT_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"activation dtype {x.dtype} not supported (float16 / bfloat16)")
    w, ws, n, k, b, bcode = _int8_operands(weight_int8, weight_scale, bias)
    shape = x.shape
    if not shape or shape[-1] != k:
        raise RuntimeError(f"x has shape {tuple(shape)}, the layer expects {k} features")
    x2 = x if len(shape) == 2 else x.reshape(-1, k)
    if not x2.is_contiguous() or x2.data_ptr() & 15:
        x2 = _aligned(x2)
    m = x2.shape[0]
    y = x2.new_empty((m, n))
    nbytes = _lib.load().nsq_int8_linear_workspace_size(m, k, n)
    work = x2.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(dev, "nsq_int8_linear", x2.data_ptr(), code, m, k, n, w.data_ptr(), ws.data_ptr(),
          None if b is None else b.data_ptr(), bcode, y.data_ptr(), None if work is None else work.data_ptr(), nbytes,
          _stream_on(dev))
    return y if len(shape) == 2 else y.reshape(*shape[:-1], n)


def int8_linear_quantized(codes: torch.Tensor, scale: torch.Tensor, weight_int8: torch.Tensor,
                          weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                          dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of ``int8_linear`` for activations already quantised by
    ``int8_quantize`` (once, for several layers that read the same x): codes
    int8 [..., K], scale float32 [...]; returns [..., N] in ``dtype``."""
    if bias is None:
        dev = _device_of("int8_linear_quantized", codes, scale, weight_int8, weight_scale)
    else:
        dev = _device_of("int8_linear_quantized", codes, scale, weight_int8, weight_scale, bias)
    shape = codes.shape
    if codes.dtype != torch.int8 or scale.dtype != torch.float32 or not shape or scale.shape != shape[:-1]:
        raise TypeError(f"codes must be int8 [..., K] with a float32 scale [...], got {codes.dtype} "
                        f"{tuple(shape)} and {scale.dtype} {tuple(scale.shape)}")
    code = _ACT_CODES.get(dtype)
    if code is None:
        raise TypeError(f"output dtype {dtype} not supported (float16 / bfloat16)")
    w, ws, n, k, b, bcode = _int8_operands(weight_int8, weight_scale, bias)
    if shape[-1] != k:
        raise RuntimeError(f"codes have {shape[-1]} features, the layer expects {k}")
    c2 = _aligned(codes.reshape(-1, k))
    s2 = scale.reshape(-1).contiguous()
    m = c2.shape[0]
    y = codes.new_empty((m, n), dtype=dtype)
    _call(dev, "nsq_int8_linear_quantized", c2.data_ptr(), s2.data_ptr(), m, k, n, w.data_ptr(), ws.data_ptr(),
          None if b is None else b.data_ptr(), bcode, y.data_ptr(), code, _stream_on(dev))
    return y if len(shape) == 2 else y.reshape(*shape[:-1], n)


# ---------------------------------------------------------------------------
# 8-bit key/value cache and decode attention over it
# ---------------------------------------------------------------------------

_KV_CODES = {torch.int8: _lib.KV_INT8, torch.float8_e4m3fn: _lib.KV_FP8}


def _kv_desc(k_cache, v_cache, k_scale, v_scale, what: str):
    """Checks the four tensors of a cache; returns the packed struct nsq_kv_cache and the cache's shape."""
    code = _KV_CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype != k_cache.dtype:
        raise TypeError(f"{what}: caches must both be int8 or both float8_e4m3fn, got {k_cache.dtype} "
                        f"and {v_cache.dtype}")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{what}: caches must be [pages, page_size, kv_heads, head_dim] of one shape, got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    rows = shape[:3]
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32 or k_scale.shape != rows or (
            v_scale.shape != rows):
        raise ValueError(f"{what}: scales must be float32 {tuple(rows)}, got {k_scale.dtype} {tuple(k_scale.shape)} "
                         f"and {v_scale.dtype} {tuple(v_scale.shape)}")
    k0, k1, k2, kd = k_cache.stride()
    v0, v1, v2, vd = v_cache.stride()
    if (kd != 1 or vd != 1) and shape[3] > 1:
        raise ValueError(f"{what}: head_dim must be contiguous in the caches")
    return _lib.KV_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *shape,
                              k0, k1, k2, v0, v1, v2, *k_scale.stride(), *v_scale.stride(), code), shape


def _kv_rows(t: torch.Tensor):
    """[T, heads, head_dim] with 16-byte aligned rows of contiguous head_dim (a
    copy only where needed), and its token and head strides."""
    s0, s1, s2 = t.stride()
    if s2 != 1 or t.data_ptr() & 15 or (s0 & 7 and t.shape[0] > 1) or (s1 & 7 and t.shape[1] > 1):
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, _ = t.stride()
    return t, s0, s1


def _slots_arg(slots: torch.Tensor, what: str) -> torch.Tensor:
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise TypeError(f"{what}: slots must be int64 [T], got {slots.dtype} {tuple(slots.shape)}")
    return slots.contiguous()


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   k_scale: torch.Tensor, v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise k and v [T, kv_heads, head_dim] (float16 or bfloat16) into an
    8-bit cache, in place.

    k_cache, v_cache: int8 or float8_e4m3fn [pages, page_size, kv_heads,
    head_dim], any strides with head_dim contiguous (token-major or head-major
    pools; no expanded ones, whose places share memory); k_scale, v_scale: float32 [pages, page_size, kv_heads]. Token t
    goes to place ``slots[t] = page * page_size + offset`` (int64); a negative
    slot is a padded token and is skipped, one past the pool is skipped and
    recorded in the status word. Slots are distinct: of two tokens with the
    same slot the stored row is unspecified. Per (token, head) row: scale =
    max|row| / 127 (int8) or / 448 (float8), 1 where that is 0; codes are the
    nearest to row / scale. A row with a NaN or an infinity reads back as NaN.
    """
    dev = _device_of("kv_cache_write", k, v, k_cache, v_cache, k_scale, v_scale, slots)
    code = _ACT_CODES.get(k.dtype)
    if code is None or v.dtype != k.dtype:
        raise TypeError(f"kv_cache_write: k and v must both be float16 or both bfloat16, got {k.dtype} and {v.dtype}")
    desc, (_, _, heads, dim) = _kv_desc(k_cache, v_cache, k_scale, v_scale, "kv_cache_write")
    slots = _slots_arg(slots, "kv_cache_write")
    n = slots.shape[0]
    if k.shape != (n, heads, dim) or v.shape != (n, heads, dim):
        raise ValueError(f"kv_cache_write: k and v must be {(n, heads, dim)}, got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    k, kt, kh = _kv_rows(k)
    v, vt, vh = _kv_rows(v)
    _call(dev, "nsq_kv_cache_write", desc, k.data_ptr(), v.data_ptr(), code, kt, kh, vt, vh, n, slots.data_ptr(),
          _stream_on(dev))


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  slots: torch.Tensor, dtype: torch.dtype):
    """The rows at ``slots`` (int64 [T]) of an 8-bit cache, as (k, v)
    [T, kv_heads, head_dim] in ``dtype`` (float16 or bfloat16): code * scale,
    rounded once; zeros where a slot is negative."""
    dev = _device_of("kv_cache_read", k_cache, v_cache, k_scale, v_scale, slots)
    code = _ACT_CODES.get(dtype)
    if code is None:
        raise TypeError(f"kv_cache_read: dtype {dtype} not supported (float16 / bfloat16)")
    desc, (_, _, heads, dim) = _kv_desc(k_cache, v_cache, k_scale, v_scale, "kv_cache_read")
    slots = _slots_arg(slots, "kv_cache_read")
    n = slots.shape[0]
    k = k_scale.new_empty((n, heads, dim), dtype=dtype)
    v = k_scale.new_empty((n, heads, dim), dtype=dtype)
    _call(dev, "nsq_kv_cache_read", desc, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code, _stream_on(dev))
    return k, v


def kv_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                        softmax_scale: Optional[float] = None, return_lse: bool = False):
    """Attention of one query token per sequence over its 8-bit cache.

    q: [B, heads, head_dim] float16 or bfloat16, heads a multiple of kv_heads
    (grouped-query); page_table int32 [B, W]: the pages of each sequence in
    order; seq_lens int32 [B]: tokens held (0 for a padded row: its output is
    0, its log-sum-exp -inf). ``softmax_scale`` defaults to head_dim ** -0.5.
    Scores and sums are float32, the weights of v float16 (relative to their
    largest: 11 bits each). The caches may be expanded views.
    Returns out [B, heads, head_dim] in q's dtype, with ``return_lse`` also the
    natural log-sum-exp of the scaled scores, float32 [B, heads]. Entries of
    page_table past a sequence's last page are never read. A page outside the
    pool or a length past the table (or below 0) is recorded in the status
    word: that page's tokens are left out, the length is clamped.
    """
    what = "kv_attention_decode"
    dev = _device_of(what, q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens)
    code = _ACT_CODES.get(q.dtype)
    if code is None:
        raise TypeError(f"{what}: query dtype {q.dtype} not supported (float16 / bfloat16)")
    desc, (_, page, heads, dim) = _kv_desc(k_cache, v_cache, k_scale, v_scale, what)
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim or shape[1] == 0 or heads == 0 or shape[1] % heads:
        raise ValueError(f"{what}: q must be [B, heads, {dim}] with heads a multiple of {heads}, got {tuple(shape)}")
    b, h, _ = shape
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b:
        raise TypeError(f"{what}: page_table must be int32 [{b}, W], got {page_table.dtype} {tuple(page_table.shape)}")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (b,):
        raise TypeError(f"{what}: seq_lens must be int32 [{b}], got {seq_lens.dtype} {tuple(seq_lens.shape)}")
    q, qs, qh = _kv_rows(q)
    width = page_table.shape[1]
    if page_table.stride(1) != 1 and width > 1:
        page_table = page_table.contiguous()
    if not seq_lens.is_contiguous():
        seq_lens = seq_lens.contiguous()
    out = q.new_empty(shape)
    lse = q.new_empty((b, h), dtype=torch.float32) if return_lse else None
    if dev == _current_device():
        nbytes = _lib.load().nsq_kv_attention_workspace_size(b, h, heads, dim, page, width)
    else:
        with torch.cuda.device(dev):
            nbytes = _lib.load().nsq_kv_attention_workspace_size(b, h, heads, dim, page, width)
    work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(dev, "nsq_kv_attention_decode", desc, q.data_ptr(), code, qs, qh, b, h, page_table.data_ptr(),
          page_table.stride(0) if b > 1 else 0, width, seq_lens.data_ptr(),
          dim ** -0.5 if softmax_scale is None else softmax_scale, out.data_ptr(),
          None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), nbytes, _stream_on(dev))
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# Fused projections for decode batches (row-streaming kernel, M <= 32)
# ---------------------------------------------------------------------------

FUSED_MAX_M = 32


def _unwrap(mod):
    """The quantized module behind a tensor-parallel wrapper (its local shard)."""
    return getattr(mod, "linear", mod)


def _ptr_array(vals, ctype=None):
    arr = (ctypes.c_void_p * len(vals))(*vals) if ctype is None else (ctype * len(vals))(*vals)
    return arr


def linear_multi(x: torch.Tensor, mods) -> Optional[list]:
    """One launch for 1..3 AWQLinear (or 1..3 FP8Linear) layers that read the
    same x, e.g. q/k/v; Int8Linear layers share one quantisation of x (any M).
    Returns their outputs as views of one [M, sum N] buffer (Int8Linear: a buffer
    each), or None when the fused kernel does not apply (M > 32, mixed formats,
    bias dtypes that differ, group sizes that differ)."""
    mods = [_unwrap(m) for m in mods]
    kinds = {type(m).__name__ for m in mods}
    if len(kinds) != 1 or x.dtype not in _ACT_CODES:
        return None
    if kinds == {"Int8Linear"}:  # one quantisation of x for all, at any batch size
        codes, scale = int8_quantize(x)
        return [int8_linear_quantized(codes, scale, mm.weight_int8, mm.scale(), mm.bias, x.dtype) for mm in mods]
    k = x.shape[-1]
    lead = x.shape[:-1]
    x2 = _aligned(x.reshape(-1, k))
    m = x2.shape[0]
    if m == 0 or m > FUSED_MAX_M:
        return None
    biases = [mm.bias for mm in mods]
    has_bias = [b is not None for b in biases]
    if any(has_bias) and not all(has_bias):
        biases = [b if b is not None else torch.zeros(mm.out_features, device=x.device, dtype=x.dtype)
                  for b, mm in zip(biases, mods)]
    bias_dtypes = {b.dtype for b in biases if b is not None}
    if len(bias_dtypes) > 1:
        return None
    biases = [b.contiguous() for b in biases] if any(has_bias) else None
    bcode = _BIAS_CODES[biases[0].dtype] if biases else _lib.DTYPE_NONE
    ns = [mm.out_features for mm in mods]
    y = torch.empty(m, sum(ns), dtype=x.dtype, device=x.device)
    n_arr = (ctypes.c_int64 * len(ns))(*ns)
    b_arr = _ptr_array([b.data_ptr() for b in biases]) if biases else None
    lib = _lib.load()
    if kinds == {"AWQLinear"}:
        gs = {mm.group_size for mm in mods}
        if len(gs) != 1 or any(mm.in_features != k for mm in mods):
            return None
        qws = [_weight(mm.qweight) for mm in mods]
        scs = [_dense(mm.scales) for mm in mods]
        zrs = [_dense(mm.zeros) for mm in mods]
        rc = lib.nsq_awq_linear_multi(_ptr(x2), _ACT_CODES[x.dtype], m, k, len(mods),
                                      _ptr_array([t.data_ptr() for t in qws]), _ptr_array([t.data_ptr() for t in scs]),
                                      _ptr_array([t.data_ptr() for t in zrs]), n_arr, gs.pop(), b_arr, bcode, _ptr(y),
                                      y.shape[1], _stream(x))
    elif kinds == {"FP8Linear"}:
        ws = [_weight(_u8(mm.weight_fp8)) for mm in mods]
        if any(w.shape[1] != k for w in ws):
            return None
        scs = [_scale_arg(mm.weight_scale) for mm in mods]
        rc = lib.nsq_fp8_linear_multi(_ptr(x2), _ACT_CODES[x.dtype], m, k, len(mods),
                                      _ptr_array([t.data_ptr() for t in ws]), _ptr_array([t.data_ptr() for t in scs]),
                                      n_arr, b_arr, bcode, _ptr(y), y.shape[1], _stream(x))
    else:
        return None
    if rc == _lib.ENOTSUP:
        return None
    _lib.check(rc, "nsq_*_linear_multi")
    outs, c0 = [], 0
    for n in ns:
        outs.append(y[:, c0:c0 + n].reshape(*lead, n))
        c0 += n
    return outs


def gate_up_silu(x: torch.Tensor, gate, up) -> Optional[torch.Tensor]:
    """SiLU(gate(x)) * up(x) in one launch (MLP.forward's inner expression,
    causal_lm.py:482) for AWQ or FP8 gate/up layers without bias; None when
    the fused kernel does not apply (M > 32, bias, mismatched layers). Int8Linear
    layers share one quantisation of x and run as two products."""
    gate, up = _unwrap(gate), _unwrap(up)
    if type(gate) is not type(up) or x.dtype not in _ACT_CODES or gate.bias is not None or up.bias is not None:
        return None
    if type(gate).__name__ == "Int8Linear":
        g, u = linear_multi(x, (gate, up))
        return torch.nn.functional.silu(g) * u
    k = x.shape[-1]
    lead = x.shape[:-1]
    x2 = _aligned(x.reshape(-1, k))
    m = x2.shape[0]
    n = gate.out_features
    if m == 0 or m > FUSED_MAX_M or up.out_features != n:
        return None
    y = torch.empty(m, n, dtype=x.dtype, device=x.device)
    lib = _lib.load()
    if type(gate).__name__ == "AWQLinear":
        if gate.group_size != up.group_size or gate.in_features != k or up.in_features != k:
            return None
        qg, qu = _weight(gate.qweight), _weight(up.qweight)
        sg, zg, su, zu = (_dense(t) for mod in (gate, up) for t in (mod.scales, mod.zeros))
        rc = lib.nsq_awq_gate_up_silu(_ptr(x2), _ACT_CODES[x.dtype], m, k, n, _ptr(qg), _ptr(sg), _ptr(zg), _ptr(qu),
                                      _ptr(su), _ptr(zu), gate.group_size, _ptr(y), _stream(x))
    elif type(gate).__name__ == "FP8Linear":
        wg, wu = _weight(_u8(gate.weight_fp8)), _weight(_u8(up.weight_fp8))
        if wg.shape[1] != k or wu.shape[1] != k:
            return None
        rc = lib.nsq_fp8_gate_up_silu(_ptr(x2), _ACT_CODES[x.dtype], m, k, n, _ptr(wg), _ptr(_scale_arg(gate.weight_scale)),
                                      _ptr(wu), _ptr(_scale_arg(up.weight_scale)), _ptr(y), _stream(x))
    else:
        return None
    if rc == _lib.ENOTSUP:
        return None
    _lib.check(rc, "nsq_*_gate_up_silu")
    return y.reshape(*lead, n)
