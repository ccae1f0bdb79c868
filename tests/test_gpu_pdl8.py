"""The 8-bit operators one behind the other with programmatic dependent launch
on: the same bits as without it, on every path of the int8 linear."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def pdl():
    from nanosglang_b200 import _lib

    def run(fn):
        prev = _lib.set_pdl(True)
        try:
            out = fn()
            torch.cuda.synchronize()
        finally:
            _lib.set_pdl(prev)
        assert _lib.device_status()[0] == 0
        return out

    return run


def make_layers(sizes, seed):
    g = torch.Generator().manual_seed(seed)
    layers = []
    for k, n in zip(sizes, sizes[1:] + sizes[:1]):
        w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
        s = torch.full((n,), 1 / (73 * k ** 0.5)).cuda()
        layers.append((w, s, s * 0.5))
    return layers


# x quantised in the product's own launch; rows of 8, 32 and 64 tokens; one-CTA tiles of 32 and 64 tokens;
# K split over a cluster; CTA pairs
@pytest.mark.parametrize("m,sizes", [(5, [512, 512]), (5, [1024, 1040]), (20, [1024, 1024]), (40, [512, 1024]),
                                     (40, [2048, 2064]), (300, [1024, 1024]), (65, [8192, 128]), (200, [12304, 528]),
                                     (1000, [2064, 2592])])
@pytest.mark.parametrize("shared", [False, True])
def test_linear_chain(m, sizes, shared, pdl):
    """Linears that read what the one ahead writes, nothing in between; with
    ``shared``, two products of one quantisation."""
    from nanosglang_b200 import ops
    layers = make_layers(sizes, m + len(sizes))
    x0 = torch.randn(m, sizes[0], generator=torch.Generator().manual_seed(m)).bfloat16().cuda()

    def chain():
        x = x0.clone()

        def once():
            y = x
            for w, s, s2 in layers * 2:
                if shared:
                    codes, scale = ops.int8_quantize(y)
                    z = ops.int8_linear_quantized(codes, scale, w, s)
                    y = ops.int8_linear_quantized(codes, scale, w, s2)
                    y = z if w.shape[0] % 32 else y + z
                else:
                    y = ops.int8_linear(y, w, s)
            x.copy_(torch.tanh(y))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            once()
        steps = []
        for _ in range(20):
            graph.replay()
            steps.append(x.clone())
        torch.cuda.synchronize()
        return torch.stack(steps)

    want = chain()
    assert want.isfinite().all() and (want[-1] != want[-2]).any()
    assert torch.equal(pdl(chain), want)


@pytest.mark.parametrize("m,k,n,dtype", [(1, 4096, 4096, torch.bfloat16), (1, 4096, 4096, torch.float32),
                                         (8, 2048, 4096, torch.float16), (64, 2048, 8192, torch.bfloat16),
                                         (300, 1024, 2000, torch.bfloat16)])
@pytest.mark.parametrize("quantized", [False, True])
def test_weight_quantised_just_ahead(m, k, n, dtype, quantized, pdl):
    """A weight whose codes are made by the kernel right ahead of the product
    that reads them, again and again from other values."""
    from nanosglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    weights = [torch.randn(n, k, generator=g, device="cuda").to(dtype) for _ in range(3)]
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    xc, xs = ops.int8_quantize(x)

    def runs():
        w = weights[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            codes, scale = ops.int8_quantize(w)
            y = ops.int8_linear_quantized(xc, xs, codes, scale) if quantized else ops.int8_linear(x, codes, scale)
        out = []
        for i in range(12):
            w.copy_(weights[i % 3])
            graph.replay()
            out.append(y.clone())
        torch.cuda.synchronize()
        return torch.stack(out)

    want = runs()
    assert torch.equal(pdl(runs), want)


@pytest.mark.parametrize("m,k,n", [(1, 512, 512), (5, 1024, 512), (100, 512, 1000)])
def test_weight_view_copied_in_the_call(m, k, n, pdl):
    """A weight that is not contiguous is copied within the call, right ahead of
    the kernel that reads the copy."""
    from nanosglang_b200 import ops
    g = torch.Generator().manual_seed(6)
    weights = [torch.randint(-127, 128, (k, n), generator=g, dtype=torch.int8).cuda() for _ in range(3)]
    scale = torch.rand(n, generator=g).cuda()
    x = torch.randn(m, k, generator=g).bfloat16().cuda()

    def runs():
        w = weights[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.int8_linear(x, w.t(), scale)
        out = []
        for i in range(12):
            w.copy_(weights[i % 3])
            graph.replay()
            out.append(y.clone())
        torch.cuda.synchronize()
        return torch.stack(out)

    want = runs()
    assert torch.equal(pdl(runs), want)


def test_a_weight_copy_is_not_right_ahead():
    """What the call launches last before a kernel that may load the weight
    early is not the copy of that weight."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from nanosglang_b200 import ops
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func._schema.name.split("::")[1])
            return func(*args, **(kwargs or {}))

    g = torch.Generator().manual_seed(7)
    w = torch.randint(-127, 128, (512, 64), generator=g, dtype=torch.int8).cuda().t()
    f8 = torch.randn(512, 64, generator=g).cuda().to(torch.float8_e4m3fn).view(torch.uint8).t()
    qw = torch.randint(-9, 9, (64, 64), generator=g, dtype=torch.int32).cuda().t()
    sz = [torch.rand(4, 64, generator=g).half().cuda().t() for _ in range(2)]
    x = torch.randn(2, 512, generator=g).half().cuda()
    codes, scale = ops.int8_quantize(x)
    ones, wide, plain = torch.ones(64, device="cuda"), torch.ones(64, 2, device="cuda"), f8.contiguous()
    for call in (lambda: ops.int8_linear(x, w, ones), lambda: ops.int8_linear_quantized(codes, scale, w, ones),
                 lambda: ops.fp8_linear(x, f8, ones[:1]), lambda: ops.awq_linear(x, qw, *sz, 128),
                 lambda: ops.fp8_linear(x, plain, ones[:1].half()),
                 lambda: ops.fp8_linear(x, plain, ones[:1], wide[:, 0])):
        seen.clear()
        with Log():
            call()
        copies = [i for i, name in enumerate(seen) if name in ("clone", "copy_", "contiguous", "_to_copy")]
        assert copies and any(name in ("zeros", "zero_", "fill_") for name in seen[copies[-1] + 1:]), seen
