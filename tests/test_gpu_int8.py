"""int8 linear on the GPU against 64-bit arithmetic.

Tolerances: the codes are compared bit for bit (IEEE float32 operations). The
sums are exact integers, so y carries the rounding of the sum to float32, two
products and the bias addition (2^-24 each) and one to y's type (eps / 2):
  |y - exact| <= 4 * 2^-24 * (|dot| + |bias|) + eps / 2 * |y|
(first order; 1.01 covers the products of roundings), plus half the smallest
subnormal where the type underflows.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def ref_quantize(x):
    """codes and scale by float32 operations on the CPU."""
    xf = x.cpu().float()
    s = xf.abs().amax(-1) / 127.0
    s = torch.where(s == 0, torch.ones_like(s), s)
    return (xf / s[..., None]).round().clamp(-127, 127).to(torch.int8), s


def check_linear(y, x, w, ws, bias):
    codes, s = ref_quantize(x)
    dot = codes.double() @ w.cpu().double().t() * s.double()[..., None] * ws.cpu().double()
    b = 0.0 if bias is None else bias.cpu().double()
    want = dot + b
    eps = torch.finfo(y.dtype).eps
    tol = 1.01 * (4 * 2.0 ** -24 * (dot.abs() + abs(b)) + eps / 2 * want.abs()) + torch.finfo(y.dtype).tiny * eps
    got = y.cpu().double()
    assert got.shape == want.shape
    worst = ((got - want).abs() / tol).max() if want.numel() else 0.0
    assert worst <= 1.0, f"worst error {worst} of the tolerance"


def make(m, k, n, dtype, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(m, k, generator=g) * (1 + 9 * (torch.rand(k, generator=g) < 0.05))).to(dtype).cuda()
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    ws = (torch.rand(n, generator=g) * 1e-3 + 1e-5).cuda()
    b = None if bias is None else torch.randn(n, generator=g).to(bias).cuda()
    return x, w, ws, b


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 16), (2, 896), (4, 2056), (3, 16384), (2, 16392), (2, 20000),
                                   (300, 64), (2, 3, 128)])
def test_quantize_bits(shape, dtype):
    from nanosglang_b200 import ops
    g = torch.Generator().manual_seed(1)
    x = torch.randn(*shape, generator=g).to(dtype)
    x.view(-1, shape[-1])[0] = 0  # an all-zero row
    codes, s = ops.int8_quantize(x.cuda())
    rc, rs = ref_quantize(x)
    assert torch.equal(codes.cpu(), rc) and torch.equal(s.cpu(), rs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_range(dtype):
    """Rows at the ends of the type's range, ties and non-finite rows."""
    from nanosglang_b200 import ops
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # smallest subnormal
    big = torch.finfo(dtype).max
    ties = torch.arange(-127, 128).float() / 2 + 0.0
    x = torch.zeros(6, 256, dtype=dtype)
    x[0, :4] = torch.tensor([tiny, -tiny, 2 * tiny, 0.0]).to(dtype)
    x[1, :3] = torch.tensor([big, -big, big / 3]).to(dtype)
    x[2, :255] = ties.to(dtype)  # max 63.5: scale 0.5, quotients whole
    x[3, :255] = (ties * 2).to(dtype)  # max 127: scale 1, whole numbers
    x[3, 255] = 0.5
    x[4] = torch.randn(256, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[4, 0] = 127.0  # scale 1: halves are ties, to even
    x[4, 1:9] = torch.tensor([0.5, 1.5, 2.5, 3.5, -0.5, -1.5, -2.5, 63.5]).to(dtype)
    codes, s = ops.int8_quantize(x.cuda())
    rc, rs = ref_quantize(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(codes.cpu(), rc)
    y = x.clone()
    y[0, 3], y[1, 5] = float("nan"), float("inf")
    codes, s = ops.int8_quantize(y.cuda())
    back = codes.cpu().float() * s.cpu()[:, None]
    assert back[:2].isnan().all() and back[2:].isfinite().all()


# one token to prefill chunks; K with a tail of every 16-byte step; N off every tile
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (1, 896, 4864), (2, 48, 15), (7, 80, 17), (8, 1040, 130), (9, 128, 64),
                                   (16, 4096, 520), (17, 112, 127), (31, 4864, 896), (32, 2048, 129), (33, 896, 1000),
                                   (63, 160, 33), (64, 512, 257), (65, 144, 255), (100, 4864, 896), (127, 256, 128),
                                   (128, 128, 512), (129, 896, 384), (255, 272, 320), (256, 1024, 256),
                                   (257, 4096, 264), (300, 64, 1), (511, 384, 2000), (777, 4864, 896),
                                   (1025, 1152, 1537), (2000, 16, 40)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(m, k, n, dtype):
    from nanosglang_b200 import ops
    bias = [None, dtype, torch.float32][(m + n) % 3]
    x, w, ws, b = make(m, k, n, dtype, bias, seed=m + k + n)
    y = ops.int8_linear(x, w, ws, b)
    assert y.dtype == dtype
    check_linear(y, x, w, ws, b)
    codes, s = ops.int8_quantize(x)
    assert torch.equal(ops.int8_linear_quantized(codes, s, w, ws, b, dtype), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(70, 128, 4728), (200, 384, 10008), (40, 256, 16000), (500, 128, 4096),
                                   (300, 896, 4864), (1300, 1040, 904)])
def test_linear_uneven_tiles(m, k, n, dtype):
    """Tiles of other than 64 or 128 rows, the last one short, 8 features to a store."""
    from nanosglang_b200 import ops
    x, w, ws, b = make(m, k, n, dtype, dtype, seed=n)
    check_linear(ops.int8_linear(x, w, ws, b), x, w, ws, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1301, 8), (1301, 1016), (1190, 1536), (1185, 1544), (1200, 2048), (1187, 4104),
                                    (1185, 8192), (1185, 8200), (20000, 136)])
def test_quantize_many_rows(rows, k, dtype):
    """Every number of threads and vectors a row takes when rows are many."""
    from nanosglang_b200 import ops
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows + k)).to(dtype)
    x[rows // 2] = 0
    codes, s = ops.int8_quantize(x.cuda())
    rc, rs = ref_quantize(x)
    assert torch.equal(codes.cpu(), rc) and torch.equal(s.cpu(), rs)


def test_linear_largest_sums():
    """The longest K with every product at its largest: 127 * 128 * 131072 is just under 2^31."""
    from nanosglang_b200 import ops
    for m in (1, 130):
        x = torch.ones(m, 131072, dtype=torch.bfloat16).cuda()
        x[0] = -1
        w = torch.full((20, 131072), -128, dtype=torch.int8).cuda()
        ws = torch.full((20,), 2.0 ** -20).cuda()
        y = ops.int8_linear(x, w, ws)
        check_linear(y, x, w, ws, None)
        with pytest.raises(RuntimeError):
            ops.int8_linear(torch.ones(1, 131088, dtype=torch.bfloat16).cuda(),
                            torch.zeros(4, 131088, dtype=torch.int8).cuda(), ws[:4])


@pytest.mark.parametrize("m", [3, 200])
def test_linear_views_and_empty(m):
    from nanosglang_b200 import ops
    x, w, ws, b = make(m, 128, 48, torch.bfloat16, torch.bfloat16)
    want = ops.int8_linear(x, w, ws, b)
    wide = torch.zeros(m, 264, dtype=torch.bfloat16).cuda()
    wide[:, 3:131] = x  # rows neither contiguous nor aligned
    assert torch.equal(ops.int8_linear(wide[:, 3:131], w, ws, b), want)
    assert torch.equal(ops.int8_linear(x.view(1, m, 128), w, ws, b), want.view(1, m, 48))
    assert torch.equal(ops.int8_linear(x, w.t().contiguous().t(), ws, b), want)
    assert ops.int8_linear(x[:0], w, ws, b).shape == (0, 48)
    # an odd N leaves every other row of y off 4-byte alignment
    x, w, ws, b = make(m, 128, 47, torch.float16, None)
    check_linear(ops.int8_linear(x, w, ws), x, w, ws, None)


@pytest.mark.parametrize("m", [4, 150])
def test_linear_nonfinite_tokens_stay_alone(m):
    from nanosglang_b200 import ops
    x, w, ws, _ = make(m, 256, 130, torch.bfloat16, None)
    want = ops.int8_linear(x, w, ws)
    x[1, 7], x[2, 0] = float("nan"), float("-inf")
    y = ops.int8_linear(x, w, ws)
    assert y[1:3].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("m", [5, 300])
def test_linear_captured_and_other_stream(m):
    from nanosglang_b200 import ops
    x, w, ws, b = make(m, 896, 272, torch.bfloat16, torch.float32)
    want = ops.int8_linear(x, w, ws, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            y = ops.int8_linear(x, w, ws, b)
    side.synchronize()
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y1 = ops.int8_linear(x, w, ws, b)
        y2 = ops.int8_linear(x * 2, w, ws, b)
    x.copy_(x.flip(0))
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    check_linear(y1, x, w, ws, b)
    check_linear(y2, x * 2, w, ws, b)


def test_refusals():
    from nanosglang_b200 import ops
    x, w, ws, b = make(4, 64, 32, torch.bfloat16, torch.bfloat16)
    for bad, err in [((x.float(), w, ws), TypeError), ((x, w.float(), ws), TypeError), ((x, w, ws.half()), TypeError),
                     ((x, w, ws[:5]), TypeError), ((x[:, :48], w, ws), RuntimeError), ((x, w, ws, b[:3]), ValueError),
                     ((x, w[0], ws), TypeError), ((x, w, ws.cpu()), RuntimeError), ((x, w, ws, b.double()), TypeError)]:
        with pytest.raises(err):
            ops.int8_linear(*bad)
    with pytest.raises(RuntimeError):  # K not a multiple of 16
        ops.int8_linear(x[:, :24].contiguous(), w[:, :24].contiguous(), ws)
    codes, s = ops.int8_quantize(x)
    for bad in [(codes.float(), s, w, ws), (codes, s[:2], w, ws), (codes, s, w, ws, b, torch.float32)]:
        with pytest.raises(TypeError):
            ops.int8_linear_quantized(*bad)
    with pytest.raises(TypeError):
        ops.int8_quantize(x.double())
    with pytest.raises(ValueError):
        ops.int8_quantize(x[:, :0])
