"""The int8 linear's forms that small layers do not reach, against 64 bits: CTA
pairs (tails of tokens, features and k-blocks, several tiles a pair), K split
over clusters, for few and for many tokens. Tolerances as in test_gpu_int8.py."""

import pytest
import torch

from test_gpu_int8 import DTYPES, make, ref_quantize

pytestmark = pytest.mark.gpu


def check(m, k, n, dtype, bias):
    from nanosglang_b200 import ops
    x, w, ws, b = make(m, k, n, dtype, bias, seed=m + k + n)
    y = ops.int8_linear(x, w, ws, b)
    codes, s = ref_quantize(x)
    dot = codes.cuda().double() @ w.double().t() * s.cuda().double()[:, None] * ws.double()
    b = torch.zeros((), dtype=torch.float64, device="cuda") if b is None else b.double()
    want = dot + b
    eps = torch.finfo(dtype).eps
    tol = 1.01 * (4 * 2.0 ** -24 * (dot.abs() + b.abs()) + eps / 2 * want.abs()) + torch.finfo(dtype).tiny * eps
    worst = float(((y.double() - want).abs() / tol).max())
    assert worst <= 1.0, f"worst error {worst} of the tolerance"
    qc, qs = ops.int8_quantize(x)
    assert torch.equal(ops.int8_linear_quantized(qc, qs, w, ws, None if b.dim() == 0 else b.to(bias), dtype), y)


# last token tile of 1, 188, 220, 232 and 255 tokens; last feature tile of 8, 40, 64 and 137 (N % 8 != 0: 2-byte
# stores), its odd CTA partly or wholly past N; 1, 2, 9, 17 and 33 k-blocks; one tile a pair and up to seven; more
# than 32 token tiles
@pytest.mark.parametrize("m,k,n", [(257, 2064, 8000), (1000, 2064, 2600), (511, 2064, 5001), (1500, 2064, 2003),
                                   (700, 2064, 4000), (3000, 144, 10007), (3000, 16, 10000), (2100, 4112, 1032),
                                   (8500, 1040, 1300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pairs(m, k, n, dtype):
    check(m, k, n, dtype, [None, dtype, torch.float32][(m + n) % 3])


# tiles of 32, 64 and 128 tokens; two and four CTAs; stages that they share evenly and not; N % 8 != 0
@pytest.mark.parametrize("m,k,n", [(65, 8192, 20), (65, 12304, 133), (200, 8192, 520), (200, 12304, 517),
                                   (130, 16384, 2000), (130, 12304, 2000), (130, 16384, 4096), (130, 12304, 4090),
                                   (300, 30000, 300)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_k_split_over_a_cluster(m, k, n, dtype, bias):
    check(m, k, n, dtype, dtype if bias else None)


# up to 8 tokens: K over 2, 4 and 8 CTAs; 9 to 64 tokens: rows of 16, 32 and 64 tokens
@pytest.mark.parametrize("m,k,n", [(1, 8192, 130), (7, 4096, 900), (8, 14336, 600), (5, 65536, 40), (3, 2064, 1000),
                                   (9, 6000, 7000), (16, 512, 7090), (32, 1040, 999), (33, 1008, 1000), (64, 80, 13000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows(m, k, n, dtype):
    check(m, k, n, dtype, [None, dtype, torch.float32][(m + n) % 3])


def test_one_token_without_a_batch_dimension():
    from nanosglang_b200 import ops
    x, w, ws, b = make(1, 512, 70, torch.bfloat16, torch.bfloat16)
    want = ops.int8_linear(x, w, ws, b)
    assert torch.equal(ops.int8_linear(x[0], w, ws, b), want[0])
    codes, s = ops.int8_quantize(x[0])
    assert codes.shape == (512,) and s.shape == ()
    assert torch.equal(ops.int8_linear_quantized(codes, s, w, ws, b), want[0])
    assert torch.equal(ops.int8_linear(x.expand(9, 512), w, ws, b), want.expand(9, 70))
