"""Decode attention near the ends of its types' ranges, against 64 bits with the
tolerances of test_gpu_kv.py. Its term for the smallest subnormal of the output's
type covers what the kernel may lose at the low end: v's scale below 2^-140 leaves
a weight fewer than 11 bits, an error of 2^-25 of 2^-126 times a code of at
most 448, 2^-142 of bf16's 2^-133."""

import pytest
import torch

from test_gpu_kv import CODES, check_attention, make_pool, tables

pytestmark = pytest.mark.gpu


def spread_to(s, c, peak):
    """Scales s times what makes the largest value of codes c ``peak``."""
    top = (c.cpu().to(torch.float16).double().abs().amax(-1) * s.cpu().double()).max()
    return (s.cpu().double() * (peak / top)).float().cuda()


# the largest bf16 is 3.39e38; scales are subnormal below 1.2e-38
@pytest.mark.parametrize("peak", [3.3e38, 1e36, 1e-30, 1e-36, 1.5e-37, 1e-39])
@pytest.mark.parametrize("lens", [[2000, 64, 500], [100, 1, 128]])
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("flat", [True, False])
def test_v_at_the_ends_of_bf16(codes, lens, peak, flat):
    """Outputs stay right although sums over many tokens pass fp32's range, and
    although the scales of v are subnormal."""
    from nanosglang_b200 import ops
    page, dim, pages = 16, 64, sum(-(-n // 16) for n in lens)
    kc, vc, ks, vs = make_pool(pages, page, 1, dim, codes, seed=61, spread=0.2)
    vs = spread_to(vs, vc, peak)
    vc.view(torch.uint8)[:] &= 0x7F  # no cancellation: the outputs are near the end of the range
    table, lens_t = tables(lens, page, pages, seed=62)
    q = torch.randn(3, 4, dim, generator=torch.Generator().manual_seed(63)).bfloat16().cuda()
    scale = 0.0 if flat else dim ** -0.5
    out, lse = ops.kv_attention_decode(q, kc, vc, ks, vs, table, lens_t, softmax_scale=scale, return_lse=True)
    assert out.isfinite().all() and (out != 0).any()
    check_attention(out, lse, q, (kc, vc, ks, vs), table, lens_t, scale)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("long", [False, True])
def test_v_scales_over_the_whole_range_of_float32(codes, long):
    """One sequence whose scales of v go from 2^-145 to 2^110, the large ones
    last, first and at weights that make all of them count."""
    from nanosglang_b200 import ops
    n, page, dim = (600 if long else 120), 16, 64
    pages = -(-n // page)
    kc, vc, ks, vs = make_pool(pages, page, 1, dim, codes, seed=64)
    table = torch.arange(pages, dtype=torch.int32)[None].cuda()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    for first, last in ((-145, 110), (110, -145)):
        e = torch.linspace(first, last, pages * page)
        v = torch.exp2(e.double()).float().view(pages, page, 1).cuda()
        # scores fall as the scales rise: k rows are multiples of one direction.
        # A probability stays above 2^-115, in fp32's normal range
        k = torch.ones(pages, page, 1, dim, dtype=torch.int8, device="cuda")
        kcode = k if codes == torch.int8 else k.half().to(codes)
        for slope in (0.0, 0.2, 0.45):
            ksc = (-(e.double() * slope / dim)).float().view(pages, page, 1)
            top = ksc.min()
            ksc = (ksc - top).cuda()  # scales are not negative
            q = torch.ones(1, 2, dim).bfloat16().cuda()
            pool = (kcode, vc, ksc, v)
            out, lse = ops.kv_attention_decode(q, *pool, table, lens, softmax_scale=0.6931471805599453, return_lse=True)
            assert out.isfinite().all()
            check_attention(out, lse, q, pool, table, lens, 0.6931471805599453)


@pytest.mark.parametrize("codes", CODES)
def test_fp16_scales_and_queries(codes):
    """Peaked and flat softmax, negative and zero softmax scales, tiny and large
    fp16 queries, every result in fp16's range."""
    from nanosglang_b200 import ops
    lens, page, dim, pages = [500, 130, 77], 16, 64, 60
    kc, vc, ks, vs = make_pool(pages, page, 1, dim, codes, seed=65, spread=0.3)
    table, lens_t = tables(lens, page, pages)
    q0 = torch.randn(3, 4, dim, generator=torch.Generator().manual_seed(66))
    for q, scale in ((q0, 0.125), (q0 * 30, 0.125), (q0 * 1e-6, 0.125), (q0, -0.5), (q0, 0.0), (q0 * 1e4, 1e-5)):
        q = q.half().cuda()
        out, lse = ops.kv_attention_decode(q, kc, vc, ks, vs, table, lens_t, softmax_scale=scale, return_lse=True)
        assert out.isfinite().all()
        check_attention(out, lse, q, (kc, vc, ks, vs), table, lens_t, scale)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("n,first", [(3000, True), (3000, False), (120, True)])
@pytest.mark.parametrize("drop", [14, 18, 22])
def test_small_weights_keep_their_bits(codes, n, first, drop):
    """One token takes nearly all of the softmax, but its v is 0 in half of the
    dims: there the output is the sum of weights ``drop`` powers of two smaller.

    Each weight is off by 2^-11 of itself, and below 2^-26 of the largest by
    2^-37 of that; the other terms as in test_gpu_kv.py."""
    from nanosglang_b200 import ops
    page, dim, pages = 16, 64, -(-n // 16)
    g = torch.Generator().manual_seed(67)
    vc = torch.randint(1, 128, (pages, page, 1, dim), generator=g, dtype=torch.int8)
    at = 7 if first else n - 3
    vc[at // page, at % page, 0, :32] = 0
    if codes != torch.int8:
        vc = vc.float().to(codes)
    kc = torch.ones(pages, page, 1, dim).to(codes)
    ks = torch.rand(pages, page, 1, generator=g) / dim
    ks[at // page, at % page] = (drop + 1) / dim
    vs = torch.full((pages, page, 1), 2.0 ** -7)
    q = torch.ones(1, 2, dim).half()
    ln2 = 0.6931471805599453
    out = ops.kv_attention_decode(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(),
                                  torch.arange(pages, dtype=torch.int32)[None].cuda(),
                                  torch.tensor([n], dtype=torch.int32).cuda(), softmax_scale=ln2)
    score = (ks.double().view(-1)[:n] * dim) * ln2
    p = torch.exp(score - score.max())
    v = vc.half().double().view(-1, dim)[:n] * 2.0 ** -7
    total = p.sum()
    want = p @ v / total
    size = score.max()
    d = size * dim * 2.0 ** -23 + (size + 7 * ln2 + 16) * 8 * 2.0 ** -24
    tol = want * (2.0 ** -11 + 2 * d + n * 2.0 ** -23) + n * 2.0 ** -37 * (p * v.amax(-1)).max() / total
    tol = 1.05 * tol + 2.0 ** -11 * want + 2.0 ** -25
    worst = ((out[0].cpu().double() - want).abs() / tol).max().item()
    assert worst <= 1.0, f"worst error {worst} of the tolerance"


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,largest,rest", [(torch.float16, 6e4, 2.0 ** -10), (torch.float16, 6e4, 2.0 ** -20),
                                                (torch.float16, 2.0 ** -20, 2.0 ** -21),
                                                (torch.bfloat16, 2.0 ** 20, 2.0 ** -4),
                                                (torch.bfloat16, 2.0 ** 100, 2.0 ** 72),
                                                (torch.bfloat16, 2.0 ** -90, 2.0 ** -118)])
def test_small_elements_of_q_count(codes, dtype, largest, rest):
    """A head whose largest element meets zeros of k: its score is made of
    elements many powers of two smaller, each of which has to be exact."""
    from nanosglang_b200 import ops
    lens, page, dim, pages = [300, 61], 16, 64, 30
    kc, vc, ks, vs = make_pool(pages, page, 1, dim, codes, seed=68, spread=0.2)
    kc.view(torch.uint8)[..., 5] = 0
    table, lens_t = tables(lens, page, pages, seed=69)
    g = torch.Generator().manual_seed(70)
    q = ((1 + torch.rand(2, 4, dim, generator=g)) * rest * torch.randn(2, 4, dim, generator=g).sign()).to(dtype)
    q[..., 5] = largest
    scale = 0.25 / rest
    out, lse = ops.kv_attention_decode(q.cuda(), kc, vc, ks, vs, table, lens_t, softmax_scale=scale, return_lse=True)
    assert (lse[0] - lse[0].min() != 0).any()
    check_attention(out, lse, q, (kc, vc, ks, vs), table, lens_t, scale)
