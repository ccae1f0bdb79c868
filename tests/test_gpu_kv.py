"""The 8-bit key/value cache and its decode attention on the GPU.

Tolerances. Codes, scales and values read back are compared bit for bit with
float32 operations on the CPU. For attention against 64 bits, with weights
p[t] = exp(score[t]), the output's error is at most (first order)
  * the fp16 rounding of each weight, half an ulp: 2^-11 relative, and below
    fp16's normal range 2^-25 of the largest weight times scale;
  * an error d of a score in the exponent changes its weight by d, in the
    numerator and in the denominator: 2 d. Products of codes and q are exact,
    a sum of D terms in fp32 is off by D 2^-23 of the sum of their magnitudes
    (2^-23 a term: the tensor core may truncate), the scalings, the maximum's
    subtraction and exp2 by 8 * 2^-24 of the largest magnitudes;
  * fp32 accumulation over n tokens: n 2^-23 relative to sum p |v|;
  * the rounding to the output's type: eps / 2.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
CODES = [torch.int8, torch.float8_e4m3fn]


def ref_encode(rows, codes):
    """float32 rows -> codes and scales by float32 operations (CPU)."""
    s = rows.abs().amax(-1) / (127.0 if codes == torch.int8 else 448.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = rows / s[..., None]
    return (q.round().clamp(-127, 127).to(torch.int8) if codes == torch.int8 else q.to(codes)), s


def make_pool(pages, page, heads, dim, codes, layout="nhd", seed=0, spread=1.0):
    """k_cache, v_cache, k_scale, v_scale on the GPU, [pages, page, heads, dim]."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        rows = torch.randn(pages, page, heads, dim, generator=g)
        rows *= torch.exp(spread * torch.randn(pages, page, heads, 1, generator=g))
        c, s = ref_encode(rows, codes)
        if layout == "hnd":
            c = c.view(torch.uint8).transpose(1, 2).contiguous().cuda().view(codes).transpose(1, 2)
            s = s.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        else:
            c, s = c.cuda(), s.cuda()
        out.append((c, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def values(c, s):
    return c.cpu().to(torch.float16).double() * s.cpu().double()[..., None]


def check_attention(out, lse, q, pool, table, lens, scale):
    kc, vc, ks, vs = pool
    page = kc.shape[1]
    k_all, v_all, q = values(kc, ks), values(vc, vs), q.cpu().double()
    heads, dim = kc.shape[2], kc.shape[3]
    group = q.shape[1] // heads
    eps = torch.finfo(out.dtype).eps
    got_out, got_lse = out.cpu().double(), lse.cpu().double()
    worst = 0.0
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            assert (got_out[b] == 0).all() and (got_lse[b] == -math.inf).all()
            continue
        pages = table[b].cpu().long()[:-(-n // page)]
        kb = k_all[pages].reshape(-1, heads, dim)[:n]
        vb = v_all[pages].reshape(-1, heads, dim)[:n]
        for h in range(q.shape[1]):
            k, v = kb[:, h // group], vb[:, h // group]
            score = k @ q[b, h] * scale
            size = (k.abs() @ q[b, h].abs() * abs(scale)).max()
            m = score.max()
            p = torch.exp(score - m)
            total = p.sum()
            want = p @ v / total
            # score error: the dot product, and the fp32 roundings of score, log2(scale), maximum and exp2
            top_v = v.abs().amax(-1)
            lg = math.log(2) * max(abs(math.log2(t)) if t > 0 else 0.0 for t in (top_v.max().item(), top_v.min().item()))
            d = size * dim * 2.0 ** -23 + (size + lg + 16) * 8 * 2.0 ** -24
            absum = (p @ v.abs()) / total
            weight = (p * top_v).max() / total
            tol = absum * (2.0 ** -11 + 2 * d + n * 2.0 ** -23) + n * 2.0 ** -25 * weight
            tol = 1.05 * tol + eps / 2 * want.abs() + torch.finfo(out.dtype).tiny * eps
            worst = max(worst, ((got_out[b, h] - want).abs() / tol).max().item())
            want_lse = m + torch.log(total)
            tol_lse = d + n * 2.0 ** -23 + 4 * 2.0 ** -24 * (1 + want_lse.abs())
            worst = max(worst, ((got_lse[b, h] - want_lse).abs() / tol_lse).item())
    assert worst <= 1.0, f"worst error {worst} of the tolerance"


def tables(lens, page, pages, seed=0, width=None):
    """Shuffled distinct pages for every sequence; -1 past its end."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    perm = torch.randperm(pages, generator=g).tolist()
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, k in enumerate(need):
        t[b, :k] = torch.tensor([perm.pop() for _ in range(k)], dtype=torch.int32)
    return t.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


# --------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("heads,dim,page,layout", [(1, 16, 1, "nhd"), (2, 64, 16, "nhd"), (2, 64, 7, "hnd"),
                                                   (8, 128, 16, "hnd"), (3, 80, 5, "nhd"), (4, 96, 32, "hnd"),
                                                   (2, 256, 16, "nhd"), (1, 144, 3, "nhd")])
def test_write_and_read(heads, dim, page, layout, codes, dtype):
    from nanosglang_b200 import ops
    pages, T = 9, min(37, 9 * page - 2)
    pool = make_pool(pages, page, heads, dim, codes, layout, seed=3)
    before = [(c.view(torch.uint8) if c.dtype == codes else c).cpu().contiguous() for c in pool]
    g = torch.Generator().manual_seed(4)
    kv = [torch.randn(T, heads, dim, generator=g).to(dtype) for _ in range(2)]
    kv[0][0] = 0
    slots = torch.randperm(pages * page, generator=g)[:T]
    skip = T > 3
    if skip:
        slots[2] = -1
    ops.kv_cache_write(kv[0].cuda(), kv[1].cuda(), *pool, slots.cuda())
    for i in range(2):
        want_c, want_s = before[i].view(-1, heads, dim), before[2 + i].view(-1, heads)
        c, s = ref_encode(kv[i].float(), codes)
        keep = slots >= 0
        want_c[slots[keep]], want_s[slots[keep]] = c.view(torch.uint8)[keep], s[keep]
        # every place that no slot names is as it was
        assert torch.equal(pool[i].view(torch.uint8).cpu().reshape(-1, heads, dim), want_c)
        assert torch.equal(pool[2 + i].cpu().reshape(-1, heads), want_s)
    at = torch.cat([slots, torch.tensor([0, pages * page - 1, -5])])
    k, v = ops.kv_cache_read(*pool, at.cuda(), dtype)
    for got, c, s in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        flat = c.cpu().float().reshape(-1, heads, dim) * s.cpu().reshape(-1, heads)[..., None]
        want = flat[at.clamp(min=0)].to(dtype)
        want[at < 0] = 0
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_range(dtype, codes):
    """Tiny, huge and non-finite rows, and every quotient a tie can reach."""
    from nanosglang_b200 import ops
    fi = torch.finfo(dtype)
    x = torch.zeros(6, 1, 64, dtype=dtype)
    x[0, 0, :3] = torch.tensor([fi.smallest_normal * fi.eps, -fi.smallest_normal * fi.eps, 0]).to(dtype)
    x[1, 0, :3] = torch.tensor([fi.max, -fi.max, fi.max / 2]).to(dtype)
    x[2, 0] = torch.arange(64).to(dtype) * 7  # 441 = 63 * 7 and its fractions
    x[2, 0, 1] = 448
    x[3, 0] = (torch.arange(64).float() / 64 * 1.75).to(dtype)  # 0.75 of the largest: a tie of e4m3 up to the scale's rounding
    x[4, 0, 5] = float("nan")
    x[5, 0, 6] = float("-inf")
    pool = make_pool(1, 6, 1, 64, codes)
    slots = torch.arange(6).cuda()
    ops.kv_cache_write(x.cuda(), x.cuda(), *pool, slots)
    c, s = ref_encode(x.float(), codes)
    assert torch.equal(pool[0].view(torch.uint8).cpu().view(6, 64)[:4], c.view(torch.uint8).view(6, 64)[:4])
    assert torch.equal(pool[3].cpu().view(-1)[:4], s.view(-1)[:4])
    k, _ = ops.kv_cache_read(*pool, slots, torch.bfloat16)
    assert k[4:].isnan().all() and k[:4].isfinite().all()


def test_write_strided_rows_and_bad_slots():
    from nanosglang_b200 import _lib, ops
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(12, 8, 64, generator=g).to(torch.bfloat16).cuda()  # 4 q, 2 k, 2 v heads in one buffer
    a, b = make_pool(2, 16, 2, 64, torch.int8), make_pool(2, 16, 2, 64, torch.int8)
    slots = torch.arange(12).cuda()
    ops.kv_cache_write(qkv[:, 4:6], qkv[:, 6:], *a, slots)
    ops.kv_cache_write(qkv[:, 4:6].contiguous(), qkv[:, 6:].contiguous(), *b, slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    odd = torch.randn(12, 2, 70, generator=g).to(torch.bfloat16).cuda()[..., 3:67]  # rows off 16-byte alignment
    ops.kv_cache_write(odd, odd, *a, slots)
    ops.kv_cache_write(odd.contiguous(), odd.contiguous(), *b, slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # a slot past the pool is skipped and recorded; nothing else changes
    _lib.device_status_reset()
    before = [x.clone() for x in a]
    ops.kv_cache_write(odd[:1] * 0, odd[:1] * 0, *a, torch.tensor([32]).cuda())
    assert _lib.device_status()[:2] == (_lib.EINVAL, 200)
    assert all(torch.equal(x, y) for x, y in zip(a, before))
    _lib.device_status_reset()
    k, v = ops.kv_cache_read(*a, torch.tensor([1 << 40, 3]).cuda(), torch.bfloat16)
    assert _lib.device_status()[:2] == (_lib.EINVAL, 201)
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[1] != 0).any()
    _lib.device_status_reset()


# --------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("heads,group,dim,page,layout", [
    (2, 7, 64, 16, "nhd"), (8, 4, 128, 16, "nhd"), (2, 8, 128, 64, "hnd"), (1, 1, 64, 1, "nhd"),
    (3, 2, 96, 5, "hnd"), (2, 12, 128, 32, "nhd"), (1, 16, 64, 16, "hnd"), (1, 33, 80, 16, "nhd"),
    (2, 3, 256, 16, "nhd"), (1, 20, 192, 24, "hnd"), (1, 9, 16, 48, "nhd"), (2, 1, 32, 128, "hnd")])
def test_attention(heads, group, dim, page, layout, codes, dtype):
    from nanosglang_b200 import ops
    # lengths: empty rows, one token, both sides of a warp's 16, of a unit of 64, of a page, and long ones
    lens = [1, 0, 15, 16, 17, page, page + 1, 63, 64, 65, 0, 333, 1500]
    pages = sum(-(-n // page) for n in lens) + 2
    pool = make_pool(pages, page, heads, dim, codes, layout, seed=dim + group)
    table, lens_t = tables(lens, page, pages, seed=6)
    g = torch.Generator().manual_seed(7)
    q = (1.5 * torch.randn(len(lens), heads * group, dim, generator=g)).to(dtype).cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    check_attention(out, lse, q, pool, table, lens_t, dim ** -0.5)
    assert torch.equal(ops.kv_attention_decode(q, *pool, table, lens_t), out)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens,heads,group,dim", [([40001], 2, 4, 128), ([9000, 1, 0, 12345], 1, 8, 64),
                                                  ([5] * 300, 1, 2, 64), ([700] * 130, 2, 2, 64),
                                                  ([0, 0, 0], 2, 4, 64), ([2500] * 5, 8, 1, 128)])
def test_attention_splits(lens, heads, group, dim, codes):
    """Items cut over many CTAs, many items per CTA, more CTAs than units; a
    second call gives the same bits."""
    from nanosglang_b200 import ops
    page = 16
    pages = sum(-(-n // page) for n in lens) + 1
    pool = make_pool(pages, page, heads, dim, codes, seed=8)
    table, lens_t = tables(lens, page, pages, seed=9)
    q = torch.randn(len(lens), heads * group, dim, generator=torch.Generator().manual_seed(10)).half().cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    check_attention(out, lse, q, pool, table, lens_t, dim ** -0.5)
    again, lse2 = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("lens", [[700], [0, 513, 1, 300], [33] * 40, [129, 0, 0, 256] * 36])
@pytest.mark.parametrize("heads,group", [(5, 1), (12, 1), (17, 9), (32, 1), (37, 1), (64, 1)])
def test_attention_many_kv_heads(heads, group, lens):
    """Heads that are walked side by side in every number (37: alone, 64: two
    rows of 32, 17 x 9: 34 items of a sequence in two rows), more items than
    workers and fewer, segments of one unit."""
    from nanosglang_b200 import ops
    dim, page, codes = 64, 16, torch.int8
    pages = sum(-(-n // page) for n in lens) + 3
    pool = make_pool(pages, page, heads, dim, codes, "nhd", seed=20)
    table, n = tables(lens, page, pages, seed=21)
    g = torch.Generator().manual_seed(22)
    q = torch.randn(len(lens), heads * group, dim, generator=g).to(torch.bfloat16).cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, n, return_lse=True)
    check_attention(out, lse, q, pool, table, n, dim ** -0.5)
    again = ops.kv_attention_decode(q, *pool, table, n)
    assert torch.equal(out, again)


@pytest.mark.parametrize("codes", CODES)
def test_attention_ranges(codes):
    """Scales of v over thirty orders of magnitude within one sequence, peaked
    and flat softmax, a large and a negative softmax scale, tiny and huge q."""
    from nanosglang_b200 import ops
    lens, page, dim = [500, 130, 77], 16, 64
    pages = 60
    kc, vc, ks, vs = make_pool(pages, page, 1, dim, codes, seed=11)
    table, lens_t = tables(lens, page, pages)
    g = torch.Generator().manual_seed(12)
    q0 = torch.randn(3, 4, dim, generator=g)
    wild = (10.0 ** (30 * torch.rand(pages, page, 1, generator=g) - 20)).cuda()
    for q, scale, v in ((q0.bfloat16(), 0.125, wild), ((q0 * 30).half(), 0.125, vs), ((q0 * 1e-6).half(), 0.125, vs),
                        ((q0 * 1e30).bfloat16(), 1e-31, vs), ((q0 * 1e-30).bfloat16(), 1e30, vs),
                        (q0.half(), -0.5, vs), (q0.half(), 0.0, vs), (q0.bfloat16(), 0.125, vs * 0)):
        pool = (kc, vc, ks, v)
        out, lse = ops.kv_attention_decode(q.cuda(), *pool, table, lens_t, softmax_scale=scale, return_lse=True)
        if out.dtype == torch.bfloat16 or float(v.max()) < 1:
            check_attention(out, lse, q, pool, table, lens_t, scale)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("page", [16, 5])
def test_attention_ignores_what_is_not_held(codes, page):
    """NaN codes and scales past a sequence's end (inside its last page too),
    table entries past its pages, and other sequences' NaN stay out."""
    from nanosglang_b200 import ops
    lens, dim = [37, 64, 0, 130], 64
    pages = 60
    pool = make_pool(pages, page, 2, dim, codes, seed=13)
    table, lens_t = tables(lens, page, pages, width=40)
    q = torch.randn(4, 6, dim, generator=torch.Generator().manual_seed(14)).bfloat16().cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    check_attention(out, lse, q, pool, table, lens_t, dim ** -0.5)
    held = torch.zeros(pages * page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            held[int(table[b, t // page]) * page + t % page] = True
    at = (~held).nonzero()[:, 0]
    for c in pool[:2]:
        c.view(torch.uint8)[at // page, at % page] = 0x7F
    for s in pool[2:]:
        s[at // page, at % page] = float("nan")
    wild = table.clone()
    wild[table < 0] = 2 ** 31 - 1
    got, got_lse = ops.kv_attention_decode(q, *pool, wild, lens_t, return_lse=True)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    # a NaN row reaches the heads that read it and no others
    p0 = int(table[1, 3])
    pool[2][p0, 2, 0] = float("nan")
    got = ops.kv_attention_decode(q, *pool, table, lens_t)
    assert got[1, :3].isnan().all() and torch.equal(got[1, 3:], out[1, 3:]) and torch.equal(got[[0, 2, 3]], out[[0, 2, 3]])
    pool[2][p0, 2, 0] = 1.0
    pool[3][p0, 2, 1] = float("nan")
    got = ops.kv_attention_decode(q, *pool, table, lens_t)
    assert got[1, 3:].isnan().all() and torch.equal(got[[0, 2, 3]], out[[0, 2, 3]])


@pytest.mark.parametrize("page", [16, 5])
def test_attention_bad_pages_and_lengths(page):
    from nanosglang_b200 import _lib, ops
    lens, dim = [70, 200], 64
    pages = 64
    pool = make_pool(pages, page, 1, dim, torch.int8, seed=15)
    table, lens_t = tables(lens, page, pages)
    q = torch.randn(2, 4, dim, generator=torch.Generator().manual_seed(16)).half().cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    for bad in (pages, -3, 2 ** 31 - 1):
        _lib.device_status_reset()
        t = table.clone()
        t[0, 1] = bad
        got, got_lse = ops.kv_attention_decode(q, *pool, t, lens_t, return_lse=True)
        assert _lib.device_status()[:2] == (_lib.EINVAL, 202)
        assert torch.equal(got[1], out[1]) and got[0].isfinite().all() and (got_lse[0] < lse[0]).all()
    width = table.shape[1]
    for n, clamped in ((width * page + 1, width * page), (-7, 0)):
        _lib.device_status_reset()
        t = torch.where(table < 0, 0, table).to(torch.int32)
        got = ops.kv_attention_decode(q, *pool, t, torch.tensor([n, 200], dtype=torch.int32).cuda())
        assert _lib.device_status()[:2] == (_lib.EINVAL, 203)
        want = ops.kv_attention_decode(q, *pool, t, torch.tensor([clamped, 200], dtype=torch.int32).cuda())
        assert torch.equal(got, want)
    _lib.device_status_reset()


def test_attention_far_pool():
    """A pool whose far pages lie past 2^32 bytes from its start."""
    from nanosglang_b200 import ops
    pages, page, heads, dim = 2 ** 21 + 3, 16, 1, 128
    kc = torch.empty(pages, page, heads, dim, dtype=torch.int8, device="cuda")
    vc = torch.empty_like(kc)
    ks = torch.empty(pages, page, heads, device="cuda")
    vs = torch.empty_like(ks)
    near = make_pool(6, page, heads, dim, torch.int8, seed=17)
    far = torch.tensor([pages - 1, 5, pages - 3, 2 ** 20, pages - 2, 0])
    g = torch.Generator().manual_seed(18)
    rows = [torch.randn(6 * page, heads, dim, generator=g).bfloat16().cuda() for _ in range(2)]
    slots = (far[:, None] * page + torch.arange(page)).view(-1).cuda()
    ops.kv_cache_write(*rows, kc, vc, ks, vs, slots)
    ops.kv_cache_write(*rows, *near, torch.arange(6 * page).cuda())
    for x, y in zip(ops.kv_cache_read(kc, vc, ks, vs, slots, torch.half),
                    ops.kv_cache_read(*near, torch.arange(6 * page).cuda(), torch.half)):
        assert torch.equal(x, y)
    q = torch.randn(1, 4, dim, generator=g).bfloat16().cuda()
    n = torch.tensor([91], dtype=torch.int32).cuda()
    a = ops.kv_attention_decode(q, kc, vc, ks, vs, far[None].int().cuda(), n)
    b = ops.kv_attention_decode(q, *near, torch.arange(6, dtype=torch.int32)[None].cuda(), n)
    assert torch.equal(a, b)


def test_attention_captured_streams_and_views():
    """A captured call follows seq_lens and the cache as they change; two
    graphs and an eager call in between do not disturb one another; q and the
    table may be strided views."""
    from nanosglang_b200 import ops
    page, heads, dim, width = 16, 2, 64, 30
    pool = make_pool(70, page, heads, dim, torch.float8_e4m3fn, seed=19)
    table, lens = tables([400, 3, 470, 0], page, 70, width=width)
    full = torch.where(table < 0, 0, table).to(torch.int32)
    g = torch.Generator().manual_seed(20)
    qkv = torch.randn(4, 12, dim, generator=g).bfloat16().cuda()
    q = qkv[:, :8]
    wide = torch.zeros(4, width + 9, dtype=torch.int32).cuda()
    wide[:, 4:4 + width] = full
    view = wide[:, 4:4 + width]
    want = ops.kv_attention_decode(q.contiguous(), *pool, full, lens)
    assert torch.equal(ops.kv_attention_decode(q, *pool, view, lens), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.kv_attention_decode(q, *pool, view, lens)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, ops.kv_attention_decode(q, *pool, full, lens, return_lse=True)))
    for new in ([1, 480, 17, 100], [0, 0, 480, 64]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        for gr, _ in graphs:
            gr.replay()
        eager = ops.kv_attention_decode(q, *pool, full, lens, return_lse=True)
        torch.cuda.synchronize()
        check_attention(*eager, q, pool, full, lens, dim ** -0.5)
        for _, (o, l) in graphs:
            assert torch.equal(o, eager[0]) and torch.equal(l, eager[1])


def test_empty_batches():
    from nanosglang_b200 import ops
    pool = make_pool(4, 16, 2, 64, torch.int8)
    none = torch.zeros(0, dtype=torch.int64).cuda()
    rows = torch.zeros(0, 2, 64, dtype=torch.half).cuda()
    before = [x.clone() for x in pool]
    ops.kv_cache_write(rows, rows, *pool, none)
    assert all(torch.equal(x, y) for x, y in zip(pool, before))
    assert ops.kv_cache_read(*pool, none, torch.half)[0].shape == (0, 2, 64)
    q = torch.zeros(0, 4, 64, dtype=torch.half).cuda()
    assert ops.kv_attention_decode(q, *pool, torch.zeros(0, 3, dtype=torch.int32).cuda(),
                                   torch.zeros(0, dtype=torch.int32).cuda()).shape == (0, 4, 64)
    # a table without columns holds no token
    q = torch.ones(2, 4, 64, dtype=torch.half).cuda()
    out, lse = ops.kv_attention_decode(q, *pool, torch.zeros(2, 0, dtype=torch.int32).cuda(),
                                       torch.zeros(2, dtype=torch.int32).cuda(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_refusals():
    from nanosglang_b200 import ops
    kc, vc, ks, vs = make_pool(4, 16, 2, 64, torch.int8)
    rows = torch.zeros(3, 2, 64, dtype=torch.half).cuda()
    slots = torch.arange(3).cuda()
    for bad, err in [((rows.float(), rows, kc, vc, ks, vs, slots), TypeError),
                     ((rows, rows.bfloat16(), kc, vc, ks, vs, slots), TypeError),
                     ((rows, rows, kc.float(), vc, ks, vs, slots), TypeError),
                     ((rows, rows, kc, vc.view(torch.float8_e4m3fn), ks, vs, slots), TypeError),
                     ((rows, rows, kc, vc[:2], ks, vs, slots), ValueError),
                     ((rows, rows, kc, vc, ks[:2], vs, slots), ValueError),
                     ((rows, rows, kc, vc, ks, vs.half(), slots), ValueError),
                     ((rows, rows, kc, vc, ks, vs, slots.int()), TypeError),
                     ((rows, rows, kc, vc, ks, vs, slots[:2]), ValueError),
                     ((rows, rows[..., :32], kc, vc, ks, vs, slots), ValueError),
                     ((rows, rows, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, ks, vs, slots), ValueError),
                     ((rows, rows, kc, vc, ks, vs, slots.cpu()), RuntimeError)]:
        with pytest.raises(err):
            ops.kv_cache_write(*bad)
    with pytest.raises(TypeError):
        ops.kv_cache_read(kc, vc, ks, vs, slots, torch.float32)
    q = torch.zeros(2, 4, 64, dtype=torch.half).cuda()
    table, lens = torch.zeros(2, 3, dtype=torch.int32).cuda(), torch.ones(2, dtype=torch.int32).cuda()
    for bad, err in [((q.float(), kc, vc, ks, vs, table, lens), TypeError),
                     ((q[:, :3], kc, vc, ks, vs, table, lens), ValueError),
                     ((q[..., :32], kc, vc, ks, vs, table, lens), ValueError),
                     ((q, kc, vc, ks, vs, table.long(), lens), TypeError),
                     ((q, kc, vc, ks, vs, table[:1], lens), TypeError),
                     ((q, kc, vc, ks, vs, table, lens.long()), TypeError),
                     ((q, kc, vc, ks, vs, table, lens[:1]), TypeError)]:
        with pytest.raises(err):
            ops.kv_attention_decode(*bad)
    with pytest.raises(RuntimeError):
        ops.kv_attention_decode(q, kc, vc, ks, vs, table, lens, softmax_scale=float("nan"))
    odd = make_pool(4, 16, 2, 24, torch.int8)  # head_dim not a multiple of 16
    with pytest.raises(RuntimeError):
        ops.kv_cache_read(*odd, slots, torch.half)
