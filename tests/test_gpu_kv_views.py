"""Caches whose pages, tokens or heads share memory (expanded tensors), as the
calls that only read them may get."""

import pytest
import torch

from test_gpu_kv import CODES, check_attention, make_pool, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("shared", ["heads", "pages", "tokens", "k heads only"])
def test_attention_over_an_expanded_pool(shared, page, dim, codes):
    """One stored head, page or token stands for all of them (stride 0): the
    same bits as the pool written out."""
    from nanosglang_b200 import ops
    heads, lens = 4, [100, 0, 1, 333]
    pages = sum(-(-n // page) for n in lens) + 1
    dims = {"heads": 2, "pages": 0, "tokens": 1, "k heads only": 2}[shared]
    pool = make_pool(pages, page, heads, dim, codes, seed=31)
    view = []
    for i, t in enumerate(pool):
        raw = t.view(torch.uint8) if t.dtype == codes else t
        if shared != "k heads only" or i in (0, 2):
            raw = raw.narrow(dims, 0, 1).clone().expand(raw.shape)
        view.append(raw.view(codes) if t.dtype == codes else raw)
    full = [t.contiguous() for t in view]
    table, lens_t = tables(lens, page, pages, seed=32)
    q = torch.randn(4, 8, dim, generator=torch.Generator().manual_seed(33)).bfloat16().cuda()
    out, lse = ops.kv_attention_decode(q, *view, table, lens_t, return_lse=True)
    check_attention(out, lse, q, full, table, lens_t, dim ** -0.5)
    want, want_lse = ops.kv_attention_decode(q, *full, table, lens_t, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    slots = torch.arange(pages * page).cuda()
    for a, b in zip(ops.kv_cache_read(*view, slots, torch.half), ops.kv_cache_read(*full, slots, torch.half)):
        assert torch.equal(a, b)


def test_write_of_half_a_thousand_million_rows():
    """More threads (16 lanes for two rows) than 32 bits count: the last tokens
    are written, and nothing but they (one row of k and v, expanded)."""
    from nanosglang_b200 import ops
    n, dim = 2 ** 29 + 1000, 256
    pool = make_pool(2, 16, 1, dim, torch.int8, seed=34)
    want = [t.clone() for t in pool]
    row = torch.randn(1, 1, dim, generator=torch.Generator().manual_seed(35)).bfloat16().cuda()
    slots = torch.full((n,), -1, device="cuda")
    slots[-3:] = torch.tensor([4, 31, 9])
    ops.kv_cache_write(row.expand(n, 1, dim), row.expand(n, 1, dim), *pool, slots)
    ops.kv_cache_write(row.expand(3, 1, dim), row.expand(3, 1, dim), *want, slots[-3:].clone())
    assert all(torch.equal(a, b) for a, b in zip(pool, want))


def test_attention_over_expanded_queries_and_tables():
    """One query for all heads, one page table for all sequences (stride 0), and
    one page named many times."""
    from nanosglang_b200 import ops
    page, heads, dim, width = 16, 2, 64, 20
    pool = make_pool(30, page, heads, dim, torch.int8, seed=36)
    g = torch.Generator().manual_seed(37)
    lens = torch.tensor([0, 1, 77, 320, 5], dtype=torch.int32).cuda()
    table = torch.randperm(30, generator=g)[:width].int().cuda()
    table[3:9] = table[3]
    q = torch.randn(5, 1, dim, generator=g).half().cuda()
    out, lse = ops.kv_attention_decode(q.expand(5, 6, dim), *pool, table.expand(5, width), lens, return_lse=True)
    full = table.repeat(5, 1)
    check_attention(out, lse, q.repeat(1, 6, 1), pool, full, lens, dim ** -0.5)
    want = ops.kv_attention_decode(q.repeat(1, 6, 1), *pool, full, lens)
    assert torch.equal(out, want)


@pytest.mark.parametrize("width", [3, 12])
def test_attention_of_thousands_of_sequences(width):
    """More sequences than a block has threads, most of them empty or short."""
    from nanosglang_b200 import ops
    b, page, dim = 5003, 16, 64
    pool = make_pool(64, page, 1, dim, torch.int8, seed=38)
    g = torch.Generator().manual_seed(39)
    lens = torch.randint(-30, 17 * width, (b,), generator=g).clamp(0, page * width).int()
    lens[-1] = page * width
    table = torch.randint(0, 64, (b, width), generator=g).int()
    q = torch.randn(b, 2, dim, generator=g).bfloat16()
    out, lse = ops.kv_attention_decode(q.cuda(), *pool, table.cuda(), lens.cuda(), return_lse=True)
    at = torch.cat([torch.arange(0, b, 61), torch.tensor([b - 1])])
    check_attention(out[at.cuda()], lse[at.cuda()], q[at], pool, table[at], lens[at], dim ** -0.5)
    assert (out[(lens == 0).cuda()] == 0).all() and out.isfinite().all()
