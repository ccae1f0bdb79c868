"""Decode attention: joining the partial results of items cut over workers, in
every form of the join."""

import pytest
import torch

from test_gpu_kv import CODES, check_attention, make_pool, tables

pytestmark = pytest.mark.gpu


# one long sequence among more than a hundred short ones: more partials than a warp takes, four pairs a block;
# many sequences of 15 to 18 partials: both sides of what a warp takes; few items of hundreds of partials
@pytest.mark.parametrize("lens", [[3] * 70 + [20000] + [40] * 60, [940 + 3 * i for i in range(112)],
                                  [1, 30001, 0], [7000]])
@pytest.mark.parametrize("dim,heads,group", [(64, 1, 2), (128, 1, 8), (256, 1, 3), (112, 1, 9)])
@pytest.mark.parametrize("codes", CODES)
def test_join(lens, dim, heads, group, codes):
    from nanosglang_b200 import ops
    page = 16
    pages = sum(-(-n // page) for n in lens) + 1
    pool = make_pool(pages, page, heads, dim, codes, seed=71)
    table, lens_t = tables(lens, page, pages, seed=72)
    q = torch.randn(len(lens), heads * group, dim, generator=torch.Generator().manual_seed(73)).half().cuda()
    out, lse = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    check_attention(out, lse, q, pool, table, lens_t, dim ** -0.5)
    again, lse2 = ops.kv_attention_decode(q, *pool, table, lens_t, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
