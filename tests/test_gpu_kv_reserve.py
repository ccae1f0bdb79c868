"""Decode attention while SMs are kept free for others (nsq_set_sm_reserve)."""

import pytest
import torch

from test_gpu_kv import check_attention, make_pool, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sized,called", [(24, 0), (0, 24), (70, 10), (24, 24)])
@pytest.mark.parametrize("lens", [[9000, 3, 700], [300] * 150])
def test_workspace_sized_under_one_reserve_serves_another(lens, sized, called):
    from nanosglang_b200 import _lib
    page, heads, dim = 16, 2, 64
    pages = sum(-(-n // page) for n in lens) + 1
    pool = make_pool(pages, page, heads, dim, torch.int8, seed=51)
    table, lens_t = tables(lens, page, pages, seed=52)
    b, h, width = len(lens), heads * 3, table.shape[1]
    q = torch.randn(b, h, dim, generator=torch.Generator().manual_seed(53)).bfloat16().cuda()
    kc, vc, ks, vs = pool
    desc = _lib.KV_CACHE.pack(*(t.data_ptr() for t in pool), *kc.shape, *kc.stride()[:3], *vc.stride()[:3], *ks.stride(),
                              *vs.stride(), _lib.KV_INT8)
    lib = _lib.load()
    out, lse = torch.empty_like(q), torch.empty(b, h, device="cuda")
    prev = lib.nsq_set_sm_reserve(sized)
    try:
        nbytes = lib.nsq_kv_attention_workspace_size(b, h, heads, dim, page, width)
        guard = 1 << 16
        work = torch.full((nbytes + guard,), 0x5A, dtype=torch.uint8, device="cuda")
        lib.nsq_set_sm_reserve(called)
        _lib.check(lib.nsq_kv_attention_decode(
            desc, q.data_ptr(), _lib.DTYPE_BF16, q.stride(0), q.stride(1), b, h, table.data_ptr(), width, width,
            lens_t.data_ptr(), dim ** -0.5, out.data_ptr(), lse.data_ptr(), work.data_ptr(), nbytes,
            torch.cuda.current_stream().cuda_stream), "nsq_kv_attention_decode")
        torch.cuda.synchronize()
    finally:
        lib.nsq_set_sm_reserve(prev)
    assert (work[nbytes:] == 0x5A).all()
    check_attention(out, lse, q, pool, table, lens_t, dim ** -0.5)
