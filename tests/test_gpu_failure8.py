"""Failure path of the 8-bit operators' bounded waits, on the GPU, without a
fault: through the test hook of the C ABI one barrier expects an arrival that
never comes, with a short limit the wait for it runs out, and the kernel must
record its tag, let its copies land and return; the context stays usable."""

import pytest
import torch

from test_gpu_kv import make_pool, tables

pytestmark = pytest.mark.gpu

ATTENTION_WAIT_TAG = 204


@pytest.fixture
def withheld():
    """A context manager's worth of a call: runs fn with one arrival withheld
    and a limit of 1 ms, returns the status word."""
    from nanosglang_b200 import _lib

    def run(fn):
        torch.cuda.synchronize()
        _lib.device_status_reset()
        _lib.set_wait_limit_ns(1_000_000)
        prev = _lib.withhold_weight_load_for_test(True)
        try:
            fn()
            torch.cuda.synchronize()  # the kernels return: no hang, no fault
        finally:
            _lib.withhold_weight_load_for_test(prev)
        status = _lib.device_status()
        _lib.device_status_reset()
        return status

    return run


# what the workspace holds beforehand: words that are no count and no slot, and words that could be
@pytest.mark.parametrize("word", [0x7F7F7F7F, -2 ** 31, -1, 3])
@pytest.mark.parametrize("lens,heads,dim,page", [([20000, 1, 700], 2, 64, 16), ([300] * 200, 4, 128, 16),
                                                 ([9000, 40, 500], 2, 64, 5)])
def test_attention_wait_runs_out(withheld, lens, heads, dim, page, word):
    """A worker that gives up leaves its items' entries in the workspace as they
    were; the join follows none that the grid cannot have written."""
    from nanosglang_b200 import _lib
    pages = sum(-(-n // page) for n in lens) + 1
    pool = make_pool(pages, page, heads, dim, torch.int8, seed=41)
    table, lens_t = tables(lens, page, pages, seed=42)
    b, h = len(lens), heads * 2
    q = torch.randn(b, h, dim, generator=torch.Generator().manual_seed(43)).bfloat16().cuda()
    lib = _lib.load()
    width = table.shape[1]
    nbytes = lib.nsq_kv_attention_workspace_size(b, h, heads, dim, page, width)
    assert nbytes > 0
    kc, vc, ks, vs = pool
    desc = _lib.KV_CACHE.pack(*(t.data_ptr() for t in (kc, vc, ks, vs)), *kc.shape, *kc.stride()[:3], *vc.stride()[:3],
                              *ks.stride(), *vs.stride(), _lib.KV_INT8)

    def call():
        work = torch.full((nbytes // 4,), word, dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)
        _lib.check(lib.nsq_kv_attention_decode(
            desc, q.data_ptr(), _lib.DTYPE_BF16, q.stride(0), q.stride(1), b, h, table.data_ptr(), width, width,
            lens_t.data_ptr(), dim ** -0.5, out.data_ptr(), None, work.data_ptr(), nbytes,
            torch.cuda.current_stream().cuda_stream), "nsq_kv_attention_decode")
        torch.cuda.synchronize()
        return out

    want = call()
    assert _lib.device_status()[0] == 0
    got = []
    code, where, _ = withheld(lambda: got.append(call()))
    assert (code, where) == (_lib.EDEVICE_TIMEOUT, ATTENTION_WAIT_TAG)
    assert torch.equal(got[0][-1], want[-1])  # far from the first worker's share
    assert torch.equal(call(), want) and _lib.device_status()[0] == 0


# a tile of one CTA, of a pair, and one whose K is split over a cluster; with and without a staged y
@pytest.mark.parametrize("m,k,n", [(300, 2048, 1024), (300, 2048, 1001), (1000, 2064, 2600), (200, 12304, 520)])
def test_int8_gemm_wait_runs_out(withheld, m, k, n):
    from nanosglang_b200 import _lib, ops
    g = torch.Generator().manual_seed(44)
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    ws = torch.rand(n, generator=g).cuda()
    want = ops.int8_linear(x, w, ws)
    code, where, _ = withheld(lambda: ops.int8_linear(x, w, ws))
    assert code == _lib.EDEVICE_TIMEOUT and 210 <= where <= 215
    assert torch.equal(ops.int8_linear(x, w, ws), want) and _lib.device_status()[0] == 0
