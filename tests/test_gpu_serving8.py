"""The 8-bit operators together, as a serving loop uses them: int8 projections,
the 8-bit cache and its decode attention inside the harness engine, against the
same engine with every operator replaced by a 64-bit form.

Tolerance: the operators agree with 64 bits up to the rounding of their output
(tested on their own), so each of the 8 operators of a layer can move its
output by one rounding of the model's dtype (eps / 2 on either side, eps in
all); over L layers the logits can be off by 8 L eps of their norm.
"""

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


def plain_quantize(x):
    s = x.float().abs().amax(-1) * torch.ones((), device=x.device)
    s = (s.double() / 127).float()
    s = torch.where(s == 0, torch.ones_like(s), s)
    return (x.double() / s.double()[..., None]).float().round().to(torch.int8), s


def plain_quantized(codes, scale, w, ws, bias=None, dtype=torch.bfloat16):
    y = codes.double() @ w.double().t() * scale.double()[..., None] * ws.double()
    return (y if bias is None else y + bias.double()).to(dtype)


def plain_linear(x, w, ws, bias=None):
    return plain_quantized(*plain_quantize(x), w, ws, bias, x.dtype)


def plain_write(k, v, kc, vc, ks, vs, slots):
    page = kc.shape[1]
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        if c.dtype == torch.int8:
            codes, scale = plain_quantize(x)
        else:
            scale = (x.double().abs().amax(-1) / 448).float()
            scale = torch.where(scale == 0, torch.ones_like(scale), scale)
            codes = (x.double() / scale.double()[..., None]).float().to(c.dtype)
        c.view(torch.uint8)[slots // page, slots % page] = codes.view(torch.uint8)
        s[slots // page, slots % page] = scale


def plain_attention(q, kc, vc, ks, vs, table, lens, softmax_scale=None, return_lse=False):
    page, heads, dim = kc.shape[1:]
    group = q.shape[1] // heads
    out = torch.zeros_like(q)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        at = table[b].long()
        k, v = ((c.view(torch.uint8)[at].view(c.dtype).to(torch.float16).double() * s[at].double()[..., None])
                .reshape(-1, heads, dim)[:n] for c, s in ((kc, ks), (vc, vs)))
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        p = torch.einsum("hd,thd->ht", q[b].double(), k).mul(dim ** -0.5).softmax(-1)
        out[b] = torch.einsum("ht,thd->hd", p, v).to(q.dtype)
    return out


@pytest.fixture
def model():
    from harness import model as H
    from nanosglang_b200.quantization import quantize_model
    m = H.build_model(H.TINY, "cuda", torch.bfloat16)
    H.init_dense(m, 11)
    quantize_model(m, "int8")
    return m


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("codes,page,fused", [("int8", 64, True), ("fp8", 16, False), ("int8", 24, False)])
def test_engine_with_8bit_cache(model, codes, page, fused, monkeypatch):
    from harness import engine as E
    from harness import model as H
    from nanosglang_b200 import ops
    from nanosglang_b200.quantization import Int8Linear
    assert sum(isinstance(x, Int8Linear) for x in model.modules()) == 7 * H.TINY.num_hidden_layers
    if fused:
        H.fuse_projections(model)
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, H.TINY.vocab_size, (n,), generator=g).cuda() for n in (33, 1, 100)]
    logits, caches = [], []
    for plain in (False, True):
        with monkeypatch.context() as mp:
            if plain:
                mp.setattr(ops, "int8_quantize", plain_quantize)
                mp.setattr(ops, "int8_linear", plain_linear)
                mp.setattr(ops, "int8_linear_quantized", plain_quantized)
                mp.setattr(ops, "kv_cache_write", plain_write)
                mp.setattr(ops, "kv_attention_decode", plain_attention)
            eng = E.DecodeEngine(model, max_slots=4, max_len=150, max_steps=20, kv_cache=codes, page_size=page)
            eng.prefill(prompts)
            rows = []
            fed = torch.arange(3, device="cuda") + 5  # the same tokens on both sides
            with torch.no_grad():
                for step in range(4):
                    pos = eng.positions[:3] + step
                    ctx = (eng.first_place[:3] + pos, eng.page_table[:3], (pos + 1).to(torch.int32))
                    rows.append(model.forward_decode(fed + step, pos, eng.caches, ctx))
            logits.append(rows)
            caches.append(eng)
    eps = torch.finfo(torch.bfloat16).eps
    for own, want in zip(*logits):
        assert rel(own, want) <= 8 * H.TINY.num_hidden_layers * eps
    # the first layer's cache rows of the prompts: the same inputs but for one rounding of k and v
    slots = torch.arange(33, device="cuda")
    a, b = caches[0].caches[0][0], caches[1].caches[0][0]
    for x, y in zip(a.read(slots, torch.bfloat16), b.read(slots, torch.bfloat16)):
        assert rel(x, y) <= (1 / 127 if codes == "int8" else 2.0 ** -4)


def test_engine_graph_equals_eager(model):
    """Captured decode steps of the 8-bit engine (padded bucket included) give
    the tokens of eager steps; a second engine's graphs do not disturb them."""
    from harness import engine as E
    from harness import model as H
    g = torch.Generator().manual_seed(13)
    prompts = [torch.randint(0, H.TINY.vocab_size, (n,), generator=g).cuda() for n in (17, 64, 5)]
    engines = [E.DecodeEngine(model, max_slots=4, max_len=120, max_steps=30, kv_cache=c) for c in ("int8", "fp8", "int8")]
    for eng in engines[:2]:
        eng.capture()
    for eng in engines:
        eng.prefill(prompts)
    for _ in range(10):
        engines[0].decode_steps([3])  # 3 requests in the bucket of 4
        engines[1].decode_steps([3])
        with torch.no_grad():
            engines[2]._step(4)
    torch.cuda.synchronize()
    assert torch.equal(engines[0].history[:11, :3], engines[2].history[:11, :3])
    for a, b in zip(engines[0].caches, engines[2].caches):
        n = (17 + 10) // 64 * 64 + 27
        places = torch.arange(n, device="cuda")
        for x, y in zip(a[0].read(places[:27], torch.bfloat16), b[0].read(places[:27], torch.bfloat16)):
            assert torch.equal(x, y)


def test_int8_linear_module_and_row_shards():
    """from_linear against the weight it came from; row-parallel shards add up
    to a product that quantises each slice of x with its own scale."""
    from nanosglang_b200 import ops
    from nanosglang_b200 import tensor_parallel as TP
    from nanosglang_b200.quantization import Int8Linear
    torch.manual_seed(14)
    lin = nn.Linear(512, 96, bias=True).cuda().bfloat16()
    m = Int8Linear.from_linear(lin)
    w = lin.weight.double()
    step = w.abs().amax(1, keepdim=True) / 127
    # half a step, and what float32 adds: the quotient (below 128, where half an
    # ulp is 2^-18) rounds before it is rounded to a whole number, and the scale
    # is off by 2^-24 of itself: (0.5 + 2^-18) (1 + 2^-24) < 0.5 + 2^-17 steps
    assert ((m.weight_int8.double() * m.weight_scale.double()[:, None] - w).abs() <= step * (0.5 + 2.0 ** -17)).all()
    x = torch.randn(2, 5, 512, device="cuda").bfloat16()
    assert torch.equal(m(x), ops.int8_linear(x, m.weight_int8, m.weight_scale, m.bias))
    cast = Int8Linear.from_linear(lin).bfloat16()  # casts weight_scale as well
    assert torch.equal(cast(x), ops.int8_linear(x, m.weight_int8, m.weight_scale.bfloat16().float(), m.bias.bfloat16()))
    shards = [TP.RowParallelLinear.from_linear(m, 2, r, reduce_output=False) for r in range(2)]
    parts = [s(x[..., 256 * r:256 * (r + 1)]).double() for r, s in enumerate(shards)]
    want = [plain_linear(x[..., 256 * r:256 * (r + 1)], m.weight_int8[:, 256 * r:256 * (r + 1)], m.weight_scale,
                         m.bias if r == 0 else None).double() for r in range(2)]
    eps = torch.finfo(torch.bfloat16).eps
    for a, b in zip(parts, want):
        assert ((a - b).abs() <= eps * b.abs() + 1e-6).all()


@pytest.mark.parametrize("captured", [False, True])
def test_chain_with_programmatic_launch(captured):
    """Projection -> cache write -> attention -> projection, step after step,
    with programmatic dependent launch on: every kernel waits for the one it
    reads from, so nothing changes."""
    from nanosglang_b200 import QuantizedKVCache, _lib, ops
    g = torch.Generator().manual_seed(15)
    heads, kvh, dim, hidden, bs = 8, 2, 64, 512, 5
    layers = []
    for n, k in ((heads * dim, hidden), (kvh * dim, hidden), (kvh * dim, hidden), (hidden, heads * dim)):
        layers.append((torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda(),
                       (torch.rand(n, generator=g) * 1e-3).cuda()))
    x0 = torch.randn(bs, hidden, generator=g).bfloat16().cuda()
    table = torch.arange(bs * 20, dtype=torch.int32).view(bs, 20).cuda()

    def run(steps):
        cache = QuantizedKVCache(bs * 20, 16, kvh, dim, "fp8", "cuda")
        lens = torch.zeros(bs, dtype=torch.int32, device="cuda")
        places = torch.arange(bs, device="cuda") * 320
        x = x0.clone()

        def step():
            q, k, v = (ops.int8_linear(x, w, s) for w, s in layers[:3])
            cache.write(k.view(bs, kvh, dim), v.view(bs, kvh, dim), places)
            lens.add_(1)
            places.add_(1)
            o = cache.attend(q.view(bs, heads, dim), table, lens)
            x.copy_(torch.tanh(ops.int8_linear(o.view(bs, -1), *layers[3]) + x))

        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                step()
            for _ in range(steps - 1):
                gr.replay()
        else:
            for _ in range(steps):
                step()
        torch.cuda.synchronize()
        return x, cache.read(torch.arange(bs * 320, device="cuda"), torch.bfloat16)

    want, want_kv = run(200)
    prev = _lib.set_pdl(True)
    try:
        got, got_kv = run(200)
    finally:
        _lib.set_pdl(prev)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(got_kv, want_kv))
    assert _lib.device_status()[0] == 0
