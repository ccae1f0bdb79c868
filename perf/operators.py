"""The 8-bit serving operators as measured cases: int8 linears, the 8-bit
key/value cache (written, read back) and decode attention over that cache.

``run`` computes each operator in its plain form (elementary torch operations
in float32) or, with ``own`` set, through ``nanosglang_b200.ops``; ``exact``
computes the same outputs in 64 bits from the definitions:

  int8 linear   codes = rint(x / s), s = max|x| / 127 per token (1 where that
                is 0); y = (codes . weight_int8^T) * s * weight_scale + bias
  cache         per (token, head) row: s = max|row| / 127, codes = rint(row / s)
                (int8), or s = max|row| / 448, codes = e4m3(row / s) (fp8);
                read back as codes * s
  attention     softmax(scale * q . k^T) . v over the first seq_lens[b] tokens
                of each sequence's pages; a sequence of length 0 gives 0 and a
                log-sum-exp of -inf
"""

import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def listed():
    return [
        # one token through the gate projection of the 0.5B model: launch latency
        {"name": "linear-1", "op": "linear", "m": 1, "k": 896, "n": 4864, "dtype": "fp16", "bias": False},
        # a decode batch of 16 through the gate projection of the 8B model: weight bandwidth
        {"name": "linear-16", "op": "linear", "m": 16, "k": 4096, "n": 14336, "dtype": "bf16", "bias": False},
        # a chunk of ragged prompts through a long-K projection with few outputs
        {"name": "linear-777", "op": "linear", "m": 777, "k": 4864, "n": 896, "dtype": "bf16", "bias": True},
        # a full prefill chunk through the gate projection of the 8B model: tensor-core rate
        {"name": "linear-8192", "op": "linear", "m": 8192, "k": 4096, "n": 14336, "dtype": "bf16", "bias": False},
        # one new token of one short sequence, its context read back
        {"name": "cache-1", "op": "cache", "tokens": 1, "slots": 48, "kv_heads": 2, "dim": 64, "page": 16,
         "codes": "int8", "dtype": "fp16", "layout": "nhd"},
        # a decode step of 64 streams, contexts of 128 tokens read back
        {"name": "cache-64", "op": "cache", "tokens": 64, "slots": 8192, "kv_heads": 8, "dim": 128, "page": 16,
         "codes": "fp8", "dtype": "bf16", "layout": "nhd"},
        # a ragged prefill chunk into head-major pages
        {"name": "cache-5001", "op": "cache", "tokens": 5001, "slots": 5056, "kv_heads": 2, "dim": 64, "page": 64,
         "codes": "int8", "dtype": "bf16", "layout": "hnd"},
        # two full prefill chunks of the 8B model's heads
        {"name": "cache-16384", "op": "cache", "tokens": 16384, "slots": 16384, "kv_heads": 8, "dim": 128,
         "page": 16, "codes": "fp8", "dtype": "bf16", "layout": "nhd"},
        # one short sequence: launch latency
        {"name": "attention-short", "op": "attention", "batch": 1, "length": 40, "ragged": False, "kv_heads": 2,
         "group": 7, "dim": 64, "page": 16, "codes": "int8", "dtype": "fp16", "layout": "nhd"},
        # 64 streams at context 2048, the 8B model's heads
        {"name": "attention-64x2048", "op": "attention", "batch": 64, "length": 2048, "ragged": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 16, "codes": "fp8", "dtype": "bf16", "layout": "nhd"},
        # a continuous batch: lengths from 0 (a padded row) to 8192, the 72B model's heads, head-major pages
        {"name": "attention-ragged", "op": "attention", "batch": 48, "length": 8192, "ragged": True,
         "kv_heads": 8, "group": 8, "dim": 128, "page": 64, "codes": "int8", "dtype": "bf16", "layout": "hnd"},
        # one very long sequence: the split over tokens
        {"name": "attention-long", "op": "attention", "batch": 1, "length": 131001, "ragged": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 16, "codes": "fp8", "dtype": "bf16", "layout": "nhd"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "cache", "attention", "attention"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "linear":
        most = 8192 * 4096 * 14336
        k = 16 * _spread(rng, 4, 1848)
        n = _spread(rng, 64, 29568)
        m = _spread(rng, 1, max(1, min(8192, most // (k * n))))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.5}
    heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128])
    page, codes, layout = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "fp8"]), rng.choice(["nhd", "hnd"])
    common = {"kv_heads": heads, "dim": dim, "page": page, "codes": codes, "dtype": dtype, "layout": layout}
    if op == "cache":
        tokens = _spread(rng, 1, 16384 * 1024 // (heads * dim) if heads * dim > 1024 else 16384)
        pages = -(-tokens // page)
        pages += rng.randint(0, max(1, min(pages, 16384 // page - pages)))
        return {"op": op, "tokens": tokens, "slots": page * pages, **common}
    most = 64 * 2048 * 8 * 128
    batch = _spread(rng, 1, 256)
    length = _spread(rng, 1, min(131072, most // (batch * heads * dim)))
    return {"op": op, "batch": batch, "length": length, "ragged": rng.random() < 0.5,
            "group": rng.choice([1, 2, 4, 7, 8, 12]), **common}


def _activations(gen, m, k, dtype):
    """Rows of unit-normal values with one channel in 64 twenty times as large."""
    loud = 1.0 + 19.0 * (torch.rand(k, generator=gen, device="cuda") < 1 / 64)
    return (torch.randn(m, k, generator=gen, device="cuda") * loud).to(dtype)


def _encode(rows, codes):
    """Rows [..., D] in float32 -> codes and float32 scales [...]."""
    s = rows.abs().amax(-1) / (127.0 if codes == "int8" else 448.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = rows / s[..., None]
    return (q.round().clamp(-127, 127).to(torch.int8) if codes == "int8" else q.to(torch.float8_e4m3fn)), s


def _pool(gen, case, pages):
    """One cache pool: codes [pages, page, heads, dim] and scales [pages, page,
    heads] (views of head-major memory for "hnd"), filled with earlier rows."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    hnd = case["layout"] == "hnd"
    c = torch.empty((pages, heads, page, dim) if hnd else (pages, page, heads, dim), dtype=_CODES[case["codes"]],
                    device="cuda")
    s = torch.empty((pages, heads, page) if hnd else (pages, page, heads), device="cuda")
    step = max(1, (1 << 25) // (page * heads * dim))
    for i in range(0, pages, step):
        rows = torch.randn(c[i:i + step].shape, generator=gen, device="cuda")
        rows[..., ::17] *= 4.0
        c[i:i + step], s[i:i + step] = _encode(rows, case["codes"])
    return (c.transpose(1, 2), s.transpose(1, 2)) if hnd else (c, s)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        w, ws = _encode(torch.randn(n, k, generator=gen, device="cuda") * 0.02, "int8")
        bias = torch.randn(n, generator=gen, device="cuda").to(dtype) if case["bias"] else None
        return {"case": case, "x": _activations(gen, m, k, dtype), "w": w, "ws": ws, "bias": bias}
    if case["op"] == "cache":
        pages = case["slots"] // case["page"]
        kc, ks = _pool(gen, case, pages)
        vc, vs = _pool(gen, case, pages)
        shape = (case["tokens"], case["kv_heads"] * case["dim"])
        kv = [_activations(gen, *shape, dtype).view(-1, case["kv_heads"], case["dim"]) for _ in range(2)]
        slots = torch.randperm(case["slots"], generator=gen, device="cuda")[:case["tokens"]]
        return {"case": case, "k": kv[0], "v": kv[1], "kc": kc, "vc": vc, "ks": ks, "vs": vs, "slots": slots,
                "all": torch.arange(case["slots"], device="cuda")}
    batch, length, page = case["batch"], case["length"], case["page"]
    width = -(-length // page)
    pages = batch * width
    kc, ks = _pool(gen, case, pages)
    vc, vs = _pool(gen, case, pages)
    table = torch.randperm(pages, generator=gen, device="cuda").view(batch, width)
    if case["ragged"]:
        lens = torch.randint(0, length + 1, (batch,), generator=gen, device="cuda")
    else:
        lens = torch.full((batch,), length, device="cuda")
    used = torch.arange(width, device="cuda")[None] * page < lens[:, None]
    table = torch.where(used, table, torch.full_like(table, -1)).to(torch.int32)  # no page past the sequence's end
    q = torch.randn(batch, case["kv_heads"] * case["group"], case["dim"], generator=gen, device="cuda").to(dtype)
    return {"case": case, "q": q, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table,
            "lens": lens.to(torch.int32)}


def _plain_linear(s):
    x = s["x"].float()
    codes, scale = _encode(x, "int8")
    y = (codes.float() @ s["w"].float().t()) * scale[:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_cache(s):
    page, dtype, out = s["case"]["page"], s["k"].dtype, {}
    for name in ("k", "v"):
        pool, scales = s[name + "c"], s[name + "s"]
        codes, scale = _encode(s[name].float(), s["case"]["codes"])
        # float8 has no indexed write: the same bytes as uint8
        pool.view(torch.uint8)[s["slots"] // page, s["slots"] % page] = codes.view(torch.uint8)
        scales[s["slots"] // page, s["slots"] % page] = scale
        rows = pool.view(torch.uint8)[s["all"] // page, s["all"] % page].view(pool.dtype)
        out[name] = (rows.float() * scales[s["all"] // page, s["all"] % page][..., None]).to(dtype)
        out[name + "_scale"] = scales
    return out


def _plain_attention(s):
    c = s["case"]
    heads, dim, page = c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long().clamp(min=0)
    batch, width = table.shape

    def gathered(codes, scales):
        rows = codes.view(torch.uint8)[table].view(codes.dtype).float() * scales[table][..., None]
        return rows.reshape(batch, width * page, heads, dim)

    q = s["q"].float().view(batch, heads, c["group"], dim)
    held = torch.arange(width * page, device="cuda")[None] < s["lens"][:, None]
    score = torch.einsum("bhgd,bthd->bhgt", q, gathered(s["kc"], s["ks"])) / math.sqrt(dim)
    score = score.masked_fill(~held[:, None, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1)
    out = torch.einsum("bhgt,bthd->bhgd", p, gathered(s["vc"], s["vs"])) / torch.where(total == 0, 1, total)[..., None]
    lse = torch.log(total) + top[..., 0]
    return {"out": out.reshape(batch, -1, dim).to(s["q"].dtype), "lse": lse.reshape(batch, -1)}


def _own(s):
    from nanosglang_b200 import ops

    op = s["case"]["op"]
    if op == "linear":
        return ops.int8_linear(s["x"], s["w"], s["ws"], s["bias"])
    if op == "cache":
        ops.kv_cache_write(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        k, v = ops.kv_cache_read(s["kc"], s["vc"], s["ks"], s["vs"], s["all"], s["k"].dtype)
        return {"k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}
    out, lse = ops.kv_attention_decode(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"],
                                       return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "cache":
        new, held = case["tokens"] * heads, case["slots"] * heads
        # new rows and slots in, their codes and scales out; all codes and scales in, 16-bit rows out
        return {"bytes": 2 * (new * (2 * dim + dim + 4) + held * (dim + 4 + 2 * dim)) + 8 * (case["tokens"] + case["slots"]),
                "flops": 2 * (2 * new * dim + held * dim)}
    tokens = case["batch"] * case["length"] // (2 if case["ragged"] else 1)
    rows = case["batch"] * heads * case["group"]
    return {"bytes": 2 * tokens * heads * (dim + 4) + rows * (4 * dim + 4) + 4 * (tokens // case["page"] + case["batch"]),
            "flops": 4 * tokens * heads * case["group"] * dim}


def _e4m3(v):
    """float64 -> the nearest e4m3 value (ties to even), still in float64."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _encode64(rows, codes):
    most = 127.0 if codes == "int8" else 448.0
    s = rows.abs().max(-1, keepdim=True).values / most
    s[s == 0] = 1.0
    q = rows / s
    return (torch.round(q) if codes == "int8" else _e4m3(q)), s


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        codes, scale = _encode64(s["x"].double(), "int8")
        y = (codes * scale) @ (s["w"].double() * s["ws"].double()[:, None]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "cache":
        out = {}
        for name in ("k", "v"):
            scales = s[name + "s"].double().reshape(case["slots"], case["kv_heads"])
            codes = s[name + "c"].to(torch.float16).double().reshape(case["slots"], case["kv_heads"], case["dim"])
            new, scale = _encode64(s[name].double(), case["codes"])
            codes[s["slots"]], scales[s["slots"]] = new, scale[..., 0]
            out[name] = codes * scales[..., None]
            out[name + "_scale"] = scales.view(-1, case["page"], case["kv_heads"])
        return out
    heads, dim, group, lens = case["kv_heads"], case["dim"], case["group"], s["lens"].tolist()
    out = torch.zeros(case["batch"], heads * group, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], heads * group), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // case["page"])].long()
        for h in range(heads):
            # one head's pages as bytes, then 64-bit rows of its n tokens
            k, v = ((c[:, :, h].view(torch.uint8)[pages].view(c.dtype).to(torch.float16).double() * t[pages, :, h].double()[..., None])
                    .reshape(-1, dim)[:n] for c, t in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            rows = slice(h * group, (h + 1) * group)
            score = (s["q"][b, rows].double() @ k.t()) * dim ** -0.5
            lse[b, rows] = torch.logsumexp(score, -1)
            out[b, rows] = torch.exp(score - lse[b, rows, None]) @ v
    return {"out": out, "lse": lse}
