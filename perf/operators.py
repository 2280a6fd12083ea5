"""The operators of a transformer layer served in few bits, as cases to measure: the root-mean-square norm that writes
8-bit integers with a scale for each token, the product of 8-bit integers that reads them, and a key/value cache held in
4 bits (e2m1 values, a power-of-two scale for each 32 of them): written, read back, and attended to.

`listed()` and `draw(rng)` give cases, `prepare(case, seed)` what a serving program has in hand before the call,
`run(state)` one pass (the operators' plain form in torch, or with `own` set the package's calls), `exact(case, seed)` the
result in 64 bits and `work(case)` what one pass has to move and to compute.  Sizes: the widths 4096, 8192, 14336 and
28672 and the head dims 64 and 128 are those of the benchmark's own workloads, the rest is generic."""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the eight magnitudes of a 4-bit float (bit 3 of a code is the sign)


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the norm in front of a projection while one user decodes: launch latency
        dict(name="norm, one token", op="norm", tokens=1, width=8192, residual=True, dtype="bf16"),
        # the same over a prompt: a stream through memory
        dict(name="norm, prompt", op="norm", tokens=8192, width=8192, residual=True, dtype="bf16"),
        # a projection while 16 users decode: the weights are read once
        dict(name="gemm, 16 tokens", op="gemm", m=16, n=28672, k=8192, bias=False, out="bf16"),
        # a mid-sized batch with ragged sizes and a bias
        dict(name="gemm, ragged", op="gemm", m=777, n=4100, k=4112, bias=True, out="fp16"),
        # a prompt through a large projection: the matrix pipes
        dict(name="gemm, prompt", op="gemm", m=8192, n=8192, k=8192, bias=False, out="bf16"),
        # 64 users append one token each and read it back
        dict(name="cache, 64 tokens", op="cache", tokens=64, kv_heads=8, dim=128, page=64, fused=False, dtype="bf16"),
        # a prompt is written from slices of a fused projection's output and read back
        dict(name="cache, prompt", op="cache", tokens=16384, kv_heads=8, dim=128, page=64, fused=True, dtype="bf16"),
        # one user's next token over a short context
        dict(name="attention, one user", op="attention", batch=1, heads=32, kv_heads=8, dim=128, page=16, context=517, queries=1,
             ragged=False, dtype="fp16"),
        # a batch of next tokens, every head with its own keys, pages of 16, sequences of length zero among them
        dict(name="attention, many heads", op="attention", batch=64, heads=32, kv_heads=32, dim=64, page=16, context=2048, queries=1,
             ragged=True, dtype="fp16"),
        # a batch of next tokens over long contexts: the cache is read once
        dict(name="attention, long", op="attention", batch=32, heads=64, kv_heads=8, dim=128, page=64, context=32768, queries=1,
             ragged=True, dtype="bf16"),
        # a mixed step: some sequences decode, some bring a piece of their prompt
        dict(name="attention, mixed", op="attention", batch=24, heads=32, kv_heads=8, dim=128, page=32, context=4000, queries=200,
             ragged=True, dtype="bf16"),
        # a piece of a prompt attends to what is cached before it
        dict(name="attention, chunk", op="attention", batch=1, heads=32, kv_heads=8, dim=128, page=64, context=10240, queries=2048,
             ragged=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "gemm", "cache", "attention", "attention"))
    if op == "norm":
        tokens = _log(rng, 1, 8192)
        return dict(op=op, tokens=tokens, width=_log(rng, 64, 16384 if tokens < 4096 else 8192), residual=rng.random() < 0.75,
                    dtype=rng.choice(("bf16", "fp16")))
    if op == "gemm":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 28672), _log(rng, 64, 14336)
        while m * n * k > 2**38:
            n = (n + 1) // 2
        if rng.random() < 0.6:  # widths of layers are multiples of 64
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        return dict(op=op, m=m, n=n, k=k, bias=rng.random() < 0.4, out=rng.choice(("bf16", "fp16", "fp32")))
    dim, page = rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "cache":
        return dict(op=op, tokens=_log(rng, 1, 16384), kv_heads=kv_heads, dim=dim, page=page, fused=rng.random() < 0.5, dtype=dtype)
    heads = kv_heads * rng.choice((1, 3, 4, 7, 8))
    context = _log(rng, 1, 32768)
    batch = _log(rng, 1, max(1, min(256, 500000 // context)))
    queries = 1 if rng.random() < 0.6 else min(context, _log(rng, 2, 1024))
    while batch > 1 and batch * heads * queries * context > 2**29:
        batch = batch // 2
    while queries > 1 and batch * heads * queries * context > 2**29:
        queries = queries // 2
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page, context=context, queries=queries,
                ragged=rng.random() < 0.6, dtype=dtype)


def _lengths(case):
    """(context length, new tokens) of every sequence; a ragged batch has short, long and empty ones among them."""
    b, c, q = case["batch"], case["context"], case["queries"]
    if not case["ragged"]:
        return [c] * b, [q] * b
    mix = [((i * 2654435761) >> 7) % 1000 / 999 for i in range(1, b + 1)]
    lens = [max(1, round(c * (0.1 + 0.9 * x))) for x in mix]
    lens[0] = c
    if b > 3:
        lens[b // 2] = 0
        lens[b // 3] = 1
    if q == 1:
        return lens, [1] * b
    news = [min(n, 1 if i % 2 else max(1, round(q * x))) for i, (n, x) in enumerate(zip(lens, reversed(mix)))]
    news[0] = min(c, q)
    return lens, news


# ------------------------------------------------------------------------------------------------ the cache's layout
# k codes  [pages, heads, page, dim/2]             byte b of a token: elements 2b (low half) and 2b + 1
# k scales [pages, heads, page, dim/32]            the exponent of two, + 127
# v codes  [pages, heads, page/4, 16, 4, dim/32]   four tokens side by side: piece r of a token is its elements r*dim/16 ..
# v scales [pages, heads, page/4, dim/32, 4]
def _encode(x):
    """fp32 [..., dim] -> codes and scales (uint8): e = floor(log2 of the largest of 32) - 2, a code is x / 2^e, to nearest even."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(-126, 125)
    y = torch.ldexp(blocks, -e.unsqueeze(-1))
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    code = (code + 8 * torch.signbit(y).byte()).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _decode(codes, scales):
    """packed codes [..., dim/2] and scales [..., dim/32] -> fp32 [..., dim]"""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    pair = table[torch.stack((codes & 15, codes >> 4), -1).to(torch.int32)].flatten(-2)
    scale = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.to(torch.int32) - 127)
    return (pair.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def _new_cache(pages, heads, page, dim, dev):
    u8 = dict(dtype=torch.uint8, device=dev)
    return (torch.zeros(pages, heads, page, dim // 2, **u8), torch.ones(pages, heads, page, dim // 32, **u8),
            torch.zeros(pages, heads, page // 4, 16, 4, dim // 32, **u8), torch.ones(pages, heads, page // 4, dim // 32, 4, **u8))


def _fill(cache, at, k, v):
    """pages `at` of the cache from k, v [pages, page, heads, dim]"""
    kc, ks = _encode(k.float().transpose(1, 2))
    cache[0][at], cache[1][at] = kc, ks
    vc, vs = _encode(v.float().transpose(1, 2))
    cache[2][at] = vc.unflatten(-1, (16, -1)).unflatten(2, (-1, 4)).transpose(3, 4)
    cache[3][at] = vs.unflatten(2, (-1, 4)).transpose(3, 4)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    if op == "norm":
        dt = DTYPES[case["dtype"]]
        t, w = case["tokens"], case["width"]
        x = torch.randn(t, w, device=dev, generator=g)
        res = torch.randn(t, w, device=dev, generator=g) * 3 if case["residual"] else None
        weight = 1 + 0.2 * torch.randn(w, device=dev, generator=g)
        return dict(op=op, x=x.to(dt), residual=None if res is None else res.to(dt), weight=weight.to(dt))
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]

        def codes(rows):  # what a gaussian row quantises to
            c = torch.empty(rows, k, dtype=torch.int8, device=dev)
            for at in range(0, rows, 4096):
                c[at:at + 4096] = (torch.randn(min(4096, rows - at), k, device=dev, generator=g) * 32).round().clamp(-127, 127)
            return c

        x, w = codes(m), codes(n)
        sa = torch.exp(0.5 * torch.randn(m, 1, device=dev, generator=g)) * 0.03
        sb = torch.exp(0.2 * torch.randn(n, 1, device=dev, generator=g)) * 0.001
        bias = torch.randn(n, device=dev, generator=g) if case["bias"] else None
        return dict(op=op, x=x, weight=w, scale_a=sa, scale_b=sb, bias=bias, out=DTYPES[case["out"]])
    dt, page, h, d = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"]
    if op == "cache":
        t = case["tokens"]
        pages = -(-t // page) + 8
        if case["fused"]:  # slices of one projection's output: queries, keys, values
            qkv = torch.randn(t, 4 * h + 2 * h, d, device=dev, generator=g).to(dt)
            k, v = qkv[:, 4 * h:5 * h], qkv[:, 5 * h:]
        else:
            k = torch.randn(t, h, d, device=dev, generator=g).to(dt)
            v = torch.randn(t, h, d, device=dev, generator=g).to(dt)
        if t <= 256:  # next tokens of many sequences: anywhere
            slots = torch.randperm(pages * page, device=dev, generator=g)[:t]
        else:  # a prompt: page after page, the pages in any order
            order = torch.randperm(pages, device=dev, generator=g)[: -(-t // page)]
            slots = (order[:, None] * page + torch.arange(page, device=dev)).flatten()[:t]
        return dict(op=op, cache=_new_cache(pages, h, page, d, dev), k=k, v=v, slots=slots, dtype=dt)
    lens, news = _lengths(case)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 2, max(need)
    cache = _new_cache(pages, h, page, d, dev)
    step = max(1, 2**25 // (page * h * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        _fill(cache, slice(at, at + n), torch.randn(n, page, h, d, device=dev, generator=g), torch.randn(n, page, h, d, device=dev, generator=g))
    order = torch.randperm(pages, device=dev, generator=g).int()
    table, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    order = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    q = (torch.randn(sum(news), case["heads"], d, device=dev, generator=g) * 1.5).to(dt)
    start = torch.tensor([0] + news).cumsum(0).int().to(dev)
    return dict(op=op, q=q, cache=cache, table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32).to(dev),
                start=start if case["queries"] > 1 else None, max_queries=max(news))


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _RUN[s["op"]](s)


def _run_norm(s):
    if own:
        import helion_amd as hx

        if s["residual"] is None:
            (q, scale), h = hx.rms_norm_int8(s["x"], s["weight"], eps=EPS), None
        else:
            q, scale, h = hx.rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        values = torch.mul(q, scale, out=torch.empty_like(s["x"]))  # the values that the integers stand for
        return dict(values=values, scale=scale, residual=h)
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    f = h.double()  # 64 bits: values next to a rounding border
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
    top = y.abs().amax(-1, keepdim=True)
    code = torch.round(y * (127 / top)).float()
    scale = (top / 127).float()
    return dict(values=(code * scale).to(h.dtype), scale=scale, residual=None if s["residual"] is None else h)


def _run_gemm(s):
    if own:
        import helion_amd as hx

        return hx.int8_gemm(s["x"], s["weight"].t(), s["scale_a"], s["scale_b"], bias=s["bias"], out_dtype=s["out"])
    y = (s["x"].float() @ s["weight"].float().t()) * s["scale_a"] * s["scale_b"].t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"])


def _run_cache(s):
    if own:
        import helion_amd as hx

        cache = hx.Kv4Cache(*s["cache"])
        hx.kv4_write(cache, s["k"], s["v"], s["slots"])
        return hx.kv4_read(cache, s["slots"], dtype=s["dtype"])
    kc, ks, vc, vs = s["cache"]
    page = kc.shape[2]
    at, inside = s["slots"] // page, s["slots"] % page
    c, e = _encode(s["k"].float())
    kc[at, :, inside], ks[at, :, inside] = c, e
    c, e = _encode(s["v"].float())
    vc[at, :, inside // 4, :, inside % 4], vs[at, :, inside // 4, :, inside % 4] = c.unflatten(-1, (16, -1)), e
    k = _decode(kc[at, :, inside], ks[at, :, inside])
    v = _decode(vc[at, :, inside // 4, :, inside % 4].flatten(-2), vs[at, :, inside // 4, :, inside % 4])
    return k.to(s["dtype"]), v.to(s["dtype"])


def _run_attention(s):
    if own:
        import helion_amd as hx

        return hx.kv4_attention(s["q"], hx.Kv4Cache(*s["cache"]), s["table"], s["lens"], query_start=s["start"],
                                max_query_len=s["max_queries"])
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    kc, ks, vc, vs = s["cache"]
    b, dev = table.shape[0], q.device
    heads, kv_heads, dim = q.shape[1], kc.shape[1], q.shape[2]
    group, n, mq = heads // kv_heads, table.shape[1] * kc.shape[2], s["max_queries"]
    k = _decode(kc[table].transpose(1, 2).flatten(2, 3), ks[table].transpose(1, 2).flatten(2, 3))  # [b, kv_heads, n, dim]
    v = _decode(vc[table].transpose(1, 2).transpose(4, 5).reshape(b, kv_heads, n, dim // 2),
                vs[table].transpose(1, 2).transpose(4, 5).reshape(b, kv_heads, n, dim // 32))
    start = torch.arange(b + 1, device=dev) if s["start"] is None else s["start"].long()
    new = start[1:] - start[:-1]
    step = torch.arange(mq, device=dev)
    there = step < new[:, None]  # [b, mq]: a row of the padded batch that is a query
    rows = (start[:-1, None] + step).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().view(b, mq, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b * kv_heads, group * mq, dim)
    w = torch.bmm(qp, k.reshape(b * kv_heads, n, dim).transpose(1, 2)).view(b, kv_heads, group, mq, n) * dim**-0.5
    last = (lens - new)[:, None] + step  # a query sees the keys up to its own
    seen = (torch.arange(n, device=dev) <= last[..., None]) & there[..., None]
    w = w.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)  # a query that sees no key gives zeros
    out = torch.bmm(w.view(b * kv_heads, group * mq, n), v.reshape(b * kv_heads, n, dim))
    out = out.view(b, kv_heads, group, mq, dim).permute(0, 3, 1, 2, 4).reshape(b, mq, heads, dim)
    return out[there].to(q.dtype)


_RUN = {"norm": _run_norm, "gemm": _run_gemm, "cache": _run_cache, "attention": _run_attention}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _e2m1_64(x):
    """the values in float64 that blocks of 32 are held as: steps of 1/2 below 2, of 1 below 4, of 2 up to 6"""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    unit = 2.0 ** (torch.floor(torch.log2(top.clamp(min=2.0**-124))) - 2).clamp(-126, 125)
    y = blocks / unit
    step = 0.5 * 2.0 ** torch.floor(torch.log2(y.abs().clamp(min=1.0)))
    return ((torch.round(y / step) * step).clamp(-6, 6) * unit).flatten(-2)


def _half_byte_64(c):
    """code -> float64: sign, two bits of exponent, one of mantissa"""
    e, m = ((c >> 1) & 3).double(), (c & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * 2.0 ** (e - 1))
    return torch.where(c >= 8, -mag, mag)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS) * s["weight"].double()
        scale = y.abs().max(-1, keepdim=True).values / 127
        return dict(values=torch.round(y / scale) * scale, scale=scale, residual=None if s["residual"] is None else h)
    if op == "gemm":
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        w = s["weight"].double().t().contiguous()
        for at in range(0, case["m"], 1024):
            out[at:at + 1024] = s["x"][at:at + 1024].double() @ w
        out *= s["scale_a"].double()
        out *= s["scale_b"].double().t()
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "cache":
        return _e2m1_64(s["k"]), _e2m1_64(s["v"])
    if case["batch"] * case["kv_heads"] > 8192:
        return None
    kc, ks, vc, vs = s["cache"]
    dim, page, group = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, news = _lengths(case)
    at = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        here = s["table"][b, : -(-n // page)].long()
        for h in range(case["kv_heads"] if n else 0):
            kb = kc[here, h].reshape(-1, dim // 2)[:n]
            k = torch.stack((_half_byte_64(kb & 15), _half_byte_64(kb >> 4)), -1).reshape(n, dim)
            k = k * (2.0 ** (ks[here, h].reshape(-1, dim // 32)[:n].double() - 127)).repeat_interleave(32, -1)
            vb = vc[here, h].permute(0, 1, 3, 2, 4).reshape(-1, dim // 2)[:n]
            v = torch.stack((_half_byte_64(vb & 15), _half_byte_64(vb >> 4)), -1).reshape(n, dim)
            v = v * (2.0 ** (vs[here, h].permute(0, 1, 3, 2).reshape(-1, dim // 32)[:n].double() - 127)).repeat_interleave(32, -1)
            q = s["q"][at:at + new, h * group:(h + 1) * group].double().transpose(0, 1)  # [group, new, dim]
            w = q @ k.t() / math.sqrt(dim)
            past = torch.arange(n, device="cuda") > torch.arange(n - new, n, device="cuda")[:, None]
            w = torch.softmax(w.masked_fill(past, float("-inf")), -1)
            out[at:at + new, h * group:(h + 1) * group] = (w @ v).transpose(0, 1)
        at += new
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":  # x and the residual read, the sum, the integers and the scales written; and the values read back
        t, w, e = case["tokens"], case["width"], BYTES[case["dtype"]]
        moved = t * w * (e * (3 if case["residual"] else 1) + 1) + t * 4 + w * e
        return dict(bytes=moved + t * w * e, flops=8 * t * w)
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=m * k + n * k + m * n * BYTES[case["out"]] + 4 * (m + n), flops=2 * m * n * k)
    h, d = case["kv_heads"], case["dim"]
    if op == "cache":  # k and v read, 4 bits and scales written; and read back
        t = case["tokens"]
        return dict(bytes=4 * t * h * d * BYTES[case["dtype"]] + 2 * t * h * (d // 2 + d // 32) + 8 * t, flops=8 * t * h * d)
    lens, news = _lengths(case)
    rows = sum(news) * case["heads"] * d
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, news) if n)
    return dict(bytes=2 * rows * BYTES[case["dtype"]] + 2 * sum(lens) * h * (d // 2 + d // 32), flops=4 * pairs * case["heads"] * d)
