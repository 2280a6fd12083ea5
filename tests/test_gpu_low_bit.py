"""The operators of a layer served in few bits on the GPU, through their Python entry points, against float64 restatements
(oracle/low_bit.py) with bounds derived from the roundings the kernels make."""
import pytest
import torch

import helion_amd as hx
from oracle import low_bit as ref
from tests import _low_bit as lb

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _dev(*ts):
    return [t.to(DEV) if t is not None else None for t in ts]


# ---------------------------------------------------------------------------------------------- norm, quantisation by rows
@pytest.mark.parametrize("rows,width,dtype,residual", [
    (1, 8192, BF, True), (1, 1, BF, False), (7, 333, HF, True), (64, 4096, BF, True), (33, 5120, F32, True), (5, 513, BF, False),
    (300, 1024, HF, True), (3, 28672, BF, False), (2, 65536, HF, True), (1000, 64, BF, True), (17, 2050, F32, False), (9, 16384, BF, True),
])
def test_rms_norm_int8(rows, width, dtype, residual):
    x, r, w = lb.norm_inputs(rows, width, dtype, residual, rows + width)
    xd, rd, wd = _dev(x, r, w)
    res = hx.rms_norm_int8(xd, wd, residual=rd, eps=1e-5)
    want = ref.add(x, r)
    if residual:
        assert torch.equal(res[2].cpu(), want)
    lb.check_rows(res[0].cpu(), res[1].cpu(), ref.rms_norm(want, w, 1e-5), ref.sqrt_rows(width))


@pytest.mark.parametrize("rows,width,dtype", [(1, 14336, BF), (500, 128, HF), (64, 4100, F32), (3, 1, BF), (28, 8192, BF)])
def test_int8_quantize_per_token(rows, width, dtype):
    x, _, _ = lb.norm_inputs(rows, width, dtype, False, 5)
    q, s = hx.int8_quantize_per_token(x.to(DEV))
    lb.check_rows(q.cpu(), s.cpu(), x.double(), 4)


def test_rows_of_any_shape_and_stride():
    g = torch.Generator().manual_seed(0)
    big = torch.randn(6, 5, 300, generator=g).to(BF).to(DEV)
    w = torch.randn(101, generator=g).to(BF).to(DEV)
    for x in (big[:, :, 7:108], big[:, 2, :101], big.transpose(0, 1)[..., :101], big[0, 0, 3:104], big[..., ::2][..., :101]):
        q, s = hx.rms_norm_int8(x, w)
        q2, s2 = hx.rms_norm_int8(x.contiguous(), w)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], 1)
        assert torch.equal(q, q2) and torch.equal(s, s2)
        a = hx.rms_norm_int8(x, w, residual=x)
        b = hx.rms_norm_int8(x.contiguous(), w, residual=x.contiguous())
        assert all(torch.equal(i, j) for i, j in zip(a, b))
    q, s = hx.int8_quantize_per_token(big[:0])
    assert q.shape == (0, 5, 300) and s.shape == (0, 5, 1)


def test_rows_specials():
    x = torch.randn(5, 700, generator=torch.Generator().manual_seed(1))
    x[0], x[1, 3], x[2, 699], x[3] = 0, float("inf"), float("nan"), x[3] * 1e-42
    q, s = (t.cpu() for t in hx.int8_quantize_per_token(x.to(DEV)))
    assert s[0] == 1 and (q[0] == 0).all() and torch.isinf(s[1]) and (q[1] == 0).all() and torch.isnan(s[2]) and (q[2] == 0).all()
    assert (q[3].double() - x[3].double() * 127 / x[3].double().abs().max()).abs().max() <= 0.5 + 1e-4
    lb.check_rows(q[4:], s[4:], x[4:].double(), 4)


def test_rows_refusals():
    x, w = torch.randn(4, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV, dtype=BF)
    for bad in (lambda: hx.rms_norm_int8(x, w[:63]), lambda: hx.rms_norm_int8(x, w.float()), lambda: hx.rms_norm_int8(x, w, residual=x[:3]),
                lambda: hx.rms_norm_int8(x, w, residual=x.half()), lambda: hx.int8_quantize_per_token(x[:, :0]),
                lambda: hx.int8_quantize_per_token(torch.zeros(1, 70000, device=DEV)), lambda: hx.int8_quantize_per_token(x[0, 0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        hx.int8_quantize_per_token(x.int())
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.rms_norm_int8(x, w.cpu())


# ---------------------------------------------------------------------------------------------- product
@pytest.mark.parametrize("m,n,k,bias,out,layout", [
    (1, 256, 128, None, BF, "col"), (16, 1000, 1024, BF, BF, "col"), (16, 1024, 8192, None, F32, "col"), (1, 64, 16384, F32, F32, "col"),
    (33, 4100, 4096, None, HF, "col"), (100, 515, 272, F32, F32, "col"), (777, 1025, 4112, HF, HF, "col"), (300, 260, 1000, BF, BF, "col"),
    (64, 100, 77, F32, F32, "row"), (257, 512, 2048, None, BF, "row"), (512, 512, 512, None, F32, "col"), (5, 3, 1, None, F32, "col"),
    (1024, 1024, 1024, BF, BF, "col"), (2050, 2056, 384, None, HF, "col"), (32, 640, 640, F32, BF, "col"), (3, 40, 4096, None, F32, "col"),
    (128, 8192, 1024, BF, BF, "col"), (20, 77, 9000, None, F32, "col"), (2304, 2048, 2048, F32, F32, "col"),
])
def test_int8_gemm(m, n, k, bias, out, layout):
    x, y, sa, sb, b = lb.gemm_inputs(m, n, k, m + n + k, bias, layout)
    xd, yd, sad, sbd, bd = _dev(x, y, sa, sb, b)
    got = hx.int8_gemm(xd, yd, sad, sbd, bias=bd, out_dtype=out)
    lb.check_gemm(got, xd, yd, sad, sbd, bd, out)
    assert torch.equal(got, hx.int8_gemm(xd, yd, sad.flatten(), sbd.flatten(), bias=bd, out_dtype=out))


@pytest.mark.parametrize("m,n,k", [(1, 40, 16), (16, 300, 1040), (30, 64, 9008), (33, 300, 1040), (64, 128, 8208), (200, 515, 48), (300, 260, 4112),
                                   (2304, 2048, 144), (2304, 2060, 2064)])
def test_int8_gemm_nothing_behind_k_counts(m, n, k):
    """k a multiple of 16 but not of 128, read in place: what stands behind k in longer rows does not matter, on either side,
    with the other one read in place too or copied"""
    x, y, sa, sb, _ = lb.gemm_inputs(m, n, k, m + k, None, "col")
    xd, yd, sad, sbd = _dev(x, y, sa, sb)
    want = ((x.to(DEV).double() @ y.to(DEV).double()).float() * sad.view(-1, 1)) * sbd.view(1, -1)
    wide = torch.full((m, k + 112), 127, dtype=torch.int8, device=DEV)
    tall = torch.full((n, k + 112), -127, dtype=torch.int8, device=DEV)
    wide[:, :k], tall[:, :k] = xd, yd.t()
    odd_a, odd_b = torch.empty(m * k + 1, dtype=torch.int8, device=DEV)[1:].view(m, k), yd.contiguous()
    odd_a.copy_(xd)
    for a in (xd, wide[:, :k], odd_a):
        for b in (yd, tall[:, :k].t(), odd_b):
            assert torch.equal(hx.int8_gemm(a, b, sad, sbd, out_dtype=F32), want)


def test_int8_gemm_strides_and_empty():
    x, y, sa, sb, _ = lb.gemm_inputs(70, 90, 256, 3)
    want = hx.int8_gemm(*_dev(x, y, sa, sb), out_dtype=F32)
    xs = torch.zeros(70, 300, dtype=torch.int8, device=DEV)
    xs[:, 5:261] = x.to(DEV)
    ys = torch.zeros(256, 2, 90, dtype=torch.int8, device=DEV)
    ys[:, 1] = y.to(DEV)
    yt = torch.zeros(90, 3, 256, dtype=torch.int8, device=DEV)
    yt[:, 1] = y.t().to(DEV)
    yo = torch.zeros(90, 260, dtype=torch.int8, device=DEV)
    yo[:, 3:259] = y.t().to(DEV)
    s = sa.to(DEV).expand(70, 3)[:, :1], sb.to(DEV)
    for a in (xs[:, 5:261], x.to(DEV), x.to(DEV).t().contiguous().t()):
        for b in (ys[:, 1], yt[:, 1].t(), yo[:, 3:259].t(), y.to(DEV).contiguous()):
            assert torch.equal(hx.int8_gemm(a, b, *s, out_dtype=F32), want)
    one = hx.int8_gemm(x.to(DEV), y[:, :1].to(DEV).expand(256, 9), sa.to(DEV), sb[:, :1].to(DEV).expand(1, 9), out_dtype=F32)
    assert torch.equal(one, want[:, :1].expand(70, 9))
    assert hx.int8_gemm(x[:0].to(DEV), y.to(DEV), sa[:0].to(DEV), sb.to(DEV)).shape == (0, 90)
    with pytest.raises(ValueError):
        hx.int8_gemm(x[:, :0].to(DEV), y[:0].to(DEV), sa.to(DEV), sb.to(DEV))


def test_int8_gemm_refusals():
    x, y, sa, sb, b = _dev(*lb.gemm_inputs(8, 16, 32, 0, F32))
    for bad in (lambda: hx.int8_gemm(x, y[:31], sa, sb), lambda: hx.int8_gemm(x, y, sa[:7], sb), lambda: hx.int8_gemm(x, y, sa, sb, bias=b[:3]),
                lambda: hx.int8_gemm(x[0], y, sa, sb), lambda: hx.int8_gemm(x, y, sa, sb, bias=b.long()),
                lambda: hx.int8_gemm(torch.zeros(1, 140000, dtype=torch.int8, device=DEV), torch.zeros(140000, 1, dtype=torch.int8, device=DEV), sa[:1], sb[:, :1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hx.int8_gemm(x.float(), y, sa, sb), lambda: hx.int8_gemm(x, y, sa.half(), sb), lambda: hx.int8_gemm(x, y, sa, sb, out_dtype=torch.int32)):
        with pytest.raises(TypeError):
            bad()


# ---------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize("tokens,heads,d,page,dtype,wide", [
    (1, 1, 128, 16, BF, True), (64, 8, 128, 64, BF, True), (100, 3, 64, 32, HF, False), (77, 2, 256, 16, F32, True), (5000, 2, 128, 128, BF, False),
    (4099, 1, 64, 1024, HF, True),
])
def test_kv4_write_and_read(tokens, heads, d, page, dtype, wide):
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    fused = torch.randn(tokens, 3 * heads, d, generator=g).to(dtype)
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, slots[tokens - 1]
    slots = slots.to(torch.int64 if wide else torch.int32)
    cache = hx.kv4_cache(pages, page, heads, d)
    for t in cache:
        t.fill_(0xA5)
    fd = fused.to(DEV)
    hx.kv4_write(cache, fd[:, heads:2 * heads], fd[:, 2 * heads:], slots.to(DEV))
    # the whole cache, bit for bit: the last token of a slot, and what was there before
    last = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            last[s] = t
    at, src = torch.tensor(list(last)), torch.tensor(list(last.values()))
    for values, x, (c, s) in ((False, k, cache[:2]), (True, v, cache[2:])):
        codes, scales = ref.from_layout(c.cpu(), s.cpu(), values)
        want_c = torch.stack((torch.full((1,), 0x5, dtype=torch.uint8), torch.full((1,), 0xA, dtype=torch.uint8)), -1).flatten().repeat(pages * page * heads * d // 2)
        want_c, want_s = want_c.view(pages * page, heads, d), torch.full((pages * page, heads, d // 32), 0xA5, dtype=torch.uint8)
        ec, es = ref.encode(x.float())
        want_c[at], want_s[at] = ec[src], es[src]
        assert torch.equal(codes.transpose(1, 2).reshape(pages * page, heads, d), want_c)
        assert torch.equal(scales.transpose(1, 2).reshape(pages * page, heads, d // 32), want_s)
    for dt in (dtype, F32):
        rk, rv = hx.kv4_read(cache, slots.to(DEV), dt)
        for r, values, (c, s) in ((rk, False, cache[:2]), (rv, True, cache[2:])):
            dec = ref.decode(*ref.from_layout(c.cpu(), s.cpu(), values)).transpose(1, 2).reshape(pages * page, heads, d)
            inside = (slots >= 0) & (slots < pages * page)
            exact = torch.where(inside[:, None, None], dec[slots.long().clamp(0, pages * page - 1)], torch.zeros(()).double())
            assert torch.equal(r.cpu(), exact.to(dt))


def test_kv4_write_every_rounding_and_specials():
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    vals = torch.cat([mids, mids * (1 - 2**-20), mids * (1 + 2**-20), torch.tensor([6.0, 6.5, 7.999, 4.0, 0.0, -0.0, 1e-9, 0.5])])
    k = torch.zeros(9, 1, 64)
    k[0, 0, :29], k[0, 0, 32:61] = vals, -vals
    k[1], k[2] = k[0] * 2.0**100, k[0] * 2.0**-130
    k[3, 0, 5], k[4, 0, 40], k[5, 0, 0], k[6, 0, 0], k[7, 0, 33] = float("inf"), float("nan"), 2.0**-149, 3.4e38, -1.5 * 2.0**-126
    cache = hx.kv4_cache(1, 16, 1, 64)
    for t in cache:
        t.zero_()
    slots = torch.arange(9)
    hx.kv4_write(cache, k.to(DEV), -k.to(DEV), slots.to(DEV))
    for values, x, (c, s) in ((False, k, cache[:2]), (True, -k, cache[2:])):
        codes, scales = ref.from_layout(c.cpu(), s.cpu(), values)
        ec, es = ref.encode(x)
        assert torch.equal(codes[0, 0, :9], ec[:, 0]) and torch.equal(scales[0, 0, :9], es[:, 0])
    rk, _ = hx.kv4_read(cache, slots.to(DEV), F32)
    assert torch.isnan(rk[3, 0, :32]).all() and (rk[3, 0, 32:] == 0).all() and torch.isnan(rk[4, 0, 32:]).all()


def test_kv4_write_the_last_token_of_a_slot_stays():
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(6000, 2, 128, generator=g).to(BF), torch.randn(6000, 2, 128, generator=g).to(BF)
    slots = torch.randint(-3, 900, (6000,), generator=g)
    cache = hx.kv4_cache(20, 64, 2, 128)
    for t in cache:
        t.zero_()
    hx.kv4_write(cache, k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = hx.kv4_read(cache, torch.arange(900, device=DEV), F32)
    last = {s: t for t, s in enumerate(slots.tolist()) if s >= 0}
    at, src = torch.tensor(list(last)), torch.tensor(list(last.values()))
    for r, x in ((rk, k), (rv, v)):
        assert torch.equal(r.cpu()[at], ref.decode(*ref.encode(x.float()))[src].float())


@pytest.mark.parametrize("heads,tokens", [(12, 5000), (2, 70000), (5, 4100)])
def test_kv4_write_many_heads_and_many_tokens(heads, tokens):
    """several heads in one go with some left over, tokens beyond one launch, slots that repeat within and across launches"""
    g = torch.Generator().manual_seed(heads)
    k, v = (torch.randn(tokens, heads, 64, generator=g).to(HF) for _ in range(2))
    n = tokens - tokens // 8
    slots = torch.cat([torch.randperm(n, generator=g), torch.randperm(n, generator=g)])[:tokens].to(torch.int32)
    slots[::97] = 5                                         # one slot again and again, in every group of tokens
    cache = hx.kv4_cache(-(-n // 32), 32, heads, 64)
    for t in cache:
        t.zero_()
    hx.kv4_write(cache, k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = hx.kv4_read(cache, torch.arange(n, device=DEV, dtype=torch.int32), F32)
    last = torch.full((n,), -1, dtype=torch.long).scatter_reduce_(0, slots.long(), torch.arange(tokens), "amax")
    for r, x in ((rk, k), (rv, v)):
        want = ref.decode(*ref.encode(x.float())).float()[last.clamp(min=0)] * (last >= 0)[:, None, None]
        assert torch.equal(r.cpu(), want)


def test_kv4_offsets_beyond_32_bits():
    """a cache of more than 4 GB of codes: its last page is written, read back and attended to"""
    heads, d, page = 8, 128, 64
    pages = 2**32 // (heads * page * d // 2) + 3
    cache = hx.kv4_cache(pages, page, heads, d)
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(40, heads, d, generator=g).to(BF), torch.randn(40, heads, d, generator=g).to(BF)
    slots = torch.arange(40) + (pages - 1) * page
    hx.kv4_write(cache, k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = hx.kv4_read(cache, slots.to(DEV), F32)
    for r, x in ((rk, k), (rv, v)):
        assert torch.equal(r.cpu(), ref.decode(*ref.encode(x.float())).float())
    q = torch.randn(1, 2 * heads, d, generator=g).to(BF)
    out = hx.kv4_attention(q.to(DEV), cache, torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV))
    small = [t[pages - 1:].cpu() for t in cache]
    lb.check_attention(out.cpu(), q, small, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([40]), None)


def test_kv4_refusals():
    c = hx.kv4_cache(4, 16, 2, 64)
    k, s = torch.zeros(3, 2, 64, device=DEV, dtype=BF), torch.arange(3, device=DEV)
    q, t, n = torch.zeros(2, 4, 64, device=DEV, dtype=BF), torch.zeros(2, 2, device=DEV, dtype=torch.int32), torch.ones(2, device=DEV, dtype=torch.int32)
    start = torch.tensor([0, 1, 2], device=DEV, dtype=torch.int32)
    for bad in (lambda: hx.kv4_write(c, k[:, :1], k[:, :1], s), lambda: hx.kv4_write(c, k, k[:2], s), lambda: hx.kv4_write(c, k, k, s[:2]),
                lambda: hx.kv4_write(c, k, k, s.float()), lambda: hx.kv4_write(c._replace(v=c.v[:3]), k, k, s),
                lambda: hx.kv4_write(c._replace(k=c.k.transpose(0, 1)), k, k, s), lambda: hx.kv4_read(c, s.view(3, 1)),
                lambda: hx.kv4_attention(q[:, :3], c, t, n), lambda: hx.kv4_attention(q[:1], c, t, n), lambda: hx.kv4_attention(q, c, t.long(), n),
                lambda: hx.kv4_attention(q, c, t, n[:1]), lambda: hx.kv4_attention(q, c, t, n, query_start=start[:2]),
                lambda: hx.kv4_attention(q, c, t, n, query_start=start, max_query_len=0), lambda: hx.kv4_attention(q, c, t, n, out=q[:1]),
                lambda: hx.kv4_attention(q, c, t, n, out=q.half()), lambda: hx.kv4_attention(q[..., :32], c, t, n)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hx.kv4_write(c, k, k.half(), s), lambda: hx.kv4_read(c, s, torch.int8), lambda: hx.kv4_attention(q.double(), c, t, n),
                lambda: hx.kv4_write(c._replace(k=c.k.view(torch.int8)), k, k, s)):
        with pytest.raises(TypeError):
            bad()


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype,dim,page,kv_heads,group,lens,news", lb.ATTENTION + [
    (BF, 128, 64, 8, 8, [2000, 1, 777, 0, 4096], None), (HF, 128, 16, 8, 4, [517], None), (HF, 64, 16, 32, 1, [300, 2048], None),
    (BF, 128, 32, 2, 4, [700, 1000, 64, 64], [1, 130, 64, 1]), (HF, 64, 1024, 1, 6, [3000], [70]), (F32, 128, 64, 2, 4, [1500, 3], [40, 3]),
    (BF, 256, 64, 2, 2, [2500], [33]), (BF, 128, 32, 8, 16, [8 * i for i in range(32)], [min(8 * i, 16 if i % 3 else 1) for i in range(32)]),
    (HF, 64, 16, 16, 2, [512] * 15 + [3], [256] * 15 + [3]), (HF, 128, 64, 8, 4, [70 + i for i in range(32)], [64 - i for i in range(32)]), (BF, 64, 16, 1, 1, [16], [16]), (HF, 256, 16, 2, 1, [1300, 5], None),
])
def test_kv4_attention(dtype, dim, page, kv_heads, group, lens, news):
    q, cache, table, n, start = lb.attention_case(dtype, dim, page, kv_heads, group, lens, news, seed=len(lens))
    qd, td, nd, sd = _dev(q, table, n, start)
    cd = hx.Kv4Cache(*_dev(*cache))
    mq = max(news) if news else 1
    out = hx.kv4_attention(qd, cd, td, nd, query_start=sd, max_query_len=mq)
    lb.check_attention(out, qd, cd, td, nd, sd, p_terms=lb.p_terms(dtype, dim, news, group))
    again = hx.kv4_attention(qd, cd, td, nd, query_start=sd, max_query_len=mq)
    assert torch.equal(out, again)


@pytest.mark.parametrize("lens,news", [
    ([(37 * i) % 61 for i in range(200)], None), ([20] * 300, None), ([17 * (i % 2) for i in range(129)], None),
    ([3 + (11 * i) % 90 for i in range(131)], [1 + (7 * i) % 3 for i in range(131)]), ([500] + [5] * 139, None)])
def test_kv4_attention_of_many_sequences(lens, news):
    """more sequences than a wave has lanes, which run in the order of their lengths: different, equal, alternating ones"""
    q, cache, table, n, start = lb.attention_case(BF, 64, 16, 8, 2, lens, news, seed=1)
    qd, td, nd, sd = _dev(q, table, n, start)
    cd = hx.Kv4Cache(*_dev(*cache))
    out = hx.kv4_attention(qd, cd, td, nd, query_start=sd, max_query_len=max(news) if news else 1)
    lb.check_attention(out, qd, cd, td, nd, sd)


@pytest.mark.parametrize("dtype,many", [(BF, False), (HF, False), (BF, True), (HF, True)])
def test_kv4_attention_masks(dtype, many):
    """many: 64 key/value heads with 16 query heads each, 112 rows, 512 workgroups of 128 (the kernel for pieces of prompts)"""
    lens, news = ([40, 33] * 4, [5, 7] * 4) if many else ([40, 33], [5, 7])
    q, cache, table, n, start = lb.attention_case(dtype, 64, 16, 64 if many else 1, 16 if many else 2, lens, news)
    qd, td, nd, sd = _dev(q, table, n, start)
    cd = hx.Kv4Cache(*_dev(*cache))
    call = lambda c=cd, t=td, ln=nd, **kw: hx.kv4_attention(qd, c, t, ln, query_start=sd, **{"max_query_len": 7, **kw}).cpu()
    check = lambda *args, **kw: lb.check_attention(*args, p_terms=1 if many and dtype == BF else 2, **kw)
    check(call(causal=False), q, cache, table, n, start, causal=False)
    check(call(scale=0.3, max_query_len=7 if many else 1), q, cache, table, n, start, scale=0.3)
    few = torch.tensor([2, 33] * (len(lens) // 2), dtype=torch.int32)
    out = call(ln=few.to(DEV))
    check(out, q, cache, table, few, start)
    assert (out[:3] == 0).all()
    holes = table.clone()
    holes[0, 1], holes[1, 0] = 10**6, -1
    check(call(t=holes.to(DEV)), q, cache, holes, n, start)
    p, i = int(table[0, 38 // 16]), 38 % 16
    vs = cache[3].clone()
    vs[p, :, i // 4, 1, i % 4] = 255
    nan = (cache[0], cache[1], cache[2], vs)
    out = call(c=hx.Kv4Cache(*_dev(*nan)))
    check(out, q, nan, table, n, start)
    assert torch.isnan(out[3:5, :, 32:]).all() and not torch.isnan(out[:3]).any()


def test_kv4_attention_strides_out_and_rows_behind_the_last_sequence():
    q, cache, table, n, start = lb.attention_case(BF, 128, 16, 2, 4, [300, 90], [40, 3])
    cd = hx.Kv4Cache(*_dev(*cache))
    fused = torch.randn(50, 3, 8, 128, device=DEV).to(BF)
    fused[:43, 1] = q.to(DEV)
    td, nd, sd = _dev(table, n, start)
    want = hx.kv4_attention(q.to(DEV), cd, td, nd, query_start=sd, max_query_len=40)
    out = torch.full((50, 8, 128), 7.0, device=DEV, dtype=BF)
    got = hx.kv4_attention(fused[:, 1], cd, td.t().contiguous().t(), nd, query_start=sd, max_query_len=40, out=out)
    assert got is out and torch.equal(out[:43], want) and (out[43:] == 7).all()
    later = sd + 4                                        # rows in front of the first sequence stay too
    out = torch.full((50, 8, 128), 7.0, device=DEV, dtype=BF)
    moved = torch.zeros(50, 8, 128, device=DEV, dtype=BF)
    moved[4:47] = q.to(DEV)
    hx.kv4_attention(moved, cd, td, nd, query_start=later, max_query_len=40, out=out)
    assert torch.equal(out[4:47], want) and (out[:4] == 7).all() and (out[47:] == 7).all()
    assert hx.kv4_attention(moved[:0], cd, td[:0], nd[:0]).shape == (0, 8, 128)


# ---------------------------------------------------------------------------------------------- together
class _Layer:
    """the attention half of a layer: norm, product, cache, attention, quantisation, product"""

    def __init__(self, width, heads, kv_heads, d, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.heads, self.kv, self.d = heads, kv_heads, d
        self.weight = (1 + 0.1 * torch.randn(width, device=DEV, generator=g)).to(BF)
        self.wqkv, self.sqkv = hx.int8_quantize_per_token(torch.randn((heads + 2 * kv_heads) * d, width, device=DEV, generator=g).to(BF) * width**-0.5)
        self.wo, self.so = hx.int8_quantize_per_token(torch.randn(width, heads * d, device=DEV, generator=g).to(BF) * (heads * d) ** -0.5)
        self.cache = hx.kv4_cache(12, 32, kv_heads, d)

    def step(self, x, residual, slots, table, lens, start=None, max_query=1):
        a, s, h = hx.rms_norm_int8(x, self.weight, residual=residual)
        qkv = hx.int8_gemm(a, self.wqkv.t(), s, self.sqkv).view(-1, self.heads + 2 * self.kv, self.d)
        hx.kv4_write(self.cache, qkv[:, self.heads:self.heads + self.kv], qkv[:, self.heads + self.kv:], slots)
        o = hx.kv4_attention(qkv[:, :self.heads], self.cache, table, lens, query_start=start, max_query_len=max_query)
        b, t = hx.int8_quantize_per_token(o.view(-1, self.heads * self.d))
        return hx.int8_gemm(b, self.wo.t(), t, self.so), h

    def plain(self, x, residual, history):
        """float64, from the formulas; history: lists of k and v rows of the sequence in front of these tokens"""
        h = ref.add(x, residual)
        y = ref.rms_norm(h, self.weight, 1e-6)
        qd = lambda v: torch.round(v / ref.row_scale(v)) * ref.row_scale(v)
        qkv = (qd(y) @ (self.wqkv.double() * self.sqkv.double()).t()).to(BF).view(-1, self.heads + 2 * self.kv, self.d)
        k, v = (ref.decode(*ref.encode(t.float())) for t in (qkv[:, self.heads:self.heads + self.kv], qkv[:, self.heads + self.kv:]))
        k, v = torch.cat([history[0], k]), torch.cat([history[1], v])
        n, new, g = k.shape[0], x.shape[0], self.heads // self.kv
        q = qkv[:, :self.heads].double()
        w = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(g, 1)) * self.d**-0.5
        w = w.masked_fill(torch.arange(n, device=DEV) > torch.arange(n - new, n, device=DEV)[:, None], float("-inf")).softmax(-1)
        o = torch.einsum("hij,jhd->ihd", w, v.repeat_interleave(g, 1)).to(BF).double().reshape(new, -1)
        return qd(o) @ (self.wo.double() * self.so.double()).t(), h, (k, v)


def test_a_prompt_and_two_steps_of_a_layer():
    """A prompt of 40 tokens, then two single tokens, through all operators in order; each output against float64 with the
    same quantisation.  A value next to a rounding border may fall to its other side: one step of an 8-bit row (1/127 of its
    largest), one of a 4-bit key or value (a sixth of its block at most), so single elements may differ by that times a
    weight; in the norm of a row these are rare, and 2 % covers one 4-bit flip in each row's 41 keys with margin."""
    layer = _Layer(512, 8, 2, 64)
    g = torch.Generator(device=DEV).manual_seed(1)
    table = torch.tensor([[5, 2, 9]], dtype=torch.int32, device=DEV)
    slot = lambda i: table[0, i // 32].long() * 32 + i % 32
    history = (torch.zeros(0, 2, 64, device=DEV).double(),) * 2
    at = 0
    for new in (40, 1, 1):
        x, r = (torch.randn(new, 512, device=DEV, generator=g).to(BF) for _ in range(2))
        pos = torch.arange(at, at + new, device=DEV)
        at += new
        lens = torch.tensor([at], dtype=torch.int32, device=DEV)
        start = torch.tensor([0, new], dtype=torch.int32, device=DEV) if new > 1 else None
        out, h = layer.step(x, r, slot(pos), table, lens, start, new)
        want, wh, history = layer.plain(x, r, history)
        assert torch.equal(h, wh)
        assert ((out.double() - want).norm(dim=-1) <= 0.02 * want.norm(dim=-1)).all()


def test_a_captured_step_on_another_stream():
    layer = _Layer(1024, 16, 4, 128)
    b = 3
    x, r = (torch.randn(b, 1024, device=DEV).to(BF) for _ in range(2))
    table = torch.tensor([[0, 1, 2], [3, 4, 5], [6, 7, 8]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([70, 33, 96], dtype=torch.int32, device=DEV)
    slots = torch.tensor([2 * 32 + 5, 4 * 32, 8 * 32 + 31], device=DEV)
    for t in layer.cache:
        t.random_(100, 130)
    want = [t.clone() for t in layer.step(x, r, slots, table, lens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.step(x, r, slots, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs = []
    for _ in range(2):                                      # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = layer.step(x, r, slots, table, lens)
        graphs.append((graph, outs))
    for replay in range(3):
        for graph, outs in graphs:
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            graph.replay()
            eager = layer.step(x, r, slots, table, lens)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs, want)) and all(torch.equal(a, c) for a, c in zip(eager, want)), replay


def test_captured_long_rows_and_split_products():
    """the paths with a workspace (split keys, split K, copied operands) in a graph"""
    q, cache, table, n, _ = lb.attention_case(BF, 128, 64, 1, 8, [4000, 2500])
    qd, td, nd = _dev(q, table, n)
    cd = hx.Kv4Cache(*_dev(*cache))
    x, y, sa, sb, _ = _dev(*lb.gemm_inputs(40, 200, 8200, 4))
    calls = lambda: (hx.kv4_attention(qd, cd, td, nd), hx.int8_gemm(x, y, sa, sb, out_dtype=F32))
    want = [t.clone() for t in calls()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_traced_entry_points():
    x, y, sa, sb, b = _dev(*lb.gemm_inputs(20, 48, 256, 0, BF))
    h, w = torch.randn(5, 96, device=DEV).to(BF), torch.ones(96, device=DEV, dtype=BF)
    q, cache, table, n, _ = lb.attention_case(BF, 64, 16, 2, 2, [20, 31])
    qd, td, nd = _dev(q, table, n)
    cd = _dev(*cache)
    k = torch.randn(3, 2, 64, device=DEV).to(BF)

    def step(cd):
        c = hx.Kv4Cache(*cd)
        hx.kv4_write(c, k, k, torch.tensor([1, 2, 3], device=DEV))
        return (hx.int8_gemm(x, y, sa, sb, bias=b), *hx.rms_norm_int8(h, w), *hx.rms_norm_int8(h, w, residual=h), *hx.int8_quantize_per_token(h),
                *hx.kv4_read(c, torch.tensor([2, 3], device=DEV)), hx.kv4_attention(qd, c, td, nd))

    want = step([t.clone() for t in cd])
    got = torch.compile(step, backend="eager", fullgraph=True)([t.clone() for t in cd])
    assert all(torch.equal(i, j) for i, j in zip(got, want))


# ---------------------------------------------------------------------------------------------- more than one launch holds
def test_more_rows_than_a_launch_holds():
    """70 million rows, more work-items than one launch may have: every row stands for itself, so a piece on its own agrees"""
    rows = 70_000_000
    x = torch.randn(rows, 8, device=DEV, dtype=HF, generator=torch.Generator(DEV).manual_seed(0))
    w = torch.linspace(0.5, 2.0, 8, device=DEV).to(HF)
    q, s = hx.int8_quantize_per_token(x)
    nq, ns, h = hx.rms_norm_int8(x, w, residual=x)
    assert torch.equal(h, x + x)
    for at in (0, 2**25 - 3, 2**26 - 3, rows - 6):
        piece = slice(at, at + 6)
        for got, want in zip((q, s, nq, ns), (*hx.int8_quantize_per_token(x[piece]), *hx.rms_norm_int8(x[piece], w, residual=x[piece])[:2])):
            assert torch.equal(got[piece], want)


def test_more_tokens_read_than_a_launch_holds():
    cache = hx.kv4_cache(2, 64, 1, 64)
    k = torch.randn(128, 1, 64, device=DEV, dtype=HF)
    hx.kv4_write(cache, k, -k, torch.arange(128, device=DEV))
    slots = (torch.arange(2**20 + 77, device=DEV) * 7) % 131 - 1
    rk, rv = hx.kv4_read(cache, slots, dtype=HF)
    one = hx.kv4_read(cache, torch.arange(-1, 130, device=DEV), dtype=HF)
    assert torch.equal(rk, one[0][slots + 1]) and torch.equal(rv, one[1][slots + 1])


@pytest.mark.parametrize("starts", [False, True])
def test_more_sequences_than_a_launch_holds(starts):
    batch, heads = 2**20 + 3, 8
    cache = hx.kv4_cache(1, 16, heads, 64)
    k = torch.randn(16, heads, 64, device=DEV, dtype=HF)
    hx.kv4_write(cache, k, k.flip(0), torch.arange(16, device=DEV))
    q = torch.randn(batch, heads, 64, device=DEV, dtype=HF)
    table = torch.zeros(batch, 1, dtype=torch.int32, device=DEV)
    lens = (torch.arange(batch, device=DEV) % 17).int()
    start = torch.arange(batch + 1, device=DEV).int() if starts else None
    out = hx.kv4_attention(q, cache, table, lens, query_start=start, max_query_len=1)
    for at in (0, 2**19 - 20, 2**20 - 20, batch - 40):
        piece = slice(at, at + 40)
        want = hx.kv4_attention(q[piece], cache, table[piece], lens[piece])
        assert torch.equal(out[piece], want) and not want[lens[piece] > 0].eq(0).all()


# ---------------------------------------------------------------------------------------------- precision of the weights
@pytest.mark.parametrize("dim,page,kv_heads,group,lens,news", [
    (128, 16, 1, 8, [90, 33], [5, 4]), (64, 32, 2, 20, [700, 1], None), (128, 64, 8, 8, [300 + 9 * i for i in range(32)], [64] * 32),
    (64, 16, 64, 16, [40, 33] * 4, [5, 7] * 4), (128, 32, 8, 4, [1000, 64] * 6, [100, 1] * 6),
])
@pytest.mark.parametrize("case", [lb.attention_case, lb.cancelling_case])
def test_kv4_attention_weights_lose_nothing_to_a_batch(case, dim, page, kv_heads, group, lens, news):
    """the weights are two bf16 terms whichever kernel a batch's rows lead to (32 rows a workgroup, or 128 where they fill the
    chip): results near zero show what they lose"""
    q, cache, table, n, start = _dev_case(case(BF, dim, page, kv_heads, group, lens, news))
    out = hx.kv4_attention(q, cache, table, n, query_start=start, max_query_len=max(news) if news else 1)
    lb.check_attention(out, q, cache, table, n, start, p_terms=2)


def _dev_case(case):
    q, cache, table, n, start = case
    return (q.to(DEV), hx.Kv4Cache(*_dev(*cache)), *_dev(table, n, start))


# ---------------------------------------------------------------------------------------------- integers next to a border
@pytest.mark.parametrize("dtype,width,norm", [(HF, 700, True), (BF, 300, True), (HF, 1500, True), (F32, 515, False), (HF, 64, False), (F32, 2100, False)])
def test_integers_are_those_of_the_formula(dtype, width, norm):
    x, w = lb.border_rows(dtype, width, norm)
    q, _ = hx.rms_norm_int8(x.to(DEV), w.to(DEV)) if norm else hx.int8_quantize_per_token(x.to(DEV))
    lb.check_border_rows(q.cpu(), x, w)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_prompt_has_the_integers_and_scales_of_the_formula(dtype):
    """every integer of 2048 rows: products are exact, so only a quotient on a middle could differ, and both sides round it
    to the even one; the scale is rounded once from 64 bits (an ulp for what the roots and sums of float64 differ by)"""
    g = torch.Generator(DEV).manual_seed(0)
    x, r = (torch.randn(2048, 8192, device=DEV, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(8192, device=DEV, generator=g)).to(dtype)
    q, scale, h = hx.rms_norm_int8(x, w, residual=r)
    want = ref.add(x, r)
    assert torch.equal(h, want)
    lb.check_border_rows(q, h, w)
    exact = ref.row_scale(ref.rms_norm(h, w, 1e-6))
    assert ((scale.double() - exact).abs() <= 2.0**-24 * (1 + 1e-6) * exact).all()


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e25, 3e38])
def test_rms_norm_int8_squares_beyond_fp32(size):
    x, _, w = lb.norm_inputs(3, 5000, F32, False, 7)
    x = x / x.abs().amax(-1, keepdim=True).clamp(min=1) * size
    q, scale = hx.rms_norm_int8(x.to(DEV), w.to(DEV))
    lb.check_rows(q.cpu(), scale.cpu(), ref.rms_norm(x, w, 1e-6), 4)


# ---------------------------------------------------------------------------------------------- weights of a module
def test_a_modules_weight_is_a_plain_argument():
    """an nn.Parameter (the usual norm weight or bias) gives what its data gives and leaves no graph"""
    x, w = torch.randn(6, 128, device=DEV).to(BF), torch.randn(128, device=DEV).to(BF)
    a, b, sa, sb, bias = _dev(*lb.gemm_inputs(6, 16, 128, 0, BF))
    call = lambda x, w, bias: (*hx.rms_norm_int8(x, w), *hx.rms_norm_int8(x, w, residual=x), *hx.int8_quantize_per_token(x),
                               hx.int8_gemm(a, b, sa, sb, bias=bias))
    want = call(x, w, bias)
    for run in (call, torch.compile(call, backend="eager", fullgraph=True)):
        got = run(x.clone().requires_grad_(), torch.nn.Parameter(w), torch.nn.Parameter(bias))
        assert all(torch.equal(i, j) and not i.requires_grad for i, j in zip(got, want))


# ---------------------------------------------------------------------------------------------- dispatch modes
def test_dispatch_modes_see_the_operators():
    """a mode (here a log, and make_fx's) sees the registered ops, and what it traces computes the same"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    x, w = torch.randn(6, 128, device=DEV).to(BF), torch.randn(128, device=DEV).to(BF)
    b, sb = hx.int8_quantize_per_token(torch.randn(32, 128, device=DEV).to(BF))

    def step(x):
        q, s, h = hx.rms_norm_int8(x, w, residual=x)
        return hx.int8_gemm(q, b.t(), s, sb), h, hx.matmul(x, w.view(128, 1).expand(128, 8).contiguous())

    want = step(x)
    with Log():
        got = step(x)
    assert all(torch.equal(i, j) for i, j in zip(got, want))
    names = {"helion_amd::add_rms_norm_int8", "helion_amd::int8_gemm", "helion_amd::matmul"}
    assert names <= set(seen)
    traced = make_fx(step)(x)
    assert names <= {str(n.target).replace(".default", "").replace(".", "::") for n in traced.graph.nodes}
    y = torch.randn_like(x)
    assert all(torch.equal(i, j) for i, j in zip(traced(y), step(y)))


# ---------------------------------------------------------------------------------------------- infinities in q
@pytest.mark.parametrize("dtype,group,kv_heads,pairs", [(BF, 2, 1, 1), (HF, 8, 2, 1), (BF, 16, 64, 4), (F32, 2, 1, 1)])
def test_kv4_attention_of_infinite_queries(dtype, group, kv_heads, pairs):
    """an infinity in q makes the row NaN, also where it takes every score to minus infinity; a row without a key stays zero"""
    q, cache, table, _, start, n = lb.infinite_queries(dtype, group, [5, 7] * pairs, kv_heads)
    cd = hx.Kv4Cache(*_dev(*cache))
    out = hx.kv4_attention(q.to(DEV), cd, table.to(DEV), n.to(DEV), query_start=start.to(DEV), max_query_len=7).cpu()
    lb.check_attention(out, q, cache, table, n, start)
    assert torch.isnan(out[3]).all() and (out[0] == 0).all() and torch.isnan(out[6]).all()


# ---------------------------------------------------------------------------------------------- every kernel, by its path
@pytest.mark.parametrize("m,n,k,bias,out,path", [
    (512, 4096, 4096, BF, BF, 2), (200, 515, 48, HF, BF, 18), (100, 512, 16000, BF, BF, 10), (130, 2048, 16400, None, HF, 26),
    (777, 4096, 4096, BF, BF, 3), (777, 4100, 4112, F32, HF, 19), (200, 4096, 16384, BF, BF, 11), (200, 4096, 16400, HF, HF, 27),
    (3500, 2560, 4096, BF, BF, 4), (3500, 2500, 4096, HF, F32, 4), (3500, 2560, 4112, F32, HF, 20),
    (1, 256, 128, None, HF, 1), (16, 1024, 8192, BF, BF, 1), (16, 1000, 16384, BF, BF, 9), (16, 300, 1040, F32, F32, 17), (30, 64, 9008, HF, BF, 25),
])
def test_int8_gemm_every_kernel(m, n, k, bias, out, path):
    """tiles of 64, 128 and 256 rows and the kernel for up to 32, unsplit and split, K a multiple of 128 and not, the output types"""
    from helion_amd import _lib

    x, y, sa, sb, b = _dev(*lb.gemm_inputs(m, n, k, m + n + k, bias))
    assert _lib.load().hx_int8_gemm_path(m, n, k, k, 1, k, x.data_ptr(), y.data_ptr()) == path
    lb.check_gemm(hx.int8_gemm(x, y, sa, sb, bias=b, out_dtype=out), x, y, sa, sb, b, out)


@pytest.mark.parametrize("dtype,dim,page,kv_heads,group,lens,news,path", [
    (BF, 128, 64, 8, 8, [300 + 10 * i for i in range(32)], [64] * 32, 3), (BF, 64, 16, 8, 8, [300 + 10 * i for i in range(32)], [64 - i for i in range(32)], 3),
    (HF, 128, 32, 8, 8, [600 - 10 * i for i in range(32)], [64] * 32, 3), (BF, 128, 32, 8, 4, [700, 65] * 4, [100, 1] * 4, 2),
    (BF, 128, 64, 8, 8, [5000, 20], None, 9), (BF, 64, 16, 2, 8, [4100], [4], 10), (BF, 128, 16, 8, 4, [200], None, 1),
])
def test_kv4_attention_every_kernel(dtype, dim, page, kv_heads, group, lens, news, path):
    """16, 32 and 128 rows a workgroup, keys split and not; maxima that move over the tiles"""
    from helion_amd import _lib

    q, cache, table, n, start = _dev_case(lb.attention_case(dtype, dim, page, kv_heads, group, lens, news))
    q = q * torch.linspace(0.2, 3, q.shape[0], device=DEV)[:, None, None].to(dtype)
    mq = max(news) if news else 1
    assert _lib.load().hx_kv4_attention_path(q.shape[0], len(lens), q.shape[1], kv_heads, dim, page, table.shape[1], mq, 1 if dtype == BF else 0) == path
    out = hx.kv4_attention(q, cache, table, n, query_start=start, max_query_len=mq)
    lb.check_attention(out, q, cache, table, n, start)


@pytest.mark.parametrize("dtype,residual,width,size,eps", [(BF, True, 130, 1.5e38, 1e-6), (BF, True, 8192, 1e-35, 1e-6), (F32, True, 33000, 1e-35, 0.0),
                                                           (BF, False, 300, 1e-36, 0.0), (F32, False, 2100, 3e38, 0.0)])
def test_rms_norm_int8_products_beyond_fp32(dtype, residual, width, size, eps):
    """rows whose products with the weight leave fp32, or come near its lower end, are worked out again with a power of two"""
    x, r, w = lb.norm_inputs(3, width, dtype, residual, 11)
    x = (x.double() / x.double().abs().amax() * size).to(dtype)
    r = (r.double() / r.double().abs().amax() * size).to(dtype) if residual else None
    x[1, 0] = size                                   # (no row of zeros: without eps it has no root)
    res = hx.rms_norm_int8(*_dev(x, w), residual=r.to(DEV) if residual else None, eps=eps)
    h = ref.add(x, r)
    lb.check_rows(res[0].cpu(), res[1].cpu(), ref.rms_norm(h, w, eps), 4)
    if dtype == BF:
        lb.check_border_rows(res[0].cpu(), h, w)
