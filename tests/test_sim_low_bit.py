"""The operators of a layer served in few bits, executed on the CPU in the host execution model (tests/sim: the kernel
sources lane by lane, operands between inaccessible pages) against float64 restatements of their formulas."""
import pytest
import torch

from oracle import low_bit as ref
from tests import _low_bit as lb
from tests.sim import simlib, simops

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


# ---------------------------------------------------------------------------------------------- norm, quantisation by rows
@pytest.mark.parametrize("rows,width,dtype,residual,stride", [
    (1, 8, BF, True, None), (5, 512, HF, False, None), (3, 513, BF, True, None), (2, 1000, F32, True, 1003), (3, 2048, BF, True, None),
    (3, 2049, HF, False, 2060), (2, 4100, BF, True, None), (1, 9000, HF, True, None), (3, 1, BF, True, None), (4, 7, F32, False, 9),
    (1, 33000, BF, False, None), (1, 17000, BF, True, None),
])
def test_rms_norm_int8(rows, width, dtype, residual, stride):
    x, r, w = lb.norm_inputs(rows, width, dtype, residual, rows + width)
    q, scale, h = simops.rms_norm_int8(x, w, r, 1e-5, stride)
    want = ref.add(x, r)
    if residual:
        assert torch.equal(h, want)
    lb.check_rows(q, scale, ref.rms_norm(want, w, 1e-5), ref.sqrt_rows(width))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quantize_rows_is_exact_where_the_maximum_is_127(dtype):
    x = torch.arange(-127, 128).repeat(3, 1).to(dtype)
    x[1] = x[1] / 4
    q, scale, _ = simops.rms_norm_int8(x)
    assert torch.equal(q[0].int(), x[0].int()) and torch.equal(q[1], q[0])
    assert scale[0] == 1 and scale[1] == 0.25


def test_quantize_rows_specials():
    x = torch.randn(6, 70, generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 69] = float("nan")
    x[3] = x[3] * 1e-42          # subnormal numbers: 127 / max is beyond fp32
    x[4] = 3.4e38
    q, scale, _ = simops.rms_norm_int8(x)
    assert scale[0] == 1 and (q[0] == 0).all()
    assert torch.isinf(scale[1]) and (q[1] == 0).all()
    assert torch.isnan(scale[2]) and (q[2] == 0).all()
    assert (q[3].double() - x[3].double() * 127 / x[3].double().abs().max()).abs().max() <= 0.5 + 1e-4
    assert (q[4] == 127).all()
    lb.check_rows(q[5:], scale[5:], x[5:].double(), 4)
    # through the norm: an infinity makes the mean infinite and the row NaN
    y = torch.randn(3, 100).to(BF)
    y[1, 5] = float("inf")
    q, scale, _ = simops.rms_norm_int8(y, torch.ones(100, dtype=BF))
    assert torch.isnan(scale[1]) and (q[1] == 0).all() and torch.isfinite(scale[[0, 2]]).all()


# ---------------------------------------------------------------------------------------------- product
@pytest.mark.parametrize("m,n,k,bias,out,layout", [
    (1, 16, 16, None, BF, "col"), (64, 128, 128, F32, F32, "col"), (17, 130, 256, BF, HF, "col"), (3, 5, 7, HF, F32, "col"),
    (65, 257, 272, None, BF, "col"), (130, 128, 1040, BF, BF, "col"), (20, 40, 2176, None, F32, "col"),     # split K
    (20, 33, 100, F32, F32, "row"), (128, 128, 640, None, HF, "row"), (1, 1, 1, None, F32, "row"),
    (40, 64, 2064, None, F32, "col"), (33, 48, 144, BF, BF, "col"),                                        # K % 128 != 0: B read on
])
@pytest.mark.parametrize("variant", ["lazy-reverse", "eager"])
def test_int8_gemm(m, n, k, bias, out, layout, variant):
    simlib.configure(variant if variant in simlib.VARIANTS else list(simlib.VARIANTS)[0])
    x, y, sa, sb, b = lb.gemm_inputs(m, n, k, m + n + k, bias, layout)
    lb.check_gemm(simops.int8_gemm(x, y, sa, sb, b, out), x, y, sa, sb, b, out)


def test_int8_gemm_largest_sum():
    """every product at its largest: 131071 * 2^14 stays below 2^31"""
    k = 131071
    x, y = torch.full((1, k), -128, dtype=torch.int8), torch.full((1, k), -128, dtype=torch.int8).t()
    one = torch.ones(1)
    assert simops.int8_gemm(x, y, one, one, None, F32).item() == float(k * 2**14)


# ---------------------------------------------------------------------------------------------- cache
def _empty(pages, heads, page, d, fill=0xA5):
    s = d // 32
    return [torch.full(shape, fill, dtype=torch.uint8) for shape in
            ((pages, heads, page, d // 2), (pages, heads, page, s), (pages, heads, page // 4, 16, 4, s), (pages, heads, page // 4, s, 4))]


def _written(cache, k, v, slots):
    """the cache after a write, token by token"""
    cache = [t.clone() for t in cache]
    page = cache[0].shape[2]
    kc, ks = ref.encode(k.float())
    vc, vs = ref.encode(v.float())
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < cache[0].shape[0] * page:
            continue
        p, i = divmod(s, page)
        cache[0][p, :, i], cache[1][p, :, i] = ref.pack(kc[t]), ks[t]
        cache[2][p, :, i // 4, :, i % 4], cache[3][p, :, i // 4, :, i % 4] = ref.pack(vc[t]).unflatten(-1, (16, -1)), vs[t]
    return cache


@pytest.mark.parametrize("tokens,heads,d,page,dtype,wide", [
    (1, 1, 64, 16, BF, True), (5, 2, 128, 16, HF, False), (19, 3, 256, 32, F32, True), (70, 1, 64, 64, HF, True), (33, 5, 128, 16, BF, False),
])
def test_kv4_write_and_read(tokens, heads, d, page, dtype, wide):
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    fused = torch.randn(tokens, 3 * heads, d, generator=g).to(dtype)   # keys and values as slices of one output
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    k[0, 0, :32] = 0
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, slots[tokens - 1]      # padding, outside, overtaken by the last token
    slots = slots.to(torch.int64 if wide else torch.int32)
    got = simops.kv4_write(_empty(pages, heads, page, d), k, v, slots)
    want = _written(_empty(pages, heads, page, d), k, v, slots)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    rk, rv = simops.kv4_read(got, slots, dtype)
    for r, values, c, s in ((rk, False, got[0], got[1]), (rv, True, got[2], got[3])):
        dec = ref.decode(*ref.from_layout(c, s, values)).transpose(1, 2).reshape(pages * page, heads, d)
        inside = (slots >= 0) & (slots < pages * page)
        exact = torch.where(inside[:, None, None], dec[slots.long().clamp(0, pages * page - 1)], torch.zeros(()).double())
        assert torch.equal(r, exact.to(dtype))


def test_kv4_write_every_rounding_and_specials():
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    vals = torch.cat([mids, mids * (1 - 2**-20), mids * (1 + 2**-20), torch.tensor([6.0, 6.5, 7.999, 4.0, 0.0, -0.0, 1e-9, 0.5])])
    rows = torch.zeros(9, 1, 64)
    rows[0, 0, :29], rows[0, 0, 32:61] = vals, -vals
    rows[1] = rows[0] * 2.0**100
    rows[2] = rows[0] * 2.0**-130           # the block's exponent is clamped: subnormal quotients
    rows[3, 0, 5] = float("inf")
    rows[4, 0, 40] = float("nan")
    rows[5, 0, 0] = 2.0**-149
    rows[6, 0, 0] = 3.4e38
    rows[7, 0, 33] = -1.5 * 2.0**-126
    k = rows
    slots = torch.arange(9)
    got = simops.kv4_write(_empty(1, 1, 16, 64), k, -k, slots)
    want = _written(_empty(1, 1, 16, 64), k, -k, slots)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    rk, _ = simops.kv4_read(got, slots, F32)
    assert torch.isnan(rk[3, 0, :32]).all() and (rk[3, 0, 32:] == 0).all() and torch.isnan(rk[4, 0, 32:]).all()
    assert not torch.isnan(rk[[0, 1, 2, 5, 6, 7, 8]]).any()


@pytest.mark.parametrize("tokens", [3, 130])
def test_kv4_write_the_last_token_of_a_slot_stays(tokens):
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(tokens, 1, 64, generator=g), torch.randn(tokens, 1, 64, generator=g)
    slots = torch.randint(0, 20, (tokens,), generator=g)
    for rev in (False, True):
        empty = _empty(2, 1, 16, 64)
        if rev:
            with simlib.workgroups_last_to_first():
                got = simops.kv4_write(empty, k, v, slots)
        else:
            got = simops.kv4_write(empty, k, v, slots)
        for a, b in zip(got, _written(empty, k, v, slots)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype,dim,page,kv_heads,group,lens,news", lb.ATTENTION)
def test_kv4_attention(dtype, dim, page, kv_heads, group, lens, news):
    q, cache, table, n, start = lb.attention_case(dtype, dim, page, kv_heads, group, lens, news)
    out = simops.kv4_attention(q, cache, table, n, start)
    lb.check_attention(out, q, cache, table, n, start, p_terms=lb.p_terms(dtype, dim, news, group))


@pytest.mark.parametrize("dtype,dim,page,kv_heads,group,lens,news", [
    (BF, 128, 16, 1, 4, [90, 20, 0, 3, 70], [33, 20, 0, 1, 4]),     # 132 rows: two workgroups; 80, none, 4 and 16 of them
    (HF, 64, 64, 2, 1, [200], [130]), (HF, 128, 32, 1, 8, [40, 150], [9, 20]), (BF, 64, 16, 1, 3, [64, 129], [64, 1]),
])
def test_kv4_attention_many_rows(dtype, dim, page, kv_heads, group, lens, news):
    """the kernel for pieces of prompts (a chip of one compute unit: it takes every batch with more than 64 rows)"""
    q, cache, table, n, start = lb.attention_case(dtype, dim, page, kv_heads, group, lens, news)
    with simlib.cus(1):
        out = simops.kv4_attention(q, cache, table, n, start)
        lb.check_attention(out, q, cache, table, n, start, p_terms=lb.p_terms(dtype, dim, news, group))
        out = simops.kv4_attention(q, cache, table, n, start, causal=False, max_query=-(-65 // group))
        lb.check_attention(out, q, cache, table, n, start, causal=False, p_terms=lb.p_terms(dtype, dim, news, group))


@pytest.mark.parametrize("dtype,news", [(BF, None), (HF, [2, 40])])
def test_kv4_attention_split_keys(dtype, news):
    """two splits of a long row (the table is wide enough), joined by the second kernel; rows behind the last sequence stay"""
    q, cache, table, n, start = lb.attention_case(dtype, 64, 256, 1, 2, [600, 130], news)
    table = torch.cat([table, torch.full((2, 3), -1, dtype=torch.int32)], 1)
    if start is not None:
        q = torch.cat([q, q[:3]])
    with simlib.cus(4):
        out = simops.kv4_attention(q, cache, table, n, start, fill=0x11)
    valid = slice(0, 42 if news else 2)
    lb.check_attention(out, q, cache, table, n, start, p_terms=2, rows=valid)
    if start is not None:
        assert (out[42:].view(torch.uint8) == 0x11).all()


@pytest.mark.parametrize("many", [False, True])
def test_kv4_attention_masks(many):
    """not causal; more new tokens than keys (rows without a key give zeros); a page that does not exist; lengths beyond the
    table; a max_query that is too small; NaN in a value that only later rows see"""
    q, cache, table, n, start = lb.attention_case(BF, 64, 16, 1, 10 if many else 2, [40, 33], [5, 7])
    check = lambda *args, **kw: lb.check_attention(*args, p_terms=1 if many else 2, **kw)
    with simlib.cus(1 if many else 256):
        out = simops.kv4_attention(q, cache, table, n, start, causal=False)
        check(out, q, cache, table, n, start, causal=False)
        out = simops.kv4_attention(q, cache, table, n, start, scale=0.3, max_query=7 if many else 1)
        check(out, q, cache, table, n, start, scale=0.3)
        few = torch.tensor([2, 33], dtype=torch.int32)
        out = simops.kv4_attention(q, cache, table, few, start)
        check(out, q, cache, table, few, start)
        assert (out[:3] == 0).all()
        holes = table.clone()
        holes[0, 1], holes[1, 0] = 10**6, -1
        out = simops.kv4_attention(q, cache, holes, n, start)
        check(out, q, cache, holes, n, start)
        far = torch.tensor([4000, 33], dtype=torch.int32)
        full = torch.zeros(2, 3, dtype=torch.int32)
        full[0], full[1] = table[0, :3], table[1, :3]
        clamped = torch.tensor([48, 33], dtype=torch.int32)
        kc, ks, vc, vs = (t.clone() for t in cache)
        ks[ks == 255] = 120
        vs[vs == 255] = 120
        out = simops.kv4_attention(q, (kc, ks, vc, vs), full, far, start)
        check(out, q, (kc, ks, vc, vs), full, clamped, start)
        p, i = int(table[0, 38 // 16]), 38 % 16   # key 38: rows 3 and 4 of sequence 0 see it
        vs2 = cache[3].clone()
        vs2[p, 0, i // 4, 1, i % 4] = 255
        nan = (cache[0], cache[1], cache[2], vs2)
        out = simops.kv4_attention(q, nan, table, n, start)
        check(out, q, nan, table, n, start)
        assert torch.isnan(out[3:5, :, 32:]).all() and not torch.isnan(out[:3]).any() and not torch.isnan(out[:, :, :32]).any()


def test_kv4_attention_no_pages():
    q = torch.randn(2, 2, 64).to(BF)
    cache = _empty(0, 1, 16, 64)
    out = simops.kv4_attention(q, cache, torch.zeros(2, 1, dtype=torch.int32), torch.tensor([5, 0], dtype=torch.int32), fill=0xFF)
    assert (out == 0).all()


# (dtype, dim, page, kv_heads, group, lens, new tokens, compute units): 32 rows a workgroup, and 128
WEIGHTS = [(BF, 128, 16, 1, 8, [90, 33], [5, 4], 256), (BF, 64, 32, 1, 20, [70], None, 256), (BF, 128, 16, 1, 4, [90, 70], [32, 4], 1),
           (BF, 64, 16, 2, 2, [129], [64], 1)]


@pytest.mark.parametrize("dtype,dim,page,kv_heads,group,lens,news,cus", WEIGHTS)
@pytest.mark.parametrize("case", [lb.attention_case, lb.cancelling_case])
def test_kv4_attention_weights_lose_nothing_to_a_batch(case, dtype, dim, page, kv_heads, group, lens, news, cus):
    """the weights are two bf16 terms whichever kernel a batch's rows lead to: results near zero show what they lose"""
    q, cache, table, n, start = case(dtype, dim, page, kv_heads, group, lens, news)
    with simlib.cus(cus):
        out = simops.kv4_attention(q, cache, table, n, start)
    lb.check_attention(out, q, cache, table, n, start, p_terms=2)


# ---------------------------------------------------------------------------------------------- integers next to a border
@pytest.mark.parametrize("dtype,width,norm", [(HF, 700, True), (BF, 300, True), (F32, 515, False), (HF, 64, False)])
def test_integers_are_those_of_the_formula(dtype, width, norm):
    x, w = lb.border_rows(dtype, width, norm)
    q, _, _ = simops.rms_norm_int8(x, w)
    lb.check_border_rows(q, x, w)


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e25, 3e38])
def test_rms_norm_int8_squares_beyond_fp32(size):
    """the mean of the squares is in 64 bits: rows whose squares leave fp32 are like others (eps: 1e-6)"""
    x, _, w = lb.norm_inputs(3, 130, F32, False, 7)
    x = x / x.abs().amax(-1, keepdim=True).clamp(min=1) * size
    q, scale, _ = simops.rms_norm_int8(x, w)
    lb.check_rows(q, scale, ref.rms_norm(x, w, 1e-6), 4)


@pytest.mark.parametrize("dtype,group,news,cus", [(BF, 2, [5, 7], 256), (HF, 8, [5, 7], 256), (BF, 16, [5, 7], 1), (F32, 2, [5, 7], 256)])
def test_kv4_attention_of_infinite_queries(dtype, group, news, cus):
    """an infinity in q makes the row NaN, also where it takes every score to minus infinity; a row without a key stays zero"""
    q, cache, table, _, start, n = lb.infinite_queries(dtype, group, news)
    with simlib.cus(cus):
        out = simops.kv4_attention(q, cache, table, n, start)
    lb.check_attention(out, q, cache, table, n, start)
    assert torch.isnan(out[3, :, :]).all() and (out[0] == 0).all() and torch.isnan(out[6]).all()


# ---------------------------------------------------------------------------------------------- every kernel of the product
# (compute units, m, n, k, bias, out, path): tiles of 64, 128 and 256 rows, unsplit and split, K a multiple of 128 and not
TILES = [
    (1, 257, 257, 1040, BF, BF, 20), (1, 300, 513, 784, HF, F32, 20), (1, 129, 256, 640, None, HF, 4), (1, 129, 256, 2048, BF, BF, 4),
    (4, 129, 256, 2064, F32, HF, 19), (4, 129, 256, 2048, BF, BF, 3), (3, 128, 128, 4096, BF, BF, 11), (8, 130, 128, 8208, None, HF, 27),
    (16, 250, 250, 4112, F32, BF, 26), (4, 100, 128, 4096, None, F32, 10), (2, 128, 128, 4096, HF, HF, 2), (2, 100, 128, 2064, None, BF, 18),
    (1, 5, 40, 8192, BF, BF, 1), (4, 5, 40, 8320, None, HF, 9), (1, 20, 40, 8208, F32, F32, 25), (256, 20, 70, 1040, HF, BF, 17),
]


@pytest.mark.parametrize("cus,m,n,k,bias,out,path", TILES)
@pytest.mark.parametrize("variant", ["lazy-reverse", "eager"])
def test_int8_gemm_every_kernel(cus, m, n, k, bias, out, path, variant):
    simlib.configure(variant)
    x, y, sa, sb, b = lb.gemm_inputs(m, n, k, m + n + k, bias)
    A = 1 << 20
    with simlib.cus(cus):
        assert simlib.load().hx_int8_gemm_path(m, n, k, k, 1, k, A, A) == path
        got = simops.int8_gemm(x, y, sa, sb, b, out)
    lb.check_gemm(got, x, y, sa, sb, b, out)


def _path(q, cache, table, news):
    pages, kv_heads, page, half = cache[0].shape
    return simlib.load().hx_kv4_attention_path(q.shape[0], table.shape[0], q.shape[1], kv_heads, 2 * half, page, table.shape[1],
                                               max(news) if news else 1, {HF: 0, BF: 1, F32: 2}[q.dtype])


@pytest.mark.parametrize("cus,case,path", [
    (256, (BF, 128, 16, 1, 8, [90, 33], [5, 4]), 2), (256, (BF, 128, 64, 1, 8, [40], None), 1), (256, (BF, 256, 16, 1, 8, [90, 33], [5, 4]), 1),
    (256, (F32, 64, 16, 1, 8, [90, 33], [5, 4]), 1), (4, (BF, 64, 256, 1, 2, [2100, 130], None), 9), (4, (HF, 64, 256, 1, 2, [2100], [20]), 10),
    # 128 rows a workgroup: sequences of 128 rows, 80, none, 4 and 16; several tiles of 64 keys; two and one workgroups of a sequence
    (1, (BF, 128, 16, 1, 4, [200, 20, 0, 1, 70, 40], [32, 20, 0, 1, 4, 4]), 3), (1, (BF, 128, 32, 2, 8, [333, 150], [16, 9]), 3),
    (1, (HF, 64, 16, 1, 4, [260, 150], [32, 20]), 3), (1, (HF, 128, 64, 2, 1, [300], [256]), 3), (1, (BF, 64, 16, 2, 2, [64, 129], [64, 1]), 3),
])
@pytest.mark.parametrize("causal", [True, False])
def test_kv4_attention_every_kernel(cus, case, path, causal):
    """the kernel a case runs; maxima that move over the tiles, both buffers, pages ahead of their use"""
    q, cache, table, n, start = lb.attention_case(*case)
    q = q * torch.linspace(0.2, 3, q.shape[0])[:, None, None].to(q.dtype)
    with simlib.cus(cus):
        assert _path(q, cache, table, case[6]) == path
        out = simops.kv4_attention(q, cache, table, n, start, causal=causal)
    lb.check_attention(out, q, cache, table, n, start, causal=causal, p_terms=3 if q.dtype == F32 else 2)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (HF, 128)])
def test_kv4_attention_masks_with_128_rows_a_workgroup(dtype, dim):
    """rows without a key, a page that does not exist, a max_query that is too small, a NaN in a value that only later rows see"""
    q, cache, table, n, start = lb.attention_case(dtype, dim, 16, 1, 16, [100, 93], [5, 7])
    check = lambda *args, **kw: lb.check_attention(*args, p_terms=2, **kw)
    with simlib.cus(1):
        assert _path(q, cache, table, [5, 7]) == 3
        check(simops.kv4_attention(q, cache, table, n, start, scale=-0.3), q, cache, table, n, start, scale=-0.3)
        few = torch.tensor([2, 93], dtype=torch.int32)
        out = simops.kv4_attention(q, cache, table, few, start)
        check(out, q, cache, table, few, start)
        assert (out[:3] == 0).all()
        holes = table.clone()
        holes[0, 1], holes[1, 0], holes[1, 4] = 10**6, -1, -1
        check(simops.kv4_attention(q, cache, holes, n, start), q, cache, holes, n, start)
        p, i = int(table[0, 98 // 16]), 98 % 16   # key 98: rows 3 and 4 of sequence 0 see it
        vs = cache[3].clone()
        vs[p, 0, i // 4, 1, i % 4] = 255
        nan = (cache[0], cache[1], cache[2], vs)
        out = simops.kv4_attention(q, nan, table, n, start)
        check(out, q, nan, table, n, start)
        assert torch.isnan(out[3:5, :, 32:64]).all() and not torch.isnan(out[:3]).any() and not torch.isnan(out[:, :, :32]).any()
        ks = cache[1].clone()
        ks[int(table[0, 1]), 0, 3, 1] = 255       # key 19: every row of sequence 0 sees it
        nan = (cache[0], ks, *cache[2:])
        out = simops.kv4_attention(q, nan, table, n, start)
        check(out, q, nan, table, n, start)
        assert torch.isnan(out[:5]).all() and not torch.isnan(out[5:]).any()


@pytest.mark.parametrize("dtype,residual,width,size,eps", [(BF, True, 130, 1.5e38, 1e-6), (BF, True, 700, 1e-35, 1e-6), (F32, True, 2100, 1e-35, 0.0),
                                                           (BF, False, 300, 1e-36, 0.0), (F32, False, 515, 3e38, 0.0)])
def test_rms_norm_int8_products_beyond_fp32(dtype, residual, width, size, eps):
    """rows whose products with the weight leave fp32, or come near its lower end, are worked out again with a power of two"""
    x, r, w = lb.norm_inputs(3, width, dtype, residual, 11)
    x = (x.double() / x.double().abs().amax() * size).to(dtype)
    r = (r.double() / r.double().abs().amax() * size).to(dtype) if residual else None
    x[1, 0] = size                                   # (no row of zeros: without eps it has no root)
    q, scale, h = simops.rms_norm_int8(x, w, r, eps)
    h = ref.add(x, r)
    lb.check_rows(q, scale, ref.rms_norm(h, w, eps), 4)
    if dtype == BF:
        lb.check_border_rows(q, h, w)
