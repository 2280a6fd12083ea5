"""Inputs and checks shared by the CPU and GPU tests of the low-bit serving operators."""
from __future__ import annotations

import math

import torch

from oracle import low_bit as ref

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def norm_inputs(rows, width, dtype, residual, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g).to(dtype)
    r = (3 * torch.randn(rows, width, generator=g)).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dtype)
    if rows > 2:
        x[1] = 0
        if residual:
            r[1] = 0
    return x, r, w


def check_rows(q, scale, y, roundings):
    """q, scale against the float64 values y: integers are within half a step and the fp32 roundings of y / scale"""
    want = ref.row_scale(y)
    assert scale.dtype == F32 and scale.shape == (*y.shape[:-1], 1)
    assert ((scale.double() - want).abs() <= (roundings + 2) * 2.0**-24 * want).all()
    steps = torch.where(y.abs().amax(-1, keepdim=True) == 0, torch.zeros_like(y), y / want)
    assert q.dtype == torch.int8
    assert ((q.double() - steps).abs() <= 0.5 + 127 * roundings * 2.0**-24).all()
    assert (q.int().abs() <= 127).all()


def gemm_inputs(m, n, k, seed, bias=None, layout="col"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    y = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).t()
    if layout == "row":
        y = y.contiguous()
    sa = torch.exp(torch.randn(m, 1, generator=g)) * 0.01
    sb = torch.exp(torch.randn(1, n, generator=g)) * 0.001
    b = torch.randn(n, generator=g).to(bias) if bias is not None else None
    return x, y, sa, sb, b


def check_gemm(out, x, y, sa, sb, b, out_dtype):
    want, size = ref.int8_gemm(x, y, sa, sb, b)
    assert out.dtype == out_dtype and out.shape == want.shape
    # the integer to fp32, two scales, the bias
    err, most = (out.double() - want).abs(), ref.float_bound(want, size, out_dtype, 4)
    assert (err <= most).all(), f"off by up to {float((err / most).max()):.2f} of the bound"


def attention_case(dtype, dim, page, kv_heads, group, lens, news=None, seed=0, spare=2):
    """A filled cache in pages of any order, garbage where no key is, tables with entries that are not to be used."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + spare, max(max(need), 1) + 1
    k = torch.randn(pages, kv_heads, page, dim, generator=g)
    v = torch.randn(pages, kv_heads, page, dim, generator=g)
    kc, ks = ref.encode(k)
    vc, vs = ref.encode(v)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = 0
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = order[at]
            used[order[at], : min(page, n - i * page)] = True
            at += 1
    # what nobody has written: NaN scales, any codes
    gone = ~used[:, None, :, None].expand(pages, kv_heads, page, dim // 32)
    ks = torch.where(gone, torch.full_like(ks, 255), ks)
    vs = torch.where(gone, torch.full_like(vs, 255), vs)
    tokens = sum(news) if news is not None else len(lens)
    q = (1.5 * torch.randn(tokens, kv_heads * group, dim, generator=g)).to(dtype)
    start = torch.tensor([0] + news).cumsum(0).int() if news is not None else None
    cache = (*ref.to_layout(kc, ks, False), *ref.to_layout(vc, vs, True))
    return q, cache, table, torch.tensor(lens, dtype=torch.int32), start


def check_attention(out, q, cache, table, lens, start, scale=None, causal=True, p_terms=2, rows=None):
    want, size, spread = ref.attention(q, *cache, table, lens, start, scale, causal)
    most = ref.attention_bound(want, size, spread, q.dtype, int(lens.max()) if lens.numel() else 0, q.shape[2], p_terms)
    got = out.double()
    if rows is not None:
        got, want, most = got[rows], want[rows], most[rows]
    assert torch.equal(got.isnan(), want.isnan())
    err = torch.where(want.isnan(), torch.zeros_like(got), (got - want).abs())
    most = torch.where(want.isnan(), torch.ones_like(most), most)
    assert (err <= most).all(), f"off by up to {float((err / most).max()):.2f} of the bound"


def p_terms(dtype, dim, news, group):
    """bf16 terms a weight is multiplied as: three for fp32; two, except where a bf16 result is rounded as coarsely itself and
    rows are many (more than 16 for a sequence, head dims up to 128): one"""
    if dtype == F32:
        return 3
    return 1 if dtype == BF and dim <= 128 and (max(news) if news else 1) * group > 16 else 2


# (dtype, dim, page, kv_heads, group, lens, new tokens or None)
ATTENTION = [
    (BF, 128, 16, 2, 4, [1], None),
    (BF, 128, 64, 1, 8, [33, 0, 16, 65], None),             # an empty sequence, a whole block, one past it
    (HF, 64, 16, 3, 1, [31, 32, 100], None),
    (F32, 128, 32, 1, 5, [70], None),
    (BF, 256, 16, 1, 2, [40, 17], None),
    (HF, 256, 32, 1, 3, [35], [3]),
    (HF, 128, 16, 1, 7, [50, 20], [3, 20]),                  # a piece of a prompt and a whole one, 60 rows and 140
    (BF, 64, 128, 2, 2, [40, 1, 0, 9], [12, 1, 0, 4]),
    (F32, 64, 16, 1, 2, [30, 5], [9, 5]),
    (BF, 128, 32, 1, 16, [90], [5]),                         # more than 16 rows
    (HF, 64, 16, 1, 3, [25], [25]),
]


def cancelling_case(dtype, dim, page, kv_heads, group, lens, news):
    """Values that cancel: the keys at even places have 1.5 times the weight of the others (as near as q's type allows) and
    values of 1 against -1.5, so a result is near zero and what its weights lose by rounding stands alone."""
    q, cache, table, n, start = attention_case(dtype, dim, page, kv_heads, group, lens, news)
    pages = cache[0].shape[0]
    k, v = torch.zeros(pages, kv_heads, page, dim), torch.ones(pages, kv_heads, page, dim)
    k[:, :, 0::2, 0] = 1
    v[:, :, 1::2] = -1.5
    cache = (*ref.to_layout(*ref.encode(k), False), *ref.to_layout(*ref.encode(v), True))
    q = torch.zeros_like(q)
    q[..., 0] = (math.log(1.5) * dim**0.5 + 0.02 * torch.arange(q.shape[0] * q.shape[1]).view(q.shape[:2]).remainder(7)).to(dtype)
    return q, cache, table, n, start


def border_rows(dtype, width, norm, seed=0):
    """(x, weight): three rows whose values x * weight * 127 / max lie next to the middle between two integers, as near as
    x's type allows, on it (a half of the maximum) and anywhere; weight is None without a norm"""
    g = torch.Generator().manual_seed(seed)
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dtype) if norm else torch.ones(width, dtype=dtype)
    x = torch.randn(3, width, generator=g).to(dtype)
    k = torch.randint(-126, 126, (2, width), generator=g) + 0.5
    for row in range(2):
        x[row, 0] = 5.3 + row
        top = x[row, 0].double() * w[0].double()
        for c in range(1, width):
            best = (k[row, c] * top / 127 / w[c].double()).to(dtype)
            if dtype != F32:  # of the numbers nearby the one whose quotient comes nearest to a middle
                near = (best.view(torch.int16) + torch.arange(-200, 201, dtype=torch.int16)).view(dtype)
                near = near[(near.double() * w[c].double()).abs() < top.abs()]
                off = (near.double() * w[c].double() * 127 / top) % 1 - 0.5
                best = near[off.abs().argmin()]
            x[row, c] = best
    if norm:
        w[width // 2] = w[0]
    x[:2, width // 2] = x[:2, 0] / 2
    return x, w if norm else None


def check_border_rows(q, x, weight):
    """The integers of the formula: products of 16-bit numbers, and 127 times them, are exact in float64, so the quotient is
    rounded once, by 2^-53 of itself, where the nearest one that is no middle is 2^-32 away."""
    y = x.double() if weight is None else x.double() * weight.double()
    assert torch.equal(q.double(), torch.round(y * 127 / y.abs().amax(-1, keepdim=True)))


def infinite_queries(dtype, group, news, kv_heads=1):
    """Sequences of 3 and 33 keys in turn (the first ones' first tokens see none) whose keys all have a positive first element;
    -inf there in token 0, which sees nothing, and token 3, inf in token 6."""
    lens = [3, 33] * (len(news) // 2)
    q, cache, table, n, start = attention_case(dtype, 64, 16, kv_heads, group, lens, news)
    codes, scales = ref.from_layout(cache[0], cache[1], False)
    codes[..., 0] = 4
    cache = (*ref.to_layout(codes, scales, False), *cache[2:])
    q[[0, 3], :, 0], q[6, :, 0] = -math.inf, math.inf
    return q, cache, table, lens, start, n
