"""The operators of a layer served in few bits, restated in float64 from their formulas (test infrastructure only; works on
CPU and device tensors alike).  Functions that a kernel must match bit for bit return the integers themselves."""
from __future__ import annotations

import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------- norm and quantisation by rows
def add(x: torch.Tensor, residual: torch.Tensor | None) -> torch.Tensor:
    """x + residual rounded once to x's dtype (the sum of two 16- or 32-bit floats is exact in float64 but for cases that
    round the same way)."""
    return x if residual is None else (x.double() + residual.double()).to(x.dtype)


def rms_norm(h: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    h = h.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()


def row_scale(y: torch.Tensor) -> torch.Tensor:
    top = y.double().abs().amax(-1, keepdim=True)
    return torch.where(top == 0, torch.ones_like(top), top / 127)


# ---------------------------------------------------------------- product of 8-bit integers
def int8_gemm(x: torch.Tensor, y: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, bias: torch.Tensor | None = None):
    """(result, size): the product in float64 and |product| + |bias|, what roundings are relative to."""
    acc = x.double() @ y.double()  # exact: below 2^53
    p = acc * scale_a.double().reshape(-1, 1) * scale_b.double().reshape(1, -1)
    b = torch.zeros(p.shape[1], dtype=torch.float64, device=p.device) if bias is None else bias.double().reshape(-1)
    return p + b, p.abs() + b.abs()


# ---------------------------------------------------------------- 4-bit cache
def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., D] -> (codes [..., D] 0..15, scale bytes [..., D/32])"""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    e = torch.floor(torch.log2(safe))
    e = e - (torch.pow(2.0, e) > safe).double() + (torch.pow(2.0, e + 1) <= safe).double()  # log2 may be off by an ulp
    e = torch.where(top == 0, torch.full_like(e, -126.0), (e - 2).clamp(-126, 125))
    y = blocks / torch.pow(2.0, e).unsqueeze(-1)
    table = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    a = torch.where(bad.unsqueeze(-1), torch.zeros_like(y), y).abs().clamp(max=6.0)
    d = (a.unsqueeze(-1) - table).abs()
    # nearest; of two equally near ones the even code
    near = d == d.amin(-1, keepdim=True)
    first = near.int().argmax(-1)
    both = near.sum(-1) == 2
    code = torch.where(both & (first % 2 == 1), first + 1, first)
    code = code + 8 * torch.signbit(x).unflatten(-1, (-1, 32)).long()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), dtype=torch.float64, device=codes.device)
    s = torch.pow(2.0, scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (table[codes.long()].unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def to_layout(codes: torch.Tensor, scales: torch.Tensor, values: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """codes [pages, heads, page, D] and scales [pages, heads, page, D/32] in the cache's layout"""
    c = pack(codes)
    if not values:
        return c.contiguous(), scales.contiguous()
    return (c.unflatten(-1, (16, -1)).unflatten(2, (-1, 4)).transpose(3, 4).contiguous(),
            scales.unflatten(2, (-1, 4)).transpose(3, 4).contiguous())


def from_layout(c: torch.Tensor, s: torch.Tensor, values: bool) -> tuple[torch.Tensor, torch.Tensor]:
    if values:
        c = c.transpose(3, 4).flatten(4, 5).flatten(2, 3)
        s = s.transpose(3, 4).flatten(2, 3)
    return unpack(c), s


def attention(q, kc, ks, vc, vs, block_table, seq_lens, query_start=None, scale=None, causal=True):
    """(out, size, spread) in float64: the result (zeros where no sequence writes), the same average over |v|, and for each
    row the largest sum_d |q_d k_d| of a key it sees, times scale (what the rounding of its scores is relative to)."""
    tokens, heads, d = q.shape
    kv_heads, page = kc.shape[1], kc.shape[2]
    group = heads // kv_heads
    scale = d**-0.5 if scale is None else scale
    k_all, v_all = decode(*from_layout(kc, ks, False)), decode(*from_layout(vc, vs, True))  # [pages, heads, page, D]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, spread = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for b, n in enumerate(seq_lens.tolist()):
        t0 = b if query_start is None else int(query_start[b])
        new = 1 if query_start is None else int(query_start[b + 1]) - t0
        pages = block_table[b, : -(-n // page)].tolist()
        if new == 0 or n <= 0:
            continue
        ok = torch.tensor([0 <= p < kc.shape[0] for p in pages], device=q.device).repeat_interleave(page)[:n]
        at = torch.tensor([p if 0 <= p < kc.shape[0] else 0 for p in pages], device=q.device)
        for h in range(kv_heads):
            k, v = k_all[at, h].reshape(-1, d)[:n], v_all[at, h].reshape(-1, d)[:n]
            for i in range(new):
                see = ok & (torch.arange(n, device=q.device) <= (n - new + i if causal else n - 1))
                if not bool(see.any()):
                    continue
                ki, vi = k[see], v[see]
                qi = q[t0 + i, h * group:(h + 1) * group].double()
                w = torch.softmax(qi @ ki.t() * scale, -1)
                out[t0 + i, h * group:(h + 1) * group] = w @ vi
                size[t0 + i, h * group:(h + 1) * group] = w @ vi.abs()
                spread[t0 + i, h * group:(h + 1) * group] = (qi.abs() @ ki.abs().t()).amax(-1) * abs(scale)
    return out, size, spread


def attention_bound(out, size, spread, dtype, keys, d, p_terms):
    """How far a kernel's result may be from `out`: the rounding to dtype, and relative to the average over |v| the errors
    of the weights (numerator and denominator: twice) and of the sums.  Scores: fp32 sums of d products, each addition
    off by at most 2^-23 of the sum of magnitudes, then two roundings; a score's error is the relative error of its weight.
    exp2: 2^-22.  Weights as p_terms bf16 numbers: 2^(-9 p_terms).  Sums over the keys: one addition in 32 at fp32 for
    each tile, and 64 for the joins."""
    half = torch.finfo(dtype).eps / 2
    score = spread.unsqueeze(-1) * ((d + 4) * 2.0**-23)
    weights = 2 * (score + 2.0**-22 + 2.0 ** (-9 * p_terms)) + (keys / 32 + 64) * 2.0**-23
    tiny = float(torch.finfo(dtype).smallest_normal) * half * 2
    return half * out.abs() + (1 + half) * weights * size + tiny


def float_bound(ref, size, dtype, roundings):
    """the rounding to dtype, and `roundings` in fp32 relative to `size`"""
    half = torch.finfo(dtype).eps / 2
    return half * ref.abs() + (1 + half) * roundings * 2.0**-24 * size + float(torch.finfo(dtype).smallest_normal) * half * 2


def sqrt_rows(width: int) -> int:
    """fp32 roundings in y / scale of the norm: the mean's (a lane's sum of up to 64 squares, ten joins, the division, eps),
    halved by the root, the root, the reciprocal, two products, the maximum's own, 127 / max and the last product"""
    return int(math.ceil((min(width, 64) + 12) / 2)) + 10
