"""A paged key/value cache held in 4 bits, and attention of new tokens over it.

The format is MXFP4: e2m1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a power-of-two scale for each 32
consecutive elements of a head, 4.25 bits an element.  The rounding is to the nearest value, ties to the even code; what a
block's exponent ``floor(log2 max|x|) - 2`` leaves above 6 becomes 6.  The layout of the four tensors is part of the C
interface (include/hx_kernels.h).  For inference: no result carries a gradient."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .ops import kv4_attention_call, kv4_attention_out_call, kv4_read_call, kv4_write_call


class Kv4Cache(NamedTuple):
    """The cache of one layer: k [pages, heads, page, head_dim / 2], k_scale [pages, heads, page, head_dim / 32],
    v [pages, heads, page / 4, 16, 4, head_dim / 32], v_scale [pages, heads, page / 4, head_dim / 32, 4], all uint8."""

    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor


def kv4_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, device: torch.device | str = "cuda") -> Kv4Cache:
    """An empty cache of ``pages`` pages of ``page_size`` tokens (a power of two from 16 to 1024) for head dims 64, 128 and
    256.  Its content is undefined until it is written; nothing reads what lies behind a sequence's length."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"kv4_cache: head_dim must be 64, 128 or 256, got {head_dim}")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"kv4_cache: page_size must be a power of two from 16 to 1024, got {page_size}")
    if pages < 0 or kv_heads < 1:
        raise ValueError(f"kv4_cache: {pages} pages of {kv_heads} heads")
    s = head_dim // 32

    def empty(*shape: int) -> torch.Tensor:
        return torch.empty(shape, dtype=torch.uint8, device=device)

    return Kv4Cache(empty(pages, kv_heads, page_size, head_dim // 2), empty(pages, kv_heads, page_size, s),
                    empty(pages, kv_heads, page_size // 4, 16, 4, s), empty(pages, kv_heads, page_size // 4, s, 4))


def kv4_write(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise k and v, [tokens, heads, head_dim] float16, bfloat16 or float32, into the cache: token t goes to
    ``slots[t] = page * page_size + place`` (int32 or int64).  k and v may be slices of one projection's output (any token and
    head strides).  A slot outside the cache (-1 for a padded token) writes nothing; of several tokens with one slot the last
    one stays.  One launch for every 32768 tokens."""
    kv4_write_call(*cache, k, v, slots)


def kv4_read(cache: Kv4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, [tokens, heads, head_dim] of ``dtype``: the values held at ``slots`` (int32 or int64), zeros for a slot outside
    the cache."""
    return kv4_read_call(*cache, slots, dtype)


def kv4_attention(q: torch.Tensor, cache: Kv4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                  query_start: torch.Tensor | None = None, max_query_len: int = 1, scale: float | None = None, causal: bool = True,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` of new tokens over the cached keys and values of their sequences.

    q: [tokens, heads, head_dim] float16, bfloat16 or float32 (any token and head strides), heads a multiple of the cache's:
    query head h reads key/value head ``h // (heads // kv_heads)``.  block_table: [sequences, width] int32, the pages of each
    sequence in order; seq_lens: [sequences] int32, its keys, the new tokens' own among them (write them first).
    Without query_start every sequence has one new token, row b of q.  With it, [sequences + 1] int32, the new tokens of sequence b
    are rows ``query_start[b] .. query_start[b + 1] - 1``, and max_query_len (a host number) is the most of one sequence; it
    sizes the launch, a larger count is computed all the same.  causal: new token i of n sees the keys up to its own,
    ``seq_lens[b] - n + i``; otherwise all keys of its sequence.  A row without a key gives zeros.  scale: ``head_dim ** -0.5``
    unless given.

    Rows of q outside ``query_start[0] .. query_start[sequences] - 1`` are left as they were in ``out``, which is allocated where it is
    not given (undefined there).  Table entries behind a sequence's last page are not used, and a page outside the cache masks
    its keys; a length beyond the table counts as the table's size.  Keys and values enter the products exactly, q and the
    weights as sums of bf16 terms (weights two, three for float32, in every batch), everything else is fp32."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    args = (q, *cache, block_table, seq_lens, query_start, max_query_len, float(scale), bool(causal))
    if out is None:
        return kv4_attention_call(*args)
    kv4_attention_out_call(out, *args)
    return out
