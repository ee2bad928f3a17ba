"""Attention next to the packed linears: of whole prompts, and over a key/value cache held in 4 bits.

Between `fused_qkv` and the output projection a model needs attention.  A prompt attends to itself:

    out = prompt_attention(q, k, v, cu_seqlens)                    # packed prompts of any lengths, causal, grouped heads

With weights of 2 to 4 bits the keys and values of past tokens are the next largest thing that a decode step reads, so
they are kept in 4 bits as well:

    cache = KV4Cache.empty(n_pages, kv_heads, head_dim)            # one for each layer
    kv4_append(cache, k, v, page_table, starts, cu_seqlens)        # new tokens, at positions starts[s], starts[s] + 1, ...
    out = kv4_attention(q, cache, page_table, lengths)             # the newest tokens over everything up to them
    k, v = kv4_read(cache, page_table, starts, cu_seqlens, n)      # values back, e.g. the history of a prompt that goes on

The format: the head_dim values of a token and head are cut into groups of `group_size`; a group keeps its smallest
value lo, scale = (largest - lo) / 15 rounded to the cache's dtype, and a 4-bit code round((x - lo) / scale) for each
value, which then stands for code * scale + lo.  Sequences own pages of `page_size` tokens: row s of `page_table` lists
the pages of sequence s in order.  All index tensors are int32 on the cache's device and are read there: a call is asynchronous,
and a captured one may be replayed with other contents.  The reference has no counterpart (it leaves attention to its host).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import ops


def _C():
    ops._check_ext()
    if not hasattr(ops._C, "kv4_block_bytes"):
        raise RuntimeError("the selected backend has no attention operators")
    return ops._C


@dataclass(frozen=True, eq=False)
class KV4Cache:
    """Keys and values of one layer in 4 bits: `pages` uint8 [n_pages, kv_heads, bytes of a page and head]."""
    pages: torch.Tensor
    head_dim: int
    page_size: int = 64
    group_size: int = 64
    dtype: torch.dtype = torch.float16

    @staticmethod
    def empty(n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, group_size: int = 64,
              dtype: torch.dtype = torch.float16, device="cuda") -> "KV4Cache":
        """A cache with room for n_pages * page_size tokens: head_dim 64 or 128; group_size 32, 64 or 128, at most
        head_dim; page_size a multiple of 16; dtype (of keys, values and queries) float16 or bfloat16."""
        c = _C()
        block = c.kv4_block_bytes(head_dim, group_size)
        if block == 0:
            raise ValueError("KV4Cache: head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim")
        if page_size <= 0 or page_size % 16:
            raise ValueError("KV4Cache: page_size must be a positive multiple of 16")
        if n_pages < 1 or kv_heads < 1:
            raise ValueError("KV4Cache: n_pages and kv_heads must be positive")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("KV4Cache: dtype must be float16 or bfloat16")
        pages = torch.empty(n_pages, kv_heads, page_size // 16 * block, dtype=torch.uint8, device=device)
        if pages.is_cuda:
            c.prepare_attention(pages.device)
        return KV4Cache(pages, int(head_dim), int(page_size), int(group_size), dtype)

    def __getstate__(self):
        return {f: v for f, v in self.__dict__.items() if f != "_record"}      # the library's record names addresses of this process

    @property
    def n_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.pages.shape[1]


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Quantise the keys and values of new tokens into the cache.

    k, v: packed [tokens, kv_heads, head_dim] with `cu_seqlens` [B + 1], the first token of each sequence; or, without it,
    [B, T, kv_heads, head_dim], or packed with as many tokens of each sequence (a decode step: one).  Any strides; rows that are not contiguous or not
    16-byte aligned are copied first.  `starts` [B]: the position of each sequence's first new token.  No position
    may be written twice in one call.  A token whose position has no page (beyond the table, or a page number outside the cache) is left out,
    and `_C.decode_status()` then reports 3001."""
    if cu_seqlens is None:
        if k.dim() == 4 or v.dim() == 4:
            if k.shape != v.shape:
                raise ValueError("kv4_append: k and v must have the same shape")
            if page_table.dim() == 2 and k.shape[0] != page_table.shape[0]:
                raise ValueError("kv4_append: page_table needs one row for each sequence of k and v")
            k, v = k.flatten(0, 1), v.flatten(0, 1)
        if page_table.dim() == 2 and page_table.shape[0] and k.shape[0] % page_table.shape[0]:
            raise ValueError("kv4_append: without cu_seqlens every sequence brings as many tokens")
    _C().kv4_append(cache, k, v, page_table, starts, cu_seqlens)


def kv4_read(cache: KV4Cache, page_table: torch.Tensor, starts: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
             n_tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) packed [n_tokens, kv_heads, head_dim] in the cache's dtype: what the cache holds for the tokens that `kv4_append`
    would write with the same `starts` and `cu_seqlens`.  Rows of tokens that have no place there are not written."""
    if cu_seqlens is None and page_table.dim() == 2 and page_table.shape[0] and n_tokens % page_table.shape[0]:
        raise ValueError("kv4_read: without cu_seqlens every sequence has as many tokens")
    return _C().kv4_read(cache, page_table, starts, cu_seqlens, n_tokens)


def kv4_attention(q: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor, lengths: torch.Tensor,
                  scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale * q K^T) V of the newest tokens over the cache (their own keys and values appended before).

    q: [B, H, head_dim], one token of each sequence, or [B, T, H, head_dim], the T newest; any strides.  H is a multiple of the
    cache's heads, and query head h reads key head h // (H // kv_heads).  `lengths` [B]: cached tokens of each sequence, q's own
    among them; token j of T sees the first lengths - T + 1 + j.  A row that sees nothing (lengths 0) is 0, one with a score
    that is NaN is NaN.  scale: finite, default head_dim ** -0.5.
    T may be any, but the cache is read once for each 16 rows (T * H / kv_heads of them) of a key head: for long pieces of
    a prompt, read the history back and use prompt attention."""
    return _C().kv4_attention(q, cache, page_table, lengths, cache.head_dim ** -0.5 if scale is None else float(scale))


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None, causal: bool = True,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q K^T) V for packed prompts of different lengths.

    q [Tq, H, head_dim], k and v [Tk, Hkv, head_dim], float16 or bfloat16, head_dim 64 or 128, H a multiple of Hkv (query head h
    reads key head h // (H // Hkv)); any strides, rows that are not contiguous or not 16-byte aligned are copied first.
    `cu_seqlens` int32 [B + 1]: the first query of each sequence and the end of the last; `cu_seqlens_k` the same for the keys where
    they differ: a piece of a prompt attends to what came before it and to itself.  causal: query r of Lq sees the first
    Lk - Lq + r + 1 keys.  A query that sees none gives 0, one with a score of NaN or +inf, or none above -inf, NaN.  Rows of no sequence are left as they are in `out` (and are
    undefined without it; it shares no memory with q, k and v).  scale: finite, default head_dim ** -0.5.  Keys and values that a query does not see do not
    touch it, infinities and NaN among them.  Scratch for tiles that are cut between SMs (on 148 SMs at head_dim 128 158 MB for long prompts, 39 MB for
    a few thousand tokens, none for up to 128) is kept for each stream that calls this eagerly, and comes from the graph's pool in a capture."""
    return _C().prompt_attention(q, k, v, cu_seqlens, cu_seqlens if cu_seqlens_k is None else cu_seqlens_k,
                                 q.shape[-1] ** -0.5 if scale is None else float(scale), causal, out)
