"""Attention between the packed projections: prompts, and a key/value cache held in 4 bits.

``fused_qkv`` ends in rotated q, k and v and the output projection takes the attention's result; these ops
are what runs between them.  A prompt attends to itself with ``prompt_attention`` while ``kv4_append``
stores its keys and values; each decode step appends its new token and attends with ``kv4_attention``:

    cache = KV4Cache.empty(num_pages, kv_heads, head_dim, page_size=64)
    kv4_append(cache, k, v, block_table, seq_lens, cu_seqlens)          # a packed batch of prompts
    o = prompt_attention(q, k, v, cu_seqlens, max_seqlen)
    ...
    seq_lens += 1
    kv4_append(cache, k, v, block_table, seq_lens)                      # one new token a sequence
    o = kv4_attention(q, cache, block_table, seq_lens)

The cache is a pool of pages that sequences share (``block_table``); lengths and the table are read on the
device, so a captured decode step follows them on replay.  The reference has no counterpart of these ops.
They are for inference: none has a backward, and an input that requires a gradient is refused under grad mode.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import ops


def _backend():
    ops._check_ext()
    return ops._C


@dataclass
class KV4Cache:
    """Pages of keys and values in 4 bits, one layer's: ``pages`` int32 [pages, kv heads, words] (the words of
    ``page_size`` tokens of one head, include/crispybits_attention.h).  A vector of one token and head is held as
    4-bit codes with a scale and a zero point of its own: about a quarter of its 16-bit size."""
    pages: torch.Tensor
    page_size: int
    head_dim: int

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, device=None) -> "KV4Cache":
        """A pool of ``num_pages`` pages of ``page_size`` tokens (a power of two from 32 on) on ``device``
        (default: the current GPU); head_dim is a multiple of 8 up to 256."""
        words = _backend().kv4_page_words(head_dim, page_size)
        pages = torch.zeros(num_pages, num_kv_heads, words, dtype=torch.int32,
                            device=torch.device(device if device is not None else "cuda"))
        return cls(pages, page_size, head_dim)

    @property
    def num_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.pages.shape[1]


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Store new tokens' k and v [rows, kv heads, head_dim] (fp16 / bf16 / fp32, rows and heads strided as they
    come).  ``seq_lens`` int32 [sequences] counts each sequence's tokens with the new ones, and
    ``block_table`` int32 [sequences, pages] names its pages.  Rows ``cu_seqlens[b] : cu_seqlens[b + 1]`` are the
    newest tokens of sequence b; without ``cu_seqlens`` row b is the newest token of b.  Rows that have no
    place (an idle slot with length 0, a table entry of -1) are left out.  A page written by a call must belong to
    one sequence."""
    _backend().kv4_append(cache.pages, cache.page_size, cache.head_dim, k, v, block_table, seq_lens, cu_seqlens)


def kv4_read(cache: KV4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
             cu_seqlens: Optional[torch.Tensor] = None, rows: Optional[int] = None,
             dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """k and v [rows, kv heads, head_dim] as the cache holds them, of the tokens that ``kv4_append`` with the same
    table, lengths and ``cu_seqlens`` stores (``rows``: the packed rows; without ``cu_seqlens`` one a sequence).  A
    whole cache is read with cumulative ``seq_lens`` as ``cu_seqlens``.  Tokens without a page are zeros."""
    if rows is None:
        if cu_seqlens is not None:
            raise ValueError("kv4_read needs the number of packed rows with cu_seqlens")
        rows = seq_lens.shape[0]
    return _backend().kv4_read(cache.pages, cache.page_size, cache.head_dim, block_table, seq_lens, cu_seqlens, rows,
                               dtype)


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q K^T) V of each sequence's newest tokens over its cached tokens.

    q is [sequences, heads, head_dim] (one new token each) or [sequences, t, heads, head_dim] (the t newest,
    which the cache already holds): query i sees positions up to ``seq_lens - t + i``.  Query heads are
    grouped over the cache's kv heads.  ``scale`` (positive, at most 2^127) defaults to head_dim ** -0.5.  A query that sees nothing
    (an idle slot) gives zeros.  Tokens whose table entry names no page take no part."""
    if q.dim() not in (3, 4):
        raise ValueError("q must be [sequences, heads, head_dim] or [sequences, new tokens, heads, head_dim]")
    if scale is None:
        scale = cache.head_dim ** -0.5
    C = _backend()
    if q.dim() == 4:
        return C.kv4_attention(q, cache.pages, cache.page_size, cache.head_dim, block_table, seq_lens, scale, out)
    o = C.kv4_attention(q.unsqueeze(1), cache.pages, cache.page_size, cache.head_dim, block_table, seq_lens, scale,
                        None if out is None else out.unsqueeze(1))
    return out if out is not None else o.squeeze(1)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     max_seqlen: Optional[int] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts over themselves: q [rows, heads, head_dim], k and v [rows, kv heads,
    head_dim] (fp16 / bf16 / fp32, rows and heads strided as they come), row i of a sequence attending to its rows
    0 .. i.  ``cu_seqlens`` int32 [sequences + 1] holds the sequences' first rows and the end of the last.
    ``max_seqlen`` is at least the longest sequence's length (default: all rows; a tight bound launches less).
    ``scale`` (positive, at most 2^127) defaults to head_dim ** -0.5.  Rows behind the last sequence come back as zeros, or stay as
    they were in ``out``.  What the causal mask hides takes no part, infinities and NaN included; a visible
    infinity or NaN in v gives an infinity or NaN, whatever its weight."""
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, head_dim]")
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if max_seqlen is None:
        max_seqlen = q.shape[0]
    return _backend().prompt_attention(q, k, v, cu_seqlens, min(int(max_seqlen), q.shape[0]), scale, out)
