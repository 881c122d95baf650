"""A key/value cache in 8 bits, in pages, for several sequences, and the two operators that a model runs on it.

A cache is four tensors (`KVCache`): k and v [pages, kv_heads, page_size, head_dim] of torch.int8 or torch.float8_e4m3fn, and
k_scale, v_scale [pages, kv_heads] of torch.float32; a value is its code times the scale of its page and head (scales are greater than zero, and those of
values below 2^-64 count as 2^-64). Next to weights
that are pruned and compressed the cache is what a decode step reads most of: half the bytes of an fp16 cache.

Which tokens belong to which sequence is said by three int32 tensors on the device, read when the kernels run (so a captured call
is replayed with new ones written into them):

  page_table [sequences, most pages]   page j of sequence i holds its tokens j * page_size ...
  lengths [sequences]                  tokens of sequence i in the cache, the rows of this call included (0: not served)
  query_start [sequences + 1]          rows query_start[i] .. query_start[i + 1] of the call are the last ones of sequence i;
                                       left out where every sequence has one row (decoding)

One step of a layer is `rope_append` with the layer's q, k and v, then `paged_attention` with the q that it returns. The reference has
no cache; its decode benchmark uses the static fp16 cache of a library (python_scripts/util_run_pruned_llm.py:51-81).
"""
from __future__ import annotations

from typing import NamedTuple

import torch


_is_compiling = torch.compiler.is_compiling


def _direct_append(*args):
    """The way past the operator dispatcher, where the package has it (see `multiply`); None: through the operator."""


def _direct_attention(*args):
    """The same for `paged_attention`."""


class KVCache(NamedTuple):
    """Codes of the keys and values and their scales. Any tuple of the four tensors is taken where one is asked for; pages may
    be strided (k and v as halves of one tensor, say), what is inside a page is contiguous."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new_cache(pages: int, kv_heads: int, page_size: int = 32, head_dim: int = 128, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> KVCache:
    """An empty cache. page_size: 16, 32, 64 or 128 tokens share a scale; head_dim: 64, 128 or 256."""
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise TypeError(f"a cache holds torch.int8 or torch.float8_e4m3fn, not {dtype}")
    if page_size not in (16, 32, 64, 128) or head_dim not in (64, 128, 256) or pages < 1 or kv_heads < 1:
        raise ValueError(f"no cache of {pages} pages of {page_size} tokens, {kv_heads} heads of {head_dim}")
    codes = [torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
    return KVCache(*codes, *scales)


def rope_append(qkv, cos_table, sin_table, cache, page_table, lengths, query_start=None):
    """Rotates q and k of the call's rows at their positions and puts k and v into the cache; returns q [rows, heads, head_dim].

    qkv [rows, (heads + 2 * kv_heads) * head_dim], fp16 or bfloat16: q, k and v of every row, not yet rotated (what a stacked
    q/k/v projection returns; rows may be strided, each 16-byte aligned). cos_table, sin_table: fp16 [positions, head_dim] with both halves equal, rows for every
    position that the page table can name (rotate-half, as in `rope_attention`).

    The scale of a page and head is the smallest power of two (2^-64 or more) with which the call's rows on that page fit the type; it
    never shrinks while a page fills, and the tokens that a page holds already are moved to the new scale where it grows. Codes are
    correctly rounded. A value that is not finite makes its page's scale NaN, so that whoever attends to it gets NaN, until the page is
    started anew. Rows at positions that the table has no page for are left out (q is rotated all the same where the table reaches),
    rows of no sequence get a q of zeros, and slots behind the last token are left as they were.

    A page may be read by many sequences but written for one: calls that write the same page must not overlap on the GPU, and the
    rows of one call must not share a page between sequences, or between two places of one."""
    if not _is_compiling():
        q = _direct_append(qkv, cos_table, sin_table, cache, page_table, lengths, query_start)   # None: not a plain call
        if q is not None:
            return q
    k, v, k_scale, v_scale = cache
    return torch.ops.macko_spmv.rope_append.default(qkv, cos_table, sin_table, k, v, k_scale, v_scale, page_table, lengths, query_start)


def paged_attention(q, cache, page_table, lengths, query_start=None, scale=None):
    """softmax(scale * q K^T) V over the cached tokens at or before each row's position; returns [rows, heads, head_dim] of q's type.

    q [rows, heads, head_dim], fp16 or bfloat16, rotated (heads and rows may be strided, all 16-byte aligned); heads must be a multiple of the cache's, and head h reads
    the cache's head h // (heads // kv_heads). scale: 1 / sqrt(head_dim) if None, else a finite number. A row that sees no token (an empty sequence, rows of no
    sequence) gives zeros. Sums and the softmax are kept in fp32; the weights of the values are rounded to fp16 on the way, by half a step or by 2^-32 of
    the row's largest product of a weight and its value's scale.

    One kernel serves the whole call, chosen by the mean number of rows of a sequence, those without rows among them: a call takes longer than its parts
    where a long prompt stands next to many single tokens or empty sequences, and is better made as two."""
    if not _is_compiling():
        out = _direct_attention(q, cache, page_table, lengths, query_start, scale)   # None: not a plain call
        if out is not None:
            return out
    k, v, k_scale, v_scale = cache
    return torch.ops.macko_spmv.paged_attention.default(q, k, v, k_scale, v_scale, page_table, lengths, query_start, scale)
