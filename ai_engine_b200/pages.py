"""Pages of a key/value cache: who holds them, and moving them
(aie_pages_* of ``include/aie_seq.h``).

The cache is one tensor ``kv`` [layers, 2, pages, page_size, kv_heads,
head_dim] (keys, then values), or one in 4 bits (``new_cache4``); its bookkeeping four int32 CUDA tensors
(``PageState``).  A row of the table is one stream.  All decisions are made on
the device, in the lists' order and lowest free page first, so a call can be
captured in a CUDA graph and nothing is copied to the host; what a call could
not do it leaves undone and says in ``status``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class PageState(NamedTuple):
    """refs [pages]: rows that hold each page; lens [rows]: tokens of each row;
    table [rows, width]: a row's pages in order, -1 behind the last; status
    [1]: _lib.PAGES_FULL | _lib.PAGES_BAD_ROW, collected."""
    refs: torch.Tensor
    lens: torch.Tensor
    table: torch.Tensor
    status: torch.Tensor


def new_state(pages: int, rows: int, width: int, device="cuda") -> PageState:
    """The state of an empty cache: `rows` streams of up to `width` pages each."""
    return PageState(torch.zeros(pages, dtype=torch.int32, device=device), torch.zeros(rows, dtype=torch.int32, device=device),
                     torch.full((rows, width), -1, dtype=torch.int32, device=device),
                     torch.zeros(1, dtype=torch.int32, device=device))


def new_cache(layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
              device="cuda") -> torch.Tensor:
    """An empty cache; kv[layer, 0] and kv[layer, 1] are a layer's k_pages and v_pages."""
    return torch.zeros((layers, 2, pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)


def new_cache4(layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An empty cache in 4 bits: uint8 [layers, 2, pages, kv_heads, page_size,
    head_dim * 5 / 8], for attention.kv4_file, kv4_load and kv4_attention and for
    fork, copy and compact.  A page and head's bytes are one block: its places'
    codes, then their groups' scales and lowest values (aie_kv4).  head_dim is a
    multiple of 32 up to 256, page_size of 8."""
    if head_dim % 32 or not 0 < head_dim <= 256 or page_size % 8 or page_size <= 0:
        raise ValueError(f"pages of {page_size} places of heads of {head_dim}: multiples of 8 and of 32, heads up to 256")
    return torch.zeros((layers, 2, pages, kv_heads, page_size, head_dim * 5 // 8), dtype=torch.uint8, device=device)


def grow(st: PageState, page_size: int, rows: torch.Tensor, counts: torch.Tensor, tokens: int, stream=None) -> torch.Tensor:
    """Row rows[i] gets counts[i] more tokens and the pages for them; returns
    slots [tokens] int64, where each new token stands (the list's order), -1
    past the counts' sum.  With too few pages nothing changes: every slot is
    -1 and status says so."""
    return _lib.seqcall().pages_grow(st, page_size, rows, counts, tokens, stream)


def fork(kv: torch.Tensor, st: PageState, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """Row dst[i] (empty, not in src) becomes a copy of row src[i]: src's whole
    pages are shared, a page that src fills in part is copied."""
    _lib.seqcall().pages_fork(kv, st, src, dst, stream)


def copy(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """Page dst[i] becomes a copy of page src[i] in every layer.  No page is a
    destination twice, nor both a source and a destination."""
    _lib.seqcall().pages_copy(kv, src, dst, stream)


def free(st: PageState, rows: torch.Tensor, stream=None) -> None:
    """The rows become empty; pages that no row holds any more are free."""
    _lib.seqcall().pages_free(st, rows, stream)


def compact(kv: torch.Tensor, st: PageState, stream=None) -> torch.Tensor:
    """The pages in use move to the front of the cache; returns remap [pages]
    int32, each page's new number, -1 for a free one."""
    return _lib.seqcall().pages_compact(kv, st, stream)
