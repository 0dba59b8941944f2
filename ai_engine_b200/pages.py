"""Pages of a key/value cache: who holds them, and moving them
(aie_pages_* of ``include/aie_seq.h``).

The cache is one tensor ``kv`` [layers, 2, pages, page_size, kv_heads,
head_dim] (keys, then values); its bookkeeping four int32 CUDA tensors
(``PageState``).  A row of the table is one stream.  All decisions are made on
the device, in the lists' order and lowest free page first, so a call can be
captured in a CUDA graph and nothing is copied to the host; what a call could
not do it leaves undone and says in ``status``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check
from .attention import DTYPE_ID, _empty, _stream, _vector


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


def _pack_kv(kv: torch.Tensor):
    if kv.dtype not in DTYPE_ID or not kv.is_cuda or kv.dim() != 6 or kv.shape[1] != 2 or not kv.is_contiguous():
        raise TypeError("kv must be a contiguous float16, bfloat16 or float32 CUDA tensor "
                        "[layers, 2, pages, page_size, kv_heads, head_dim]")
    layers, _, pages, size, heads, dim = kv.shape
    return kv.data_ptr(), size * heads * dim * kv.element_size(), layers, pages, size


def _args(kv: Optional[torch.Tensor], st: PageState, n: int, stream, page_size: int = 0):
    """The packed aie_pages, and the scratch it points to (kept by the caller over the launch)."""
    refs, lens, table, status = st
    dev = refs.get_device()
    r, ln, tb, sp = (_vector(refs, "refs", torch.int32, dev), _vector(lens, "lens", torch.int32, dev),
                     _vector(table, "table", torch.int32, dev, 2), _vector(status, "status", torch.int32, dev))
    pages, rows, width = refs.shape[0], lens.shape[0], table.shape[1]
    if dev < 0 or table.shape[0] != rows or status.shape[0] != 1:
        raise ValueError("the state is refs [pages], lens [rows], table [rows, width] and status [1] on a CUDA device")
    data = page_bytes = layers = 0
    if kv is not None:
        data, page_bytes, layers, has, page_size = _pack_kv(kv)
        if has != pages or kv.get_device() != dev:
            raise ValueError(f"kv has {has} pages on {kv.device}, the state {pages} on {refs.device}")
    ws = _empty(_lib.load().aie_pages_workspace(pages, n) // 4, torch.int32, refs.device, stream)
    return _lib.PAGES.pack(data, r, ln, tb, sp, ws.data_ptr(), page_bytes, layers, pages, page_size, rows, width, 0), ws


def _lists(a: torch.Tensor, b: torch.Tensor, names, device) -> int:
    for t, name in zip((a, b), names):
        _vector(t, name, torch.int32, device)
    if a.shape != b.shape:
        raise ValueError(f"{a.shape[0]} {names[0]} but {b.shape[0]} {names[1]}")
    return a.shape[0]


def grow(st: PageState, page_size: int, rows: torch.Tensor, counts: torch.Tensor, tokens: int, stream=None) -> torch.Tensor:
    """Row rows[i] gets counts[i] more tokens and the pages for them; returns
    slots [tokens] int64, where each new token stands (the list's order), -1
    past the counts' sum.  With too few pages nothing changes: every slot is
    -1 and status says so."""
    dev = st.refs.get_device()
    n = _lists(rows, counts, ("rows", "counts"), dev)
    args, ws = _args(None, st, n, stream, page_size)
    slots = _empty(tokens, torch.int64, st.refs.device, stream)
    check(_lib.load().aie_pages_grow(args, rows.data_ptr(), counts.data_ptr(), n, slots.data_ptr(), tokens,
                                     _stream(stream, dev)), "aie_pages_grow")
    return slots


def fork(kv: torch.Tensor, st: PageState, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """Row dst[i] (empty, not in src) becomes a copy of row src[i]: src's whole
    pages are shared, a page that src fills in part is copied."""
    dev = st.refs.get_device()
    n = _lists(src, dst, ("src", "dst"), dev)
    args, ws = _args(kv, st, n, stream)
    check(_lib.load().aie_pages_fork(args, src.data_ptr(), dst.data_ptr(), n, _stream(stream, dev)), "aie_pages_fork")


def copy(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """Page dst[i] becomes a copy of page src[i] in every layer.  No page is a
    destination twice, nor both a source and a destination."""
    n = _lists(src, dst, ("src", "dst"), kv.get_device())
    data, page_bytes, layers, pages, size = _pack_kv(kv)
    args = _lib.PAGES.pack(data, 0, 0, 0, 0, 0, page_bytes, layers, pages, size, 0, 0, 0)
    check(_lib.load().aie_pages_copy(args, src.data_ptr(), dst.data_ptr(), n, _stream(stream, kv.get_device())), "aie_pages_copy")


def free(st: PageState, rows: torch.Tensor, stream=None) -> None:
    """The rows become empty; pages that no row holds any more are free."""
    dev = st.refs.get_device()
    _vector(rows, "rows", torch.int32, dev)
    args, _ = _args(None, st, 0, stream)
    check(_lib.load().aie_pages_free(args, rows.data_ptr(), rows.shape[0], _stream(stream, dev)), "aie_pages_free")


def compact(kv: torch.Tensor, st: PageState, stream=None) -> torch.Tensor:
    """The pages in use move to the front of the cache; returns remap [pages]
    int32, each page's new number, -1 for a free one."""
    dev = st.refs.get_device()
    args, ws = _args(kv, st, 0, stream)
    remap = _empty(st.refs.shape[0], torch.int32, st.refs.device, stream)
    check(_lib.load().aie_pages_compact(args, remap.data_ptr(), _stream(stream, dev)), "aie_pages_compact")
    return remap
