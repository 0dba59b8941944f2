"""Attention for serving sequences, over the C ABI (``include/aie_seq.h``).

``qk_norm_rope`` norms and rotates the heads of a projection and files keys
and values into a paged cache; ``prompt_attention`` attends whole packed
prompts; ``prefix_attention`` makes a one-token step for a batch of streams
that share the front of their contexts.  ``pages`` keeps the cache.

Tensors are CUDA tensors ``[tokens, heads, head_dim]`` in float16, bfloat16 or
float32 with any strides, so long as a head's elements lie side by side.
Every call runs on the current (or given) CUDA stream and waits for nothing.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import check

DTYPE_ID = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}


def _stream(stream, device: int) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype: torch.dtype, device, stream) -> torch.Tensor:
    """Memory for a call on `stream`: from that stream's pool, not from blocks
    that work queued on the current stream may still use."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.stream(s):
        return torch.empty(shape, dtype=dtype, device=device)


def _empty_like(t: torch.Tensor, stream) -> torch.Tensor:
    if stream is None:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    return _empty(t.shape, t.dtype, t.device, stream)


def _heads(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int):
    """(data, token stride, head stride) of a [tokens, heads, head_dim] tensor."""
    if t.dtype is not dtype or t.get_device() != dev:
        raise TypeError(f"{name} must be a {dtype} tensor on cuda:{dev}, as q is: got {t.dtype} on {t.device}")
    ts, hs, ds = t.stride()
    if ds != 1 and t.shape[2] != 1:
        raise ValueError(f"{name}'s heads must be contiguous (stride 1 in the last dimension)")
    return t.data_ptr(), ts, hs


def _dtype(t: torch.Tensor, name: str) -> int:
    dt = DTYPE_ID.get(t.dtype)
    if dt is None or not t.is_cuda or t.dim() != 3:
        raise TypeError(f"{name} must be a float16, bfloat16 or float32 CUDA tensor [tokens, heads, head_dim]")
    return dt


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int, dims: int = 1) -> int:
    if t.dtype is not dtype or t.get_device() != dev or t.dim() != dims or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dims}-D {dtype} tensor on cuda:{dev}")
    return t.data_ptr()


def _cache(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype: torch.dtype, dev: int, kv_heads: int, dim: int):
    """(k, v, page, token and head strides, pages, page size) of [pages, page_size, kv_heads, head_dim] tensors."""
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if t.dtype is not dtype or t.get_device() != dev or t.dim() != 4:
            raise TypeError(f"{name} must be a {dtype} tensor [pages, page_size, kv_heads, head_dim] on cuda:{dev}")
    shape, (ps, ts, hs, ds) = k_pages.shape, k_pages.stride()
    if v_pages.shape != shape or v_pages.stride() != (ps, ts, hs, ds):
        raise ValueError("k_pages and v_pages must have the same shape and strides")
    pages, size, heads, d = shape
    if heads != kv_heads or d != dim:
        raise ValueError(f"the cache holds {heads} heads of {d}, not {kv_heads} of {dim}")
    if ds != 1 and dim != 1:
        raise ValueError("a cached head must be contiguous (stride 1 in the last dimension)")
    return k_pages.data_ptr(), v_pages.data_ptr(), ps, ts, hs, pages, size


_NO_PAGES = (0, 0, 0, 0, 0, 0, 0)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, v: Optional[torch.Tensor] = None, k_pages: Optional[torch.Tensor] = None,
                 v_pages: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                 q_out: Optional[torch.Tensor] = None, k_out: Union[torch.Tensor, bool, None] = None,
                 stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head of q and k over its elements, times a [head_dim]
    float32 weight (None: that tensor is not normed), and the rotation of its
    first ``cos_sin.shape[1]`` elements by its token's position, in one pass
    (aie_qk_norm_rope).  cos_sin is a float32 [positions, rot_dim] table, the
    cosines of a position's angles, then their sines; pair i is elements
    (i, i + rot_dim / 2), or (2i, 2i + 1) when interleaved.  positions is
    int32 [tokens]; one outside the table gives NaN.

    With k_pages, v_pages, v and slots (int64 [tokens]) the new keys and v are
    also filed into the cache at slot page * page_size + place; -1 files
    nothing.  k_out False: the keys go to the cache only.  q_out may be q and
    k_out may be k.  Returns (q_out, k_out)."""
    dt = _dtype(q, "q")
    tokens, hq, d = q.shape
    dt_, dev = q.dtype, q.get_device()
    if k.dim() != 3 or k.shape[0] != tokens or k.shape[2] != d:
        raise ValueError(f"q is {tuple(q.shape)} but k is {tuple(k.shape)}")
    hk = k.shape[1]
    pos = _vector(positions, "positions", torch.int32, dev)
    cs = _vector(cos_sin, "cos_sin", torch.float32, dev, 2)
    if positions.shape[0] != tokens:
        raise ValueError(f"{positions.shape[0]} positions for {tokens} tokens")
    wq = wk = 0
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (d,):
            raise ValueError(f"a weight of shape {tuple(w.shape)} for heads of {d}")
    if q_weight is not None:
        wq = _vector(q_weight, "q_weight", torch.float32, dev)
    if k_weight is not None:
        wk = _vector(k_weight, "k_weight", torch.float32, dev)
    pages, vh, sl = _NO_PAGES, (0, 0, 0), 0
    if k_pages is not None:
        if v is None or v_pages is None or slots is None:
            raise ValueError("filing into the cache takes v, v_pages and slots")
        if v.shape != k.shape:
            raise ValueError(f"k is {tuple(k.shape)} but v is {tuple(v.shape)}")
        if slots.shape != (tokens,):
            raise ValueError(f"slots of shape {tuple(slots.shape)} for {tokens} tokens")
        pages, vh = _cache(k_pages, v_pages, dt_, dev, hk, d), _heads(v, "v", dt_, dev)
        sl = _vector(slots, "slots", torch.int64, dev)
    elif v is not None or v_pages is not None or slots is not None or k_out is False:
        raise ValueError("v, v_pages, slots and k_out=False go with a cache (k_pages)")
    if q_out is None:
        q_out = _empty_like(q, stream)
    elif q_out.shape != q.shape:
        raise ValueError(f"q is {tuple(q.shape)} but q_out is {tuple(q_out.shape)}")
    if k_out is None:
        k_out = _empty_like(k, stream)
    elif k_out is not False and k_out.shape != k.shape:
        raise ValueError(f"k is {tuple(k.shape)} but k_out is {tuple(k_out.shape)}")
    ko = (0, 0, 0) if k_out is False else _heads(k_out, "k_out", dt_, dev)
    args = _lib.QK_ROPE.pack(*_heads(q, "q", dt_, dev), *_heads(k, "k", dt_, dev), *vh, *_heads(q_out, "q_out", dt_, dev), *ko, *pages,
                             wq, wk, cs, pos, sl, tokens, hq, hk, d, cos_sin.shape[1], cos_sin.shape[0],
                             dt, interleaved, eps, 0)
    check(_lib.load().aie_qk_norm_rope(args, _stream(stream, dev)), "aie_qk_norm_rope")
    return q_out, (None if k_out is False else k_out)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, *, causal: bool = True,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v over packed sequences (aie_prompt_attn): sequence
    s is tokens cu[s] .. cu[s + 1] of q [tokens, heads, head_dim] and of k, v
    [tokens, kv_heads, head_dim]; with causal a token sees its sequence up to
    itself.  cu is an int32 CUDA tensor [sequences + 1]; it is not copied to
    the host.  scale defaults to head_dim ** -0.5."""
    dt = _dtype(q, "q")
    tokens, hq, d = q.shape
    dt_, dev = q.dtype, q.get_device()
    if k.dim() != 3 or k.shape[0] != tokens or k.shape[2] != d or v.shape != k.shape:
        raise ValueError(f"q is {tuple(q.shape)} but k and v are {tuple(k.shape)} and {tuple(v.shape)}")
    c = _vector(cu, "cu", torch.int32, dev)
    if cu.shape[0] < 1:
        raise ValueError("cu holds at least one entry")
    if out is None:
        out = _empty_like(q, stream)
    elif out.shape != q.shape:
        raise ValueError(f"q is {tuple(q.shape)} but out is {tuple(out.shape)}")
    args = _lib.PROMPT.pack(*_heads(q, "q", dt_, dev), *_heads(k, "k", dt_, dev), *_heads(v, "v", dt_, dev), *_heads(out, "out", dt_, dev), c, tokens,
                            cu.shape[0] - 1, hq, k.shape[1], d, dt, causal, d ** -0.5 if scale is None else scale)
    check(_lib.load().aie_prompt_attn(args, _stream(stream, dev)), "aie_prompt_attn")
    return out


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix: Optional[torch.Tensor],
                     prefix_len: int, table: torch.Tensor, lens: torch.Tensor, *, max_len: Optional[int] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """One query token for each of q's streams [batch, heads, head_dim] over a
    paged cache (aie_prefix_attn).  Stream b attends to its first lens[b]
    places (int32 CUDA tensor): those below prefix_len stand in the shared
    pages ``prefix`` (int32, in order) and are read once for all streams; the
    rest in its own pages, table[b, place // page_size].  As pages.fork leaves
    them, ``prefix`` is any stream's row.  A stream without places gives
    zeros.  max_len bounds lens (default: what a table row holds); longer
    streams are cut off there."""
    dt = _dtype(q, "q")
    b, hq, d = q.shape
    dt_, dev = q.dtype, q.get_device()
    hk = k_pages.shape[2] if k_pages.dim() == 4 else 0
    pages = _cache(k_pages, v_pages, dt_, dev, hk, d)
    size = pages[6]
    tb = _vector(table, "table", torch.int32, dev, 2)
    ln = _vector(lens, "lens", torch.int32, dev)
    if table.shape[0] != b or lens.shape[0] != b:
        raise ValueError(f"{b} streams, but {table.shape[0]} table rows and {lens.shape[0]} lengths")
    if prefix_len < 0:
        raise ValueError(f"prefix_len is {prefix_len}")
    pre = 0
    if prefix_len:
        pre = _vector(prefix, "prefix", torch.int32, dev)
        if prefix.shape[0] * size < prefix_len:
            raise ValueError(f"{prefix.shape[0]} pages of {size} do not hold a prefix of {prefix_len}")
    if max_len is None:
        max_len = max(table.shape[1] * size, prefix_len)
    if out is None:
        out = _empty_like(q, stream)
    elif out.shape != q.shape:
        raise ValueError(f"q is {tuple(q.shape)} but out is {tuple(out.shape)}")
    lib = _lib.load()
    head = (*_heads(q, "q", dt_, dev), *_heads(out, "out", dt_, dev), *pages, pre, tb, ln)
    tail = (b, hq, hk, d, prefix_len, max_len, table.shape[1], dt, d ** -0.5 if scale is None else scale, 0)
    need = lib.aie_prefix_attn_workspace(_lib.PREFIX.pack(*head, 0, 0, *tail))
    ws = _empty(need, torch.uint8, q.device, stream)
    check(lib.aie_prefix_attn(_lib.PREFIX.pack(*head, ws.data_ptr(), need, *tail), _stream(stream, dev)), "aie_prefix_attn")
    return out
