"""Attention for serving sequences, over the C ABI (``include/aie_seq.h``).

``qk_norm_rope`` norms and rotates the heads of a projection and files keys
and values into a paged cache; ``prompt_attention`` attends whole packed
prompts; ``prefix_attention`` makes a one-token step for a batch of streams
that share the front of their contexts.  ``pages`` keeps the cache.

Tensors are CUDA tensors ``[tokens, heads, head_dim]`` in float16, bfloat16 or
float32 with any strides, so long as a head's elements lie side by side.
Every call runs on the current (or given) CUDA stream and waits for nothing;
outputs come from that stream's memory.  There is no backward pass: where
gradients are recorded, a tensor that requires one is refused.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, v: Optional[torch.Tensor] = None, k_pages: Optional[torch.Tensor] = None,
                 v_pages: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                 q_out: Optional[torch.Tensor] = None, k_out: Union[torch.Tensor, bool, None] = None,
                 pair_axis: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head of q and k over its elements, times a [head_dim]
    float32 weight (None: that tensor is not normed), and the rotation of its
    first ``cos_sin.shape[1]`` elements by its token's position, in one pass
    (aie_qk_norm_rope).  cos_sin is a float32 [positions, rot_dim] table, the
    cosines of a position's angles, then their sines; pair i is elements
    (i, i + rot_dim / 2), or (2i, 2i + 1) when interleaved.  positions is
    int32 [tokens]; one outside the table gives NaN.

    With pair_axis (uint8 [rot_dim / 2]) tokens stand on several axes, as a
    frame's do in time, height and width: positions is int32 [tokens, axes], and
    pair i takes its angle from column i of the table's row for the position
    along axis pair_axis[i] (aie_qk_norm_rope_axes).  Sections of a head, axes
    taking turns, and axes with frequencies of their own (columns of the table)
    are all such a list.

    With k_pages, v_pages, v and slots (int64 [tokens]) the new keys and v are
    also filed into the cache at slot page * page_size + place; -1 files
    nothing.  k_out False: the keys go to the cache only.  q_out may be q and
    k_out may be k.  Returns (q_out, k_out)."""
    return _lib.seqcall().qk_norm_rope(q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, v, k_pages, v_pages,
                                       slots, q_out, k_out, stream, pair_axis)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, *, causal: bool = True,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v over packed sequences (aie_prompt_attn): sequence
    s is tokens cu[s] .. cu[s + 1] of q [tokens, heads, head_dim] and of k, v
    [tokens, kv_heads, head_dim]; with causal a token sees its sequence up to
    itself.  cu is an int32 CUDA tensor [sequences + 1]; it is not copied to
    the host.  scale defaults to head_dim ** -0.5.  Tokens of no sequence are
    left as they are in out, undefined without it.  With causal, a NaN or
    infinity in v may reach earlier tokens of its sequence too."""
    return _lib.seqcall().prompt_attention(q, k, v, cu, causal, scale, out, stream)


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix: Optional[torch.Tensor],
                     prefix_len: int, table: torch.Tensor, lens: torch.Tensor, *, max_len: Optional[int] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """One query token for each of q's streams [batch, heads, head_dim] over a
    paged cache (aie_prefix_attn).  Stream b attends to its first lens[b]
    places (int32 CUDA tensor): those below prefix_len stand in the shared
    pages ``prefix`` (int32, in order) and are read once for all streams; the
    rest in its own pages, table[b, place // page_size].  As pages.fork leaves
    them, ``prefix`` is any stream's row.  A stream without places gives
    zeros; what stands behind a stream's places, NaN and infinities too, never
    reaches its result.  max_len bounds lens (default: what a table row
    holds); longer streams are cut off there."""
    return _lib.seqcall().prefix_attention(q, k_pages, v_pages, prefix, prefix_len, table, lens, max_len, scale, out, stream)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_k: torch.Tensor, *, cu_q: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v of packed tokens over the states of their
    sequence, all of which each token sees (aie_cross_attn): tokens cu_q[s] ..
    cu_q[s + 1] of q [tokens, heads, head_dim] attend to states cu_k[s] ..
    cu_k[s + 1] of k, v [states, kv_heads, head_dim].  Without cu_q token s is
    sequence s's one token, as in a step of a batch.  cu_q and cu_k are int32
    CUDA tensors [sequences + 1]; they are not copied to the host.  scale
    defaults to head_dim ** -0.5.  A sequence without states gives zeros; tokens
    of no sequence are left as they are in out, undefined without it.  out
    overlaps no input."""
    return _lib.seqcall().cross_attention(q, k, v, cu_k, cu_q, scale, out, stream)


def kv4_file(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor,
             stream=None) -> None:
    """k and v [tokens, kv_heads, head_dim] into a 4-bit cache (aie_kv4_file) at
    slots (int64 [tokens], page * page_size + place; -1 files nothing): groups of
    32 elements with a scale and a lowest value each.  k_pages and v_pages are
    kv[layer, 0] and kv[layer, 1] of ``pages.new_cache4``.  Two tokens with one
    slot leave that place undefined.  Groups with a NaN or an infinity read as
    NaN; finite values count up to 65504."""
    _lib.seqcall().kv4_file(k, v, k_pages, v_pages, slots, stream)


def kv4_load(k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16,
             stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values at slots of a 4-bit cache (aie_kv4_load) as k and v [tokens,
    kv_heads, head_dim]; a slot outside the cache (-1) gives zeros.  A prompt's
    next part attends to its first by prompt_attention over both, the first
    part's keys and values read back and its queries handed in again."""
    return _lib.seqcall().kv4_load(k_pages, v_pages, slots, dtype, stream)


def kv4_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
                  max_len: Optional[int] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """One query token for each of q's streams [batch, heads, head_dim], float16
    or bfloat16, over a 4-bit cache (aie_kv4_attn).  Stream b attends to its
    first lens[b] places (int32 CUDA tensor), in pages table[b, place //
    page_size].  A stream without places gives zeros; what stands behind a
    stream's places never reaches its result.  max_len bounds lens (default: what
    a table row holds); longer streams are cut off there.  out overlaps no input."""
    return _lib.seqcall().kv4_attention(q, k_pages, v_pages, table, lens, max_len, scale, out, stream)
