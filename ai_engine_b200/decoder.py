"""A small attention decoder over frame features: many streams behind one prompt.

What the sequence operators look like in use.  A prompt (features of an
instruction, or of a reference clip) is attended once and filed into the
cache; every stream forks from it; each step attends one new token per stream
to the shared prompt and the stream's own past; ended streams give their
pages back.  Projections are plain matrix products; everything else of a
layer is ``attention`` and ``pages``.

    python -m ai_engine_b200.decoder [streams] [prompt tokens] [steps]
"""
from __future__ import annotations

import sys
from typing import List, Sequence

import torch

from . import attention, pages


def angles(positions: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """The [positions, rot_dim] table of cosines, then sines, that qk_norm_rope takes."""
    f = base ** (-torch.arange(rot_dim // 2, dtype=torch.float64, device=device) / (rot_dim // 2))
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


class StreamDecoder:
    """Layers of x += attention(x) wo over a paged cache.  Row 0 of the cache
    holds the prompt, rows 1 .. streams the streams forked from it.  A row
    holds up to max_len tokens, rounded up to whole pages."""

    def __init__(self, layers: int, dim: int, q_heads: int, kv_heads: int, head_dim: int, *, streams: int, pages_: int,
                 page_size: int = 16, max_len: int = 4096, dtype=torch.bfloat16, device="cuda", seed: int = 0):
        self.dim, self.hq, self.hk, self.d = dim, q_heads, kv_heads, head_dim
        width = -(-max_len // page_size)
        self.page_size, self.max_len, self.dtype, self.device = page_size, width * page_size, dtype, torch.device(device)
        g = torch.Generator(device).manual_seed(seed)
        heads = (q_heads + 2 * kv_heads) * head_dim

        def weight(*shape):
            return (torch.randn(shape, generator=g, device=device) * shape[0] ** -0.5).to(dtype)
        self.wqkv = [weight(dim, heads) for _ in range(layers)]
        self.wo = [weight(q_heads * head_dim, dim) for _ in range(layers)]
        self.norms = [1.0 + 0.1 * torch.randn(2, head_dim, generator=g, device=device) for _ in range(layers)]
        self.table = angles(self.max_len, head_dim, device=device)
        self.kv = pages.new_cache(layers, pages_, page_size, kv_heads, head_dim, dtype, device)
        self.state = pages.new_state(pages_, streams + 1, width, device)
        self.prompt_len, self.live = 0, set()  # rows that hold tokens

    def _int(self, x) -> torch.Tensor:
        return torch.as_tensor(x, dtype=torch.int32, device=self.device)

    def _layer(self, i: int, x: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, keep_k: bool):
        """Projected, normed and rotated heads of a layer, keys and values filed."""
        qkv = (x @ self.wqkv[i]).view(x.shape[0], self.hq + 2 * self.hk, self.d)
        q, k, v = qkv.split([self.hq, self.hk, self.hk], 1)
        q, k = attention.qk_norm_rope(q, k, positions, self.table, q_weight=self.norms[i][0], k_weight=self.norms[i][1], v=v,
                                      k_pages=self.kv[i, 0], v_pages=self.kv[i, 1], slots=slots, q_out=q,
                                      k_out=k if keep_k else False)
        return q, k, v

    def _out(self, i: int, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
        return x + o.reshape(x.shape[0], -1) @ self.wo[i]

    def prompt(self, x: torch.Tensor) -> torch.Tensor:
        """The prompt's features [tokens, dim] through the layers and into row 0,
        which is empty, as all rows are."""
        if self.prompt_len or self.live:
            raise ValueError("rows hold a prompt or streams: end them first")
        t = x.shape[0]
        slots = pages.grow(self.state, self.page_size, self._int([0]), self._int([t]), t)
        positions, cu = torch.arange(t, dtype=torch.int32, device=self.device), self._int([0, t])
        for i in range(len(self.wqkv)):
            q, k, v = self._layer(i, x, positions, slots, True)
            x = self._out(i, x, attention.prompt_attention(q, k, v, cu))
        self.prompt_len = t
        return x

    def fork(self, rows: Sequence[int]) -> None:
        """The rows become streams that have seen the prompt."""
        if self.prompt_len:
            self.live.update(rows)
        pages.fork(self.kv, self.state, self._int([0] * len(rows)), self._int(list(rows)))

    def step(self, rows: Sequence[int], x: torch.Tensor) -> torch.Tensor:
        """One token for each of the rows [rows, dim]."""
        self.live.update(rows)
        r = self._int(list(rows))
        at = r.long()
        positions = self.state.lens[at]
        slots = pages.grow(self.state, self.page_size, r, torch.ones_like(r), len(rows))
        table, lens = self.state.table[at], self.state.lens[at]
        for i in range(len(self.wqkv)):
            q, _, _ = self._layer(i, x, positions, slots, False)
            x = self._out(i, x, attention.prefix_attention(q, self.kv[i, 0], self.kv[i, 1], self.state.table[0],
                                                           self.prompt_len, table, lens, max_len=self.max_len))
        return x

    def end(self, rows: Sequence[int], compact: bool = True) -> None:
        """The rows' streams end; the pages in use move to the front of the cache.
        Streams outlive the prompt's row: from then on each goes by its own."""
        self.live.difference_update(rows)
        if 0 in rows:
            self.prompt_len = 0
        pages.free(self.state, self._int(list(rows)))
        if compact:
            pages.compact(self.kv, self.state)

    def status(self) -> int:
        """What the cache's calls could not do (waits for the device)."""
        return int(self.state.status.item())


def main(argv: List[str]) -> None:
    streams, prompt, steps = (int(v) for v in (argv + ["32", "2000", "64"][len(argv):]))
    need = -(-prompt // 16) + streams * (steps // 16 + 2) + 8
    m = StreamDecoder(4, 1024, 16, 4, 128, streams=streams, pages_=need, max_len=prompt + steps + 1)
    g = torch.Generator("cuda").manual_seed(1)
    m.prompt(torch.randn(prompt, 1024, generator=g, device="cuda").bfloat16())
    rows = list(range(1, streams + 1))
    m.fork(rows)
    x = torch.randn(streams, 1024, generator=g, device="cuda").bfloat16()
    m.step(rows, x)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(steps - 1):
        x = m.step(rows, x)
    b.record()
    b.synchronize()
    m.end(rows[::2])
    used = int((m.state.refs > 0).sum())
    print(f"{streams} streams behind {prompt} tokens: {a.elapsed_time(b) / max(1, steps - 1) * 1e3:.0f} us a step of 4 layers; "
          f"{used} of {need} pages in use after half of them ended; status {m.status()}")


if __name__ == "__main__":
    main(sys.argv[1:])
