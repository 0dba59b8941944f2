"""The sequence operators together: prompt, forks, steps, ended streams and
compaction against the same decoder in plain 64-bit torch over lists of
keys and values."""
import math

import pytest
import torch

from ai_engine_b200.decoder import StreamDecoder

pytestmark = pytest.mark.gpu


class Plain:
    """The same layers in 64 bits on the same weights; a cache is a list of keys and values per row."""

    def __init__(self, m):
        self.m, self.rows = m, {}

    def _heads(self, i, x, pos):
        m = self.m
        q, k, v = (x @ m.wqkv[i].double()).view(x.shape[0], -1, m.d).split([m.hq, m.hk, m.hk], 1)
        half, cs = m.d // 2, m.table[pos].double()[:, None]

        def turn(y, w):
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            a, b, c, s = y[..., :half], y[..., half:], cs[..., :half], cs[..., half:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        return turn(q, m.norms[i][0]), turn(k, m.norms[i][1]), v

    def run(self, row, x, causal_from):
        """Tokens x of one row behind what it holds."""
        m = self.m
        cache = self.rows.setdefault(row, [(torch.zeros(0, m.hk, m.d, dtype=torch.float64, device="cuda"),) * 2
                                           for _ in m.wqkv])
        pos = torch.arange(causal_from, causal_from + x.shape[0], device="cuda")
        for i in range(len(m.wqkv)):
            q, k, v = self._heads(i, x, pos)
            cache[i] = tuple(torch.cat(p) for p in zip(cache[i], (k, v)))
            kk, vv = (t.repeat_interleave(m.hq // m.hk, 1).transpose(0, 1) for t in cache[i])
            s = q.transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(m.d)
            s = s.masked_fill(torch.arange(kk.shape[1], device="cuda") > pos[:, None], -math.inf)
            o = (torch.softmax(s, -1) @ vv).transpose(0, 1).reshape(x.shape[0], -1)
            x = x + o @ m.wo[i].double()
        return x


def _near(got, want, layers):
    # each layer rounds its projections, heads, weights and sum a few times to
    # f16 (2^-11): under 16 roundings a layer, adding up as independent ones do
    err = float((got.double() - want).norm() / want.norm())
    assert err <= 16 * layers * 2.0 ** -11, err


def test_streams_behind_one_prompt(cuda_ok):
    layers, streams = 3, 5
    m = StreamDecoder(layers, 192, 6, 2, 64, streams=streams, pages_=40, max_len=200, dtype=torch.float16)
    p = Plain(m)
    g = torch.Generator("cuda").manual_seed(3)

    def feats(n):
        return torch.randn(n, 192, generator=g, device="cuda").half()
    x = feats(77)  # ends inside a page
    _near(m.prompt(x), p.run(0, x.double(), 0), layers)
    rows = [1, 2, 3, 4, 5]
    m.fork(rows)
    for r in rows:
        p.rows[r] = list(p.rows[0])
    length = {r: 77 for r in rows}

    def step(rows):
        x = feats(len(rows))
        want = torch.cat([p.run(r, x[i:i + 1].double(), length[r]) for i, r in enumerate(rows)])
        for r in rows:
            length[r] += 1
        _near(m.step(rows, x), want, layers)
    for _ in range(5):
        step(rows)
    step([4, 2])  # some streams only, in another order
    m.end([1, 3])
    for _ in range(20):
        step([5, 2, 4])
    m.fork([3])  # a place that was given back
    p.rows[3] = list(p.rows[0])
    length[3] = 77
    step([2, 3])
    used = sum(-(-length[r] // 16) for r in (2, 3, 4, 5)) - 4 * (77 // 16) + -(-77 // 16)
    assert m.status() == 0 and int((m.state.refs > 0).sum()) == used
    assert m.state.lens.tolist() == [77, 0] + [length[r] for r in (2, 3, 4, 5)]


def test_command(cuda_ok, capsys):
    from ai_engine_b200 import decoder
    decoder.main(["3", "40", "4"])
    assert "status 0" in capsys.readouterr().out


def test_calls_see_what_the_last_one_wrote(cuda_ok):
    """Launches are set up while the last one runs: chains of calls, each on the
    last one's results, with and without a wait between them."""
    from ai_engine_b200 import attention, pages
    kv = pages.new_cache(2, 40, 16, 2, 64, torch.float16)
    kv[:, :, 0] = torch.randn(2, 2, 16, 2, 64, device="cuda").half()
    at = torch.arange(40, dtype=torch.int32, device="cuda")
    for i in range(39):
        pages.copy(kv, at[i:i + 1], at[i + 1:i + 2])
    assert bool((kv == kv[:, :, :1]).all())

    def chain(wait):
        g = torch.Generator("cuda").manual_seed(1)
        q = torch.randn(300, 4, 64, generator=g, device="cuda").half()
        pos, table = torch.arange(300, dtype=torch.int32, device="cuda"), torch.randn(300, 64, generator=g, device="cuda")
        w, cu = torch.ones(64, device="cuda"), torch.tensor([0, 120, 300], dtype=torch.int32, device="cuda")
        cache = pages.new_cache(1, 20, 16, 4, 64, torch.float16)
        rows = torch.arange(19, dtype=torch.int32, device="cuda")[None]
        for _ in range(12):
            k = torch.empty_like(q)
            attention.qk_norm_rope(q, q, pos, table, q_weight=w, k_weight=w, v=q, k_pages=cache[0, 0], v_pages=cache[0, 1],
                                   slots=torch.arange(300, device="cuda"), q_out=k, k_out=False)
            q = attention.prompt_attention(k, k, q, cu)
            one = attention.prefix_attention(q[-1:], cache[0, 0], cache[0, 1], rows[0], 200, rows, pos[-1:])
            q = torch.cat([q[:-1], one])
            if wait:
                torch.cuda.synchronize()
        return q
    assert torch.equal(chain(False), chain(True))
