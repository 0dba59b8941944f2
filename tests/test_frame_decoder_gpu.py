"""A decoder that reads frames: rotation on three axes, a 4-bit cache and
attention to the frames' states together, each call against its plain form in 64
bits on what the decoder hands it."""
import pytest
import torch

from ai_engine_b200 import attention, decoder, pages
from tests import _read, _seq

pytestmark = pytest.mark.gpu


@pytest.fixture
def checked(monkeypatch):
    """Every call of the operators checked as it is made; counts them."""
    count = {}
    real = {name: getattr(attention, name) for name in ("qk_norm_rope", "kv4_file", "kv4_attention", "cross_attention")}

    def rope(q, k, positions, table, **kw):
        half = kw["pair_axis"].shape[0]
        i = torch.arange(half, device="cuda")
        at = positions.long()[:, kw["pair_axis"].long()]
        own = torch.cat([table[at, i], table[at, i + half]], 1)
        rows = torch.arange(q.shape[0], device="cuda")
        want = [_seq.norm_rope(x, kw[w], rows, own, 2 * half, False, 1e-6) for x, w in ((q, "q_weight"), (k, "k_weight"))]
        got = real["qk_norm_rope"](q, k, positions, table, **kw)
        for a, b in zip(got, want):
            _seq.check_norm_rope(a, *b)
        count["qk_norm_rope"] = count.get("qk_norm_rope", 0) + 1
        return got

    def file(k, v, kp, vp, slots):
        real["kv4_file"](k, v, kp, vp, slots)
        for x, y in zip((k, v), attention.kv4_load(kp, vp, slots, dtype=torch.float32)):
            assert torch.equal(y, _read.values(x).float())
        count["kv4_file"] = count.get("kv4_file", 0) + 1

    def one_token(q, kp, vp, table, lens, max_len):
        got = real["kv4_attention"](q, kp, vp, table, lens, max_len=max_len)
        _seq.check(got, *_read.kv4_attend(q, kp, vp, table, lens.tolist()))
        count["kv4_attention"] = count.get("kv4_attention", 0) + 1
        return got

    def cross(q, k, v, cu_k, cu_q):
        got = real["cross_attention"](q, k, v, cu_k, cu_q=cu_q)
        q_lens = cu_q.diff().tolist() if cu_q is not None else [1] * q.shape[0]
        _seq.check(got, *_read.cross(q, k, v, q_lens, cu_k.diff().tolist()))
        count["cross_attention"] = count.get("cross_attention", 0) + 1
        return got

    for name, fn in (("qk_norm_rope", rope), ("kv4_file", file), ("kv4_attention", one_token), ("cross_attention", cross)):
        monkeypatch.setattr(attention, name, fn)
    return count


def _make(dtype, head_dim=64, layers=2):
    m = decoder.FrameDecoder(layers, 96, 4, 2, head_dim, streams=3, pages_=60, page_size=8, max_len=120, dtype=dtype)
    g = torch.Generator("cuda").manual_seed(5)

    def rand(n):
        return torch.randn(n, 96, generator=g, device="cuda").to(dtype)
    m.watch(rand(2 * 45 + 7), [90, 0, 7])  # one stream has no frames
    coarse = decoder.grid(2, 3, 5)
    text = torch.arange(8, 30, dtype=torch.int32, device="cuda")[:, None].expand(-1, 3)
    pos = [torch.cat([coarse, text[:11]]), text[:1], torch.cat([coarse[:15], text[:22]])]
    lens = [p.shape[0] for p in pos]
    return m, rand, torch.cat(pos).contiguous(), lens


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim", [64, 96, 128])
def test_every_call(cuda_ok, checked, dtype, head_dim):
    m, rand, pos, lens = _make(dtype, head_dim)
    m.prompt(rand(sum(lens)), pos, lens)
    for i in range(9):  # past the end of a page
        m.step(rand(3), torch.full((3, 3), 30 + i, dtype=torch.int32, device="cuda"))
    assert m.status() == 0 and m.state.lens.tolist() == [n + 9 for n in lens]
    assert checked == dict(qk_norm_rope=20, kv4_file=20, kv4_attention=18, cross_attention=20)


def test_captured_steps(cuda_ok):
    """A step captured in a graph and replayed goes on as eager steps do."""
    (m, rand, pos, lens), (n, _, _, _) = _make(torch.bfloat16), _make(torch.bfloat16)
    x, s = rand(sum(lens)), rand(3)
    at = torch.full((3, 3), 40, dtype=torch.int32, device="cuda")
    for d in (m, n):
        d.prompt(x, pos, lens)
        d.step(s, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(s, at)
    for _ in range(3):
        graph.replay()
        want = n.step(s, at)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(m.kv, n.kv) and torch.equal(m.state.table, n.state.table)
    del graph


def test_refusals(cuda_ok):
    m, rand, pos, lens = _make(torch.float16)
    with pytest.raises(ValueError):
        m.watch(rand(10), [5, 5])
    with pytest.raises(ValueError):
        m.prompt(rand(sum(lens)), pos, lens[:2])
    fresh = decoder.FrameDecoder(1, 96, 4, 2, 64, streams=3, pages_=60)
    with pytest.raises(ValueError):
        fresh.prompt(rand(sum(lens)), pos, lens)
    with pytest.raises(ValueError):
        fresh.step(rand(3), pos[:3])
    m.prompt(rand(sum(lens)), pos, lens)
    with pytest.raises(ValueError):
        m.prompt(rand(sum(lens)), pos, lens)
    with pytest.raises(ValueError):
        decoder.FrameDecoder(1, 96, 4, 2, 80, streams=3, pages_=60)


def test_cached_prompt_in_parts(cuda_ok):
    """The first part of a prompt read back from the cache in front of the next:
    as attention over those values."""
    size, hk, d, a, b = 16, 2, 64, 37, 12
    kv, st = pages.new_cache4(1, 8, size, hk, d), pages.new_state(8, 1, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(a + b, h, d, generator=g, device="cuda").half() for h in (4, hk, hk))
    slots = pages.grow(st, size, i32([0]), i32([a]), a)
    attention.kv4_file(k[:a], v[:a], kv[0, 0], kv[0, 1], slots)
    ck, cv = attention.kv4_load(kv[0, 0], kv[0, 1], slots, dtype=torch.float16)
    ks, vs = torch.cat([ck, k[a:]]), torch.cat([cv, v[a:]])
    got = attention.prompt_attention(torch.cat([q[:a], q[a:]]), ks, vs, i32([0, a + b]))[a:]
    for h in range(4):
        want, limit = _seq.attend(q[a:, h], ks[:, h // 2], vs[:, h // 2], torch.arange(a + 1, a + b + 1, device="cuda"), d ** -0.5, torch.float16)
        _seq.check(got[:, h], want, limit)
