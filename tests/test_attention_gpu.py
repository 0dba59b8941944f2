"""Norm and rotation, prompt attention and shared-prefix attention against
plain forms in 64 bits."""
import math

import pytest
import torch

from ai_engine_b200 import _lib, attention
from tests import _seq

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dt)


def _table(top, rot, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    a = 100.0 * torch.rand(top, rot // 2, generator=g, device="cuda", dtype=torch.float64)
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


# ------------------------------------------------------- norm, rotation ---

@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("tokens, hq, hk, d, rot, interleaved", [
    (1, 1, 1, 64, 64, False), (7, 8, 2, 128, 128, False), (33, 6, 3, 96, 48, True), (5, 4, 4, 80, 80, False),
    (9, 2, 1, 72, 18, False), (3, 3, 3, 20, 10, True), (130, 16, 4, 128, 64, True), (4, 2, 2, 256, 256, False),
    (2, 5, 5, 512, 510, False), (6, 7, 1, 64, 0, False), (3, 2, 1, 1, 0, False),
])
def test_norm_rope(cuda_ok, dt, tokens, hq, hk, d, rot, interleaved):
    q, k = _rand((tokens, hq, d), dt, 1, 3.0), _rand((tokens, hk, d), dt, 2, 0.5)
    wq, wk = _rand((d,), F32, 3), _rand((d,), F32, 4)
    table = _table(50, rot) if rot else torch.zeros(50, 0, device="cuda")
    pos = torch.randint(0, 50, (tokens,), device="cuda", dtype=torch.int32)
    qo, ko = attention.qk_norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    _seq.check_norm_rope(qo, *_seq.norm_rope(q, wq, pos, table, rot, interleaved, 1e-5))
    _seq.check_norm_rope(ko, *_seq.norm_rope(k, wk, pos, table, rot, interleaved, 1e-5))


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("d, rot, off", [(64, 64, 0), (128, 64, 0), (64, 32, 1), (40, 24, 3)])
def test_norm_rope_views_cache_and_place(cuda_ok, dt, d, rot, off):
    """Views of one buffer, at odd offsets too; results in place; keys and
    values into pages of heads that stand in another order than usual."""
    t, hq, hk, size, n = 19, 4, 2, 8, 5
    raw = _rand((t * (hq + 2 * hk) * d + off,), dt, 5)
    x = raw[off:].view(t, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    wk = _rand((d,), F32, 6)
    pos = torch.arange(t, device="cuda", dtype=torch.int32)
    table = _table(t, rot)
    pages = torch.zeros(2, n, hk, size, d, dtype=dt, device="cuda").transpose(2, 3)  # [.., size, heads, d] views
    slots = torch.randperm(n * size, device="cuda")[:t]
    slots[3], slots[4] = -1, n * size
    wq_, wk_ = _seq.norm_rope(q, None, pos, table, rot, False, 1e-6), _seq.norm_rope(k, wk, pos, table, rot, False, 1e-6)
    v0, rest = v.clone(), pages.clone()
    qo, ko = attention.qk_norm_rope(q, k, pos, table, k_weight=wk, v=v, k_pages=pages[0], v_pages=pages[1], slots=slots,
                                    q_out=q, k_out=k)
    assert qo is q and ko is k
    _seq.check_norm_rope(qo, *wq_)
    _seq.check_norm_rope(ko, *wk_)
    assert torch.equal(v, v0)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < n * size:
            assert torch.equal(pages[0, s // size, s % size], ko[i])
            assert torch.equal(pages[1, s // size, s % size], v[i])
            rest[0, s // size, s % size], rest[1, s // size, s % size] = ko[i], v[i]
    assert torch.equal(pages, rest)
    # into the cache only
    again = torch.zeros_like(pages)
    k2 = _rand((t, hk, d), dt, 9)
    _, none = attention.qk_norm_rope(q, k2, pos, table, k_weight=wk, v=v, k_pages=again[0], v_pages=again[1], slots=slots,
                                     k_out=False)
    want, size_ = _seq.norm_rope(k2, wk, pos, table, rot, False, 1e-6)
    assert none is None
    keep = [i for i, s in enumerate(slots.tolist()) if 0 <= s < n * size]
    at = slots[keep]
    _seq.check_norm_rope(again[0][at // size, at % size], want[keep], size_[keep])


def test_norm_rope_positions_outside_the_table(cuda_ok):
    q, k = _rand((4, 2, 64), F16, 1), _rand((4, 1, 64), F16, 2)
    pos = torch.tensor([0, -1, 10, 9], dtype=torch.int32, device="cuda")
    qo, ko = attention.qk_norm_rope(q, k, pos, _table(10, 32))
    for o in (qo, ko):
        assert torch.isfinite(o[[0, 3]]).all() and torch.isfinite(o[..., 32:]).all()
        assert torch.isnan(o[[1, 2], :, :32]).all()


def test_norm_rope_zero_rows_and_tokens(cuda_ok):
    z = torch.zeros(3, 2, 64, dtype=F16, device="cuda")
    w = torch.ones(64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    qo, ko = attention.qk_norm_rope(z, z, pos, _table(4, 64), q_weight=w, k_weight=w)
    assert not qo.any() and not ko.any()
    qo, ko = attention.qk_norm_rope(z[:0], z[:0], pos[:0], _table(4, 64), q_weight=w, k_weight=w)
    assert qo.shape == (0, 2, 64)


def test_norm_rope_refuses(cuda_ok):
    q, k = _rand((3, 4, 64), F16, 1), _rand((3, 2, 64), F16, 2)
    pos, table = torch.zeros(3, dtype=torch.int32, device="cuda"), _table(4, 64)
    call = attention.qk_norm_rope
    with pytest.raises(TypeError):
        call(q, k.float(), pos, table)
    with pytest.raises(TypeError):
        call(q, k, pos.long(), table)
    with pytest.raises(TypeError):
        call(q, k, pos, table.double())
    with pytest.raises(ValueError):
        call(q, k[:2], pos, table)
    with pytest.raises(ValueError):
        call(q, k, pos[:2], table)
    with pytest.raises(ValueError):
        call(q, k, pos, table, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        call(q, k, pos, table, k_out=False)
    with pytest.raises(ValueError):
        call(q.transpose(1, 2), k.transpose(1, 2), pos, table)
    with pytest.raises(ValueError):
        call(q, k, pos, table, k_pages=torch.zeros(2, 8, 2, 64, dtype=F16, device="cuda"))
    with pytest.raises(_lib.AieError):
        call(q, _rand((3, 3, 64), F16, 2), pos, table)


# ------------------------------------------------------ prompt attention ---

def _prompt_want(q, k, v, lens, causal, scale):
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lim = torch.zeros_like(out)
    g, at = q.shape[1] // k.shape[1], 0
    for n in lens:
        seen = torch.arange(1, n + 1, device="cuda") if causal else torch.full((n,), n, device="cuda")
        for h in range(q.shape[1]):
            out[at:at + n, h], lim[at:at + n, h] = _seq.attend(q[at:at + n, h], k[at:at + n, h // g], v[at:at + n, h // g],
                                                               seen, scale, q.dtype)
        at += n
    return out, lim


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


PROMPTS = [
    ([1], 1, 1, 64), ([5], 4, 4, 64), ([128], 2, 1, 64), ([129, 127], 2, 2, 128), ([256], 8, 2, 128),
    ([0, 3, 0, 200, 1, 0], 6, 2, 64), ([700], 8, 1, 128), ([130, 64, 513], 12, 4, 80), ([300], 20, 4, 128),
    ([33, 1000], 7, 1, 96), ([257], 3, 3, 40), ([1, 1, 1, 2], 16, 1, 64), ([90], 64, 1, 64), ([77, 140], 32, 2, 8),
    ([1500], 4, 2, 64), ([40], 130, 1, 64), ([65, 3], 2, 2, 256), ([50], 6, 2, 68),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens, hq, hk, d", PROMPTS)
def test_prompt(cuda_ok, lens, hq, hk, d, dt, causal):
    t = sum(lens)
    x = _rand((t, hq + 2 * hk, d), dt, 10 + t, 1.5)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    got = attention.prompt_attention(q, k, v, _cu(lens), causal=causal)
    _seq.check(got, *_prompt_want(q, k, v, lens, causal, d ** -0.5))


@pytest.mark.parametrize("n, hq, hk, d", [(31, 4, 2, 64), (128, 2, 1, 64), (129, 4, 4, 128), (300, 8, 2, 64)])
def test_prompt_many_sequences(cuda_ok, n, hq, hk, d):
    lens = [(i * 37) % 90 if i % 5 else 0 for i in range(n)]
    x = _rand((sum(lens), hq + 2 * hk, d), F16, n)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    _seq.check(attention.prompt_attention(q, k, v, _cu(lens)), *_prompt_want(q, k, v, lens, True, d ** -0.5))


def test_prompt_broadcast_values_and_starts_out_of_range(cuda_ok):
    """Values expanded over heads (stride 0); entries of cu outside the tokens are cut to them."""
    t, d = 90, 64
    q, k = _rand((t, 4, d), F16, 1), _rand((t, 4, d), F16, 2)
    v = _rand((t, 1, d), F16, 3).expand(t, 4, d)
    _seq.check(attention.prompt_attention(q, k, v, _cu([t])), *_prompt_want(q, k, v, [t], True, d ** -0.5))
    out = torch.full_like(q, 5.0)
    cu = torch.tensor([-7, 40, 2000], dtype=torch.int32, device="cuda")
    attention.prompt_attention(q, k, k, cu, out=out)
    _seq.check(out, *_prompt_want(q, k, k, [40, 50], True, d ** -0.5))


@pytest.mark.parametrize("lens, hq, hk, d", [([70, 3], 4, 2, 64), ([33], 3, 1, 24), ([9, 9], 2, 2, 256)])
def test_prompt_f32(cuda_ok, lens, hq, hk, d):
    t = sum(lens)
    q, k, v = _rand((t, hq, d), F32, 1), _rand((t, hk, d), F32, 2), _rand((t, hk, d), F32, 3)
    got = attention.prompt_attention(q, k, v, _cu(lens), scale=0.3)
    _seq.check(got, *_prompt_want(q, k, v, lens, True, 0.3))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_prompt_steep_scores(cuda_ok, dt):
    """Scores of a wide range whose maximum keeps growing along the keys: the
    running maximum moves in every tile; and a large negative scale."""
    t, d = 900, 64
    q, v = _rand((t, 2, d), dt, 1, 1.0), _rand((t, 1, d), dt, 3)
    k = (_rand((t, 1, d), F32, 2, 0.2) + torch.linspace(0, 2.0, t, device="cuda")[:, None, None] * q[-1:, :1].float()).to(dt)
    for scale in (1.0, -0.7):
        got = attention.prompt_attention(q, k, v, _cu([t]), causal=False, scale=scale)
        _seq.check(got, *_prompt_want(q, k, v, [t], False, scale))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_neighbours_do_not_leak(cuda_ok, dt, causal):
    """Infinities and NaN in the sequences around, and behind the packed
    tokens, reach nothing; the first tokens of a causal sequence do not see
    keys behind them that are not finite."""
    lens, hq, hk, d = [37, 101, 50], 4, 2, 64
    t = sum(lens)
    x = _rand((t + 60, hq + 2 * hk, d), dt, 3)
    x[:37], x[138:] = math.nan, math.inf
    q, k, v = x[:t, :hq], x[:t, hq:hq + hk], x[:t, hq + hk:]
    got = attention.prompt_attention(q, k, v, _cu(lens), causal=causal)
    want, lim = _prompt_want(q[37:138], k[37:138], v[37:138], [101], causal, d ** -0.5)
    _seq.check(got[37:138], want, lim)
    if causal:
        k2 = k.clone()
        k2[37 + 90:138] = math.nan
        got = attention.prompt_attention(q, k2, v, _cu(lens))
        _seq.check(got[37:127], want[:90], lim[:90])
        assert torch.isnan(got[127:138]).all()


def test_prompt_masked_scores_of_minus_infinity(cuda_ok):
    """Keys whose scores are -inf carry no weight; a row of such scores alone is NaN, as the formula says."""
    t, d = 200, 64
    q = torch.ones(t, 1, d, dtype=F16, device="cuda")
    k, v = _rand((t, 1, d), F16, 2, 0.1), _rand((t, 1, d), F16, 3)
    k[:150, :, 0] = -math.inf
    got = attention.prompt_attention(q, k, v, _cu([t]))
    assert torch.isnan(got[:150]).all()
    k2 = k.clone()
    k2[:150] = 0
    s = (q[150:, 0].double() @ k2[:, 0].double().T) / 8.0
    mask = (torch.arange(t, device="cuda") >= 150) & (torch.arange(t, device="cuda") <= torch.arange(150, t, device="cuda")[:, None])
    w = torch.softmax(torch.where(mask, s, -math.inf), -1)
    err = (got[150:, 0].double() - w @ v[:, 0].double()).abs().max()
    assert err <= 2 * 2.0 ** -11 * float(v.abs().max())


def test_prompt_tokens_outside_are_left(cuda_ok):
    q = _rand((50, 2, 64), F16, 1)
    out = torch.full_like(q, 7.0)
    cu = torch.tensor([10, 30, 30, 41], dtype=torch.int32, device="cuda")
    attention.prompt_attention(q, q, q, cu, out=out)
    assert (out[:10] == 7).all() and (out[41:] == 7).all()
    _seq.check(out[10:41], *_prompt_want(q[10:41], q[10:41], q[10:41], [20, 11], True, 0.125))


@pytest.mark.parametrize("d, off", [(64, 0), (128, 0), (64, 3), (36, 0)])
def test_prompt_layouts(cuda_ok, d, off):
    """Head-major and token-major memory, odd offsets, a strided output."""
    t, hq, hk = 150, 6, 2
    base = _rand(((hq + 2 * hk) * t * d + off,), BF16, 4)[off:].view(hq + 2 * hk, t, d).transpose(0, 1)
    q, k, v = base[:, :hq], base[:, hq:hq + hk], base[:, hq + hk:]
    wide = torch.zeros(t, 2 * hq, d + 4 if off else d, dtype=BF16, device="cuda")
    out = wide[:, ::2, :d]
    got = attention.prompt_attention(q, k, v, _cu([t]), out=out)
    assert got is out and not wide[:, 1::2].any()
    _seq.check(got.contiguous(), *_prompt_want(q, k, v, [t], True, d ** -0.5))


def test_prompt_repeats_and_other_stream(cuda_ok):
    q = _rand((800, 8, 128), BF16, 1)
    k, v = _rand((800, 2, 128), BF16, 2), _rand((800, 2, 128), BF16, 3)
    cu = _cu([300, 500])
    a = attention.prompt_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = attention.prompt_attention(q, k, v, cu, stream=s)
    s.synchronize()
    assert torch.equal(a, b) and torch.equal(a, attention.prompt_attention(q, k, v, cu))


def test_prompt_refuses(cuda_ok):
    q = _rand((10, 4, 64), F16, 1)
    cu = _cu([10])
    with pytest.raises(TypeError):
        attention.prompt_attention(q, q.float(), q, cu)
    with pytest.raises(TypeError):
        attention.prompt_attention(q, q, q, cu.long())
    with pytest.raises(TypeError):
        attention.prompt_attention(q.double(), q.double(), q.double(), cu)
    with pytest.raises(ValueError):
        attention.prompt_attention(q, q[:5], q[:5], cu)
    with pytest.raises(ValueError):
        attention.prompt_attention(q, q, q[:, :2], cu)
    with pytest.raises(ValueError):
        attention.prompt_attention(q, q, q, cu, out=q[:3])
    with pytest.raises(_lib.AieError):
        attention.prompt_attention(q, q[:, :3], q[:, :3], cu)


# ------------------------------------------------------ prefix attention ---

def _prefix_case(b, hq, hk, d, size, shared, lens, dt, seed, head_major=False):
    """A cache of randomly ordered pages; what no stream holds is NaN."""
    whole, npre = shared // size, -(-shared // size)
    top = max(max(lens), shared, 1)
    width = -(-top // size) + 1
    n = npre + b * (width - whole) + 3
    shape = (2, n, hk, size, d) if head_major else (2, n, size, hk, d)
    kv = torch.full(shape, math.nan, dtype=dt, device="cuda")
    if head_major:
        kv = kv.transpose(2, 3)
    data = _rand((2, n, size, hk, d), dt, seed, 1.2)
    order = torch.randperm(n, device="cuda").to(torch.int32)
    prefix, table = order[:npre].contiguous(), torch.full((b, width), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, whole:] = order[npre:npre + b * (width - whole)].view(b, -1)
    for p in range(npre):
        used = min(size, shared - p * size)
        kv[:, prefix[p], :used] = data[:, prefix[p], :used]
    for i, m in enumerate(lens):
        for p in range(whole, -(-m // size)):
            lo, hi = max(shared - p * size, 0), min(size, m - p * size)
            if hi > lo:
                kv[:, table[i, p], lo:hi] = data[:, table[i, p], lo:hi]
    q = _rand((b, hq, d), dt, seed + 1, 1.2)
    return q, kv, prefix, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _prefix_want(q, kv, prefix, table, lens, shared, scale):
    b, hq, d = q.shape
    size, hk = kv.shape[2], kv.shape[3]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lim = torch.zeros_like(out)
    for i, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        j = torch.arange(n, device="cuda")
        row = table[i].long()
        page = torch.where(j < shared, prefix.long()[(j // size).clamp(max=max(prefix.numel() - 1, 0))] if prefix.numel()
                           else row[j // size], row[j // size])
        k, v = kv[0][page, j % size], kv[1][page, j % size]
        for h in range(hq):
            out[i, h:h + 1], lim[i, h:h + 1] = _seq.attend(q[i, h:h + 1], k[:, h * hk // hq], v[:, h * hk // hq],
                                                           torch.tensor([n], device="cuda"), scale, q.dtype)
    return out, lim


PREFIXES = [  # batch, q heads, kv heads, head size, page size, shared places, each stream's places
    (1, 1, 1, 64, 16, 0, [1]), (1, 4, 2, 64, 16, 5, [5]), (3, 8, 2, 128, 16, 100, [100, 101, 140]),
    (4, 8, 8, 64, 32, 64, [64, 65, 300, 96]), (5, 6, 2, 128, 16, 37, [0, 12, 37, 38, 90]),
    (2, 16, 1, 128, 64, 1000, [1000, 1200]), (3, 7, 7, 80, 8, 0, [0, 200, 17]), (9, 32, 4, 128, 16, 300, [300 + 41 * i for i in range(9)]),
    (40, 8, 1, 64, 16, 257, [257 + (i * 13) % 50 for i in range(40)]), (2, 20, 4, 96, 128, 130, [130, 700]),
    (3, 4, 2, 64, 24, 50, [50, 80, 55]), (2, 3, 1, 36, 16, 20, [33, 20]), (2, 130, 1, 64, 16, 40, [60, 41]),
    (2, 2, 1, 256, 16, 40, [60, 41]), (130, 4, 2, 64, 16, 48, [48 + i % 3 for i in range(130)]),
    (2, 8, 2, 64, 256, 300, [900, 301]), (1, 8, 2, 128, 16, 0, [5000]), (2, 24, 1, 128, 16, 30, [2000, 31]),
]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("b, hq, hk, d, size, shared, lens", PREFIXES)
def test_prefix(cuda_ok, b, hq, hk, d, size, shared, lens, dt):
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, dt, 3)
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    _seq.check(got, *_prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5))


@pytest.mark.parametrize("b, hq, hk, d, size, shared, lens", [PREFIXES[4], PREFIXES[2]])
def test_prefix_f32_and_scale(cuda_ok, b, hq, hk, d, size, shared, lens):
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, F32, 3)
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln, scale=0.5)
    _seq.check(got, *_prefix_want(q, kv, prefix, table, ln, shared, 0.5))


def test_prefix_layouts(cuda_ok):
    """Head-major pages, strided queries and outputs, a bound on the lengths."""
    b, hq, hk, d, size, shared = 6, 8, 2, 64, 16, 70
    lens = [70, 75, 200, 3, 0, 90]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, BF16, 8, head_major=True)
    wide = torch.zeros(b, 2 * hq, d, dtype=BF16, device="cuda")
    qq = wide.clone()[:, ::2]
    qq.copy_(q)
    got = attention.prefix_attention(qq, kv[0], kv[1], prefix, shared, table, ln, max_len=120, out=wide[:, 1::2])
    assert not wide[:, ::2].any()
    _seq.check(got.contiguous(), *_prefix_want(q, kv, prefix, table, ln.clamp(max=120), shared, d ** -0.5))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_prefix_equals_no_prefix(cuda_ok, dt):
    """The same contexts, with and without the shared part named."""
    b, hq, hk, d, size, shared = 12, 16, 4, 128, 16, 320
    lens = [320 + 17 * i for i in range(b)]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, dt, 5)
    table[:, : shared // size] = prefix
    one = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    two = attention.prefix_attention(q, kv[0], kv[1], None, 0, table, ln)
    want, lim = _prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5)
    _seq.check(one, want, lim)
    _seq.check(two, want, lim)


def test_prefix_steep_scores(cuda_ok):
    """The largest score in the shared part, in the own part, or in neither by much."""
    b, hq, hk, d, size, shared = 3, 4, 1, 64, 16, 400
    lens = [700, 700, 700]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, BF16, 5)
    kv[0, prefix[3], 2] = (8 * q[0, :1].float()).to(BF16)
    kv[0, table[1, shared // size + 5], 2] = (8 * q[1, :1].float()).to(BF16)
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    _seq.check(got, *_prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5))


def test_prefix_bad_pages_are_not_followed(cuda_ok):
    """Page numbers outside the cache spoil their own stream's result only."""
    b, hq, hk, d, size, shared = 4, 4, 2, 64, 16, 32
    lens = [100, 100, 100, 100]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, F16, 5)
    want, lim = _prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5)
    table[1, 4], table[1, 5] = -7, 2 ** 31 - 1
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    keep = [0, 2, 3]
    _seq.check(got[keep], want[keep], lim[keep])


def test_prefix_in_a_graph_and_repeatable(cuda_ok):
    """Captured once, replayed with other lengths and queries; bit for bit the direct call's."""
    b, hq, hk, d, size, shared = 8, 16, 2, 128, 16, 500
    lens = [500 + 90 * i for i in range(b)]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, BF16, 5)
    attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    for k in range(2):
        q.copy_(_rand(q.shape, BF16, 20 + k))
        ln.copy_(torch.tensor([n - 11 * k for n in lens]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln))
    _seq.check(out, *_prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5))


def test_prefix_refuses(cuda_ok):
    q, kv, prefix, table, ln = _prefix_case(2, 4, 2, 64, 16, 20, [30, 25], F16, 1)
    call = attention.prefix_attention
    with pytest.raises(TypeError):
        call(q, kv[0].float(), kv[1].float(), prefix, 20, table, ln)
    with pytest.raises(TypeError):
        call(q, kv[0], kv[1], prefix.long(), 20, table, ln)
    with pytest.raises(TypeError):
        call(q, kv[0], kv[1], prefix, 20, table, ln.long())
    with pytest.raises(ValueError):
        call(q, kv[0], kv[1], prefix, 33, table, ln)
    with pytest.raises(ValueError):
        call(q, kv[0], kv[1], prefix, -1, table, ln)
    with pytest.raises(ValueError):
        call(q, kv[0], kv[1], prefix, 20, table[:1], ln)
    with pytest.raises(ValueError):
        call(q, kv[0], kv[1, :, :8], prefix, 20, table, ln)
    with pytest.raises(_lib.AieError):
        call(q, kv[0], kv[1], prefix, 20, table, ln, max_len=1000)
    with pytest.raises(_lib.AieError):
        call(q[:, :3], kv[0], kv[1], prefix, 20, table, ln)
