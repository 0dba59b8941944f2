"""Attention of tokens to states of another length against the plain form in 64
bits."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _read, _seq

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dt)


def _inputs(q_lens, k_lens, hq, hk, d, dt, seed=1):
    q = _rand((sum(q_lens), hq, d), dt, seed, 2.0)
    kv = _rand((sum(k_lens), 2, hk, d), dt, seed + 1)
    return q, kv[:, 0], kv[:, 1]


HEADS = [(4, 4, 64, F16), (8, 2, 128, BF16), (6, 1, 80, F16), (5, 5, 32, BF16), (3, 3, 128, F32), (7, 1, 20, F32), (16, 1, 64, BF16),
         (20, 1, 128, F16), (4, 2, 256, BF16), (12, 1, 192, F16), (9, 3, 96, F16), (40, 2, 64, F16), (2, 1, 72, BF16)]


@pytest.mark.parametrize("hq, hk, d, dt", HEADS)
@pytest.mark.parametrize("k_lens", [[1], [180, 180, 180], [5, 0, 33, 1, 16, 17, 0, 700], [2000], [0, 0]])
def test_one_token_each(cuda_ok, hq, hk, d, dt, k_lens):
    q, k, v = _inputs([1] * len(k_lens), k_lens, hq, hk, d, dt)
    got = attention.cross_attention(q, k, v, _read.starts(k_lens))
    _seq.check(got, *_read.cross(q, k, v, [1] * len(k_lens), k_lens))


@pytest.mark.parametrize("hq, hk, d, dt", HEADS)
@pytest.mark.parametrize("q_lens, k_lens", [
    ([1], [1]), ([3, 0, 40], [7, 9, 0]), ([130, 1], [127, 1300]), ([0, 2, 300], [5, 2500, 129]), ([65, 66, 67], [128, 256, 1])])
def test_packed_tokens(cuda_ok, hq, hk, d, dt, q_lens, k_lens):
    q, k, v = _inputs(q_lens, k_lens, hq, hk, d, dt)
    got = attention.cross_attention(q, k, v, _read.starts(k_lens), cu_q=_read.starts(q_lens))
    _seq.check(got, *_read.cross(q, k, v, q_lens, k_lens))


@pytest.mark.parametrize("seqs", [129, 700])
@pytest.mark.parametrize("each", [False, True])
def test_many_sequences(cuda_ok, seqs, each):
    k_lens = [(i * 37) % 50 for i in range(seqs)]
    q_lens = [1] * seqs if each else [(i * 11) % 4 for i in range(seqs)]
    q, k, v = _inputs(q_lens, k_lens, 8, 2, 64, F16)
    got = attention.cross_attention(q, k, v, _read.starts(k_lens), cu_q=None if each else _read.starts(q_lens))
    _seq.check(got, *_read.cross(q, k, v, q_lens, k_lens))


@pytest.mark.parametrize("q_lens, k_lens", [([1], [40000]), ([20], [40000]), ([1, 1, 1], [30000, 0, 5])])
def test_long_states(cuda_ok, q_lens, k_lens):
    for cu_q in (None, _read.starts(q_lens)) if max(q_lens) == 1 else (_read.starts(q_lens),):
        q, k, v = _inputs(q_lens, k_lens, 8, 2, 128, BF16)
        _seq.check(attention.cross_attention(q, k, v, _read.starts(k_lens), cu_q=cu_q), *_read.cross(q, k, v, q_lens, k_lens))


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("each", [False, True])
def test_others_values_and_rows_outside(cuda_ok, dt, each):
    """States of no sequence and of others, NaN and infinities too, reach no
    result; tokens of no sequence stay as they are."""
    q_lens, k_lens = ([1, 1, 1], [30, 0, 70]) if each else ([5, 3, 9], [30, 0, 70])
    t, n = sum(q_lens), 130
    q, kv = _rand((t + 4, 8, 64), dt, 1), _rand((n, 2, 2, 64), dt, 2)
    k, v = kv[:, 0].clone(), kv[:, 1].clone()
    k[5 + 100:], v[5 + 100:] = float("nan"), float("inf")
    k[:5], v[:5] = float("inf"), float("nan")
    cu_k = _read.starts(k_lens) + 5
    want, limit = _read.cross(q[2:2 + t], k[5:105], v[5:105], q_lens, k_lens)
    if each:
        got = attention.cross_attention(q[2:2 + t], k, v, cu_k)
    else:
        out = torch.full_like(q, 7.0)
        attention.cross_attention(q, k, v, cu_k, cu_q=_read.starts(q_lens) + 2, out=out)
        assert bool((out[:2] == 7).all()) and bool((out[2 + t:] == 7).all())
        got = out[2:2 + t]
    _seq.check(got, want, limit)
    # a sequence's own NaN reaches its own tokens, no others
    v[5] = float("nan")
    cu_q = None if each else _read.starts(q_lens) + 2
    got = attention.cross_attention(q[2:2 + t] if each else q, k, v, cu_k, cu_q=cu_q)
    got = got if each else got[2:2 + t]
    assert bool(torch.isnan(got[:q_lens[0]]).all())
    _seq.check(got[q_lens[0]:], want[q_lens[0]:], limit[q_lens[0]:])


@pytest.mark.parametrize("dt, off", [(F16, 0), (F16, 1), (BF16, 8)])
@pytest.mark.parametrize("each", [False, True])
def test_views(cuda_ok, dt, off, each):
    """Views at odd offsets, heads in another order, a broadcast head, results into a view."""
    q_lens, k_lens = ([1] * 3, [40, 3, 90]) if each else ([10, 1, 4], [40, 3, 90])
    t, n, d = sum(q_lens), sum(k_lens), 64
    q = _rand((8 * t * d + off,), dt, 1)[off:].view(8, t, d).transpose(0, 1)
    k = _rand((2 * n * d + off,), dt, 2)[off:].view(2, n, d).transpose(0, 1)
    v = _rand((n * d + off,), dt, 3)[off:].view(n, 1, d).expand(n, 2, d)
    out = torch.full((t, 3, 8, d), 5.0, dtype=dt, device="cuda")
    cu_q = None if each else _read.starts(q_lens)
    attention.cross_attention(q, k, v, _read.starts(k_lens), cu_q=cu_q, out=out[:, 1])
    _seq.check(out[:, 1].contiguous(), *_read.cross(q, k, v, q_lens, k_lens))
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 2] == 5).all())


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-3])
@pytest.mark.parametrize("each", [False, True])
def test_scales(cuda_ok, dt, scale, each):
    q_lens, k_lens = ([1] * 2, [300, 70]) if each else ([20, 7], [300, 70])
    q, k, v = _inputs(q_lens, k_lens, 4, 2, 64, dt)
    got = attention.cross_attention(q, k, v, _read.starts(k_lens), cu_q=None if each else _read.starts(q_lens), scale=scale)
    _seq.check(got, *_read.cross(q, k, v, q_lens, k_lens, scale))


@pytest.mark.parametrize("each", [False, True])
def test_scores_of_minus_infinity(cuda_ok, each):
    """Keys of -inf have no weight, also where they fill whole tiles and parts."""
    n = 3000
    q = torch.ones(1 if each else 5, 4, 64, device="cuda", dtype=F16)
    k, v = _rand((n, 2, 64), F16, 2, 0.1), _rand((n, 2, 64), F16, 3)
    k[:2500] = -float("inf")
    cu_q = None if each else _read.starts([5])
    got = attention.cross_attention(q, k, v, _read.starts([n]), cu_q=cu_q)
    _seq.check(got, *_read.cross(q, k[2500:], v[2500:], [q.shape[0]], [500]))


def test_streams_graphs_and_repeats(cuda_ok):
    """On another stream, captured and replayed, and bit for bit again."""
    for q_lens, each in (([1] * 9, True), ([3] * 9, False)):
        k_lens = [(i * 977) % 3001 for i in range(9)]
        q, k, v = _inputs(q_lens, k_lens, 8, 2, 128, BF16)
        cu_k, cu_q = _read.starts(k_lens), None if each else _read.starts(q_lens)
        want = attention.cross_attention(q, k, v, cu_k, cu_q=cu_q)
        assert all(torch.equal(want, attention.cross_attention(q, k, v, cu_k, cu_q=cu_q)) for _ in range(3))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = attention.cross_attention(q, k, v, cu_k, cu_q=cu_q, stream=side)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = attention.cross_attention(q, k, v, cu_k, cu_q=cu_q)
            b = attention.cross_attention(q, k, v, cu_k, cu_q=cu_q)
        for _ in range(2):
            a.zero_()
            b.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, want) and torch.equal(b, want)
        del graph


def test_refusals(cuda_ok):
    q, k, v = _inputs([3, 2], [7, 9], 4, 2, 64, F16)
    cu_q, cu_k = _read.starts([3, 2]), _read.starts([7, 9])
    attention.cross_attention(q, k, v, cu_k, cu_q=cu_q)
    for args, kw, error in [
        ((q, k, v, cu_k), {}, ValueError), ((q, k, v, cu_k), dict(cu_q=cu_q[:2]), ValueError),
        ((q, k, v, cu_k.long()), dict(cu_q=cu_q), TypeError), ((q, k, v[:5], cu_k), dict(cu_q=cu_q), ValueError),
        ((q, k.bfloat16(), v, cu_k), dict(cu_q=cu_q), TypeError), ((q, k[..., :32], v[..., :32], cu_k), dict(cu_q=cu_q), ValueError),
        ((q[:, :3], k, v, cu_k), dict(cu_q=cu_q), RuntimeError), ((q, k, v, cu_k), dict(cu_q=cu_q, out=q[:4]), ValueError),
        ((q.cpu(), k, v, cu_k), dict(cu_q=cu_q), TypeError), ((q, k, v, cu_k[:0]), dict(cu_q=cu_q), ValueError),
        ((q.clone().requires_grad_(), k, v, cu_k), dict(cu_q=cu_q), ValueError),
        ((q, k, v, cu_k), dict(cu_q=cu_q, scale=float("nan")), RuntimeError),
    ]:
        with pytest.raises(error):
            attention.cross_attention(*args, **kw)


@pytest.mark.parametrize("dt, d", [(F16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("each", [False, True])
def test_lists_that_are_no_starts(cuda_ok, dt, d, each):
    """Starts that decrease or lie outside: results are unspecified, but nothing
    outside out is written, and the next call is as ever."""
    bad = torch.tensor([0, 160, 0, 160, -7, 1 << 30, 0, 160, 90], dtype=torch.int32, device="cuda")
    q, k, v = _inputs([1] * 8 if each else [160], [160], 8, 2, d, dt)
    around = torch.full((q.shape[0] + 8, 8, d), 7.0, dtype=dt, device="cuda")
    cu_q = None if each else bad
    attention.cross_attention(q, k, v, bad, cu_q=cu_q, out=around[4:-4])
    assert bool((around[:4] == 7.0).all()) and bool((around[-4:] == 7.0).all())
    k_lens = [20] * 8
    cu, t = _read.starts(k_lens), q.shape[0] // 8
    got = attention.cross_attention(q, k, v, cu, cu_q=None if each else _read.starts([t] * 8))
    _seq.check(got, *_read.cross(q, k, v, [t] * 8, k_lens))


@pytest.mark.parametrize("q_lens", [[1, 1], [40, 3], None])
def test_states_beyond_32_bits(cuda_ok, q_lens):
    """States more than 2^31 elements into k and v, and the same ones alone."""
    n, k_lens = 2_200_000, [1000, 77]
    kv = torch.zeros(n, 2, 8, 128, dtype=BF16, device="cuda")
    few = _rand((sum(k_lens), 2, 8, 128), BF16, 1)
    kv[-few.shape[0] - 1:-1] = few
    cu = _read.starts(k_lens)
    far = cu + (n - few.shape[0] - 1)
    q = _rand((sum(q_lens or [1, 1]), 32, 128), BF16, 2)
    cu_q = None if q_lens is None else _read.starts(q_lens)
    assert torch.equal(attention.cross_attention(q, kv[:, 0], kv[:, 1], far, cu_q=cu_q),
                       attention.cross_attention(q, few[:, 0], few[:, 1], cu, cu_q=cu_q))


@pytest.mark.parametrize("rows", [1, 5, 70])
@pytest.mark.parametrize("dt, d", [(F32, 64), (F32, 100), (BF16, 256)])
def test_scores_of_minus_infinity_in_f32(cuda_ok, rows, dt, d):
    """The same where the tensor cores take no part, with a last tile that is not whole."""
    n = 333
    q = torch.ones(rows, 4, d, device="cuda", dtype=dt)
    k, v = _rand((n, 2, d), dt, 2, 0.1), _rand((n, 2, d), dt, 3)
    k[:100] = k[200:250] = -float("inf")
    seen = torch.cat([torch.arange(100, 200), torch.arange(250, n)]).cuda()
    for cu_q in (_read.starts([rows]),) if rows > 1 else (None, _read.starts([1])):
        got = attention.cross_attention(q, k, v, _read.starts([n]), cu_q=cu_q)
        _seq.check(got, *_read.cross(q, k[seen], v[seen], [rows], [len(seen)]))
