"""The 4-bit cache: what is filed, to the bit, and one-token attention over it
against the plain form in 64 bits."""
import pytest
import torch

from ai_engine_b200 import attention, pages
from tests import _read, _seq

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dt)


def _file(x, hk, size, d, spare=2, slots=None):
    """k alone into a new cache (v the same): the cache and its slots."""
    n = -(-x.shape[0] // size) + spare
    kv = pages.new_cache4(1, n, size, hk, d)
    if slots is None:
        slots = torch.randperm(n * size, device="cuda")[: x.shape[0]]
    attention.kv4_file(x, x, kv[0, 0], kv[0, 1], slots)
    return kv, slots


def _same(got, x):
    """What was filed, in f32 once rounded: equal in every element."""
    want = _read.values(x).float()
    assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()} differ"


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("d, hk, size, tokens", [(32, 1, 8, 1), (64, 3, 16, 37), (96, 2, 24, 100), (128, 8, 64, 513), (160, 1, 8, 9),
                                                 (192, 2, 16, 30), (224, 1, 8, 17), (256, 4, 32, 65)])
def test_file_and_load(cuda_ok, dt, d, hk, size, tokens):
    k, v = _rand((tokens, hk, d), dt, 1), _rand((tokens, hk, d), dt, 2, 0.01)
    n = -(-tokens // size) + 2
    kv = pages.new_cache4(2, n, size, hk, d)
    slots = torch.randperm(n * size, device="cuda")[:tokens]
    attention.kv4_file(k, v, kv[1, 0], kv[1, 1], slots)
    assert not bool(kv[0].any())
    a, b = attention.kv4_load(kv[1, 0], kv[1, 1], slots, dtype=F32)
    _same(a, k)
    _same(b, v)
    # the places that were not filed are as they were
    for half, x in zip(kv[1], (k, v)):
        whole = _read.read_cache(half, d).transpose(1, 2).reshape(n * size, hk, d)
        assert torch.equal(whole[slots].float(), _read.values(x).float())
        whole[slots] = 0
        assert not bool(whole.any())
    for out in (F16, BF16):
        c, e = attention.kv4_load(kv[1, 0], kv[1, 1], slots, dtype=out)
        assert c.dtype == out and torch.equal(c, a.to(out)) and torch.equal(e, b.to(out))


def test_many_values_to_the_bit(cuda_ok):
    """Enough groups that some scales and codes stand next to a border."""
    for dt in (F32, BF16, F16):
        for scale in (1.0, 1e-4, 300.0):
            x = _rand((20000, 2, 128), dt, 3, scale)
            kv, slots = _file(x, 2, 64, 128)
            _same(attention.kv4_load(kv[0, 0], kv[0, 1], slots, dtype=F32)[0], x)


def test_borders(cuda_ok):
    """Elements on the border between two codes, and one step of f32 to either
    side: ties to even, as in 64 bits."""
    s = torch.tensor(0.0999755859375, device="cuda")  # an f16
    code = torch.arange(15, device="cuda")
    on = (code + 0.5) * s
    rows = []
    for x in (on, torch.nextafter(on, on + 1), torch.nextafter(on, on - 1)):
        rows.append(torch.cat([torch.zeros(1, device="cuda"), 15 * s[None], x, torch.zeros(15, device="cuda")]))
    x = torch.stack(rows)[:, None].contiguous()
    kv, slots = _file(x, 1, 8, 32)
    got = attention.kv4_load(kv[0, 0], kv[0, 1], slots, dtype=F32)[0]
    _same(got, x)
    assert torch.equal((got[0, 0, 2:17] / s).round().long(), code + code % 2)
    assert torch.equal((got[1, 0, 2:17] / s).round().long(), code + 1)
    assert torch.equal((got[2, 0, 2:17] / s).round().long(), code)


def test_odd_values(cuda_ok):
    """Equal elements, tiny and large ones, beyond f16; NaN and infinities take
    their own group and no other."""
    x = torch.zeros(9, 1, 64, device="cuda")
    x[0] = 3.7
    x[1, 0, ::2] = 1e-7
    x[2] = 60000 * torch.sign(_rand((1, 64), F32, 1))
    x[3] = 1e30 * torch.sign(_rand((1, 64), F32, 2))
    x[4] = -0.0
    x[5], x[6], x[7] = _rand((1, 64), F32, 3), _rand((1, 64), F32, 4), _rand((1, 64), F32, 5)
    x[5, 0, 40], x[6, 0, 3], x[7, 0, 63] = float("nan"), float("inf"), -float("inf")
    x[8] = 1000 + _rand((1, 64), F32, 6, 1e-3)
    kv, slots = _file(x, 1, 8, 64)
    got = attention.kv4_load(kv[0, 0], kv[0, 1], slots, dtype=F32)[0]
    clean = x.clone()
    clean[5, 0, 32:], clean[6, 0, :32], clean[7, 0, 32:] = 0, 0, 0
    lost = torch.isnan(got)
    assert bool(lost[5, 0, 32:].all()) and bool(lost[6, 0, :32].all()) and bool(lost[7, 0, 32:].all()) and int(lost.sum()) == 96
    _same(torch.nan_to_num(got), clean)


@pytest.mark.parametrize("dt, off", [(F16, 0), (BF16, 3), (F32, 1)])
def test_views_and_slots(cuda_ok, dt, off):
    """Views of one projection; slots outside the cache; pages with a gap between them."""
    t, hk, d, size = 21, 2, 64, 16
    x = _rand((t * 5 * d + off,), dt, 1)[off:].view(t, 5, d)
    k, v = x[:, 1:3], x[:, 3:]
    room = torch.full((2, 4, 3, hk, size, d * 5 // 8), 255, dtype=torch.uint8, device="cuda")
    kp, vp = room[0, :, 1], room[1, :, 1]
    slots = torch.randperm(4 * size, device="cuda")[:t]
    slots[2], slots[5], slots[7] = -1, 4 * size, -(1 << 40)
    before = room.clone()
    attention.kv4_file(k, v, kp, vp, slots)
    a, b = attention.kv4_load(kp, vp, slots, dtype=F32)
    for got, want in ((a, k), (b, v)):
        want = _read.values(want).float()
        want[2], want[5], want[7] = 0, 0, 0
        assert torch.equal(got, want)
    assert torch.equal(room[:, :, ::2], before[:, :, ::2])


def _cache(lens, hk, d, size, seed=1, spoil=True):
    """A cache that holds streams of these lengths, NaN in every place behind them."""
    need = [-(-max(n, 0) // size) for n in lens]
    n, width = sum(need) + 3, max(need + [1]) + 1
    kv = pages.new_cache4(1, n, size, hk, d)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    every = torch.arange(n * size, device="cuda")
    k, v = _rand((n * size, hk, d), BF16, seed + 1), _rand((n * size, hk, d), BF16, seed + 2)
    k[..., ::16] *= 3
    if spoil:
        junk = torch.full_like(k, float("nan"))
        attention.kv4_file(junk, junk, kv[0, 0], kv[0, 1], every)
    used = 0
    for i, (m, length) in enumerate(zip(need, lens)):
        table[i, :m] = order[used:used + m]
        at = torch.arange(max(length, 0), device="cuda")
        slots = table[i].long()[at // size] * size + at % size
        attention.kv4_file(k[slots], v[slots], kv[0, 0], kv[0, 1], slots)
        used += m
    return kv[0, 0], kv[0, 1], table


def _check(q, kp, vp, table, lens, **kw):
    got = attention.kv4_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), **kw)
    _seq.check(got, *_read.kv4_attend(q, kp, vp, table, lens, kw.get("scale")))
    return got


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d, hq, hk, size", [(32, 1, 1, 8), (64, 8, 2, 16), (96, 5, 1, 24), (128, 8, 1, 64), (128, 9, 1, 16), (64, 16, 1, 8),
                                             (128, 20, 1, 16), (160, 2, 1, 8), (192, 6, 2, 16), (224, 1, 1, 8), (256, 12, 1, 32),
                                             (64, 40, 2, 16), (32, 3, 3, 40)])
def test_attention(cuda_ok, dt, d, hq, hk, size):
    lens = [1, 0, 7, 8, 9, 31, 32, 33, 64, 100, -3, 700]
    kp, vp, table = _cache(lens, hk, d, size)
    _check(_rand((len(lens), hq, d), dt, 9, 2.0), kp, vp, table, lens)


@pytest.mark.parametrize("lens", [[20000], [9001, 3], [1] * 300, [(i * 131) % 200 for i in range(140)], [0, 0, 0]])
def test_lengths(cuda_ok, lens):
    kp, vp, table = _cache(lens, 2, 128, 16)
    _check(_rand((len(lens), 8, 128), BF16, 9), kp, vp, table, lens)


def test_more_heads_than_warps(cuda_ok):
    """More (stream, key head) pairs than there is work to share."""
    lens = [40, 3, 17]
    kp, vp, table = _cache(lens, 1000, 32, 8)
    _check(_rand((3, 1000, 32), F16, 9), kp, vp, table, lens)


def test_max_len_cuts(cuda_ok):
    lens = [100, 40, 64]
    kp, vp, table = _cache(lens, 2, 64, 16)
    q = _rand((3, 4, 64), F16, 3)
    got = attention.kv4_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=50)
    _seq.check(got, *_read.kv4_attend(q, kp, vp, table, [min(n, 50) for n in lens]))
    nothing = attention.kv4_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=0)
    assert not bool(nothing.any())


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-4, 2.0])
@pytest.mark.parametrize("size", [1.0, 1e-30, 1e30])
def test_scales(cuda_ok, scale, size):
    """Queries far outside f16, and scales of either sign."""
    lens = [300, 33]
    kp, vp, table = _cache(lens, 2, 64, 16)
    q = _rand((2, 8, 64), BF16, 3, size)
    q[0, 0] = 0
    _check(q, kp, vp, table, lens, scale=scale / size if size > 1 else scale)


def test_views_streams_graphs_repeats(cuda_ok):
    lens = [(i * 977) % 3001 for i in range(9)]
    kp, vp, table = _cache(lens, 2, 128, 16)
    q = _rand((8, 9, 128 + 3), BF16, 1)[..., 3:].transpose(0, 1)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((9, 2, 8, 128 + 1), 5.0, dtype=BF16, device="cuda")
    attention.kv4_attention(q, kp, vp, table, n, out=out[:, 1, :, 1:])
    want = out[:, 1, :, 1:].clone()
    _seq.check(want, *_read.kv4_attend(q, kp, vp, table, lens))
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1, :, 0] == 5).all())
    assert all(torch.equal(want, attention.kv4_attention(q, kp, vp, table, n)) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = attention.kv4_attention(q, kp, vp, table, n, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = attention.kv4_attention(q, kp, vp, table, n)
        b = attention.kv4_attention(q, kp, vp, table, n)
    for _ in range(2):
        a.zero_()
        b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
    del graph


def test_pages_that_do_not_exist_are_not_read(cuda_ok):
    """Their stream's result is unspecified; the others' are as ever."""
    lens = [50, 50, 50]
    kp, vp, table = _cache(lens, 2, 64, 16)
    q = _rand((3, 4, 64), F16, 3)
    want, limit = _read.kv4_attend(q, kp, vp, table, lens)
    table[1, 0], table[1, 1], table[1, 2] = -5, kp.shape[0], 2 ** 31 - 1
    got = attention.kv4_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    _seq.check(got[::2], want[::2], limit[::2])


def test_fork_and_compact(cuda_ok):
    """The pages' upkeep moves 4-bit pages: streams attend as before."""
    size, d, hk, t = 16, 64, 2, 37
    kv, st = pages.new_cache4(2, 40, size, hk, d), pages.new_state(40, 6, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages.grow(st, size, i32([5]), i32([3 * size]), 0)
    slots = pages.grow(st, size, i32([0]), i32([t]), t)
    k, v, q = _rand((t, hk, d), F16, 1), _rand((t, hk, d), F16, 2), _rand((1, 4, d), F16, 3)
    for layer in kv:
        attention.kv4_file(k, v, layer[0], layer[1], slots)

    def look(row):
        return [attention.kv4_attention(q, x[0], x[1], st.table[row:row + 1].clone(), st.lens[row:row + 1].clone()) for x in kv]
    want = look(0)[0]
    pages.fork(kv, st, i32([0, 0]), i32([1, 2]))
    pages.free(st, i32([0, 5]))
    pages.compact(kv, st)
    assert int(st.status) == 0
    for row in (1, 2):
        assert all(torch.equal(x, want) for x in look(row))


def test_refusals(cuda_ok):
    kp, vp, table = _cache([20, 5], 2, 64, 16)
    q, lens = _rand((2, 4, 64), F16, 1), torch.tensor([20, 5], dtype=torch.int32, device="cuda")
    k, slots = _rand((2, 2, 64), F16, 2), torch.tensor([0, 1], device="cuda")
    attention.kv4_attention(q, kp, vp, table, lens)
    for args, kw, error in [
        ((q.float(), kp, vp, table, lens), {}, RuntimeError), ((q[..., :32], kp, vp, table, lens), {}, ValueError),
        ((q[:, :3], kp, vp, table, lens), {}, RuntimeError), ((q, kp.short(), vp, table, lens), {}, TypeError),
        ((q, kp[:, :, ::2], vp[:, :, ::2], table, lens), {}, ValueError), ((q, kp, vp[1:], table, lens), {}, ValueError),
        ((q, kp[..., :10], vp[..., :10], table, lens), {}, ValueError), ((q, kp, vp, table[:1], lens), {}, ValueError),
        ((q, kp, vp, table, lens.long()), {}, TypeError), ((q, kp, vp, table, lens), dict(max_len=10 ** 6), RuntimeError),
        ((q, kp, vp, table, lens), dict(out=q[:1]), ValueError), ((q, kp, vp, table, lens), dict(scale=float("nan")), RuntimeError),
        ((q.clone().requires_grad_(), kp, vp, table, lens), {}, ValueError), ((q, kp.cpu(), vp, table, lens), {}, TypeError),
    ]:
        with pytest.raises(error):
            attention.kv4_attention(*args, **kw)
    for args, error in [
        ((k[..., :32], k[..., :32], kp, vp, slots), ValueError), ((k, k[:1], kp, vp, slots), ValueError),
        ((k, k, kp, vp, slots.int()), TypeError), ((k, k, kp, vp, slots[:1]), ValueError), ((k[:, :1], k[:, :1], kp, vp, slots), ValueError),
        ((k.clone().requires_grad_(), k, kp, vp, slots), ValueError), ((k.double(), k.double(), kp, vp, slots), TypeError),
    ]:
        with pytest.raises(error):
            attention.kv4_file(*args)
    for args, kw, error in [((kp, vp, slots), dict(dtype=torch.float64), TypeError), ((kp, vp, slots.int()), {}, TypeError),
                            ((kp, vp, slots), dict(dtype="half"), TypeError), ((kp, vp.cpu(), slots), {}, TypeError)]:
        with pytest.raises(error):
            attention.kv4_load(*args, **kw)
    with pytest.raises(ValueError):
        pages.new_cache4(1, 4, 12, 2, 64)
    with pytest.raises(ValueError):
        pages.new_cache4(1, 4, 16, 2, 80)


def test_offsets_beyond_32_bits(cuda_ok):
    """The same pages far into a cache of 4.5 GB a half: filed, read and attended to as near its start."""
    lens, size, hk, d = [700, 64, 1], 64, 8, 128
    kp, vp, table = _cache(lens, hk, d, size)
    n = kp.shape[0]
    kv = pages.new_cache4(1, 110000, size, hk, d)
    far = 110000 - 1 - 3571 * torch.arange(n, device="cuda")  # on both sides of 2^31 and of 2^32 bytes
    assert int(far.min()) * kv.stride(2) > 2 ** 31 and int(far.max()) * kv.stride(2) > 2 ** 32
    kv[0, 0][far], kv[0, 1][far] = kp, vp
    moved = torch.where(table >= 0, far[table.long().clamp(min=0)].int(), table)
    q, cu = _rand((3, 32, d), BF16, 9), torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert torch.equal(attention.kv4_attention(q, kv[0, 0], kv[0, 1], moved, cu), attention.kv4_attention(q, kp, vp, table, cu))
    near = torch.arange(n * size, device="cuda")
    slots = far[near // size] * size + near % size
    k, v = _rand((n * size, hk, d), F16, 3), _rand((n * size, hk, d), F16, 4)
    attention.kv4_file(k, v, kv[0, 0], kv[0, 1], slots)
    for got, x in zip(attention.kv4_load(kv[0, 0], kv[0, 1], slots, dtype=F32), (k, v)):
        _same(got, x)
