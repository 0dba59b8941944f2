"""Norm and rotation by positions along several axes against the plain form in
64 bits."""
import pytest
import torch

from ai_engine_b200 import attention
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


def _axes(pairs, axes, kind):
    if kind == "turns":
        return (torch.arange(pairs, device="cuda") % axes).to(torch.uint8)
    if kind == "even":  # sections of eight pairs
        return (torch.arange(pairs, device="cuda") // 8 % axes).to(torch.uint8)
    g = torch.Generator("cuda").manual_seed(pairs)
    return torch.randint(0, axes, (pairs,), generator=g, device="cuda").sort().values.to(torch.uint8)


def _own_table(table, pos, axis):
    """Each token's own row of angles."""
    half = axis.shape[0]
    i = torch.arange(half, device="cuda")
    at = pos.long()[:, axis.long()]
    return torch.cat([table[at, i], table[at, i + half]], 1), torch.arange(pos.shape[0], device="cuda")


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("tokens, hq, hk, d, rot, axes, kind, interleaved", [
    (1, 1, 1, 64, 64, 3, "even", False), (7, 8, 2, 128, 128, 3, "sorted", False), (33, 6, 3, 96, 48, 3, "turns", True),
    (5, 4, 4, 80, 80, 2, "sorted", False), (9, 2, 1, 72, 18, 3, "turns", False), (3, 3, 3, 20, 10, 4, "sorted", True),
    (130, 16, 4, 128, 64, 3, "turns", True), (4, 2, 2, 256, 256, 2, "even", False), (2, 5, 5, 512, 510, 3, "sorted", False),
    (6, 7, 1, 64, 0, 3, "turns", False), (700, 20, 5, 64, 64, 3, "even", False), (6, 3, 1, 64, 64, 1, "even", False),
    (3, 2, 1, 128, 128, 255, "turns", False),
])
def test_axes(cuda_ok, dt, tokens, hq, hk, d, rot, axes, kind, interleaved):
    q, k = _rand((tokens, hq, d), dt, 1, 3.0), _rand((tokens, hk, d), dt, 2, 0.5)
    wq, wk = _rand((d,), F32, 3), _rand((d,), F32, 4)
    table = _table(50, rot) if rot else torch.zeros(50, 0, device="cuda")
    axis = _axes(rot // 2, axes, kind)
    pos = torch.randint(0, 50, (tokens, axes), device="cuda", dtype=torch.int32)
    qo, ko = attention.qk_norm_rope(q, k, pos, table, pair_axis=axis, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    own, at = _own_table(table, pos, axis)
    _seq.check_norm_rope(qo, *_seq.norm_rope(q, wq, at, own, rot, interleaved, 1e-5))
    _seq.check_norm_rope(ko, *_seq.norm_rope(k, wk, at, own, rot, interleaved, 1e-5))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d, rot, off", [(80, 40, 0), (24, 8, 0), (72, 40, 0), (120, 56, 0), (8, 8, 0), (128, 24, 0), (64, 64, 4), (80, 40, 4), (80, 40, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", [None, "sorted", "turns"])
def test_pieces_of_four(cuda_ok, dt, d, rot, off, interleaved, kind):
    """Heads and rotations in multiples of 8, rows aligned to 8 bytes and less;
    with one position a token too, filed."""
    t, hq, hk, size, n = 37, 6, 3, 8, 6
    raw = _rand((t * (hq + 2 * hk) * d + off,), dt, 5, 2.0)
    x = raw[off:].view(t, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    wq, wk, table = _rand((d,), F32, 3), _rand((d,), F32, 4), _table(50, rot)
    axis = _axes(rot // 2, 3, kind or "even")
    pos = torch.randint(0, 50, (t, 3), device="cuda", dtype=torch.int32)
    if kind is None:
        pos[:, 1], pos[:, 2] = pos[:, 0], pos[:, 0]
    own, at = _own_table(table, pos, axis)
    pages = torch.zeros(2, n, size, hk, d, dtype=dt, device="cuda")
    slots = torch.randperm(n * size, device="cuda")[:t]
    qo, ko = attention.qk_norm_rope(q, k, pos[:, 0].contiguous() if kind is None else pos, table, pair_axis=axis if kind else None,
                                    q_weight=wq, k_weight=wk, interleaved=interleaved, v=v, k_pages=pages[0], v_pages=pages[1],
                                    slots=slots)
    _seq.check_norm_rope(qo, *_seq.norm_rope(q, wq, at, own, rot, interleaved, 1e-6))
    _seq.check_norm_rope(ko, *_seq.norm_rope(k, wk, at, own, rot, interleaved, 1e-6))
    assert torch.equal(pages[0, slots // size, slots % size], ko) and torch.equal(pages[1, slots // size, slots % size], v)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("off", [0, 1])
def test_one_axis_is_the_plain_call(cuda_ok, dt, off):
    """All pairs on one of three axes: as with that axis's positions alone, to the bit."""
    t, d = 37, 64
    raw = _rand((t * 6 * d + off,), dt, 5)
    x = raw[off:].view(t, 6, d)
    table, pos = _table(60, d), torch.randint(0, 60, (t, 3), device="cuda", dtype=torch.int32)
    for axis in range(3):
        a = attention.qk_norm_rope(x[:, :4], x[:, 4:], pos, table, pair_axis=torch.full((32,), axis, dtype=torch.uint8, device="cuda"))
        b = attention.qk_norm_rope(x[:, :4], x[:, 4:], pos[:, axis].contiguous(), table)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("d, off", [(64, 0), (40, 1)])
def test_filed_and_in_place(cuda_ok, d, off):
    t, hq, hk, size, n = 19, 4, 2, 8, 5
    raw = _rand((t * (hq + 2 * hk) * d + off,), F16, 5)
    x = raw[off:].view(t, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    wk, table = _rand((d,), F32, 6), _table(t, d)
    pos = torch.randint(0, t, (t, 3), device="cuda", dtype=torch.int32)
    axis = _axes(d // 2, 3, "sorted")
    own, at = _own_table(table, pos, axis)
    pages = torch.zeros(2, n, size, hk, d, dtype=F16, device="cuda")
    slots = torch.randperm(n * size, device="cuda")[:t]
    slots[3], slots[4] = -1, n * size
    want_q, want_k = _seq.norm_rope(q, None, at, own, d, False, 1e-6), _seq.norm_rope(k, wk, at, own, d, False, 1e-6)
    rest = pages.clone()
    qo, ko = attention.qk_norm_rope(q, k, pos, table, pair_axis=axis, k_weight=wk, v=v, k_pages=pages[0], v_pages=pages[1],
                                    slots=slots, q_out=q, k_out=k)
    _seq.check_norm_rope(qo, *want_q)
    _seq.check_norm_rope(ko, *want_k)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < n * size:
            rest[0, s // size, s % size], rest[1, s // size, s % size] = ko[i], v[i]
    assert torch.equal(pages, rest)


@pytest.mark.parametrize("d, kind", [(64, "even"), (64, "turns"), (36, "turns")])
def test_positions_and_axes_that_do_not_exist(cuda_ok, d, kind):
    """NaN in the pairs that they turn, nowhere else."""
    t, half = 6, d // 2
    q = _rand((t, 2, d), F16, 1)
    table, axis = _table(20, d), _axes(half, 3, kind)
    pos = torch.randint(0, 20, (t, 3), device="cuda", dtype=torch.int32)
    good, _ = attention.qk_norm_rope(q, q, pos, table, pair_axis=axis)
    pos[1, 0], pos[2, 1], pos[3, 2] = -1, 20, 2 ** 31 - 1
    bad_axis = axis.clone()
    bad_axis[half - 1] = 3
    got, _ = attention.qk_norm_rope(q, q, pos, table, pair_axis=bad_axis)
    for i in range(t):
        for p in range(half):
            lost = p == half - 1 or (1 <= i <= 3 and int(axis[p]) == i - 1)
            for e in (p, p + half):
                assert bool(torch.isnan(got[i, :, e]).all()) == lost
                assert lost or torch.equal(got[i, :, e], good[i, :, e])


def test_refusals(cuda_ok):
    q, table = _rand((4, 2, 64), F16, 1), _table(20, 64)
    pos, axis = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.zeros(32, dtype=torch.uint8, device="cuda")
    attention.qk_norm_rope(q, q, pos, table, pair_axis=axis)
    for bad_pos, bad_axis, error in [
        (pos[:, 0].contiguous(), axis, TypeError), (pos.t(), axis, TypeError), (pos.long(), axis, TypeError),
        (pos[:3], axis, ValueError), (pos, axis[:31], ValueError), (pos, axis.int(), TypeError), (pos, axis.cpu(), TypeError),
        (torch.zeros(4, 0, dtype=torch.int32, device="cuda"), axis, RuntimeError),
        (torch.zeros(4, 256, dtype=torch.int32, device="cuda"), axis, RuntimeError), (pos, None, TypeError),
    ]:
        with pytest.raises(error):
            attention.qk_norm_rope(q, q, bad_pos, table, pair_axis=bad_axis)
