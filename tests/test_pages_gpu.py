"""Upkeep of the cache's pages against plain Python lists: every integer and
every copied value has to be equal."""
import pytest
import torch

from ai_engine_b200 import _lib, pages

pytestmark = pytest.mark.gpu


class Plain:
    """The bookkeeping as lists; kv as a tensor that moves page by page."""

    def __init__(self, kv, n, rows, width, size):
        self.kv, self.n, self.size, self.width = kv.clone(), n, size, width
        self.refs, self.lens, self.table, self.status = [0] * n, [0] * rows, [[] for _ in range(rows)], 0

    def free_pages(self):
        return [p for p in range(self.n) if self.refs[p] == 0]

    def grow(self, rows, counts, tokens):
        if len(set(rows)) < len(rows) or any(not 0 <= r < len(self.lens) for r in rows):
            self.status |= 2
            return [-1] * tokens
        need = [-(-(self.lens[r] + c) // self.size) - len(self.table[r]) for r, c in zip(rows, counts)]
        free = self.free_pages()
        if sum(need) > len(free) or any(len(self.table[r]) + m > self.width for r, m in zip(rows, need)):
            self.status |= 1
            return [-1] * tokens
        slots = []
        for r, c, m in zip(rows, counts, need):
            for _ in range(m):
                p = free.pop(0)
                self.refs[p] = 1
                self.table[r].append(p)
            slots += [self.table[r][i // self.size] * self.size + i % self.size for i in range(self.lens[r], self.lens[r] + c)]
            self.lens[r] += c
        return (slots + [-1] * tokens)[:tokens]

    def fork(self, src, dst):
        bad = any(not 0 <= r < len(self.lens) for r in src + dst) or len(set(dst)) < len(dst) or set(src) & set(dst)
        if bad or any(self.lens[r] for r in dst):
            self.status |= 2
            return
        free = self.free_pages()
        if sum(self.lens[r] % self.size > 0 for r in src) > len(free):
            self.status |= 1
            return
        for a, b in zip(src, dst):
            whole = self.lens[a] // self.size
            self.table[b] = self.table[a][:whole]
            for p in self.table[b]:
                self.refs[p] += 1
            if self.lens[a] % self.size:
                p = free.pop(0)
                self.refs[p] = 1
                self.kv[:, :, p] = self.kv[:, :, self.table[a][whole]]
                self.table[b].append(p)
            self.lens[b] = self.lens[a]

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.lens):
                for p in self.table[r]:
                    self.refs[p] -= 1
                self.table[r], self.lens[r] = [], 0

    def compact(self):
        live = [p for p in range(self.n) if self.refs[p]]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        remap = [p if self.refs[p] else -1 for p in range(self.n)]
        for a, b in zip([p for p in live if p >= len(live)], holes):
            self.kv[:, :, b] = self.kv[:, :, a]
            self.refs[b], self.refs[a], remap[a] = self.refs[a], 0, b
        self.table = [[remap[p] for p in row] for row in self.table]
        return remap

    def same(self, kv, st):
        assert st.refs.tolist() == self.refs
        assert st.lens.tolist() == self.lens
        assert st.table.tolist() == [r + [-1] * (self.width - len(r)) for r in self.table]
        assert st.status.tolist() == [self.status]
        assert torch.equal(kv, self.kv)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _both(layers=2, n=40, size=16, heads=2, dim=8, rows=10, width=8, dtype=torch.float16, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    kv = pages.new_cache(layers, n, size, heads, dim, dtype)
    kv.copy_(torch.randn(kv.shape, generator=g, device="cuda"))
    return kv, pages.new_state(n, rows, width), Plain(kv, n, rows, width, size)


@pytest.mark.parametrize("size, heads, dim, dtype", [(16, 2, 64, torch.float16), (8, 1, 8, torch.bfloat16), (24, 3, 20, torch.float32),
                                                     (1, 1, 8, torch.float16), (64, 2, 128, torch.bfloat16)])
def test_a_life_of_the_cache(cuda_ok, size, heads, dim, dtype):
    """A seeded run of calls, compared after each: growth by nothing, one and
    many tokens, forks of whole and partly filled pages, ends, compaction."""
    import random
    rng = random.Random(size)
    kv, st, p = _both(3, 50, size, heads, dim, 12, 9, dtype)
    for step in range(40):
        act = rng.choice(["grow", "grow", "fork", "free", "compact"])
        if act == "grow":
            rows = rng.sample(range(12), rng.randint(1, 5))
            counts = [rng.choice([0, 1, size, rng.randint(0, 2 * size)]) for _ in rows]
            tokens = sum(counts) + rng.choice([0, 0, 3])
            got = pages.grow(st, size, _i32(rows), _i32(counts), tokens)
            assert got.tolist() == p.grow(rows, counts, tokens)
        elif act == "fork":
            empty = [r for r in range(12) if not p.lens[r]]
            full = [r for r in range(12) if p.lens[r]]
            if not empty or not full:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(full) for _ in dst]
            pages.fork(kv, st, _i32(src), _i32(dst))
            p.fork(src, dst)
        elif act == "free":
            rows = [rng.randint(-1, 12) for _ in range(rng.randint(1, 4))]
            pages.free(st, _i32(rows))
            p.free(rows)
        else:
            assert pages.compact(kv, st).tolist() == p.compact()
        p.same(kv, st)


def test_too_few_pages_change_nothing(cuda_ok):
    kv, st, p = _both(n=6, width=8)
    for rows, counts in (([0], [70]), ([1], [33]), ([1], [17]), ([0], [16 * 9]), ([0, 1], [30, 30])):
        n = sum(counts)
        assert pages.grow(st, 16, _i32(rows), _i32(counts), n).tolist() == p.grow(rows, counts, n)
        p.same(kv, st)
    assert p.status == 1
    pages.fork(kv, st, _i32([0]), _i32([2]))  # its last page is partly filled and none is free
    p.fork([0], [2])
    p.same(kv, st)


@pytest.mark.parametrize("src, dst", [([0], [0]), ([0, 0], [3, 3]), ([0], [1]), ([10], [4]), ([0], [-1]), ([-1], [4]), ([0, 4], [4, 5])])
def test_bad_forks_change_nothing(cuda_ok, src, dst):
    kv, st, p = _both()
    pages.grow(st, 16, _i32([0, 1]), _i32([20, 5]), 25)
    p.grow([0, 1], [20, 5], 25)
    pages.fork(kv, st, _i32(src), _i32(dst))
    p.fork(src, dst)
    assert p.status == 2
    p.same(kv, st)


@pytest.mark.parametrize("rows", [[3, 3], [0, 99], [-1]])
def test_bad_growth_changes_nothing(cuda_ok, rows):
    kv, st, p = _both()
    assert pages.grow(st, 16, _i32(rows), _i32([4] * len(rows)), 8).tolist() == p.grow(rows, [4] * len(rows), 8) == [-1] * 8
    p.same(kv, st)


def test_many_pages_and_rows(cuda_ok):
    """More pages, rows and list entries than one pass of a block covers."""
    n, rows, width = 5000, 2500, 4
    kv, st, p = _both(1, n, 8, 1, 8, rows, width)
    order = list(range(0, 2 * 1200, 2))
    counts = [(i * 7) % 17 for i in range(1200)]
    total = sum(counts)
    assert pages.grow(st, 8, _i32(order), _i32(counts), total).tolist() == p.grow(order, counts, total)
    p.same(kv, st)
    src, dst = order[:1100], [r + 1 for r in order[:1100]]
    pages.fork(kv, st, _i32(src), _i32(dst))
    p.fork(src, dst)
    p.same(kv, st)
    gone = order[::3] + dst[::2]
    pages.free(st, _i32(gone))
    p.free(gone)
    assert pages.compact(kv, st).tolist() == p.compact()
    p.same(kv, st)


def test_copy(cuda_ok):
    kv, _, p = _both(3, 20)
    src, dst = [1, 5, 5, 19, 3, 77, -1], [2, 6, 7, 0, 20, 8, 9]
    pages.copy(kv, _i32(src), _i32(dst))
    for a, b in list(zip(src, dst))[:4]:
        p.kv[:, :, b] = p.kv[:, :, a]
    assert torch.equal(kv, p.kv)
    pages.copy(kv, _i32([]), _i32([]))
    assert torch.equal(kv, p.kv)


def test_empty_and_full_cache_compact(cuda_ok):
    kv, st, p = _both(n=8, width=8)
    assert pages.compact(kv, st).tolist() == p.compact() == [-1] * 8
    pages.grow(st, 16, _i32([0]), _i32([128]), 128)
    p.grow([0], [128], 128)
    assert pages.compact(kv, st).tolist() == p.compact() == list(range(8))
    p.same(kv, st)


def test_offsets_beyond_32_bits(cuda_ok):
    """A cache of more than 2^32 bytes and 2^31 elements: the last pages of the last layer move."""
    n = 36000
    kv = torch.empty(2, 2, n, 16, 8, 128, dtype=torch.float16, device="cuda")
    assert kv.numel() > 2 ** 31 and kv.numel() * 2 > 2 ** 32
    st = pages.new_state(n, 2, 4)
    kv[:, :, n - 1] = 3.0
    kv[:, :, n - 2] = torch.arange(8 * 128, device="cuda").view(8, 128).half()
    kv[:, :, 0] = 0
    st.refs[n - 2], st.refs[n - 1] = 1, 1
    st.table[1, 0], st.table[1, 1], st.lens[1] = n - 1, n - 2, 20
    remap = pages.compact(kv, st)
    assert remap[n - 2] == 0 and remap[n - 1] == 1 and st.table[1].tolist() == [1, 0, -1, -1]
    assert (kv[:, :, 1] == 3).all() and torch.equal(kv[:, :, 0], kv[:, :, n - 2])


@pytest.mark.parametrize("rows, more", [(4096, 0), (4097, 3)])
def test_growth_beyond_32_bits(cuda_ok, rows, more):
    """Lists that ask for 2^31 pages and tokens, or some more, find too few."""
    width = 1 << 19
    st = pages.new_state(64, rows, width)
    counts = [width] * 4096 + [more] * (rows - 4096)
    slots = pages.grow(st, 1, torch.arange(rows, dtype=torch.int32, device="cuda"), _i32(counts), 100)
    assert (slots == -1).all() and st.status.item() == _lib.PAGES_FULL
    assert not st.refs.any() and not st.lens.any() and st.table.max() == -1
    slots = pages.grow(st, 1, _i32([rows - 1, 0]), _i32([5, 2]), 8)
    assert slots.tolist() == [0, 1, 2, 3, 4, 5, 6, -1]


def test_calls_in_a_graph(cuda_ok):
    kv, st, p = _both()
    pages.grow(st, 16, _i32([0]), _i32([37]), 37)
    p.grow([0], [37], 37)
    src, dst, gone = _i32([0, 0]), _i32([1, 2]), _i32([0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pages.fork(kv, st, src, dst)
        pages.free(st, gone)
        remap = pages.compact(kv, st)
    g.replay()
    torch.cuda.synchronize()
    p.fork([0, 0], [1, 2])
    p.free([0])
    assert remap.tolist() == p.compact()
    p.same(kv, st)


def test_refuses(cuda_ok):
    kv, st, _ = _both()
    with pytest.raises(ValueError):
        pages.fork(kv, st, _i32([0, 1]), _i32([2]))
    with pytest.raises(TypeError):
        pages.fork(kv, st, _i32([0]).long(), _i32([2]))
    with pytest.raises(TypeError):
        pages.copy(kv.transpose(2, 3), _i32([0]), _i32([1]))
    with pytest.raises(ValueError):
        pages.compact(kv[:, :, :20].contiguous(), st)
    with pytest.raises(ValueError):
        pages.free(st._replace(table=st.table[:3].contiguous()), _i32([0]))
    with pytest.raises(_lib.AieError):
        pages.grow(st, 0, _i32([0]), _i32([2]), 2)
    odd = pages.new_cache(1, 40, 1, 1, 4, torch.float16)  # pages of 8 bytes
    with pytest.raises(_lib.AieError):
        pages.copy(odd, _i32([0]), _i32([1]))
