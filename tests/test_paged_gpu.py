"""The paged cache's operators and the prompt attention on the GPU, against their definitions in 64 bits
(paged_helpers.py) and, for the pages, against a cache kept in Python lists."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_helpers as ph  # noqa: E402
import pocketforge_b200 as pf  # noqa: E402
from paged_helpers import BF16, F16, F32, I8, TYPES, Cache, check, ints, latched, ok  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def need_device():
    if not torch.cuda.is_available() or pf.device_count() == 0:
        pytest.skip("no sm_100 device")


@pytest.fixture(autouse=True)
def no_latched_error():
    latched()
    yield
    torch.cuda.synchronize()
    assert latched() == 0


def randn(shape, t, seed, by=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * by).to(t)


def offsets_of(lens, start=0):
    return [start] + [start + sum(lens[:i + 1]) for i in range(len(lens))]


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------
class Model:
    """The page operations in Python lists; the contents of pages are followed by copying the cache's tensors."""

    def __init__(self, c):
        self.c = c
        self.table = [[] for _ in range(c.seqs)]
        self.lens = [0] * c.seqs
        self.refs = [0] * c.pages
        self.data = [x.clone() for x in self.tensors()]

    def tensors(self):
        c = self.c
        return [c.k, c.v] + ([c.ks, c.vs] if c.ks is not None else [])

    def lowest(self, n):
        got = [i for i, r in enumerate(self.refs) if r == 0][:n]
        return got if len(got) == n else None

    def reserve(self, seqs, counts):
        asked, free, flags = 0, [i for i, r in enumerate(self.refs) if r == 0], 0
        for s, n in zip(seqs, counts):
            total = -(-(self.lens[s] + n) // self.c.page)
            if total > self.c.max_pages:
                flags |= 8
                continue
            need = total - len(self.table[s])
            mine = free[asked:asked + need]
            asked += need
            if len(mine) < need:
                flags |= 8
                continue
            for p in mine:
                self.refs[p] = 1
            self.table[s] += mine
            self.lens[s] += n
        return flags

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.lens[s] = [], 0

    def fork(self, parents, children):
        free, flags = [i for i, r in enumerate(self.refs) if r == 0], 0
        todo = list(zip(parents, children))
        for p, k in todo:
            rest = self.lens[p] % self.c.page
            full = self.table[p][:self.lens[p] // self.c.page]
            if rest:
                if not free:
                    flags |= 8
                    continue
                new = free.pop(0)
                self.refs[new] = 1
                for x in self.data:
                    x[new, :, :, :rest] = x[self.table[p][-1], :, :, :rest]
            for q in full:
                self.refs[q] += 1
            self.table[k] = full + ([new] if rest else [])
            self.lens[k] = self.lens[p]
        return flags

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [i for i in range(live, self.c.pages) if self.refs[i]]
        dst = [i for i in range(live) if not self.refs[i]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[a], self.refs[b] = 0, self.refs[a]
            for x in self.data:
                x[b] = x[a]
        self.table = [[to.get(p, p) for p in row] for row in self.table]

    def same(self):
        torch.cuda.synchronize()
        assert self.c.lens.tolist() == self.lens
        assert self.c.refs.tolist() == self.refs
        got = self.c.table.tolist()
        for s, row in enumerate(self.table):
            assert got[s][:len(row)] == row, s
        for x, y in zip(self.tensors(), self.data):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,layers,kv_heads,dim,page,pages,seqs,max_pages",
                         [(I8, 2, 2, 64, 16, 40, 8, 12), (BF16, 3, 1, 64, 32, 70, 16, 9), (F16, 1, 3, 128, 128, 25, 5, 40),
                          (I8, 5, 8, 128, 64, 300, 33, 20), (I8, 1, 1, 64, 16, 5000, 64, 200)])
def test_pages_follow_the_model(dtype, layers, kv_heads, dim, page, pages, seqs, max_pages):
    """Random operations one after another; after each, lengths, counts, tables and every byte of the pages agree."""
    c = Cache(dtype, layers, kv_heads, dim, page, pages, seqs, max_pages)
    m, rng, seen = Model(c), random.Random(pages), set()
    for step in range(60):
        used = [s for s in range(seqs) if m.lens[s]]
        empty = [s for s in range(seqs) if not m.lens[s]]
        op = rng.choice(["reserve", "reserve", "reserve", "fork", "fork", "free", "compact"])
        flags = 0
        if op == "reserve":
            some = rng.sample(range(seqs), rng.randint(1, seqs))
            counts = [rng.choice([0, 1, 5, page, rng.randint(0, 4 * page), rng.randint(0, max_pages * page)]) for _ in some]
            c.reserve(some, counts)
            flags = m.reserve(some, counts)
        elif op == "fork" and used and empty:
            kids = rng.sample(empty, rng.randint(1, len(empty)))
            par = [rng.choice(used) for _ in kids]
            c.fork(par, kids)
            flags = m.fork(par, kids)
        elif op == "free" and used:
            some = rng.sample(used, rng.randint(1, max(1, len(used) // 2)))
            c.free(some)
            m.free(some)
        elif op == "compact":
            c.compact()
            m.compact()
        m.same()
        assert latched() == flags, (step, op)
        seen.add((op, flags))
    assert {o for o, _ in seen} == {"reserve", "fork", "free", "compact"}


def test_pages_many_of_them():
    """More pages than one pass of the deciding CTA takes (65,536), the ones in use at the end."""
    c = Cache(I8, 1, 1, 64, 16, 150_000, 4, 90_000, fill=False)
    c.k.zero_(), c.v.zero_(), c.ks.zero_(), c.vs.zero_()
    m = Model(c)
    for seqs, counts in (([0], [70_000 * 16]), ([1], [79_990 * 16]), ([2], [9 * 16 + 1])):
        c.reserve(seqs, counts)
        assert m.reserve(seqs, counts) == 0
        m.same()
    c.k[m.table[1]] = randn((len(m.table[1]), 1, 1, 16, 64), torch.float32, 1, 40).to(torch.int8)
    m.data[0].copy_(c.k)
    c.free([0]), m.free([0])
    c.compact(), m.compact()
    m.same()
    c.reserve([3], [75_000 * 16 + 3])  # 150,000 - 79,990 - 10 pages are free: too few
    assert m.reserve([3], [75_000 * 16 + 3]) == latched() == 8
    m.same()
    c.reserve([3], [69_999 * 16 + 3])  # every one of them
    assert m.reserve([3], [69_999 * 16 + 3]) == 0
    m.same()


def test_pages_copy():
    c = Cache(BF16, 2, 3, 64, 32, 20, 2, 4)
    k, v = c.k.clone(), c.v.clone()
    c.copy([3, 3, 7, 0], [19, 1, 2, 11])
    k[[19, 1, 2, 11]], v[[19, 1, 2, 11]] = k[[3, 3, 7, 0]], v[[3, 3, 7, 0]]
    torch.cuda.synchronize()
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    c.copy([5, 20, -1], [6, 8, 9])  # pages that are none are left out
    k[6], v[6] = k[5], v[5]
    assert latched() == 1
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_pages_lists_that_are_wrong():
    c = Cache(I8, 1, 1, 64, 16, 12, 6, 8)
    c.reserve([0, 1], [20, 16])
    assert latched() == 0
    c.reserve([2, 2, 6, -1, 3], [5, 9, 1, 1, -4])  # named again; no such sequence (twice); a count below zero
    assert latched() == 1
    assert c.lens.tolist() == [20, 16, 5, 0, 0, 0] and c.refs.tolist() == [1] * 4 + [0] * 8
    c.fork([0, 1, 0, 9, 1], [3, 3, 1, 4, 0])  # child named again, child in use, no such parent, child in use
    assert latched() == 1
    assert c.lens.tolist() == [20, 16, 5, 20, 0, 0] and c.table[3, :2].tolist() == [0, 4]
    c.fork([3, 4], [4, 5])  # a parent that is a child of the same call; the other's parent too
    assert latched() == 1
    assert c.lens.tolist() == [20, 16, 5, 20, 0, 0]
    c.free([3, 3, 5, 77])  # named again: once; empty: nothing; no such sequence
    assert latched() == 1
    assert c.lens.tolist() == [20, 16, 5, 0, 0, 0] and c.refs.tolist() == [1] * 4 + [0] * 8
    c.lens[1] = 1000  # no such length: left out, the others served
    c.reserve([1, 4], [1, 1])
    assert latched() == 1
    assert c.lens.tolist() == [20, 1000, 5, 0, 1, 0]
    for n in (0,):
        ok("pf_paged_reserve", c.ref, None, None, n, None)
        ok("pf_paged_free", c.ref, None, n, None)
        ok("pf_paged_fork", c.ref, None, None, n, None)
        ok("pf_paged_copy", c.ref, None, None, n, None)


def test_pages_a_request_too_large():
    """Pages are given out in the list's order: behind an entry for which they run out, only entries that need none are served."""
    c = Cache(I8, 1, 1, 64, 16, 10, 5, 12)
    c.reserve([4], [10])
    c.reserve([0, 1, 4, 2], [10 * 16, 1, 6, 1])  # nine are free, the first asks for ten
    assert latched() == 8
    assert c.lens.tolist() == [0, 0, 0, 0, 16] and c.refs.tolist() == [1] + [0] * 9
    c.reserve([0, 1, 2], [13 * 16, 1, 1])  # more than a sequence holds: takes no one's place
    assert latched() == 8
    assert c.lens.tolist() == [0, 1, 1, 0, 16] and c.table[1, 0] == 1 and c.table[2, 0] == 2


def test_pages_free_leaves_a_length_that_is_none():
    c = Cache(I8, 1, 1, 64, 16, 12, 4, 4).place([20, 5, 64, 1])
    c.lens[0], c.lens[2] = -7, 65
    refs, table = c.refs.tolist(), c.table.tolist()
    c.free([0, 1, 2, 0])
    assert latched() == 1
    refs[table[1][0]] = 0
    table[1][0] = -1
    assert c.lens.tolist() == [-7, 0, 65, 1] and c.refs.tolist() == refs and c.table.tolist() == table


def test_pages_lengths_that_the_caller_lowers():
    """Rejected tokens are given back by a lower length: the sequence keeps its pages for the next ones."""
    c = Cache(I8, 1, 1, 64, 16, 12, 4, 4)
    c.table.copy_(ints([[3, 7, 1, 9], [0, 0, 0, 0], [11, 10, 9, 8], [2, 4, 6, 8]]))  # contents do not matter
    c.reserve([0], [14])
    for _ in range(9):  # 5 tokens into the second page and 4 of them back
        c.reserve([0], [5])
        assert c.table[0, :2].tolist() == [0, 1] and int(c.refs.sum()) == 2
        c.lens[0] -= 5
        c.reserve([0], [1])
        c.lens[0] -= 1
    assert c.lens.tolist() == [14, 0, 0, 0] and c.refs.tolist() == [1, 1] + [0] * 10
    c.reserve([0], [40])  # 54 tokens: two pages held, two more
    assert c.table[0].tolist() == [0, 1, 2, 3]
    c.lens[0] = 20  # pages 2 and 3 held behind the length, in a row that is full
    c.fork([0], [1])  # the child has what the length counts
    assert c.lens.tolist() == [20, 20, 0, 0] and c.refs.tolist() == [2, 1, 1, 1, 1] + [0] * 7
    assert c.table[1, :2].tolist() == [0, 4]
    c.free([1])
    assert c.refs.tolist() == [1, 1, 1, 1] + [0] * 8
    c.reserve([2, 3], [16, 17])  # pages 4, 5 and 6
    c.free([2])
    c.lens[3] = 3
    c.compact()  # the page behind a length moves with the others
    assert c.refs.tolist() == [1] * 6 + [0] * 6
    assert c.table[0].tolist() == [0, 1, 2, 3] and c.table[3, :2].tolist() == [5, 4]
    c.reserve([3], [20])
    assert c.lens[3] == 23 and c.refs.tolist() == [1] * 6 + [0] * 6
    c.free([0, 3])
    assert c.lens.tolist() == [0, 0, 0, 0] and not c.refs.any()
    assert c.table[0].tolist() == [-1] * 4 and c.table[3, :2].tolist() == [-1, -1]
    assert latched() == 0


class Held(Model):
    """The model where a sequence may hold more pages than its length asks for."""

    def reserve(self, seqs, counts):
        asked, free, flags = 0, [i for i, r in enumerate(self.refs) if r == 0], 0
        for s, n in zip(seqs, counts):
            total = -(-(self.lens[s] + n) // self.c.page)
            if total > self.c.max_pages:
                flags |= 8
                continue
            need = max(total - len(self.table[s]), 0)
            mine = free[asked:asked + need]
            asked += need
            if len(mine) < need:
                flags |= 8
                continue
            for p in mine:
                self.refs[p] = 1
            self.table[s] += mine
            self.lens[s] += n
        return flags

    def fork(self, parents, children):
        held = {p: self.table[p] for p in parents}
        for p in held:
            self.table[p] = held[p][:-(-self.lens[p] // self.c.page)]
        flags = super().fork(parents, children)
        for p in held:
            self.table[p] = held[p]
        return flags


@pytest.mark.parametrize("dtype,layers,kv_heads,page,pages,seqs,max_pages", [(I8, 2, 2, 16, 60, 9, 7), (F16, 1, 1, 32, 900, 40, 300)])
def test_pages_follow_the_model_with_lengths_lowered(dtype, layers, kv_heads, page, pages, seqs, max_pages):
    """Random operations, some lengths lowered between them (never into a page that a fork has shared)."""
    c = Cache(dtype, layers, kv_heads, 64, page, pages, seqs, max_pages)
    m, rng = Held(c), random.Random(pages)
    c.table.copy_(ints([[rng.randrange(pages) for _ in range(max_pages)] for _ in range(seqs)]))
    for step in range(150):
        used = [s for s in range(seqs) if m.lens[s]]
        empty = [s for s in range(seqs) if not m.lens[s]]
        op = rng.choice(["reserve", "reserve", "reserve", "lower", "lower", "fork", "fork", "free", "compact"])
        flags = 0
        if op == "reserve":
            some = rng.sample(range(seqs), rng.randint(1, seqs))
            counts = [rng.choice([0, 1, 5, page, rng.randint(0, 4 * page), rng.randint(0, max_pages * page)]) for _ in some]
            c.reserve(some, counts)
            flags = m.reserve(some, counts)
        elif op == "lower" and used:
            for s in rng.sample(used, rng.randint(1, len(used))):
                shared = sum(m.refs[p] > 1 for p in m.table[s])
                m.lens[s] = rng.randint(min(max(1, shared * page), m.lens[s]), m.lens[s])
            c.lens.copy_(ints(m.lens))
        elif op == "fork" and used and empty:
            kids = rng.sample(empty, rng.randint(1, len(empty)))
            par = [rng.choice(used) for _ in kids]
            c.fork(par, kids)
            flags = m.fork(par, kids)
        elif op == "free" and used:
            some = rng.sample(used, rng.randint(1, max(1, len(used) // 2)))
            c.free(some)
            m.free(some)
        elif op == "compact":
            c.compact()
            m.compact()
        m.same()
        assert latched() == flags, (step, op)
    c.free(list(range(seqs)))
    assert not c.refs.any() and latched() == 0


def test_pages_many_held_behind_a_length():
    """A whole context reserved at once and given back: the next tokens' room does not take a walk past all of its pages."""
    c = Cache(I8, 1, 1, 64, 16, 90_000, 2, 88_000, fill=False)
    c.reserve([0, 1], [85_000 * 16, 5])
    c.lens[0] = 1
    seqs, counts = ints([0, 1]), ints([0, 1])

    def call():
        ok("pf_paged_reserve", c.ref, seqs.data_ptr(), counts.data_ptr(), 2, ph.stream())

    ms = elapsed(call)
    assert ms < 0.5, ms
    c.reserve([0], [32])
    assert c.lens.tolist() == [33, 7] and int(c.refs.sum()) == 85_001
    c.reserve([0], [85_000 * 16])  # three pages more than it holds
    assert int(c.lens[0]) == 85_000 * 16 + 33 and int(c.refs.sum()) == 85_004
    assert c.table[0, 85_000:85_004].tolist() == [85_001, 85_002, 85_003, -1]
    c.free([0, 1])
    assert not c.refs.any() and latched() == 0


def test_store_does_not_write_a_shared_page():
    """A sequence that got no room, or whose length was lowered into a page that a fork shares: bit 1, the page stays."""
    for cache in (I8, F16):
        c = Cache(cache, 1, 2, 64, 16, 4, 3, 4)
        c.reserve([0, 1], [32, 32])
        c.free([1])
        c.fork([0], [1])
        c.reserve([2], [32])
        c.reserve([1], [1])
        assert latched() == 8 and c.lens.tolist() == [32, 32, 32]
        x = randn((2, 128), TYPES[F32], 3)
        want = [t.clone() for t in (c.k, c.v)]
        c.store(0, x, x, [0, 0, 1], F32)  # position 31 of a page that sequence 0 holds as well
        assert latched() == 1
        assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
        c.lens[1] = 20
        c.store(0, x, x, [0, 0, 2], F32)
        assert latched() == 1
        assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
        c.free([0])  # now the pages are sequence 1's alone
        c.store(0, x, x, [0, 0, 2], F32)
        assert latched() == 0
        page = int(c.table[1, 1])
        if cache == F16:
            assert torch.equal(c.k[page, 0, :, 2:4], x.half().view(2, 2, 64).transpose(0, 1))
        else:
            assert not torch.equal(c.k[page, 0, :, 2:4], want[0][page, 0, :, 2:4])
        assert torch.equal(c.k[page, 0, :, 4:], want[0][page, 0, :, 4:])


def test_pages_compact_and_a_page_that_no_one_holds():
    """A table that names a free page behind those in use: bit 1, and the entry stays."""
    c = Cache(I8, 1, 1, 64, 16, 12, 3, 4)
    c.work.fill_(7)
    c.reserve([0, 1, 2], [32, 32, 32])
    c.free([0])
    c.table[1, 1] = 9
    c.compact()
    assert latched() == 1
    assert c.table[1, :2].tolist() == [2, 9] and c.table[2, :2].tolist() == [0, 1]


# ---------------------------------------------------------------------------
# Store
# ---------------------------------------------------------------------------
def store_codes(x):
    """(codes, scales) of rows [..][dim], by numpy in fp32, each step rounded once."""
    x = x.float().cpu().numpy()
    big = np.abs(x).max(-1)
    one = np.float32(1)
    scale = np.where(big == 0, one, big / np.float32(127)).astype(np.float32)
    mul = np.where(big == 0, one, np.float32(127) / np.where(big == 0, one, big)).astype(np.float32)
    y = x * mul[..., None]
    low = np.floor(np.abs(y))
    return (np.sign(y) * (low + (np.abs(y) - low >= np.float32(0.5)))).astype(np.int8), scale


@pytest.mark.parametrize("rows", [F32, BF16, F16])
@pytest.mark.parametrize("cache,dim,kv_heads,page,layers", [(I8, 64, 2, 16, 2), (I8, 128, 3, 64, 1), (I8, 64, 8, 128, 1),
                                                            (BF16, 64, 5, 32, 2), (F16, 128, 1, 16, 1)])
@pytest.mark.parametrize("new", [[1], [5, 0, 3, 17, 1], [0, 40, 0, 0, 129]])
def test_store(rows, cache, dim, kv_heads, page, layers, new):
    if cache != I8 and rows not in (F32, cache):
        pytest.skip("refused")
    before = [(7 * i) % 50 for i in range(len(new))]
    total = [a + b for a, b in zip(before, new)]
    c = Cache(cache, layers, kv_heads, dim, page, 80, len(new) + 1, 12).place(total)
    start, pad = 2, 3  # rows before the first sequence and behind the last one
    off = offsets_of(new, start)
    width = kv_heads * dim
    both = randn((off[-1] + pad, 2 * width + 16), TYPES[rows], sum(new) + dim)
    k, v = both[:, 16:16 + width], both[:, 16 + width:]
    k[start, :dim] = 0  # a row of zeros
    want = [x.clone() for x in (c.k, c.v) + ((c.ks, c.vs) if cache == I8 else ())]
    table, layer = c.table.tolist(), layers - 1
    for b in range(len(new)):
        for r in range(new[b]):
            pos = before[b] + r
            at = (table[b][pos // page], layer, slice(None), pos % page)
            for i, x in enumerate((k, v)):
                row = x[off[b] + r].view(kv_heads, dim)
                if cache == I8:
                    code, scale = store_codes(row)
                    want[i][at] = torch.from_numpy(code).cuda()
                    want[2 + i][at] = torch.from_numpy(scale).cuda()
                else:
                    want[i][at] = row.to(TYPES[cache])
    c.store(layer, k, v, off, rows)
    torch.cuda.synchronize()
    for x, y in zip((c.k, c.v, c.ks, c.vs), want):
        assert torch.equal(x, y)


def test_store_halves_and_extremes():
    """Ties go away from zero; the largest and smallest values; a row with inf or NaN reads back as NaN."""
    c = Cache(I8, 1, 2, 64, 16, 4, 1, 2).place([5])
    k = torch.zeros(5, 128, device="cuda")
    k[0, :8] = torch.tensor([127.0, 0.5, -0.5, 1.5, -2.5, 126.5, 0.49999997, -127.0])
    k[0, 64:68] = torch.tensor([3e38, -1e38, 1e30, 0.0])
    k[1, 0], k[1, 70] = math.inf, math.nan
    k[2, 3], k[2, 64] = -math.inf, 1e-38
    k[3, :64] = 1e-45  # the largest value is the smallest there is
    v = k.flip(0).contiguous()
    c.store(0, k, v, [0, 5], F32)
    torch.cuda.synchronize()
    for x, codes, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
        p = int(c.table[0, 0])
        for t in range(5):
            for g in range(2):
                row = x[t, g * 64:(g + 1) * 64]
                if not torch.isfinite(row).all():
                    assert torch.isnan(scales[p, 0, g, t]) and not codes[p, 0, g, t].any()
                    continue
                with np.errstate(all="ignore"):
                    big = np.abs(row.cpu().numpy()).max()
                if big and not np.isfinite(np.float32(127) / big):  # 127 / 1e-45 is no fp32 number: codes saturate
                    assert scales[p, 0, g, t] == torch.tensor(float(big / np.float32(127)))
                    continue
                code, scale = store_codes(row)
                assert torch.equal(codes[p, 0, g, t].cpu(), torch.from_numpy(code)), (t, g)
                assert scales[p, 0, g, t].cpu() == torch.tensor(float(scale))
    assert c.k[int(c.table[0, 0]), 0, 0, 0, :8].tolist() == [127, 1, -1, 2, -3, 127, 0, -127]


@pytest.mark.parametrize("big", [5e-37, 2.0 ** -121, 1e-38, 3e-41, 1e-45])
def test_store_rows_of_tiny_values(big):
    """Rows whose 127 / largest passes fp32's range: the codes are those of the row times 2^64, the scale its own."""
    one = np.float32(big)
    parts = np.array([1, -1, 0, 0.5, -0.25, 0.9, -0.3, 0.004, 0.0039, -0.0], np.float32)
    row = np.resize(parts, 64) * one
    k = torch.from_numpy(np.stack([row, -row[::-1]])).cuda().contiguous()
    c = Cache(I8, 1, 1, 64, 16, 2, 1, 2).place([2])
    c.store(0, k, k, [0, 2], F32)
    torch.cuda.synchronize()
    page = int(c.table[0, 0])
    for t in range(2):
        x = k[t].cpu().numpy()
        code, _ = store_codes(torch.from_numpy(x * np.float32(2.0 ** 64)))
        assert np.abs(code).max() == 127
        for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
            assert torch.equal(codes[page, 0, 0, t].cpu(), torch.from_numpy(code))
            assert scales[page, 0, 0, t].cpu() == torch.tensor(np.abs(x).max() / np.float32(127))


def test_store_leaves_out_what_has_no_place():
    c = Cache(F16, 1, 1, 64, 16, 8, 3, 2).place([16, 20, 4])
    c.table[1, 1] = 99  # no such page
    c.lens[2] = 1       # fewer than the rows given
    want = c.k.clone()
    x = randn((9, 64), torch.float16, 3)
    c.store(0, x, x, [0, 2, 6, 9], F16)
    assert latched() == 1
    for r in range(2):
        want[int(c.table[0, 0]), 0, 0, 14 + r] = x[r]
    want[int(c.table[2, 0]), 0, 0, 0] = x[8]  # the last row is position 0; the two before it have none
    torch.cuda.synchronize()
    assert torch.equal(c.k, want)
    ok("pf_paged_store", c.ref, 0, None, 64, None, 64, F16, None, 0, 0, None)


def test_store_offsets_that_go_back():
    """Bit 1; the rows of sequences whose offsets are in order are where they belong, the others nowhere else."""
    c = Cache(F16, 1, 1, 64, 16, 8, 4, 2).place([8, 8, 8, 8])
    want = c.k.clone()
    x = randn((8, 64), torch.float16, 3)
    c.store(0, x, x, [0, 6, 4, 4, 8], F16)
    assert latched() == 1
    torch.cuda.synchronize()
    page = [int(p) for p in c.table[:, 0]]
    want[page[3], 0, 0, 4:8] = x[4:8]
    free = torch.ones_like(c.k, dtype=torch.bool)
    free[page[0], 0, 0, 2:8] = free[page[3], 0, 0, 4:6] = False  # (rows 4 and 5 are named by two)
    assert torch.equal(c.k[free], want[free])


def test_store_many_sequences():
    """Sequence search over 3,000 offsets, most of them of empty sequences."""
    rng = random.Random(1)
    new = [rng.choice([0, 0, 0, 1, 2]) for _ in range(3000)]
    c = Cache(BF16, 1, 1, 64, 16, 3000, 3000, 1).place([n if n else 0 for n in new])
    x = randn((sum(new), 64), torch.bfloat16, 5)
    c.store(0, x, x, offsets_of(new), BF16)
    torch.cuda.synchronize()
    table, at = c.table.tolist(), 0
    for b, n in enumerate(new):
        if n:
            assert torch.equal(c.v[table[b][0], 0, 0, :n], x[at:at + n]), b
        at += n


@pytest.mark.parametrize("cache,rows,dim,kv_heads", [(I8, F32, 64, 8), (I8, BF16, 128, 3), (I8, F16, 64, 1), (BF16, F32, 64, 2), (F16, F16, 128, 5)])
def test_store_many_tokens(cache, rows, dim, kv_heads):
    """A whole batch's prompts, for which a CTA takes more tokens: empty sequences, ends inside a CTA's tokens."""
    rng = random.Random(dim + kv_heads)
    new = [rng.choice([0, 0, 1, 7, 16, rng.randint(1, 90)]) for _ in range(320)]
    before = [rng.randint(0, 40) if n else 0 for n in new]
    total = [a + b for a, b in zip(before, new)]
    c = Cache(cache, 2, kv_heads, dim, 16, sum(-(-x // 16) for x in total) + 3, 320, 9).place(total)
    off, tokens = offsets_of(new), sum(new)
    assert tokens > 2368
    k, v = (randn((tokens, kv_heads * dim), TYPES[rows], i) for i in (1, 2))
    want = [x.clone() for x in (c.k, c.v) + ((c.ks, c.vs) if cache == I8 else ())]
    seq = torch.repeat_interleave(torch.arange(320), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)]).cuda()
    page, slot = c.table[seq, pos // 16].long(), pos % 16
    for i, x in enumerate((k, v)):
        row = x.view(tokens, kv_heads, dim)
        if cache == I8:
            code, scale = store_codes(row)
            want[i][page, 1, :, slot] = torch.from_numpy(code).cuda()
            want[2 + i][page, 1, :, slot] = torch.from_numpy(scale).cuda()
        else:
            want[i][page, 1, :, slot] = row.to(TYPES[cache])
    c.store(1, k, v, off, rows)
    torch.cuda.synchronize()
    for x, y in zip((c.k, c.v, c.ks, c.vs), want):
        assert torch.equal(x, y)


def elapsed(f):
    f()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b)


def test_store_among_very_many_empty_sequences():
    """Two tokens a million sequences apart: found by halving, not by a walk past each of them (30 ms)."""
    n = 1 << 20
    c = Cache(F16, 1, 1, 64, 16, 4, n, 1)
    busy = [0, 5, n // 2, n - 1]
    for i, b in enumerate(busy):
        c.table[b, 0] = i
        c.lens[b] = 3
    c.refs.fill_(1)
    new = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    for b in busy:
        new[b + 1:] += 1
    x = randn((6, 64), torch.float16, 3)  # (rows behind the last sequence's stay out)
    want = c.k.clone()
    for i in range(4):
        want[i, 0, 0, 2] = x[i]

    def call():
        ok("pf_paged_store", c.ref, 0, x.data_ptr(), 64, x.data_ptr(), 64, F16, new.data_ptr(), n, 6, ph.stream())

    ms = elapsed(call)
    assert torch.equal(c.k, want)
    assert ms < 2.0, ms
    new[n // 2 + 7] = 1  # goes back, far from any CTA's own tokens
    call()
    assert latched() == 1


# ---------------------------------------------------------------------------
# Attention over the cache
# ---------------------------------------------------------------------------
def attend(c, t, n_seqs, rows, heads, layer=0, seed=3, by=1.5, work=None, out=None):
    q = randn((n_seqs * rows, heads * c.dim), TYPES[t], seed, by)
    out = torch.full_like(q, math.nan) if out is None else out
    c.attend(layer, q, out, t, n_seqs, rows, heads, c.dim ** -0.5, work)
    torch.cuda.synchronize()
    check(out, c.attention(layer, q, n_seqs, rows, heads, c.dim ** -0.5), TYPES[t])
    return q, out


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 200]


@pytest.mark.parametrize("rows", [1, 2, 5, 8])
@pytest.mark.parametrize("group", [1, 3, 4])
@pytest.mark.parametrize("cache,t,dim,page", [(I8, F32, 64, 16), (I8, F32, 128, 64), (I8, BF16, 64, 32), (I8, F16, 128, 128),
                                              (BF16, BF16, 64, 64), (BF16, BF16, 128, 16), (F16, F16, 64, 128),
                                              (F16, F16, 128, 32)])
def test_attention(cache, t, dim, page, group, rows):
    c = Cache(cache, 2, 2, dim, page, 140, len(EDGES), 14).place(EDGES)
    attend(c, t, len(EDGES), rows, 2 * group, layer=1)


@pytest.mark.parametrize("cache,t,dim", [(I8, F32, 64), (I8, F32, 128), (I8, BF16, 128), (BF16, BF16, 128), (F16, F16, 64)])
@pytest.mark.parametrize("kv_heads,group", [(1, 8), (1, 16), (8, 1), (2, 7), (1, 40), (3, 2)])
def test_attention_head_layouts(cache, t, dim, kv_heads, group):
    c = Cache(cache, 1, kv_heads, dim, 32, 60, 4, 30).place([333, 2, 900, 90])
    for rows in (1, 8):
        attend(c, t, 4, rows, kv_heads * group)


@pytest.mark.parametrize("cache,t", [(I8, F32), (I8, F16), (BF16, BF16), (F16, F16)])
def test_attention_long(cache, t):
    """Rows long enough to be split many ways, beside short ones."""
    c = Cache(cache, 1, 2, 64, 64, 1500, 5, 1100).place([70_001, 3, 0, 12_345, 640])
    for rows in (1, 4):
        attend(c, t, 5, rows, 8)
    c = Cache(cache, 1, 1, 128, 16, 2100, 1, 2100).place([33_333])
    attend(c, t, 1, 1, 1)


@pytest.mark.parametrize("seqs", [1, 2, 64, 300])
def test_attention_batches(seqs):
    rng = random.Random(seqs)
    lens = [rng.randint(0, 150) for _ in range(seqs)]
    c = Cache(I8, 1, 2, 64, 16, 10 * seqs + 1, seqs, 10).place(lens)
    attend(c, F32, seqs, 1, 8)
    c = Cache(BF16, 1, 2, 64, 16, 10 * seqs + 1, seqs, 10).place(lens)
    attend(c, BF16, seqs, 3, 4)


def test_attention_one_work_for_many_shapes():
    """Calls of other shapes one after another on one workspace."""
    big = Cache(I8, 1, 8, 64, 16, 900, 8, 300).place([4000, 1, 77, 3000, 0, 500, 2000, 900])
    small = Cache(F16, 1, 1, 128, 128, 40, 2, 30).place([3800, 9])
    work = torch.cat([big.work_for(8, 8, 64), small.work_for(2, 1, 4)])
    for _ in range(3):
        attend(big, F32, 8, 8, 64, work=work)
        attend(small, F16, 2, 1, 4, work=work)
        attend(big, F32, 3, 1, 32, work=work)
        attend(small, F16, 1, 8, 1, work=work)


def test_attention_scores_of_all_sizes():
    """Scores so large that one entry takes the row, and so small that all entries are alike."""
    for by in (40.0, 1e-3, 0.0):
        for cache, t in ((I8, F32), (BF16, BF16)):
            c = Cache(cache, 1, 1, 64, 16, 60, 2, 40).place([500, 37])
            attend(c, t, 2, 3, 4, by=by)


@pytest.mark.parametrize("n_seqs,heads,kv_heads,rows", [(95, 2, 1, 1), (96, 2, 1, 1), (159, 2, 2, 1), (160, 4, 4, 1), (500, 1, 1, 2),
                                                        (1030, 1, 1, 1)])
@pytest.mark.parametrize("cache,t", [(I8, F32), (BF16, BF16)])
def test_attention_many_sequences(cache, t, n_seqs, heads, kv_heads, rows):
    """As many as have their pieces planned by a launch of its own, and a few less; empty ones, long ones, one that is none."""
    rng = random.Random(n_seqs)
    lens = [rng.choice([0, 1, rng.randint(2, 60), rng.randint(60, 130)]) for _ in range(n_seqs)]
    lens[0], lens[n_seqs // 2], lens[-1] = 3000, 700, 1900
    c = Cache(cache, 1, kv_heads, 64, 16, sum(-(-n // 16) for n in lens), n_seqs, 200).place(lens)
    work = c.work_for(n_seqs, 8, heads)
    attend(c, t, n_seqs, rows, heads, work=work)
    attend(c, t, 5, rows, heads, work=work)  # the same work for a few
    attend(c, t, n_seqs, rows, heads, work=work, seed=9)
    assert latched() == 0
    c.lens[7] = 200 * 16 + 1
    q = randn((n_seqs * rows, heads * 64), TYPES[t], 3)
    out = torch.empty_like(q)
    c.attend(0, q, out, t, n_seqs, rows, heads, 0.125, work)
    assert latched() == 1
    c.lens[7] = 0
    check(out, c.attention(0, q, n_seqs, rows, heads, 0.125), TYPES[t])


def test_attention_many_sequences_in_a_graph():
    """The plan is made anew at every replay, on lengths that have changed, and again on another stream."""
    n = 170
    c = Cache(BF16, 1, 2, 64, 16, n * 12, n, 12).place([12 * 16] * n)
    q = randn((n, 4 * 64), torch.bfloat16, 5)
    out, work = torch.empty_like(q), c.work_for(n, 1, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, q, out, BF16, n, 1, 4, 0.125, work)
    rng, other = random.Random(3), torch.cuda.Stream()
    for most in (1, 60, 12 * 16):
        c.lens.copy_(ints([rng.randint(0, most) for _ in range(n - 1)] + [12 * 16]))
        out.fill_(7)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other if most == 60 else torch.cuda.current_stream()):
            for _ in range(3):
                graph.replay()
        torch.cuda.synchronize()
        check(out, c.attention(0, q, n, 1, 4, 0.125), torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 4])
def test_attention_numbers_near_the_largest(rows):
    """fp32 queries and int8 scales of 2^112 and more: the powers of two that take them into fp16's range reach there."""
    c = Cache(I8, 1, 1, 64, 16, 40, 2, 30).place([12, 37])
    c.ks *= 2.0 ** 6
    c.vs *= 2.0 ** 118
    q = randn((2 * rows, 4 * 64), torch.float32, 3, 2.0 ** 118)
    out = torch.empty_like(q)
    c.attend(0, q, out, F32, 2, rows, 4, 2.0 ** -125)
    torch.cuda.synchronize()
    check(out, c.attention(0, q, 2, rows, 4, 2.0 ** -125), torch.float32)


@pytest.mark.parametrize("cache,t", [(I8, F32), (I8, BF16), (BF16, BF16), (F16, F16)])
def test_attention_rows_of_unlike_sizes(cache, t):
    """A head whose queries are large, small or no numbers leaves the heads beside it as they are."""
    c = Cache(cache, 1, 1, 64, 16, 40, 2, 30).place([400, 21])
    q = randn((4, 8 * 64), TYPES[t], 3)
    plain, out = torch.empty_like(q), torch.empty_like(q)
    c.attend(0, q, plain, t, 2, 2, 8, 0.125)
    q.view(4, 8, 64)[:, 1] *= 1e-4
    q.view(4, 8, 64)[:, 2] *= 3e3
    q.view(4, 8, 64)[:, 4, 9] = math.inf
    q.view(4, 8, 64)[:, 5, 3] = math.nan
    q.view(4, 8, 64)[:, 7] = 0
    if t != F16:
        q.view(4, 8, 64)[:, 6] *= 1e18
    c.attend(0, q, out, t, 2, 2, 8, 0.125)
    torch.cuda.synchronize()
    a, b = out.view(4, 8, 64), plain.view(4, 8, 64)
    assert torch.equal(a[:, [0, 3]], b[:, [0, 3]])
    assert torch.isnan(a[:, 5]).all()
    few = [0, 1, 3, 7]
    want = c.attention(0, torch.nan_to_num(q, 0, 0, 0), 2, 2, 8, 0.125)
    check(a[:, few].contiguous(), tuple(x[:, few] for x in want), TYPES[t])


@pytest.mark.parametrize("cache,t", [(I8, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("rows", [1, 4])
def test_attention_does_not_read_behind_the_end(cache, t, rows):
    """NaN and inf in slots behind a sequence's length, in pages that are not its own, and in what a row may not see."""
    lens = [1, 16, 40, 333]
    c = Cache(cache, 1, 2, 64, 16, 80, 4, 40).place(lens)
    clean = Cache(cache, 1, 2, 64, 16, 80, 4, 40).place(lens)
    used = torch.zeros(80, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for p in range(n):
            used[c.table[b, p // 16], p % 16] = True
    for x in (c.k, c.v) if cache != I8 else (c.ks, c.vs):
        x.movedim(3, 1)[~used] = math.nan
    q = randn((4 * rows, 8 * 64), TYPES[t], 3)
    out, ref = torch.empty_like(q), torch.empty_like(q)
    c.attend(0, q, out, t, 4, rows, 8, 0.125)
    clean.attend(0, q, ref, t, 4, rows, 8, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    if rows == 1:
        return
    # the newest position's value: only the last row of its sequence sees it
    b, n = 3, lens[3]
    page, slot = int(c.table[b, (n - 1) // 16]), (n - 1) % 16
    for bad in (math.inf, math.nan):
        (c.v if cache != I8 else c.vs)[page, 0, :, slot] = bad
        (c.k if cache != I8 else c.ks)[page, 0, :, slot] = bad
        c.attend(0, q, out, t, 4, rows, 8, 0.125)
        torch.cuda.synchronize()
        assert torch.equal(out[:-1], ref[:-1]), bad
        assert torch.isnan(out[-1]).all()


def test_attention_infinities_of_its_own():
    """An inf among a row's own values, and a score of -inf, as the definition has them."""
    c = Cache(BF16, 1, 1, 64, 16, 8, 1, 4).place([50])
    page = int(c.table[0, 1])
    q = randn((1, 64), torch.bfloat16, 1)
    out = torch.empty_like(q)
    c.v[page, 0, 0, 3, 7] = math.inf
    c.attend(0, q, out, BF16, 1, 1, 1, 0.125)
    torch.cuda.synchronize()
    assert out[0, 7] == math.inf and torch.isfinite(out[0, :7]).all() and torch.isfinite(out[0, 8:]).all()
    c.v[page, 0, 0, 3, 7] = 0
    c.k[page, 0, 0, 3] = 0
    c.k[page, 0, 0, 3, 0] = math.inf
    q[0, 0] = -1
    c.attend(0, q, out, BF16, 1, 1, 1, 0.125)
    torch.cuda.synchronize()
    k, v = c.history(0, 0, 0)
    keep = [i for i in range(50) if i != 19]
    want = ph.softmax_mean(q[0].double() @ k[keep].T * 0.125, v[keep])
    check(out, (want.view(1, 1, 64), v.abs().amax().view(1, 1, 1), (q.double().abs() @ k[keep].abs().T * 0.125).max().view(1, 1, 1)),
          torch.bfloat16)


def test_attention_pages_and_lengths_that_are_none():
    c = Cache(I8, 1, 2, 64, 16, 60, 4, 8).place([100, 100, 100, 100])
    q = randn((4, 512), torch.float32, 1)
    ref, out = torch.empty_like(q), torch.empty_like(q)
    c.attend(0, q, ref, F32, 4, 1, 8, 0.125)
    c.table[0, 3], c.table[1, 2] = 60, -1
    c.lens[2] = 129  # more than a sequence can hold
    c.attend(0, q, out, F32, 4, 1, 8, 0.125)
    assert latched() == 1
    assert torch.equal(out[3], ref[3])
    assert torch.isfinite(out).all()
    assert not out[2].any()


def test_attention_strides():
    c = Cache(BF16, 1, 2, 64, 16, 60, 3, 20).place([100, 7, 300])
    wide = randn((6, 4 * 64 + 200), torch.bfloat16, 2)
    q = wide[:, 8:8 + 256]
    out = torch.full((6, 4 * 64 + 40), 7.0, dtype=torch.bfloat16, device="cuda")
    c.attend(0, q, out[:, 16:272], BF16, 3, 2, 4, 0.125)
    torch.cuda.synchronize()
    check(out[:, 16:272], c.attention(0, q.contiguous(), 3, 2, 4, 0.125), torch.bfloat16)
    assert (out[:, :16] == 7).all() and (out[:, 272:] == 7).all()


def test_attention_far_pages():
    """Pages whose elements pass 2^31 and 2^32."""
    c = Cache(I8, 1, 8, 128, 128, 36_000, 2, 12, fill=False)
    c.k.fill_(99), c.v.fill_(99)
    pages = [35_999, 16_383, 16_384, 0, 32_768]
    c.table[0, :5] = ints(pages)
    c.lens.copy_(ints([600, 0]))
    for p in pages:
        c.k[p] = randn((1, 8, 128, 128), torch.float32, p, 40).clamp(-127, 127).to(torch.int8)
        c.v[p] = randn((1, 8, 128, 128), torch.float32, p + 1, 40).clamp(-127, 127).to(torch.int8)
    attend(c, F32, 1, 1, 8)
    x = randn((600, 8 * 128), torch.float32, 8)
    c.store(0, x, x, [0, 600], F32)
    attend(c, F32, 1, 1, 8)
    code, _ = store_codes(x.view(600, 8, 128))
    assert torch.equal(c.k[35_999, 0].transpose(0, 1).cpu(), torch.from_numpy(code[:128]))
    c.copy([35_999], [20_000])
    torch.cuda.synchronize()
    assert torch.equal(c.k[20_000], c.k[35_999]) and torch.equal(c.v[20_000], c.v[35_999])


def test_attention_in_graphs_and_streams():
    """Captured once and replayed as the cache grows; two streams at once, each with its own workspace."""
    c = Cache(I8, 1, 2, 64, 16, 400, 4, 80).place([10, 600, 0, 1200])
    q = randn((4, 512), torch.float32, 1)
    out = torch.empty_like(q)
    work = c.work_for(4, 1, 8)
    c.attend(0, q, out, F32, 4, 1, 8, 0.125, work)  # first call on this device outside the capture
    torch.cuda.synchronize()
    grow, one = ints([0, 1, 2, 3]), ints([1, 1, 1, 1])
    off = ints([0, 1, 2, 3, 4])
    new = randn((4, 128), torch.float32, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok("pf_paged_reserve", c.ref, grow.data_ptr(), one.data_ptr(), 4, ph.stream())
        ok("pf_paged_store", c.ref, 0, new.data_ptr(), 128, new.data_ptr(), 128, F32, off.data_ptr(), 4, 4, ph.stream())
        c.attend(0, q, out, F32, 4, 1, 8, 0.125, work)
    for i in range(20):
        new.copy_(randn((4, 128), torch.float32, 10 + i))
        q.copy_(randn((4, 512), torch.float32, 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert c.lens.tolist() == [11 + i, 601 + i, 1 + i, 1201 + i]
        check(out, c.attention(0, q, 4, 1, 8, 0.125), torch.float32)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    works = [c.work_for(4, 1, 8), c.work_for(4, 1, 8)]
    outs = [torch.empty_like(q), torch.empty_like(q)]
    torch.cuda.synchronize()
    for _ in range(50):
        for s, w, o in zip((a, b), works, outs):
            with torch.cuda.stream(s):
                c.attend(0, q, o, F32, 4, 1, 8, 0.125, w)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, out)


def test_attention_answers_do_not_depend_on_the_run():
    c = Cache(I8, 1, 4, 64, 16, 2000, 3, 1000).place([9000, 55, 14_000])
    q, first = attend(c, F32, 3, 2, 16)
    work = c.work_for(3, 2, 16)
    for _ in range(20):
        out = torch.empty_like(q)
        c.attend(0, q, out, F32, 3, 2, 16, 0.125, work)
        torch.cuda.synchronize()
        assert torch.equal(out, first)


@pytest.mark.parametrize("cache,t", [(I8, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows", [1, 5])
def test_attention_a_real_step(cache, t, rows):
    """64 sequences, 32 heads over 8, one token and a verify step's five."""
    rng = random.Random(rows)
    lens = [rng.randint(512, 1024) for _ in range(64)]
    c = Cache(cache, 1, 8, 64, 64, sum(-(-n // 64) for n in lens), 64, 16).place(lens)
    q = randn((64 * rows, 32 * 64), TYPES[t], 3, 1.5)
    out = torch.empty_like(q)
    c.attend(0, q, out, t, 64, rows, 32, 0.125)
    torch.cuda.synchronize()
    for b in range(64):
        for g in range(8):
            k, v = c.history(b, 0, g)
            at = (slice(b * rows, (b + 1) * rows), slice(4 * g, 4 * g + 4))
            x = q.view(-1, 32, 64)[at].double() @ k.T * 0.125  # [row][head][entry]
            seen = torch.arange(lens[b], device="cuda") < (lens[b] - rows + 1 + torch.arange(rows, device="cuda"))[:, None, None]
            p = torch.softmax(torch.where(seen, x, -math.inf), -1)
            big_s = (q.view(-1, 32, 64)[at].double().abs() @ k.abs().T * 0.125).amax(-1, keepdim=True)
            big_v = v.abs().max().expand(rows, 4, 1)
            check(out.view(-1, 32, 64)[at].contiguous(), (p @ v, big_v, big_s), TYPES[t])


def one_dim_keys(c, n, nats):
    """Sequence 0's keys have one dim other than 0, and queries of 8 there score `nats[j]` over key j at scale 1/8."""
    page, slot = c.table[0, torch.arange(n, device="cuda") // c.page].long(), torch.arange(n, device="cuda") % c.page
    c.k.zero_()
    if c.ks is None:
        c.k[page, 0, :, slot, 0] = nats.to(c.k.dtype)[:, None]
        return page, slot, c.k[page, 0, 0, slot, 0].double()
    c.k[page, 0, :, slot, 0] = (127 * nats.sign()).to(torch.int8)[:, None]
    c.ks[page, 0, :, slot] = (nats.abs() / 127)[:, None]
    return page, slot, c.ks[page, 0, 0, slot].double() * c.k[page, 0, 0, slot, 0].double()


@pytest.mark.parametrize("dim,rows", [(64, 1), (64, 3), (128, 1), (128, 5)])
@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("at,nats", [(0, 17.4), (0, 18.0), (40_000, 17.4), (65_529, 21.0), (0, 4.0)])
def test_attention_one_key_takes_nearly_all(cache, dim, rows, at, nats):
    """A key far above 65,535 others whose values are all that comes out: each weight is far below fp16's range beside the
    largest one, and together they are the answer."""
    n = 65_536
    c = Cache(cache, 1, 1, dim, 64, 1024, 1, 1024).place([n])
    scores = torch.zeros(n, device="cuda")
    scores[at] = nats
    page, slot, s = one_dim_keys(c, n, scores)
    c.v.copy_(torch.rand(c.v.shape, generator=torch.Generator("cuda").manual_seed(5), device="cuda") * 0.5 + 0.5)
    c.v[page[at], 0, 0, slot[at]] = 0
    q = torch.zeros(rows, 2 * dim, dtype=TYPES[cache], device="cuda")
    q[:, 0] = q[:, dim] = 8
    out = torch.empty_like(q)
    c.attend(0, q, out, cache, 1, rows, 2, 0.125)
    torch.cuda.synchronize()
    v = c.v[page, 0, 0, slot].double()
    # a weight and the output are rounded to the type (eps / 2 each; fp16 weights are 2^9 times what they are to the largest, so
    # those too small for its normal numbers are off by 2^-34 of it); 2^-16 of a weight for its score, which has one product
    # (31 x 2^-24 in each of four roundings at most), the exponential and the sums; fp16 outputs below 2^-14 are off by 2^-25
    half = torch.finfo(TYPES[cache]).eps / 2
    for r in range(rows):
        m = n - rows + 1 + r
        want = ph.softmax_mean(s[:m], v[:m])
        for h in range(2):
            got = out[r, h * dim:(h + 1) * dim].double()
            tol = (2 * half + 2.0 ** -16) * want + (2.0 ** -25 + m * 2.0 ** -34 if cache == F16 else 0.0)
            assert ((got - want).abs() <= tol).all(), ((got - want).abs() / want).max()


@pytest.mark.parametrize("cache,t,dim", [(F16, F16, 64), (F16, F16, 128), (BF16, BF16, 64), (I8, F32, 64), (I8, F32, 128),
                                         (I8, F16, 64)])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("nats", [16.4, 21.2])
def test_attention_a_few_keys_take_nearly_all_of_long_ones(cache, t, dim, rows, nats):
    """The same where a warp walks over a third or a quarter of a whole sequence: as many segments as CTAs, none of them cut,
    and keys far above the others among the first ones of every warp."""
    n, seqs, kv_heads = 65_536, 64, 8
    c = Cache(cache, 1, kv_heads, dim, 64, 1024, seqs, 1024).place([n])
    c.table.copy_(c.table[:1].expand(seqs, 1024).contiguous())  # every sequence has the same pages
    c.lens.fill_(n)
    scores, high = torch.full((n,), -1.0, device="cuda"), torch.tensor([0, 16, 32, 48, 64, 96], device="cuda")
    scores[high] = nats
    page, slot, s = one_dim_keys(c, n, scores)
    if cache == I8:
        c.v.fill_(100)
        c.vs.fill_(0.0123)
    else:
        c.v.fill_(0.75)
    c.v[page[high], 0, :, slot[high]] = 0
    q = torch.zeros(seqs * rows, kv_heads * dim, dtype=TYPES[t], device="cuda")
    q[:, ::dim] = 8
    out = torch.empty_like(q)
    c.attend(0, q, out, t, seqs, rows, kv_heads, 0.125)
    torch.cuda.synchronize()
    v = c.v[page, 0, 0, slot, 0].double() * (c.vs[page, 0, 0, slot].double() if cache == I8 else 1)
    # beside the weights' and the output's rounding: fp16 weights too small for its normal numbers are off by 2^-34 of the
    # largest, int8 ones (with their scales, all alike) by 2^-33, and there are six of the largest.  2^-15 of a weight for its
    # score (23 x 1.44 x 2^-24 in each of four roundings), exponential and sums
    half = torch.finfo(TYPES[t]).eps / 2
    for r in range(rows):
        m = n - rows + 1 + r
        want = ph.softmax_mean(s[:m], v[:m, None])
        got = out.view(seqs, rows, -1)[:, r].double()
        tol = (2.0 ** -15 + half) * want + (2.0 ** -25 if t == F16 else 0.0)
        tol += m / 6 * v.max() * {I8: 2.0 ** -33, F16: 2.0 ** -34, BF16: 0.0}[cache] + (half * want if cache != I8 else 0.0)
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("dim,rows,group", [(64, 1, 4), (128, 1, 8), (64, 2, 4), (128, 2, 3), (64, 8, 1)])
def test_attention_weights_keep_more_than_16_bits(cache, dim, rows, group):
    """Up to eight rows a kv head over a 16-bit cache: the output's rounding is the only one to 16 bits."""
    c = Cache(cache, 1, 2, dim, 16, 400, 5, 200).place([40, 333, 7, 2900, 90])
    t, heads = TYPES[cache], 2 * group
    q = randn((5 * rows, heads * dim), t, 3)
    out = torch.empty_like(q)
    c.attend(0, q, out, cache, 5, rows, heads, dim ** -0.5)
    torch.cuda.synchronize()
    want, big_v, big_s = c.attention(0, q, 5, rows, heads, dim ** -0.5)
    # a weight's second plane is rounded to 16 bits: 2^-16 of the weight in bf16, 2^-21 in fp16, or 2^-24 of what is 2^9 for the
    # largest; scores, sums and exponentials as in tolerance()
    half = torch.finfo(t).eps / 2
    tol = (2.0 ** -17 * big_s + 2.0 ** -18 + 2.0 ** -16) * big_v + half * want.abs()
    d = (out.double().view_as(want) - want).abs()
    assert (d <= tol).all(), (d / tol).max()


@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 1), (64, 2), (128, 2), (64, 5)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_attention_an_infinity_stays_one(cache, dim, rows, bad):
    """An inf among the values of any entry, whatever part of its weight a plane holds: that dim of the rows that see it."""
    n, heads = 150, 4
    c = Cache(cache, 1, 1, dim, 16, 40, 1, 20).place([n])
    q = randn((rows, heads * dim), TYPES[cache], 3, 0.5)
    q[:, :dim] = 0  # weights that are powers of two: nothing is left for a second plane
    for at in range(0, n, 7):
        page, slot = int(c.table[0, at // 16]), at % 16
        c.v[page, 0, 0, slot, at % dim] = bad
    out = torch.empty_like(q)
    c.attend(0, q, out, cache, 1, rows, heads, dim ** -0.5)
    torch.cuda.synchronize()
    got = out.view(rows, heads, dim)
    for r in range(rows):
        hit = sorted({at % dim for at in range(0, n, 7) if at < n - rows + 1 + r})
        assert (got[r][:, hit] == bad).all()
        rest = [d for d in range(dim) if d not in hit]
        assert torch.isfinite(got[r][:, rest]).all()


# ---------------------------------------------------------------------------
# Prompt attention
# ---------------------------------------------------------------------------
def run_prompt(t, dim, heads, kv_heads, lens, fused=False, start=0, behind=0, by=1.0, seed=0):
    off = offsets_of(lens, start)
    n = off[-1] + behind
    cols = [heads * dim, kv_heads * dim, kv_heads * dim]
    if fused:
        q, k, v = randn((n, sum(cols) + 24), TYPES[t], seed, by)[:, 8:8 + sum(cols)].split(cols, dim=1)
    else:
        q, k, v = (randn((n, w), TYPES[t], seed + i, by) for i, w in enumerate(cols))
    out = torch.full((n, cols[0] + (16 if fused else 0)), 5.0, dtype=TYPES[t], device="cuda")[:, :cols[0]]
    o = ints(off)
    prompt(q, k, v, out, t, o, len(lens), n, heads, kv_heads, dim)
    torch.cuda.synchronize()
    assert (out[:start] == 5).all() and (out[off[-1]:] == 5).all()
    want = ph.prompt(q, k, v, off, heads, kv_heads, dim, dim ** -0.5)
    rows = slice(start, off[-1])
    check(out[rows].contiguous(), tuple(x[rows] for x in want), TYPES[t])
    return q, k, v, out


def prompt(q, k, v, out, t, offsets, n_seqs, n, heads, kv_heads, dim):
    ok("pf_prompt_attention", q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
       out.data_ptr(), out.stride(0), t, offsets.data_ptr(), n_seqs, n, heads, kv_heads, dim, dim ** -0.5, ph.stream())


LENS = [[1], [128], [129], [127, 1, 0, 2], [0, 0, 64, 0], [255, 256, 257], [700], [5] * 40, [384, 1, 500]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("t,dim,heads,kv_heads", [(BF16, 64, 4, 2), (F16, 128, 3, 1), (BF16, 128, 2, 2), (F16, 64, 7, 1)])
def test_prompt(t, dim, heads, kv_heads, lens):
    run_prompt(t, dim, heads, kv_heads, lens)
    run_prompt(t, dim, heads, kv_heads, lens, fused=True, start=3, behind=70)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (5, 1), (12, 4), (32, 8), (33, 3)])
@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128)])
def test_prompt_head_layouts(t, dim, heads, kv_heads):
    run_prompt(t, dim, heads, kv_heads, [300, 17])


@pytest.mark.parametrize("heads,kv_heads", [(6, 1), (16, 1), (24, 2), (32, 1), (64, 1), (40, 1)])
@pytest.mark.parametrize("t,dim", [(F16, 64), (BF16, 128)])
def test_prompt_groups(t, dim, heads, kv_heads):
    """Tiles of 2 to 32 heads: sequences that end and begin anywhere in them, values that a head's rows may not see."""
    lens = [1, 3, 4, 5, 31, 33, 63, 65, 130]
    q, k, v, out = run_prompt(t, dim, heads, kv_heads, lens, fused=True, behind=9)
    v = v.contiguous()
    v[sum(lens) - 1] = math.nan  # the last token's
    again = out.clone()
    prompt(q, k, v, again, t, ints(offsets_of(lens)), len(lens), q.shape[0], heads, kv_heads, dim)
    torch.cuda.synchronize()
    n = sum(lens)
    want = ph.prompt(q, k, torch.nan_to_num(v, 0), offsets_of(lens), heads, kv_heads, dim, dim ** -0.5)
    check(again[:n - 1].contiguous(), tuple(x[:n - 1] for x in want), TYPES[t])
    assert torch.isnan(again[n - 1]).all()


@pytest.mark.parametrize("t,dim", [(BF16, 64), (BF16, 128), (F16, 64), (F16, 128)])
def test_prompt_long(t, dim):
    run_prompt(t, dim, 2, 1, [2500, 4097])


def test_prompt_scores_of_all_sizes():
    """Rows whose largest score keeps rising, and scores all alike."""
    for t in (BF16, F16):
        for by in (6.0, 1e-3):
            run_prompt(t, 64, 4, 2, [600, 3], by=by)
    n, dim = 1200, 64
    q = torch.ones(n, dim, device="cuda").half()
    k = (torch.arange(n, device="cuda")[:, None] / 40 * torch.ones(dim, device="cuda")).half()  # scores rise by 0.2 an entry
    v = randn((n, dim), torch.float16, 4)
    out = torch.empty_like(q)
    prompt(q, k, v, out, F16, ints([0, n]), 1, n, 1, 1, dim)
    torch.cuda.synchronize()
    check(out, ph.prompt(q, k, v, [0, n], 1, 1, dim, dim ** -0.5), torch.float16)


@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_prompt_does_not_mix_what_is_masked(t, dim, bad):
    """inf and NaN in a later position's key and value, and in another sequence, reach no row that may not see them."""
    heads, kv_heads, lens = 4, 2, [200, 150, 131]
    q, k, v, ref = run_prompt(t, dim, heads, kv_heads, lens)
    k, v = k.clone(), v.clone()
    for where in (60, 190, 345):  # positions 60 and 190 of the first sequence, 145 of the second
        k[where], v[where] = bad, bad
    out = torch.empty_like(ref)
    prompt(q, k, v, out, t, ints(offsets_of(lens)), 3, q.shape[0], heads, kv_heads, dim)
    torch.cuda.synchronize()
    fine = [*range(0, 60), *range(200, 345), *range(350, 481)]
    want = ph.prompt(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), offsets_of(lens), heads, kv_heads,
                     dim, dim ** -0.5)
    check(out[fine].contiguous(), tuple(x[fine] for x in want), TYPES[t])
    # an inf in one dim of a value alone: that dim of the rows from there on
    k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    v[60, 5] = bad
    prompt(q, k, v, out, t, ints(offsets_of(lens)), 3, q.shape[0], heads, kv_heads, dim)
    torch.cuda.synchronize()
    assert torch.isfinite(out[:60]).all() and torch.isfinite(out[200:]).all()
    seen = out[60:200, [5, dim + 5]]
    assert (torch.isnan(seen) if math.isnan(bad) else seen == bad).all()
    others = out[60:200].view(140, heads, dim)[:, :, [i for i in range(dim) if i != 5]]
    assert torch.isfinite(others).all()


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 2), (8, 1), (6, 1), (33, 1)])
@pytest.mark.parametrize("t,dim", [(F16, 64), (BF16, 128)])
def test_prompt_infinities_of_its_own(t, dim, heads, kv_heads):
    """inf, -inf and NaN among the values of any block: each dim of a row takes what the row has seen of them."""
    lens, rng = [300, 9, 140], random.Random(heads)
    q, k, v, ref = run_prompt(t, dim, heads, kv_heads, lens, by=0.25)
    where = [(r, d) for r in (5, 64, 100, 127, 128, 200, 255, 299, 300, 308, 309, 400, 448)
             for d in rng.sample(range(kv_heads * dim), 3)] + [(60, 7), (130, 7), (280, 7)]
    v = v.clone()
    for i, (r, d) in enumerate(where):
        v[r, d] = (math.inf, -math.inf, math.nan)[i % 3]
    out = torch.empty_like(ref)
    prompt(q, k, v, out, t, ints(offsets_of(lens)), 3, q.shape[0], heads, kv_heads, dim)
    torch.cuda.synchronize()
    want, big_v, big_s = ph.prompt(q, k, torch.nan_to_num(v, 0, 0, 0), offsets_of(lens), heads, kv_heads, dim, dim ** -0.5)
    odd = torch.where(torch.isfinite(v.float()), 0.0, v.float()).view(-1, kv_heads, dim)
    seen = torch.cat([x.cumsum(0) for x in odd.split(lens)]).repeat_interleave(heads // kv_heads, 1)
    got, fine = out.view(-1, heads, dim).float(), seen == 0
    assert torch.equal(torch.isnan(got), torch.isnan(seen))
    assert torch.equal(got[torch.isinf(seen)], seen[torch.isinf(seen)])
    check(torch.where(fine, got, 0.0).to(TYPES[t]), (torch.where(fine, want, 0.0), big_v, big_s), TYPES[t])


def test_prompt_infinity_at_the_end_of_a_long_one():
    """An inf among the last tokens' values costs its rows a walk over their own block, not over the whole prompt."""
    n, dim = 100_000, 64
    q, k, v = (randn((n, dim), torch.bfloat16, i, 0.5) for i in range(3))
    v[n - 3, 11] = -math.inf
    out = torch.empty_like(q)
    prompt(q, k, v, out, BF16, ints([0, n]), 1, n, 1, 1, dim)
    torch.cuda.synchronize()
    assert latched() == 0
    assert torch.isfinite(out[:n - 3]).all() and (out[n - 3:, 11] == -math.inf).all()
    few, v0 = [0, 5000, n - 130, n - 3, n - 2, n - 1], torch.nan_to_num(v, 0, 0, 0).double()
    for i in few:
        x = q[i].double() @ k[:i + 1].double().T * dim ** -0.5
        want = ph.softmax_mean(x, v0[:i + 1])
        got = torch.where(torch.isfinite(out[i].float()), out[i].float(), want.float()).bfloat16()
        got[11] = want[11] if i >= n - 3 else got[11]
        check(got, (want.view(1, 1, dim), v0[:i + 1].abs().amax().view(1, 1, 1),
                    (q[i].double().abs() @ k[:i + 1].double().abs().T * dim ** -0.5).amax().view(1, 1, 1)), torch.bfloat16)


@pytest.mark.parametrize("t,dim,heads", [(F16, 64, 1), (F16, 64, 2), (F16, 128, 1), (BF16, 64, 1), (BF16, 128, 2)])
@pytest.mark.parametrize("at,nats", [(0, 17.4), (200, 18.0), (0, 4.0)])
def test_prompt_one_key_takes_nearly_all(t, dim, heads, at, nats):
    """A key far above all others whose values are all that comes out of the rows that see it."""
    n = 65_536
    q = torch.zeros(n, heads * dim, dtype=TYPES[t], device="cuda")
    q.view(n, heads, dim)[:, :, 0] = 8
    k = torch.zeros(n, dim, dtype=TYPES[t], device="cuda")
    k[at, 0] = nats
    v = (torch.rand(n, dim, generator=torch.Generator("cuda").manual_seed(5), device="cuda") * 0.5 + 0.5).to(TYPES[t])
    v[at] = 0
    out = torch.empty_like(q)
    ok("pf_prompt_attention", q.data_ptr(), q.stride(0), k.data_ptr(), dim, v.data_ptr(), dim, out.data_ptr(), out.stride(0),
       t, ints([0, n]).data_ptr(), 1, n, heads, 1, dim, 0.125, ph.stream())
    torch.cuda.synchronize()
    # a weight and the output are rounded to the type, and each of a row's products of 16 keys is added to 24 bits and may be
    # cut there (4,096 x 2^-23); scores and exponentials, and what is below fp16's normal numbers, as in the paged attention's
    half = torch.finfo(TYPES[t]).eps / 2
    for i in (300, 5_000, 33_333, n - 1):
        want = ph.softmax_mean(k[:i + 1, 0].double(), v[:i + 1].double())
        for h in range(heads):
            got = out[i, h * dim:(h + 1) * dim].double()
            tol = (2 * half + 2.0 ** -11 + 2.0 ** -16) * want + (2.0 ** -25 + i * 2.0 ** -34 if t == F16 else 0.0)
            assert ((got - want).abs() <= tol).all(), (i, ((got - want).abs() / want).max())


def test_prompt_many_sequences():
    rng = random.Random(2)
    run_prompt(BF16, 64, 2, 1, [rng.choice([0, 1, 2, 3, 9]) for _ in range(1500)])


def test_prompt_offsets_that_are_none():
    n, dim = 300, 64
    q, k, v = (randn((n, dim), torch.bfloat16, i) for i in range(3))
    out = torch.full_like(q, 5.0)
    prompt(q, k, v, out, BF16, ints([0, 100, 90, 200, 301]), 4, n, 1, 1, dim)  # the second goes back, the last passes the end
    assert latched() == 1
    for a, b in ((0, 100), (90, 200)):
        if a == 0:
            a, b = 0, 90  # rows 90..99 are the third sequence's too
        want = ph.prompt(q, k, v, [0, 100] if a == 0 else [90, 200], 1, 1, dim, dim ** -0.5)
        rows = list(range(a, b)) if a == 0 else list(range(100, 200))
        check(out[rows].contiguous(), tuple(x[rows] for x in want), torch.bfloat16)
    assert (out[200:] == 5).all()
    prompt(q, k, v, out, BF16, ints([0, 0]), 1, n, 1, 1, dim)
    prompt(q, k, v, out, BF16, ints([-5, 10]), 1, n, 1, 1, dim)
    assert latched() == 1
    ok("pf_prompt_attention", None, 64, None, 64, None, 64, None, 64, BF16, None, 0, 0, 1, 1, 64, 0.125, None)


def test_prompt_in_graphs_and_streams():
    lens = [500, 3, 260]
    n, heads, kv_heads, dim = sum(lens), 4, 2, 64
    q, k, v, ref = run_prompt(BF16, dim, heads, kv_heads, lens)
    off = ints(offsets_of(lens))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.empty_like(ref), torch.empty_like(ref)]
    torch.cuda.synchronize()
    for _ in range(30):
        for s, o in zip((a, b), outs):
            with torch.cuda.stream(s):
                prompt(q, k, v, o, BF16, off, 3, n, heads, kv_heads, dim)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(ref)
    with torch.cuda.graph(graph):
        prompt(q, k, v, out, BF16, off, 3, n, heads, kv_heads, dim)
    for new in ([500, 3, 260], [1, 700, 40], [0, 0, 763]):
        off.copy_(ints(offsets_of(new)))
        q.copy_(randn(q.shape, torch.bfloat16, sum(new) + new[0]))
        graph.replay()
        torch.cuda.synchronize()
        rows = slice(0, sum(new))
        want = ph.prompt(q, k, v, offsets_of(new), heads, kv_heads, dim, dim ** -0.5)
        check(out[rows], tuple(x[rows] for x in want), torch.bfloat16)


# ---------------------------------------------------------------------------
# All of them, as a server uses them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache,t,dim,page", [(BF16, BF16, 64, 16), (F16, F16, 128, 64), (I8, BF16, 64, 32)])
def test_a_run_of_them_together(cache, t, dim, page):
    """Prompts in, prompt attention and the cache agree; forks, steps of one and of five tokens, a free and a
    compaction in between; every step's attention is the definition's over the tokens fed so far."""
    heads, kv_heads, layers = 8, 2, 2
    c = Cache(cache, layers, kv_heads, dim, page, 120, 6, 20)
    lens = [page, 75, 1]
    off = offsets_of(lens)
    fed = {s: [[], []] for s in range(6)}

    def feed(seqs, counts, seed):
        """New tokens of the sequences, in every layer; returns their keys and values."""
        c.reserve(seqs, counts)
        rows = sum(counts)
        new = [0] * 6
        for s, n in zip(seqs, counts):
            new[s] = n
        both = []
        for layer in range(layers):
            k, v = (randn((rows, kv_heads * dim), TYPES[t], seed + 10 * layer + i) for i in range(2))
            c.store(layer, k, v, offsets_of(new), t)
            both.append((k, v))
            at = 0
            for s in range(6):
                fed[s][layer].append((k[at:at + new[s]], v[at:at + new[s]]))
                at += new[s]
        return both

    def agree(rows, seed):
        for layer in range(layers):
            q = randn((6 * rows, heads * dim), TYPES[t], seed + layer)
            out = torch.empty_like(q)
            c.attend(layer, q, out, t, 6, rows, heads, dim ** -0.5)
            torch.cuda.synchronize()
            check(out, c.attention(layer, q, 6, rows, heads, dim ** -0.5), TYPES[t])
            for s in range(6):  # the cache holds what was fed
                k = torch.cat([x for x, _ in fed[s][layer]]) if fed[s][layer] else None
                n = int(c.lens[s])
                assert n == (0 if k is None else k.shape[0])
                if not n:
                    continue
                for g in range(kv_heads):
                    have, _ = c.history(s, layer, g)
                    want = k[:, g * dim:(g + 1) * dim].double()
                    # int8: half a code of the row's largest value / 127, and the scale's and product's roundings
                    off_by = want.abs().amax(1, keepdim=True) / 127 * (0.5 + 2.0 ** -15) if cache == I8 else 0.0
                    assert ((have - want).abs() <= off_by).all()

    (k, v), _ = feed([0, 1, 2], lens, 1)
    q = randn((off[-1], heads * dim), TYPES[t], 77)
    o = torch.empty_like(q)
    prompt(q, k, v, o, t, ints(off), 3, off[-1], heads, kv_heads, dim)
    torch.cuda.synchronize()
    check(o, ph.prompt(q, k, v, off, heads, kv_heads, dim, dim ** -0.5), TYPES[t])
    if cache != I8:  # the last rows of the prompts, over the cache
        last = q[[x - 1 for x in off[1:]]].contiguous()
        out = torch.empty_like(last)
        c.attend(0, last, out, t, 3, 1, heads, dim ** -0.5)
        torch.cuda.synchronize()
        ref, big_v, big_s = ph.prompt(q, k, v, off, heads, kv_heads, dim, dim ** -0.5)
        check(out, tuple(x[[y - 1 for y in off[1:]]] for x in (ref, big_v, big_s)), TYPES[t])
    agree(1, 100)
    c.fork([1, 1, 0], [3, 4, 5])
    for p, s in ((1, 3), (1, 4), (0, 5)):
        fed[s] = [list(fed[p][0]), list(fed[p][1])]
    agree(1, 200)
    feed([0, 1, 2, 3, 4, 5], [5, 1, 5, 5, 5, 5], 300)
    agree(5, 400)
    c.free([1, 2])
    fed[1], fed[2] = [[], []], [[], []]
    c.compact()
    assert (c.refs > 0).int().tolist() == sorted((c.refs > 0).int().tolist(), reverse=True)
    agree(1, 500)
    feed([2, 3], [2 * page + 3, 1], 600)
    agree(3, 700)
    assert latched() == 0


@pytest.mark.parametrize("cache,t", [(I8, F32), (BF16, BF16)])
def test_verify_steps_that_give_tokens_back(cache, t):
    """Steps of five tokens, captured once, of which the host takes back 0 to 4: the cache holds what was kept, attention is the
    definition's, and no page is lost."""
    heads, kv_heads, dim, page, n = 8, 2, 64, 16, 3
    c = Cache(cache, 1, kv_heads, dim, page, 40, n + 1, 12)
    c.table.fill_(3)
    c.reserve([0, 1, 2], [30, 1, 16])
    first = randn((47, kv_heads * dim), TYPES[t], 1)
    c.store(0, first, first, [0, 30, 31, 47], t)
    fed = [x.clone() for x in first.split([30, 1, 16])]
    new, q = randn((5 * n, kv_heads * dim), TYPES[t], 2), randn((5 * n, heads * dim), TYPES[t], 3)
    out, work, back = torch.empty_like(q), c.work_for(n, 5, heads), ints([0] * (n + 1))
    seqs, five, off = ints([0, 1, 2]), ints([5] * n), ints([0, 5, 10, 15])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.lens.sub_(back)
        ok("pf_paged_reserve", c.ref, seqs.data_ptr(), five.data_ptr(), n, ph.stream())
        ok("pf_paged_store", c.ref, 0, new.data_ptr(), kv_heads * dim, new.data_ptr(), kv_heads * dim, t, off.data_ptr(), n, 5 * n,
           ph.stream())
        c.attend(0, q, out, t, n, 5, heads, 0.125, work)
    rng = random.Random(4)
    for step in range(25):
        new.copy_(randn(new.shape, TYPES[t], 100 + step))
        q.copy_(randn(q.shape, TYPES[t], 200 + step))
        graph.replay()
        torch.cuda.synchronize()
        check(out, c.attention(0, q, n, 5, heads, 0.125), TYPES[t])
        less = [rng.randint(0, 4) for _ in range(n)]
        back.copy_(ints(less + [0]))
        for b in range(n):
            fed[b] = torch.cat([fed[b], new[5 * b:5 * b + 5]])
            have = torch.cat([c.history(b, 0, g)[0] for g in range(kv_heads)], 1)
            want = fed[b].double().view(-1, kv_heads, dim)
            # int8: half a code of the row's largest value / 127, and the scale's and product's roundings
            off_by = want.abs().amax(2, keepdim=True) / 127 * (0.5 + 2.0 ** -15) if cache == I8 else 0.0
            assert ((have.view_as(want) - want).abs() <= off_by).all(), (step, b)
            fed[b] = fed[b][:fed[b].shape[0] - less[b]]
    most = c.lens.tolist()  # each step's last length is at least any before it
    assert int(c.refs.sum()) == sum(-(-x // page) for x in most[:n])
    c.free([0, 1, 2])
    assert not c.refs.any() and latched() == 0
