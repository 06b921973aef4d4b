"""Pages of a paged cache on the device (no reference counterpart) against the
same bookkeeping and moves in plain Python."""
import pytest
import torch

import runtherder_amd as R
from batch_util import ints, normal
from gpu_util import DEV, step, sync

pytestmark = pytest.mark.gpu


def filled(layers, blocks, block, hkv, d, seed):
    c = R.PagedKVCache(layers, blocks, block, hkv, d)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in (c.k, c.v):
        t.random_(0, 256, generator=g)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device=DEV))
    return c


class Slabs:
    """Host copy of a cache's slabs, for the plain moves."""

    def __init__(self, c):
        self.block, self.t = c.block_size, [x.cpu().clone() for x in (c.k, c.v, c.k_scale, c.v_scale)]

    def move(self, src, dst, rows=None):
        for x in self.t:
            a, b = src * self.block, dst * self.block
            n = self.block if rows is None else rows
            x[:, b:b + n] = x[:, a:a + n].clone()

    def same(self, c):
        for x, y in zip(self.t, (c.k, c.v, c.k_scale, c.v_scale)):
            assert torch.equal(x, y.cpu())


@pytest.mark.parametrize("layers,blocks,block,hkv,d,count", [
    (1, 8, 32, 1, 8, 1), (3, 20, 32, 2, 128, 7), (2, 40, 256, 8, 64, 20), (1, 70, 64, 3, 24, 35),
])
def test_copy(layers, blocks, block, hkv, d, count):
    c = filled(layers, blocks, block, hkv, d, count)
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(count)).tolist()
    src, dst = order[:count], order[blocks - count:]
    want = Slabs(c)
    for a, b in zip(src, dst):
        want.move(a, b)
    step(f"copy {count} pages")
    c.copy_pages(ints(src), ints(dst))
    sync()
    want.same(c)
    c.copy_pages(ints([-1, 3, blocks, 2]), ints([0, -5, 1, 1 << 30]))   # none names a pair of pages
    c.copy_pages(ints([]), ints([]))
    sync()
    want.same(c)


class Plain:
    """The pool's rules in plain Python."""

    def __init__(self, blocks, block):
        self.refs, self.block = [0] * blocks, block

    def take(self, n):
        got = [p for p, r in enumerate(self.refs) if r <= 0][:n]
        if len(got) < n:
            return None
        for p in got:
            self.refs[p] = 1
        return got

    def reserve(self, tables, lens, n_new):
        want = [(b, i) for b, (n, m) in enumerate(zip(lens, n_new)) if m > 0 and n >= 0
                for i in range(n // self.block, -(-(n + m) // self.block))]
        if any(i >= len(tables[b]) for b, i in want):
            return 2
        want = [(b, i) for b, i in want if tables[b][i] < 0]
        got = self.take(len(want))
        if got is None:
            return 1
        for (b, i), p in zip(want, got):
            tables[b][i] = p
        return 0

    def fork(self, slabs, tables, lens, parents):
        width = len(tables[0])
        length = [lens[p] if 0 <= p < len(lens) else 0 for p in parents]
        tails = [i for i, n in enumerate(length) if n % self.block]
        own = self.take(len(tails))
        if own is None:
            return None
        out = [[-1] * width for _ in parents]
        for i, (p, n) in enumerate(zip(parents, length)):
            for j in range(n // self.block):
                out[i][j] = tables[p][j]
                self.refs[tables[p][j]] += 1
        for i, page in zip(tails, own):
            j = length[i] // self.block
            out[i][j] = page
            slabs.move(tables[parents[i]][j], page, length[i] % self.block)
        return out, length

    def free(self, tables, lens, drop):
        for b, row in enumerate(tables):
            if drop[b]:
                for j, p in enumerate(row):
                    if p >= 0:
                        self.refs[p] -= 1
                    row[j] = -1
                lens[b] = 0

    def compact(self, slabs, tables):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] <= 0]
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                to = holes.pop(0)
                slabs.move(p, to)
                self.refs[to], self.refs[p] = self.refs[p], 0
                for row in tables:
                    row[:] = [to if x == p else x for x in row]


@pytest.mark.parametrize("seqs,blocks,block,width,layers,hkv,d", [
    (3, 40, 32, 9, 2, 2, 64), (20, 300, 64, 12, 1, 1, 8), (70, 9000, 32, 70, 1, 1, 8), (1, 5, 128, 5, 3, 3, 24),
])
def test_life_of_a_pool(seqs, blocks, block, width, layers, hkv, d):
    """Reserve, fork, free, compact, one behind the other, against the plain rules."""
    g = torch.Generator().manual_seed(seqs)

    def rand(lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()

    c = filled(layers, blocks, block, hkv, d, seqs)
    slabs, plain = Slabs(c), Plain(blocks, block)
    pool = R.PagePool(blocks, block)
    tables, lens = pool.new_tables(seqs, width), ints([0] * seqs)
    rows, held = tables.tolist(), lens.tolist()
    for turn in range(4):
        step(f"pool turn {turn}")
        n_new = [min(x, width * block - n) for x, n in zip(rand(-1, width * block // 3, seqs), held)]
        pool.reserve(tables, lens, ints(n_new))
        assert plain.reserve(rows, held, n_new) == 0
        held = [n + max(m, 0) for n, m in zip(held, n_new)]
        lens.copy_(ints(held))
        assert tables.tolist() == rows and pool.refs.tolist() == plain.refs
        parents = rand(-1, seqs, max(1, seqs // 2))
        kids, klens = pool.new_tables(len(parents), width), ints([9] * len(parents))
        pool.fork(c, kids, klens, tables, lens, ints(parents))
        krows, kheld = plain.fork(slabs, rows, held, parents)
        assert kids.tolist() == krows and klens.tolist() == kheld
        assert pool.refs.tolist() == plain.refs
        slabs.same(c)
        drop = rand(0, 1, seqs)
        pool.free(tables, lens, ints(drop))
        plain.free(rows, held, drop)
        assert tables.tolist() == rows and lens.tolist() == held and pool.refs.tolist() == plain.refs
        both = torch.cat([tables, kids])
        every = rows + krows
        pool.compact(c, both)
        plain.compact(slabs, every)
        assert both.tolist() == every and pool.refs.tolist() == plain.refs
        slabs.same(c)
        tables, kids = both[:seqs].contiguous(), both[seqs:].contiguous()
        pool.free(kids, klens)
        plain.free(krows, kheld, [1] * len(krows))
        assert pool.refs.tolist() == plain.refs and klens.tolist() == kheld
    assert pool.status.item() == 0


def test_a_pool_that_is_too_small_changes_nothing():
    pool, c = R.PagePool(4, 32), filled(1, 4, 32, 1, 8, 1)
    slabs = Slabs(c)
    tables, lens = pool.new_tables(2, 3), ints([0, 0])
    step("out of pages")
    pool.reserve(tables, lens, ints([90, 64]))      # 3 + 2 pages of 4
    assert pool.status.item() == R.PagePool.OUT_OF_PAGES
    assert (tables == -1).all() and (pool.refs == 0).all()
    pool.status.zero_()
    pool.reserve(tables, lens, ints([10, 97]))      # a row of 3 entries
    assert pool.status.item() == R.PagePool.TABLE_TOO_SHORT
    assert (tables == -1).all() and (pool.refs == 0).all()
    pool.status.zero_()
    pool.reserve(tables, lens, ints([65, 32]))      # all 4
    pool.reserve(tables, lens, ints([90, 1]))       # nothing more is needed
    assert pool.status.item() == 0 and (pool.refs == 1).all()
    assert tables.tolist() == [[0, 1, 2], [3, -1, -1]]
    lens.copy_(ints([65, 32]))
    kids, klens = pool.new_tables(2, 3), ints([5, 5])
    pool.fork(c, kids, klens, tables, lens, ints([1, 0]))   # the second needs a page
    assert pool.status.item() == R.PagePool.OUT_OF_PAGES
    assert (kids == -1).all() and klens.tolist() == [5, 5] and (pool.refs == 1).all()
    slabs.same(c)
    pool.status.zero_()
    pool.fork(c, kids, klens, tables, lens, ints([1, 1]))
    assert pool.status.item() == 0 and pool.refs.tolist() == [1, 1, 1, 3]
    assert kids.tolist() == [[3, -1, -1]] * 2


def test_lengths_and_tables_out_of_range():
    pool, c = R.PagePool(8, 32), filled(1, 8, 32, 1, 8, 2)
    tables, lens = ints([[0, 99, 1], [-3, 2, 1 << 30]]), ints([10 ** 9, -5])
    pool.refs[:3] = 1
    kids, klens = pool.new_tables(3, 3), ints([0, 0, 0])
    step("fork of strange tables")
    pool.fork(c, kids, klens, tables, lens, ints([0, 1, 7]))
    assert kids.tolist() == [[0, -1, 1], [-1] * 3, [-1] * 3] and klens.tolist() == [96, 0, 0]
    assert pool.refs.tolist() == [2, 2, 1, 0, 0, 0, 0, 0]
    pool.compact(c, tables)
    assert tables.tolist() == [[0, 99, 1], [-3, 2, 1 << 30]]
    pool.free(tables, lens)
    assert pool.refs.tolist() == [1, 1, 0, 0, 0, 0, 0, 0] and (tables == -1).all()
    assert pool.status.item() == 0


def test_captured_step():
    """A beam step (free, fork) in one graph, replayed, against eager ones."""
    pool, c = R.PagePool(30, 32), filled(2, 30, 32, 2, 64, 3)
    src, slens = pool.new_tables(2, 5), ints([0, 0])
    pool.reserve(src, slens, ints([70, 150]))
    slens.copy_(ints([70, 150]))
    kids, klens, parents = pool.new_tables(4, 5), ints([0] * 4), ints([0, 1, 1, 0])

    def beam():
        pool.free(kids, klens)
        pool.fork(c, kids, klens, src, slens, parents)

    step("captured beam step")
    beam()
    sync()
    want = kids.clone(), klens.clone(), pool.refs.clone(), Slabs(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        beam()
    for _ in range(3):
        g.replay()
        sync()
        assert torch.equal(kids, want[0]) and torch.equal(klens, want[1])
        assert torch.equal(pool.refs, want[2])
        want[3].same(c)
        beam()
        sync()
        assert torch.equal(kids, want[0]) and torch.equal(pool.refs, want[2])
