"""Decode of a batch over a paged cache with a shared prefix (no reference
counterpart) against the formula in 64 bits on the values the cache holds."""
import math

import pytest
import torch

import runtherder_amd as R
from batch_util import (assert_attention, attend64, dequantize, ints, normal, quantize, score_size)
from gpu_util import DEV, step, sync

pytestmark = pytest.mark.gpu


class Batch:
    """A cache with shuffled pages; sequence b holds own[b] keys behind the prefix
    (total < 0: an unused slot). Rows that no sequence holds are NaN codes and NaN scales."""

    def __init__(self, own, prefix, hq, hkv, d, block, seed, size=1.0, unused=()):
        self.hq, self.hkv, self.d, self.block, self.prefix = hq, hkv, d, block, prefix
        whole = prefix // block
        holds = [-(-(prefix + max(n, 0)) // block) - whole for n in own]
        shared = -(-prefix // block)
        blocks = shared + sum(holds) + 2
        g = torch.Generator().manual_seed(seed)
        pages = 1 + torch.randperm(blocks - 1, generator=g).int()   # the first page holds NaN
        width = max(1, whole + max(holds))
        t = torch.full((len(own), width), -1, dtype=torch.int32)
        t[:, :whole] = pages[:whole]
        pt, at = pages[:max(1, shared)].clone(), shared
        for b, n in enumerate(holds):
            t[b, whole:whole + n] = pages[at:at + n]
            at += n
        self.lens = [prefix + n for n in own]
        for b in unused:
            self.lens[b] = -b
            t[b] = 1 << 20
        c = R.PagedKVCache(1, blocks, block, hkv, d)
        rows = blocks * block
        k8, ks = quantize(normal((rows, hkv, d), seed + 1, size))
        v8, vs = quantize(normal((rows, hkv, d), seed + 2))
        used = torch.zeros(rows, dtype=torch.bool)
        self.at = []
        p = torch.arange(prefix)
        pre = pt[p // block].long() * block + p % block
        for b, n in enumerate(self.lens):
            m = torch.arange(prefix, max(n, prefix))
            mine = t[b][m // block].long() * block + m % block if n > prefix else m[:0]
            self.at.append(torch.cat([pre[:max(n, 0)], mine]))
            used[self.at[-1]] = True
        used[pre] = True
        k8[~used], v8[~used] = 0x7f, 0xff
        ks[~used], vs[~used] = math.nan, math.nan
        self.kv = dequantize(k8, ks), dequantize(v8, vs)
        c.k[0].copy_(k8), c.v[0].copy_(v8), c.k_scale[0].copy_(ks), c.v_scale[0].copy_(vs)
        self.cache, self.tables, self.prefix_table = c, t.to(DEV), pt.to(DEV)
        self.q = normal((len(own), hq, d), seed + 3, size)
        self.attn = R.BatchAttention(R.AttnConfig.for_heads(hq, hkv, d), len(own))

    def run(self, q=None, out=None, shared=True, stream=None):
        q = self.q.to(DEV) if q is None else q
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
        args = (self.prefix_table, ints([self.prefix])) if shared else ()
        self.attn.run_decode(out, q, self.cache.batch_view(0, self.tables), ints(self.lens), *args,
                             stream=stream)
        return out

    def check(self, got, only=None):
        scale = self.d ** -0.5
        for b in range(len(self.lens)) if only is None else only:
            k, v = self.kv[0][self.at[b]], self.kv[1][self.at[b]]
            want, weight = attend64(self.q[b], k, v, scale)
            if not len(k):
                assert (got[b] == 0).all()
                continue
            assert_attention(got[b], want, weight, score_size(self.q[b], k, scale))


@pytest.mark.parametrize("own,prefix", [
    ([1], 0), ([1], 32), ([0], 64), ([1, 2, 33], 100), ([5] * 9, 1000), ([31, 32, 33, 64, 65, 0], 63),
    ([700, 1, 64, 0, 300], 257), ([100, 2000, 7], 0), ([3] * 70, 300), ([0] * 33, 96),
    ([40, 1, 900] * 12, 2049), ([0, 0], 0),
])
def test_lengths(own, prefix):
    t = Batch(own, prefix, 8, 2, 128, 64, 1000 + prefix + len(own))
    step(f"batch decode own={own[:6]} prefix={prefix}")
    out = t.run()
    sync()
    t.check(out.cpu())


@pytest.mark.parametrize("hq,hkv,d", [
    (4, 4, 64), (16, 2, 64), (7, 1, 64), (32, 8, 64), (8, 8, 128), (24, 8, 128), (28, 4, 128), (40, 1, 128),
    (66, 2, 128), (5, 1, 128), (16, 16, 128), (4, 2, 256), (16, 4, 256), (9, 3, 256), (33, 1, 256),
])
@pytest.mark.parametrize("block", [32, 128])
def test_heads(hq, hkv, d, block):
    t = Batch([30, 1, 77, 0, 140], 200, hq, hkv, d, block, 2000 + hq + d)
    step(f"batch decode hq={hq} hkv={hkv} d={d} block={block}")
    out = t.run()
    sync()
    t.check(out.cpu())


def test_long():
    t = Batch([800, 3000, 10, 64] * 3, 9000, 32, 8, 128, 64, 3000)
    step("batch decode long")
    out = t.run()
    sync()
    t.check(out.cpu())


def test_many_sequences():
    t = Batch([i % 50 for i in range(300)], 500, 4, 2, 64, 32, 3100)
    step("batch decode 300 sequences")
    out = t.run()
    sync()
    t.check(out.cpu())


def test_unused_slots_and_short_sequences():
    """Unused slots (whatever their tables hold) give zeros; a sequence shorter than
    the prefix sees its own length of it."""
    t = Batch([20, 5, 100, 7], 150, 8, 2, 128, 32, 3200, unused=(1, 3))
    t.lens[0] = 40
    t.at[0] = t.at[0][:40]
    step("batch decode unused slots")
    out = t.run()
    sync()
    t.check(out.cpu())


def test_shared_prefix_equals_own_tables():
    """The same keys read through the prefix or through every table alike."""
    t = Batch([90, 1, 200], 256, 16, 4, 128, 64, 3300)   # whole pages: the tables hold the prefix
    step("batch decode shared against apart")
    a, b = t.run(), t.run(shared=False)
    sync()
    t.check(a.cpu())
    t.check(b.cpu())


def test_missing_pages_are_left_out():
    t = Batch([100, 60], 128, 8, 2, 128, 32, 3400)
    tables, pt = t.tables.cpu(), t.prefix_table.cpu()
    tables[0, 5] = -1            # keys 160..191 of sequence 0
    pt[1] = 1 << 30              # keys 32..63 of the prefix
    t.tables, t.prefix_table = tables.to(DEV), pt.to(DEV)
    for b in range(2):
        p = torch.arange(t.lens[b])
        gone = ((p >= 32) & (p < 64)) | ((p >= 160) & (p < 192) & (b == 0))
        t.at[b] = t.at[b][~gone]
    t.lens[1] = 100000           # past the table's end
    width = tables.shape[1] * 32
    p = torch.arange(128, width)
    held = tables[1][p // 32] >= 0
    rest = (tables[1][p // 32].long() * 32 + p % 32)[held]
    t.at[1] = torch.cat([t.at[1][:96], rest])
    t.kv[0][rest], t.kv[1][rest] = 0.5, 0.25
    codes, s = quantize(torch.full((1, 128), 0.5).to(torch.bfloat16))
    for c, sc, x in ((t.cache.k, t.cache.k_scale, 0.5), (t.cache.v, t.cache.v_scale, 0.25)):
        codes, s = quantize(torch.full((1, 128), x).to(torch.bfloat16))
        c[0, rest.to(DEV)] = codes[0].to(DEV)
        sc[0, rest.to(DEV)] = s[0].item()
        (t.kv[0] if x == 0.5 else t.kv[1])[rest] = dequantize(codes, s)[0]
    step("batch decode missing pages")
    out = t.run()
    sync()
    t.check(out.cpu())


@pytest.mark.parametrize("seqs", [2, 20, 70])
def test_missing_prefix_pages_with_many_rows(seqs):
    """A prefix page that is not there, where the first page holds NaN, in each of the
    ways a prefix is multiplied (few rows, blocks of 128, of 256)."""
    t = Batch([3] * seqs, 700, 16, 2, 128, 32, 3450)
    pt = t.prefix_table.cpu()
    for c, s in ((t.cache.k, t.cache.k_scale), (t.cache.v, t.cache.v_scale)):
        if not (pt == 0).any() and not (t.tables == 0).any():
            c[0, :32], s[0, :32] = 0x7f, math.nan
    pt[[0, 5, 6, 21]] = -1
    t.prefix_table = pt.to(DEV)
    for b in range(seqs):
        p = torch.arange(t.lens[b])
        block = p // 32
        gone = (p < 700) & ((block == 0) | (block == 5) | (block == 6) | (block == 21))
        t.at[b] = t.at[b][~gone]
    step(f"batch decode missing prefix pages seqs={seqs}")
    out = t.run()
    sync()
    t.check(out.cpu())


def test_score_ranges():
    for size, seed in ((6.0, 3500), (0.01, 3510)):
        t = Batch([200, 3, 64], 400, 8, 2, 128, 64, seed, size=size)
        step(f"batch decode size {size}")
        out = t.run()
        sync()
        t.check(out.cpu())


def test_strided_rows_streams_and_repeats():
    t = Batch([50, 1, 300, 8], 321, 8, 2, 128, 64, 3600)
    wide = torch.zeros((4, 12, 128), dtype=torch.bfloat16, device=DEV)
    wide[:, :8] = t.q.to(DEV)
    owide = torch.full((4, 10, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    step("batch decode strided")
    a = t.run()
    t.run(q=wide[:, :8], out=owide[:, :8])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = t.run()
    s.synchronize()
    sync()
    assert torch.equal(a, owide[:, :8]) and torch.equal(a, b) and (owide[:, 8:] == 3.0).all()
    t.check(a.cpu())


def test_nan_reaches_its_rows_only():
    """A NaN key of one sequence reaches that sequence's rows of its kv head."""
    t = Batch([50, 60], 128, 8, 2, 128, 32, 3700)
    row = t.at[1][150]
    t.cache.k_scale[0, row, 1] = math.nan
    step("batch decode NaN key")
    out = t.run().float().cpu()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :4]).all()
    assert torch.isnan(out[1, 4:]).all()


def test_graph_replays():
    t = Batch([40, 1, 200, 8] * 4, 700, 16, 4, 128, 64, 3800)
    q, out = t.q.to(DEV), torch.zeros((16, 16, 128), dtype=torch.bfloat16, device=DEV)
    view, lens = t.cache.batch_view(0, t.tables), ints(t.lens)
    plen = ints([700])
    step("batch decode graph")
    t.attn.run_decode(out, q, view, lens, t.prefix_table, plen)
    sync()
    want = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.attn.run_decode(out, q, view, lens, t.prefix_table, plen)
    for rep in range(3):
        out.zero_()
        g.replay()
        sync()
        assert torch.equal(out, want), rep
        lens.fill_(10)          # lengths live on the device: a replay takes them as they are
        g.replay()
        sync()
        assert not torch.equal(out, want)
        lens.copy_(ints(t.lens))
        t.attn.run_decode(out, q, view, lens, t.prefix_table, plen)   # eager work between
        sync()
        assert torch.equal(out, want)


# Without a shared prefix; at head_dim 64 an odd kv head has no neighbour in its tile.
@pytest.mark.parametrize("hq,hkv,d", [
    (3, 3, 64), (9, 3, 64), (20, 1, 64), (35, 5, 64), (32, 8, 64), (6, 2, 64), (24, 8, 128), (7, 7, 128), (40, 2, 128),
    (4, 2, 256),
])
def test_apart(hq, hkv, d):
    t = Batch([300, 1, 77, 0, 140, 33, 1000], 0, hq, hkv, d, 32, 4000 + hq + d)
    step(f"batch decode apart hq={hq} hkv={hkv} d={d}")
    out = t.run(shared=False)
    sync()
    t.check(out.cpu())


@pytest.mark.parametrize("hq,hkv", [(3, 3), (9, 3), (20, 1), (35, 5)])
@pytest.mark.parametrize("own,prefix", [([30, 1, 77, 0, 140], 200), ([5, 40, 0, 65] * 20, 333)])
def test_odd_heads_of_64(hq, hkv, own, prefix):
    t = Batch(own, prefix, hq, hkv, 64, 64, 4300 + hq + len(own))
    step(f"batch decode hq={hq} hkv={hkv} own={own[:5]}")
    out = t.run()
    sync()
    t.check(out.cpu())


# More rows than the merge's four waves a row fill the chip with; more sequences
# than the bisection of the runs takes (its bound).
@pytest.mark.parametrize("seqs,hq,hkv,d,prefix", [
    (150, 16, 4, 128, 300), (150, 16, 4, 128, 0), (257, 8, 2, 64, 0), (256, 16, 2, 64, 100), (80, 32, 8, 256, 70)])
def test_many_rows(seqs, hq, hkv, d, prefix):
    t = Batch([(37 * i) % 190 for i in range(seqs)], prefix, hq, hkv, d, 32, 4500 + seqs + d)
    step(f"batch decode {seqs} sequences hq={hq} d={d} prefix={prefix}")
    out = t.run(shared=prefix > 0)
    sync()
    t.check(out.cpu())
