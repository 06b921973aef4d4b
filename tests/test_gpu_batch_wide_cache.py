"""The batch operators where offsets pass 32 bits: slabs larger than 4 GiB, and
rows of a projection that end past 4 GiB. A page's number and a row's stride are
no part of an operator's arithmetic, so the results equal, bit for bit, those of
the same rows in a small cache, or without gaps."""
import pytest
import torch

import runtherder_amd as R
from batch_util import ints, normal
from gpu_util import DEV, step, sync

pytestmark = pytest.mark.gpu

HKV, D, BLOCK = 64, 128, 256          # 2 MiB of codes per page
PAGES = 2048 + 40                     # 2^32 bytes and 40 pages
HIGH = [2087, 5, 2060, 2049, 2050, 2086]   # pages of the wide cache ...
LOW = [0, 1, 2, 3, 4, 5]                   # ... and of the small one


def slabs(c):
    return (c.k, c.v, c.k_scale, c.v_scale)


def test_cache_past_4_gib():
    wide = R.PagedKVCache(2, PAGES, BLOCK, HKV, D, device=DEV)
    small = R.PagedKVCache(2, 8, BLOCK, HKV, D, device=DEV)
    lens, shared = [700, 1000], 300
    attn = R.BatchAttention(R.AttnConfig(HKV, HKV, D, D ** -0.5), 2, device=DEV)
    tables = {}
    for c, ids in ((wide, HIGH), (small, LOW)):
        # Both begin on pages 0 and 1 of the list.
        tables[c] = ints([ids[:2] + [ids[2], -1], ids[:2] + ids[3:5]])
    k, v, q = (normal((sum(lens), HKV, D), s).to(DEV) for s in (1, 2, 3))
    out = {}
    for c in (wide, small):
        step(f"append and decode in {c.num_blocks} pages")
        for layer in range(2):
            # (The first two pages, which both hold, are written by the second alone.)
            c.append_batch(layer, k[700:], v[700:], ints([0]), tables[c][1:], ints([0, 1000]))
            c.append_batch(layer, k[:188], v[:188], ints([512]), tables[c][:1], ints([0, 188]))
        for layer in range(2):
            for prefix in (None, tables[c][1]):
                o = torch.empty((2, HKV, D), dtype=torch.bfloat16, device=DEV)
                attn.run_decode(o, q[:2], c.batch_view(layer, tables[c]), ints([700 - 1, 1000]), prefix,
                                None if prefix is None else ints([shared]))
                sync()
                out[c, layer, prefix is None] = o
    for layer in range(2):
        for apart in (True, False):
            assert torch.equal(out[wide, layer, apart], out[small, layer, apart])
    page = lambda x, layer, p: x[layer].view(-1, BLOCK, *x.shape[2:])[p]
    for layer in range(2):
        for x, y in zip(slabs(wide), slabs(small)):
            for hi, lo in zip(HIGH[:2], LOW):   # (the pages that are filled whole)
                assert torch.equal(page(x, layer, hi), page(y, layer, lo))
    step("pages past 4 GiB")
    wide.copy_pages(ints([2087, 5]), ints([2055, 2056]))
    sync()
    for layer in range(2):
        for x in slabs(wide):
            assert torch.equal(page(x, layer, 2055), page(x, layer, 2087))
            assert torch.equal(page(x, layer, 2056), page(x, layer, 5))
    # The pool: in use are the tables' pages; two children, then all moved down.
    pool = R.PagePool(PAGES, BLOCK, device=DEV)
    for p in tables[wide].flatten().tolist():
        if p >= 0:
            pool.refs[p] += 1
    kids, kid_lens = pool.new_tables(2, 4), ints([0, 0])
    pool.fork(wide, kids, kid_lens, tables[wide], ints([700, 1000]), ints([1, 0]))
    pool.compact(wide, torch.cat((tables[wide], kids)))
    sync()
    assert pool.status.item() == 0 and kid_lens.tolist() == [1000, 700]
    assert (pool.refs > 0).nonzero().flatten().tolist() == list(range(7))


def test_compacted_pages_past_4_gib_keep_their_rows():
    wide = R.PagedKVCache(2, PAGES, BLOCK, HKV, D, device=DEV)
    k, v = (normal((600, HKV, D), s).to(DEV) for s in (4, 5))
    tables = ints([[2087, 2070, 2050]])
    for layer in range(2):
        wide.append_batch(layer, k, v, ints([0]), tables, ints([0, 600]))
    pool = R.PagePool(PAGES, BLOCK, device=DEV)
    pool.refs[[2050, 2070, 2087]] = 1
    rows = lambda t: [x[:, torch.cat([p * BLOCK + torch.arange(BLOCK, device=DEV) for p in t[0]])[:600].long()]
                      for x in slabs(wide)]
    before = [x.clone() for x in rows(tables)]
    step("compact past 4 GiB")
    pool.compact(wide, tables)
    sync()
    assert tables.tolist() == [[2, 1, 0]]
    for a, b in zip(before, rows(tables)):
        assert torch.equal(a, b)


def test_rows_past_4_gib():
    n, stride, hq, hkv, d = 16500, 1 << 17, 4, 1, 128   # the last row ends past 2^32 bytes
    wide = torch.empty((n, stride), dtype=torch.bfloat16, device=DEV)
    parts = {"q": (0, hq), "k": (hq * d, hkv), "v": ((hq + hkv) * d, hkv), "out": ((hq + 2 * hkv) * d, hq)}
    rows = {name: wide[:, at:at + h * d].view(n, h, d) for name, (at, h) in parts.items()}
    for i, name in enumerate("qkv"):
        rows[name].copy_(normal(tuple(rows[name].shape), 20 + i))
    cu = ints([0, 9000, n])
    want = torch.empty((n, hq, d), dtype=torch.bfloat16, device=DEV)
    step("packed rows past 4 GiB")
    R.flash_packed_bf16(want, *(rows[x].contiguous() for x in "qkv"), cu, hq, hkv, d, d ** -0.5)
    R.flash_packed_bf16(rows["out"], rows["q"], rows["k"], rows["v"], cu, hq, hkv, d, d ** -0.5)
    sync()
    assert torch.equal(rows["out"], want)
    caches = [R.PagedKVCache(1, 80, BLOCK, hkv, d, device=DEV) for _ in range(2)]
    tables = torch.arange(80, dtype=torch.int32, device=DEV).view(2, 40)
    for c, (k, v) in zip(caches, ((rows["k"], rows["v"]), (rows["k"].contiguous(), rows["v"].contiguous()))):
        for x in slabs(c):
            x.zero_()
        c.append_batch(0, k, v, ints([0, 0]), tables, cu)
    sync()
    for a, b in zip(slabs(caches[0]), slabs(caches[1])):
        assert torch.equal(a, b)
