"""Append of a batch into its sequences' pages (no reference counterpart): bytes
and scales equal, bit for bit, what PagedKVCache.append writes sequence by
sequence, which the oracle pins; rows without a page are not stored."""
import pytest
import torch

import runtherder_amd as R
from batch_util import cu_of, ints, normal
from gpu_util import DEV, int_dev, step, sync

pytestmark = pytest.mark.gpu


def tables_of(holds, width, seed):
    g = torch.Generator().manual_seed(seed)
    pages, at = torch.randperm(sum(holds), generator=g).int(), 0
    t = torch.full((len(holds), width), -1, dtype=torch.int32)
    for b, n in enumerate(holds):
        t[b, :n] = pages[at:at + n]
        at += n
    return t.to(DEV)


def fresh(blocks, block, hkv, d):
    c = R.PagedKVCache(2, blocks, block, hkv, d)
    c.k.fill_(0x55), c.v.fill_(0x2a), c.k_scale.fill_(-3.0), c.v_scale.fill_(-5.0)
    return c


def same(a, b):
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scale.view(torch.int32), b.k_scale.view(torch.int32)),
                 (a.v_scale.view(torch.int32), b.v_scale.view(torch.int32))):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lens,at,hkv,d,block,fused,pad", [
    ([5, 0, 1, 70], [0, 3, 31, 60], 8, 128, 32, False, 0),
    ([1], [0], 1, 64, 64, False, 3), ([300, 1, 2], [7, 1000, 0], 4, 256, 64, True, 2),
    ([1] * 130, list(range(130)), 3, 64, 32, False, 0), ([33, 64], [31, 0], 5, 8, 32, False, 1),
    ([20, 9], [0, 127], 2, 512, 128, False, 0), ([17, 3], [0, 5], 2, 24, 32, False, 0),
    ([0, 0, 2], [9, 9, 9], 16, 128, 32, True, 4),
])
def test_equals_sequence_by_sequence(lens, at, hkv, d, block, fused, pad):
    holds = [-(-(n + a) // block) for n, a in zip(lens, at)]
    t = tables_of(holds, max(holds) + 1, sum(lens))
    n = sum(lens) + pad
    x = normal((n, 2 * hkv + (3 if fused else 0), d), sum(at)).to(DEV)
    k, v = x[:, :hkv], x[:, hkv:2 * hkv]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    a, b = fresh(sum(holds) + 1, block, hkv, d), fresh(sum(holds) + 1, block, hkv, d)
    step(f"append batch lens={lens[:6]} hkv={hkv} d={d} block={block}")
    a.append_batch(1, k, v, ints(at), t, ints(cu_of(lens)))
    cu = cu_of(lens)
    for i, m in enumerate(lens):
        if m:
            b.append(1, k[cu[i]:cu[i] + m].contiguous(), v[cu[i]:cu[i] + m].contiguous(), m,
                     int_dev(at[i]), t[i].contiguous())
    sync()
    same(a, b)


@pytest.mark.parametrize("seqs,hkv,d", [(1, 8, 128), (64, 8, 128), (7, 3, 64), (200, 1, 256)])
def test_one_row_each(seqs, hkv, d):
    """Without cu_seqlens: as with cu_seqlens 0, 1, 2, ..; special rows as the
    single append has them (zeros, subnormals, infinities, NaN)."""
    at = [(37 * b) % 200 for b in range(seqs)]
    t = tables_of([7] * seqs, 7, seqs)
    x = normal((seqs, 2 * hkv, d), seqs)
    x[0, 0] = 0.0
    x[-1, 1, 3] = float("nan")
    x[seqs // 2, -1, 1] = float("inf")
    x[seqs // 2, 0] = 2.0 ** -130
    x = x.to(DEV)
    k, v = x[:, :hkv], x[:, hkv:]
    a, b, c = (fresh(7 * seqs, 32, hkv, d) for _ in range(3))
    step(f"append one row each seqs={seqs}")
    a.append_batch(0, k, v, ints(at), t)
    b.append_batch(0, k, v, ints(at), t, ints(list(range(seqs + 1))))
    for i in range(seqs):
        c.append(0, k[i:i + 1].contiguous(), v[i:i + 1].contiguous(), 1, int_dev(at[i]), t[i].contiguous())
    sync()
    same(a, b)
    same(a, c)


def test_rows_without_a_page_are_not_stored():
    hkv, d, block = 2, 64, 32
    k = normal((40, hkv, d), 1).to(DEV)
    t = ints([[0, -1], [2, 99], [1, 3], [-7, 3]])
    a, b = fresh(4, block, hkv, d), fresh(4, block, hkv, d)
    step("append to missing pages")
    # Positions 28..37 of a table that ends inside, 64.. past a table's end, below zero.
    a.append_batch(0, k, k, ints([28, 60, -4, 30]), t, ints([0, 10, 20, 30, 40]))
    b.append(0, k[:4].contiguous(), k[:4].contiguous(), 4, int_dev(28), ints([0]))
    b.append(0, k[24:30].contiguous(), k[24:30].contiguous(), 6, int_dev(0), ints([1]))
    b.append(0, k[32:40].contiguous(), k[32:40].contiguous(), 8, int_dev(0), ints([3]))
    sync()
    same(a, b)
