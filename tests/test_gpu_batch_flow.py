"""The batch operators together, as a serving loop calls them: prompts packed
one behind the other, their K and V into pages, sequences freed and forked,
decode steps over the shared pages, compaction; eager, as a replayed graph, and
through the C++ layer. Against 64-bit attention over the codes of each row."""
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import oracle_lib as O
import runtherder_amd as R
from batch_util import (F64, assert_attention, attend64, cu_of, dequantize, ints, normal, score_size)
from gpu_util import DEV, step, sync

pytestmark = pytest.mark.gpu

EXE = Path(__file__).resolve().parent / "cpp" / "bin" / "test_batch"


def stored(x):
    """The oracle's codes and scales of bf16 rows [..., hkv, d]."""
    *lead, d = x.shape
    codes, scale = O.quantize_kv_fp8(x.reshape(-1, d).view(torch.int16).numpy().view(np.uint16), d)
    return torch.from_numpy(codes).view(x.shape), torch.from_numpy(scale).view(lead)


class Serving:
    """A cache, its pool, the batch's device state, and every sequence's rows on the host."""

    def __init__(self, seqs, layers, pages, block, width, hq, hkv, d):
        self.hq, self.hkv, self.d, self.layers, self.block = hq, hkv, d, layers, block
        self.scale = d ** -0.5
        self.cache = R.PagedKVCache(layers, pages, block, hkv, d, device=DEV)
        self.pool = R.PagePool(pages, block, device=DEV)
        self.attn = R.BatchAttention(R.AttnConfig(hq, hkv, d, self.scale), 64, device=DEV)
        self.tables, self.lens = self.pool.new_tables(seqs, width), ints([0] * seqs)
        self.rows = [[] for _ in range(seqs)]   # per sequence: (k, v) [hkv, d] float64, per layer
        self.seed = 100

    def draw(self, *shape):
        self.seed += 1
        return normal(shape, self.seed)

    def keep(self, b, k, v):
        """k, v [layers, n, hkv, d] bf16: what the cache holds of them."""
        kd, vd = (dequantize(*stored(x)) for x in (k, v))
        self.rows[b] += [(kd[:, t], vd[:, t]) for t in range(k.shape[1])]

    def prompts(self, n):
        """Prefill: attention from the bf16 rows (checked at the ends of each prompt), then the cache."""
        total, cu = sum(n), cu_of(n)
        q, k, v = (self.draw(self.layers, total, h, self.d) for h in (self.hq, self.hkv, self.hkv))
        dn, dcu = ints(n), ints(cu)
        self.pool.reserve(self.tables, self.lens, dn)
        for layer in range(self.layers):
            dq, dk, dv = (x[layer].to(DEV) for x in (q, k, v))
            out = torch.empty_like(dq)
            self.attn.run_packed(out, dq, dk, dv, dcu)
            self.cache.append_batch(layer, dk, dv, self.lens, self.tables, dcu)
            sync()
            for b in range(len(n)):
                for t in {cu[b], (cu[b] + cu[b + 1]) // 2, cu[b + 1] - 1} if n[b] else ():
                    kk, vv = k[layer, cu[b]:t + 1], v[layer, cu[b]:t + 1]
                    assert_attention(out[t].cpu(), *attend64(q[layer, t], kk, vv, self.scale),
                                     score_size(q[layer, t], kk, self.scale))
        self.lens += dn
        for b in range(len(n)):
            self.keep(b, k[:, cu[b]:cu[b + 1]], v[:, cu[b]:cu[b + 1]])

    def token_inputs(self):
        b = len(self.rows)
        return [self.draw(self.layers, b, h, self.d) for h in (self.hq, self.hkv, self.hkv)]

    def device_step(self, q, k, v, out, ones, prefix_table=None, prefix_len=None):
        """One token of each sequence, all on the device (as a graph would capture it)."""
        self.pool.reserve(self.tables, self.lens, ones)
        for layer in range(self.layers):
            self.cache.append_batch(layer, k[layer], v[layer], self.lens, self.tables)
        self.lens += ones
        for layer in range(self.layers):
            self.attn.run_decode(out[layer], q[layer], self.cache.batch_view(layer, self.tables),
                                 self.lens, prefix_table, prefix_len)

    def check(self, q, out):
        out = out.cpu()
        for layer in range(self.layers):
            for b, rows in enumerate(self.rows):
                kk = torch.stack([r[0][layer] for r in rows]) if rows else torch.zeros(0, self.hkv, self.d, dtype=F64)
                vv = torch.stack([r[1][layer] for r in rows]) if rows else kk
                size = score_size(q[layer, b], kk, self.scale) if rows else 0.0
                assert_attention(out[layer, b], *attend64(q[layer, b], kk, vv, self.scale), size)


@pytest.mark.parametrize("hq,hkv,d,block,n,shared", [
    (32, 8, 128, 64, [130, 1, 77, 300], 256), (6, 2, 64, 32, [31, 33, 64, 100], 96), (4, 4, 256, 128, [5, 128, 1, 260], 256)])
def test_serving_loop(hq, hkv, d, block, n, shared):
    s = Serving(4, 2, 64, block, 16, hq, hkv, d)
    step(f"serving loop {hq} {hkv} {d}")
    s.prompts(n)
    # The second sequence ends; five beams of the last and one of the first go on.
    s.pool.free(s.tables, s.lens, ints([0, 1, 0, 0]))
    s.rows[1] = []
    parents = [3, 3, 0, 3, 1, 3]
    old_tables, old_lens = s.tables, s.lens
    s.tables, s.lens = s.pool.new_tables(6, 16), ints([0] * 6)
    s.pool.fork(s.cache, s.tables, s.lens, old_tables, old_lens, ints(parents))
    s.rows = [list(s.rows[p]) for p in parents]
    s.pool.free(old_tables, old_lens)
    ones = ints([1] * 6)
    for i in range(4):
        q, k, v = s.token_inputs()
        out = torch.empty((2, 6, hq, d), dtype=torch.bfloat16, device=DEV)
        s.device_step(*(x.to(DEV) for x in (q, k, v)), out, ones)
        sync()
        for b in range(6):
            s.keep(b, k[:, b:b + 1], v[:, b:b + 1])
        s.check(q, out)
        if i == 1:
            s.pool.compact(s.cache, s.tables)
            assert int((s.pool.refs > 0).sum()) == int(s.tables.max()) + 1
    # The beams of one parent alone, their prompt's whole pages as a shared prefix.
    beams = [0, 1, 3, 5]
    s.tables, s.lens = s.tables[beams].contiguous(), s.lens[beams].contiguous()
    s.rows = [s.rows[b] for b in beams]
    ones, plen = ints([1] * 4), ints([shared])
    for _ in range(2):
        q, k, v = s.token_inputs()
        out = torch.empty((2, 4, hq, d), dtype=torch.bfloat16, device=DEV)
        s.device_step(*(x.to(DEV) for x in (q, k, v)), out, ones, s.tables[1], plen)
        sync()
        for b in range(4):
            s.keep(b, k[:, b:b + 1], v[:, b:b + 1])
        s.check(q, out)
    assert s.pool.status.item() == 0


def test_captured_step_of_a_batch():
    """A whole decode step (pages, append, attention of two layers) as one graph,
    replayed with new tokens; pages run over block ends between replays, and the
    program's own eager work runs between them."""
    hq, hkv, d, block = 16, 4, 128, 32
    s = Serving(3, 2, 40, block, 12, hq, hkv, d)
    step("captured serving step")
    s.prompts([95, 31, 64])
    ones = ints([1] * 3)
    dq, dk, dv = (torch.zeros((2, 3, h, d), dtype=torch.bfloat16, device=DEV) for h in (hq, hkv, hkv))
    out = torch.zeros((2, 3, hq, d), dtype=torch.bfloat16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    for rep in range(7):
        q, k, v = s.token_inputs()
        for to, x in ((dq, q), (dk, k), (dv, v)):
            to.copy_(x)
        if rep == 1:
            lens, tables, refs = s.lens.clone(), s.tables.clone(), s.pool.refs.clone()
            with torch.cuda.graph(graph):
                s.device_step(dq, dk, dv, out, ones)
            assert torch.equal(lens, s.lens) and torch.equal(tables, s.tables)
            assert torch.equal(refs, s.pool.refs)
        if rep in (0, 3):
            s.device_step(dq, dk, dv, out, ones)   # eager, before and between replays
        else:
            graph.replay()
        sync()
        for b in range(3):
            s.keep(b, k[:, b:b + 1], v[:, b:b + 1])
        s.check(q, out)
        out.zero_()
    assert s.lens.tolist() == [102, 38, 71] and s.pool.status.item() == 0


def test_captured_prefill():
    """Packed prompts and their append as one graph, replayed over other prompts:
    the bounds are read on the device; rows behind the last prompt stay."""
    hq, hkv, d, rows = 8, 2, 128, 400
    cache = R.PagedKVCache(1, 64, 32, hkv, d, device=DEV)
    attn = R.BatchAttention(R.AttnConfig(hq, hkv, d, d ** -0.5), 8, device=DEV)
    tables = torch.arange(64, dtype=torch.int32, device=DEV).view(4, 16)
    q, k, v = (torch.zeros((rows, h, d), dtype=torch.bfloat16, device=DEV) for h in (hq, hkv, hkv))
    out, cu, at = torch.zeros_like(q), ints([0] * 5), ints([0] * 4)

    def run():
        attn.run_packed(out, q, k, v, cu)
        cache.append_batch(0, k, v, at, tables, cu)

    step("captured prefill")
    run()
    sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for rep, lens in enumerate([[100, 0, 7, 293], [1, 1, 1, 1], [400, 0, 0, 0], [33, 64, 130, 31]]):
        for i, x in enumerate((q, k, v)):
            x.copy_(normal(tuple(x.shape), 7 * rep + i))
        cu.copy_(ints(cu_of(lens)))
        got = []
        for call in (graph.replay, run):
            out.fill_(3.0)
            cache.k.zero_(), cache.v.zero_(), cache.k_scale.zero_(), cache.v_scale.zero_()
            call()
            sync()
            got.append([x.clone() for x in (out, cache.k, cache.v, cache.k_scale, cache.v_scale)])
        for a, b in zip(*got):
            assert torch.equal(a, b), rep
        n = sum(lens)
        assert (out[n:] == 3.0).all() and not (out[:n] == 3.0).all()


def test_cpp_batch_driver():
    assert EXE.exists(), "build first: __graft_entry__.build()"
    step("cpp batch driver")
    res = subprocess.run([str(EXE)], capture_output=True, text=True, timeout=100)
    print(res.stdout[-4000:], res.stderr[-2000:])
    assert res.returncode == 0
    assert "ALL OK" in res.stdout


def test_a_captured_decode_takes_the_prefix_as_it_is():
    """The prefix's length lives on the device: replays with other lengths of it, from none
    to the whole prompt, give what the eager calls give; the keys are the same ones, so
    all agree within the outputs' bounds."""
    s = Serving(3, 1, 64, 64, 16, 16, 4, 128)
    step("captured decode, prefix lengths")
    s.prompts([600, 0, 0])
    tables, lens = s.pool.new_tables(20, 16), ints([0] * 20)
    s.pool.fork(s.cache, tables, lens, s.tables, s.lens, ints([0] * 20))
    s.rows = [list(s.rows[0]) for _ in range(20)]
    q = s.draw(1, 20, 16, 128)
    dq, out, plen = q[0].to(DEV), torch.zeros((20, 16, 128), dtype=torch.bfloat16, device=DEV), ints([64])
    view = s.cache.batch_view(0, tables)

    def run():
        s.attn.run_decode(out, dq, view, lens, tables[3], plen)

    run()
    sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for n in (0, 1, 64, 300, 576, 600, 5000, 0):
        plen.fill_(n)
        got = []
        for call in (run, graph.replay):
            out.zero_()
            call()
            sync()
            got.append(out.clone())
        assert torch.equal(*got), n
        s.check(q, got[0][None])   # (what lies behind the 600 keys was never written)


def test_two_streams_at_once():
    """Calls that overlap, each with a scratch of its own, over one cache."""
    s = Serving(6, 1, 64, 64, 16, 32, 8, 128)
    step("two streams")
    s.prompts([500, 33, 800, 64, 1, 250])
    q = [s.draw(6, 32, 128).to(DEV) for _ in range(8)]
    k, v = (s.draw(1649, 8, 128).to(DEV) for _ in range(2))
    qp, cu = s.draw(1649, 32, 128).to(DEV), ints(cu_of([1000, 249, 400]))
    view = s.cache.batch_view(0, s.tables)
    attns = [R.BatchAttention(R.AttnConfig(32, 8, 128, s.scale), 6, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = []
    for x in q:
        o = torch.empty_like(x)
        attns[0].run_decode(o, x, view, s.lens)
        want.append(o)
    wp = torch.empty_like(qp)
    attns[0].run_packed(wp, qp, k, v, cu)
    sync()
    outs = [[torch.zeros_like(x) for x in q] for _ in range(2)]
    packed = [torch.zeros_like(qp) for _ in range(2)]
    sync()
    for i, x in enumerate(q):
        for j in range(2):
            attns[j].run_decode(outs[j][i], x, view, s.lens, stream=streams[j])
            if i == 3 + j:
                attns[j].run_packed(packed[j], qp, k, v, cu, stream=streams[j])
    sync()
    for j in range(2):
        assert torch.equal(packed[j], wp)
        for a, b in zip(outs[j], want):
            assert torch.equal(a, b)
