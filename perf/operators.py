"""The operators that serve a batch of sequences, as cases that can be timed.

Four operators over one paged FP8 cache, through the public Python entry points
(`own`), and in a plain form of elementary torch operations:

  packed   causal attention over whole prompts of different lengths, packed one
           behind the other: BatchAttention.run_packed
  append   the K and V rows of a packed batch (or one token of each sequence)
           into the pages of their sequences: PagedKVCache.append_batch
  decode   one token of each sequence, over a prefix whose pages all share and
           the sequence's own pages: BatchAttention.run_decode
  pages    copying, forking (and freeing), compacting pages of all layers:
           PagedKVCache.copy_pages, PagePool.fork / free / compact
"""
import math
import random

import torch

own = False   # run() calls the framework's operators instead of the plain forms

DEV = "cuda:0"

# (q heads, kv heads, head_dim): head shapes of the repository's configurations
# and tests.
H32, H64, MHA, G7, D64, D256 = ((32, 8, 128), (64, 8, 128), (16, 16, 128), (28, 4, 128),
                                (32, 8, 64), (16, 4, 256))
MOST_PACKED_FLOPS = 2.3e12    # of a drawn case: those of the largest listed one
MOST_DECODE_FLOPS = 6.8e10
MOST_PAGE_BYTES = 2.2e9


def _heads(h):
    return {"hq": h[0], "hkv": h[1], "d": h[2]}


def _packed(heads, seqs, lo, hi, fused=False, pad=0):
    """seqs prompts of lo..hi tokens; fused: q, k, v are slices of one
    projection's rows; pad: rows behind the last prompt."""
    return {"op": "packed", **_heads(heads), "seqs": seqs, "lo": lo, "hi": hi, "fused": fused,
            "pad": pad}


def _append(heads, seqs, lo, hi, cached, block=64):
    """lo..hi new tokens of each sequence behind 0..cached earlier ones."""
    return {"op": "append", **_heads(heads), "seqs": seqs, "lo": lo, "hi": hi, "cached": cached,
            "block": block}


def _decode(heads, seqs, prefix, lo, hi, block=64):
    """A prefix that all share, lo..hi own keys of each sequence behind it."""
    return {"op": "decode", **_heads(heads), "seqs": seqs, "prefix": prefix, "lo": lo, "hi": hi,
            "block": block}


def _pages(what, heads, layers, pages, count, block=64):
    """fork: count children of sequences on `pages` pages; copy: count pages;
    compact: a pool with count of its pages in use."""
    return {"op": "pages", "what": what, **_heads(heads), "layers": layers, "pages": pages,
            "count": count, "block": block}


def listed():
    cases = {
        # The smallest call: one short prompt, all latency.
        "packed_one_37": _packed(H32, 1, 37, 37),
        # An ordinary scheduler step: ragged prompts out of a fused projection,
        # padded up to a captured graph's row count.
        "packed_12_ragged": _packed(H32, 12, 40, 1100, fused=True, pad=19),
        # One long prompt (the configurations' longest).
        "packed_one_16384": _packed(H32, 1, 16384, 16384),
        # One new token of each sequence, every decode step and layer.
        "append_64_tokens": _append(H32, 64, 1, 1, 3000),
        # K and V of packed prompts.
        "append_9_prompts": _append(H32, 9, 100, 2000, 0),
        # A few samples of one ordinary prompt.
        "decode_4_after_1000": _decode(H32, 4, 1000, 1, 60),
        # A service's system prompt, ragged turns behind it.
        "decode_32_after_8192": _decode(H32, 32, 8192, 20, 900),
        # The largest: a long document, many questions about it.
        "decode_128_after_32768": _decode(H32, 128, 32768, 30, 400),
        # A batch that shares nothing, narrow heads.
        "decode_48_apart_d64": _decode(D64, 48, 0, 100, 6000),
        # A beam step: free the last one's children, fork 8 from the best, all
        # layers of a 28-layer model.
        "fork_8_beams": _pages("fork", H32, 28, 96, 8),
        # Pages to copy as a cache is split between two pools' halves.
        "copy_48_pages": _pages("copy", H32, 32, 128, 48),
        # A pool after many requests left it.
        "compact_256": _pages("compact", H32, 32, 256, 120),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["packed", "packed", "append", "decode", "decode", "decode", "pages"])
    block = rng.choice([32, 64, 64, 128, 256])
    if op == "packed":
        heads = rng.choice([H32, H32, H64, MHA, G7, D64, D256])
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 16384)
        lo = rng.randint(0, hi) if rng.random() < 0.7 else hi
        # The plain form holds a score for each pair of rows.
        while (seqs * hi > 16384 or 4.0 * heads[0] * heads[2] * seqs * hi * hi > MOST_PACKED_FLOPS
               or heads[0] * (seqs * hi) ** 2 > 8.6e9):
            seqs, hi = max(1, seqs * 3 // 4), max(1, hi * 4 // 5)
            lo = min(lo, hi)
        return _packed(heads, seqs, lo, hi, fused=heads[2] == 128 and rng.random() < 0.4,
                       pad=rng.choice([0, 0, 1, 40]))
    if op == "append":
        seqs = _log_int(rng, 1, 256)
        hi = 1 if rng.random() < 0.3 else _log_int(rng, 1, max(2, 16384 // seqs))
        return _append(rng.choice([H32, MHA, G7, D64, D256]), seqs, rng.randint(min(1, hi), hi), hi,
                       _log_int(rng, 1, 4000), block)
    if op == "decode":
        heads = rng.choice([H32, H32, H64, MHA, G7, D64, D256])
        seqs = _log_int(rng, 1, 192)
        prefix = 0 if rng.random() < 0.2 else _log_int(rng, 30, 131072)
        hi = _log_int(rng, 1, 8000)
        lo = rng.randint(0 if prefix else 1, hi)
        while (4.0 * heads[0] * heads[2] * seqs * (prefix + hi) > MOST_DECODE_FLOPS or
               seqs * hi * heads[1] * heads[2] > 2.6e8):
            seqs, hi, prefix = max(1, seqs * 4 // 5), max(1, hi * 4 // 5), prefix * 9 // 10
            lo = min(lo, hi)
        return _decode(heads, seqs, prefix, lo, hi, block)
    heads = rng.choice([H32, MHA, G7, D64, D256])
    what = rng.choice(["fork", "copy", "compact"])
    layers, pages = rng.randint(1, 32), _log_int(rng, 24, 512)
    while 2.0 * layers * pages * block * heads[1] * heads[2] > MOST_PAGE_BYTES / 2:
        layers, pages = max(1, layers * 4 // 5), max(24, pages * 4 // 5)
        block = 32 if pages == 24 and layers == 1 else block
    most = pages // 8 if what == "fork" else pages // 2
    return _pages(what, heads, layers, pages, rng.randint(1, max(1, most)), block)


# ---- sizes that follow from a case ---------------------------------------------

def _lens(case):
    """lo..hi per sequence, the first of them hi, spread evenly."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["lo"], case["hi"]))
    return [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]


def _cached(case):
    rng = random.Random("cached %d %d" % (case["seqs"], case["cached"]))
    return [rng.randint(0, case["cached"]) for _ in range(case["seqs"])]


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _up(n, block):
    return (n + block - 1) // block


def _held(case):
    """pages, compact: how many pages of the pool each of its sequences holds."""
    rng, left, held = random.Random("held %d" % case["count"]), case["count"], []
    while left:
        held.append(min(left, rng.randint(1, 12)))
        left -= held[-1]
    return held


def _fork_lens(case):
    """pages, fork: the lengths of the four sequences that are forked from."""
    rng = random.Random("fork %d" % case["pages"])
    most = (case["pages"] - case["count"]) // 4 * case["block"]
    return [rng.randint(max(1, most // 2), most) for _ in range(4)]


def _fork_parents(case):
    rng = random.Random("parents %d" % case["count"])
    return [rng.randrange(4) for _ in range(case["count"])]


def _perm(n, seed, salt):
    gen = torch.Generator().manual_seed(7919 * seed + salt)
    return torch.randperm(n, generator=gen)


# ---- inputs ------------------------------------------------------------------------

def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * seed + salt)


def _keys(gen, n, case):
    """Key rows whose channels differ in size, as a trained model's do."""
    gain = torch.exp(0.5 * torch.randn((case["hkv"], case["d"]), generator=gen, device=DEV))
    return torch.randn((n, case["hkv"], case["d"]), generator=gen, device=DEV) * gain


def _normal(gen, n, h, d):
    return torch.randn((n, h, d), generator=gen, device=DEV)


def _e4m3(x):
    """(codes as uint8, scale) of the cache format: scale = amax / 448 per row."""
    amax = x.abs().amax(-1)
    inv = torch.where(amax > 0, 448.0 / amax, torch.zeros_like(amax))
    codes = (x * inv[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), amax / 448.0


def _new_slabs(case, layers, pages):
    """The slabs of a paged cache, zeroed: of a PagedKVCache, where there is one."""
    shape = (layers, pages * case["block"], case["hkv"], case["d"])
    if own:
        import runtherder_amd as R
        cache = R.PagedKVCache(layers, pages, case["block"], case["hkv"], case["d"], device=DEV)
        slabs = [cache.k, cache.v, cache.k_scale, cache.v_scale]
        for t in slabs:
            t.zero_()
        return cache, slabs
    return None, [torch.zeros(shape, dtype=torch.uint8, device=DEV),
                  torch.zeros(shape, dtype=torch.uint8, device=DEV),
                  torch.zeros(shape[:3], dtype=torch.float32, device=DEV),
                  torch.zeros(shape[:3], dtype=torch.float32, device=DEV)]


def _handle(case, most_seqs):
    """What a program keeps for its batches: the backend with its scratch."""
    if not own:
        return None
    import runtherder_amd as R
    return R.BatchAttention(R.AttnConfig.for_heads(case["hq"], case["hkv"], case["d"]),
                            most_seqs, device=DEV)


def _prepare_packed(case, seed):
    cu, hq, hkv, d = _cu(_lens(case)), case["hq"], case["hkv"], case["d"]
    n, gen = cu[-1] + case["pad"], _gen(seed, 1)
    q, k, v = _normal(gen, n, hq, d), _keys(gen, n, case), _normal(gen, n, hkv, d)
    if case["fused"]:
        rows = torch.cat([q, k, v], 1).to(torch.bfloat16)
        q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    else:
        q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    return {"q": q, "k": k, "v": v, "cu": _int(cu), "attn": _handle(case, case["seqs"]),
            "out": torch.zeros((n, hq, d), dtype=torch.bfloat16, device=DEV)}


def _tables(case, seed, holds):
    """A table row for each sequence: holds[b] pages, shuffled over the pool,
    -1 behind them."""
    pages, at = _perm(sum(holds), seed, 2).to(torch.int32), 0
    tables = torch.full((len(holds), max(max(holds), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(holds):
        tables[b, :n] = pages[at:at + n]
        at += n
    return tables.to(DEV)


def _prepare_append(case, seed):
    lens, cached = _lens(case), _cached(case)
    holds = [_up(a + b, case["block"]) for a, b in zip(lens, cached)]
    cache, slabs = _new_slabs(case, 1, sum(holds))
    gen, n = _gen(seed, 3), sum(lens)
    k = _keys(gen, n, case).to(torch.bfloat16)
    v = _normal(gen, n, case["hkv"], case["d"]).to(torch.bfloat16)
    return {"cache": cache, "slabs": slabs, "block": case["block"], "k": k, "v": v,
            "cu": _int(_cu(lens)), "one": max(lens) == 1 == min(lens),
            "at_pos": _int(cached),
            "tables": _tables(case, seed, holds)}


def _prepare_decode(case, seed):
    block, prefix, lens = case["block"], case["prefix"], _lens(case)
    shared = prefix // block   # whole pages of the prefix: in every table
    # A last, part-filled page of the prefix: each sequence has its own copy,
    # as forking leaves it, and the prefix's table names the first one's.
    holds = [_up(prefix + n, block) - shared for n in lens]
    pages = _perm(shared + sum(holds) + 1, seed, 4).to(torch.int32)
    tables = torch.full((len(lens), max(1, shared + max(holds))), -1, dtype=torch.int32)
    tables[:, :shared] = pages[:shared]
    at = shared
    for b, n in enumerate(holds):
        tables[b, shared:shared + n] = pages[at:at + n]
        at += n
    cache, slabs = _new_slabs(case, 1, shared + sum(holds) + 1)
    rows = slabs[0].shape[1]
    gen = _gen(seed, 5)
    for t, s, x in ((slabs[0], slabs[2], _keys(gen, rows, case)),
                    (slabs[1], slabs[3], _normal(gen, rows, case["hkv"], case["d"]))):
        codes, scale = _e4m3(x)
        t[0].copy_(codes)
        s[0].copy_(scale)
    tables = tables.to(DEV)
    return {"cache": cache, "slabs": slabs, "tables": tables, "prefix": prefix,
            "prefix_table": tables[0].clone(), "prefix_len": _int([prefix]),
            "longest": prefix + max(lens), "block": block,
            "lens": _int([prefix + n for n in lens]),
            "view": cache.batch_view(0, tables) if cache is not None else None,
            "attn": _handle(case, case["seqs"]),
            "q": _normal(gen, len(lens), case["hq"], case["d"]).to(torch.bfloat16),
            "out": torch.zeros((len(lens), case["hq"], case["d"]), dtype=torch.bfloat16,
                               device=DEV)}


def _prepare_pages(case, seed):
    what, block, pages = case["what"], case["block"], case["pages"]
    cache, slabs = _new_slabs(case, case["layers"], pages)
    gen = _gen(seed, 6)
    for t in slabs[:2]:   # any codes but the two NaNs; whole numbers below 2^15 as scales
        t.random_(0, 0x7f, generator=gen)
    for t in slabs[2:]:
        t.copy_(torch.randint(1, 32768, t.shape, generator=gen, device=DEV))
    s = {"cache": cache, "slabs": slabs, "what": what, "block": block}
    if what == "copy":
        order = _perm(pages, seed, 7).to(torch.int32).to(DEV)
        s["src"], s["dst"] = order[:case["count"]].clone(), order[pages - case["count"]:].clone()
        return s
    if what == "fork":
        lens = _fork_lens(case)
        holds = [_up(n, block) for n in lens]
    else:
        holds = _held(case)
        lens = [n * block for n in holds]
    place, at = _perm(pages, seed, 8), 0
    tables = torch.full((len(holds), max(holds)), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for b, n in enumerate(holds):
        tables[b, :n] = place[at:at + n].to(torch.int32)
        refs[place[at:at + n]] = 1
        at += n
    s.update(tables=tables.to(DEV), lens=_int(lens), refs=refs.to(DEV))
    if own:
        import runtherder_amd as R
        s["pool"] = R.PagePool(pages, block, device=DEV)
        s["pool"].refs.copy_(s["refs"])
    if what == "fork":
        s["refs"] = s["pool"].refs if own else s["refs"]
        s["parents"] = _int(_fork_parents(case))
        s["child_tables"] = torch.full((case["count"], max(holds)), -1, dtype=torch.int32,
                                       device=DEV)
        s["child_lens"] = torch.zeros(case["count"], dtype=torch.int32, device=DEV)
    else:
        # The bookkeeping as the server hands it over; a pass renames copies.
        s["tables0"], s["refs0"] = s["tables"], s["refs"]
        s["tables"] = s["tables0"].clone()
        s["refs"] = s["pool"].refs if own else s["refs0"].clone()
    return s


def prepare(case, seed):
    make = {"packed": _prepare_packed, "append": _prepare_append, "decode": _prepare_decode,
            "pages": _prepare_pages}[case["op"]]
    return {"op": case["op"], **make(case, seed)}


# ---- the plain forms -----------------------------------------------------------------

def _plain_packed(s):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"]
    (n, hq, d), hkv = q.shape, k.shape[1]
    at = torch.arange(n, device=DEV, dtype=torch.int32)
    seq = (at[:, None] >= cu[None, 1:]).sum(1)
    unseen = (seq[:, None] != seq[None]) | (at[None] > at[:, None])
    qh = q.float().view(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    p = torch.matmul(qh * (1.0 / math.sqrt(d)), k.float().permute(1, 2, 0).contiguous())
    p = p.view(hkv, hq // hkv, n, n).masked_fill_(unseen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1)
    o = torch.matmul(p.view(hkv, -1, n), v.float().permute(1, 0, 2).contiguous())
    o = o.view(hkv, -1, n, d) / total[..., None]
    o = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(torch.bfloat16)
    return torch.where((at < cu[-1])[:, None, None], o, s["out"])


def _plain_append(s):
    k, v, cu, tables = s["k"], s["v"], s["cu"], s["tables"]
    at = torch.arange(k.shape[0], device=DEV)
    seq = (at[:, None] >= cu[None, 1:]).sum(1)
    pos = s["at_pos"][seq] + at - cu[seq]
    block = s["block"]
    row = tables[seq, pos // block].long() * block + pos % block
    codes, scale = _e4m3(k.float())
    s["slabs"][0][0, row], s["slabs"][2][0, row] = codes, scale
    codes, scale = _e4m3(v.float())
    s["slabs"][1][0, row], s["slabs"][3][0, row] = codes, scale


def _plain_decode(s):
    q, tables, lens, block, prefix = s["q"], s["tables"], s["lens"], s["block"], s["prefix"]
    k8, v8, ks, vs = (t[0] for t in s["slabs"])
    (b, hq, d), hkv = q.shape, k8.shape[1]
    g = hq // hkv
    at = torch.arange(prefix, device=DEV)
    row = s["prefix_table"][at // block].long() * block + at % block
    mine = torch.arange(prefix, s["longest"], device=DEV)
    rows = tables[:, mine // block].long() * block + mine % block
    there = mine < lens[:, None]
    rows = torch.where(there, rows, 0)

    def values(codes, scale, r):
        return codes[r].view(torch.float8_e4m3fn).float() * scale[r][..., None]

    qg = q.float().view(b, hkv, g, d) * (1.0 / math.sqrt(d))
    qs = qg.permute(1, 0, 2, 3).reshape(hkv, b * g, d)
    s1 = torch.matmul(qs, values(k8, ks, row).permute(1, 2, 0).contiguous())
    s1 = s1.view(hkv, b, g, prefix).permute(1, 0, 2, 3)
    s2 = torch.matmul(qg, values(k8, ks, rows).permute(0, 2, 3, 1).contiguous())
    p = torch.cat([s1.masked_fill(~(at < lens[:, None])[:, None, None], -math.inf),
                   s2.masked_fill(~there[:, None, None], -math.inf)], -1)
    top = p.amax(-1, keepdim=True)
    p = (p - torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p1 = p[..., :prefix].permute(1, 0, 2, 3).reshape(hkv, b * g, prefix)
    o = torch.matmul(p1, values(v8, vs, row).permute(1, 0, 2).contiguous())
    o = o.view(hkv, b, g, d).permute(1, 0, 2, 3)
    o = o + torch.matmul(p[..., prefix:], values(v8, vs, rows).permute(0, 2, 1, 3).contiguous())
    return (o / torch.where(total > 0, total, 1.0)).reshape(b, hq, d).to(torch.bfloat16)


def _as_pages(t, block):
    return t.view(t.shape[0], -1, block, *t.shape[2:])


def _plain_fork(s):
    refs, block = s["refs"], s["block"]
    # The children of the last pass are freed.
    slot = torch.arange(s["child_tables"].shape[1], device=DEV)
    held = slot < ((s["child_lens"] + block - 1) // block)[:, None]
    refs.index_add_(0, torch.where(held, s["child_tables"], 0).view(-1), -held.int().view(-1))
    # Shared whole pages, then a page of its own for what is part-filled.
    lens, rows = s["lens"][s["parents"]], s["tables"][s["parents"]]
    full, rest = lens // block, lens % block
    shared, tail = slot < full[:, None], rest > 0
    refs.index_add_(0, torch.where(shared, rows, 0).view(-1), shared.int().view(-1))
    free = torch.argsort((refs > 0).int(), stable=True)[:len(lens)]
    new = free[(tail.cumsum(0) - tail.int())]
    last = rows.gather(1, (full - 1 + tail.int()).clamp(min=0)[:, None])[:, 0].long()
    to = torch.where(tail, new, last)   # without a tail: the last whole page onto itself
    refs.index_add_(0, to, tail.int())
    filled = torch.arange(block, device=DEV) < rest[:, None]
    k, v, ks, vs = (_as_pages(t, block) for t in s["slabs"])
    wide = filled[None, :, :, None, None]
    k[:, to], v[:, to] = (torch.where(wide, k[:, last], k[:, to]),
                          torch.where(wide, v[:, last], v[:, to]))
    ks[:, to], vs[:, to] = (torch.where(wide[..., 0], ks[:, last], ks[:, to]),
                            torch.where(wide[..., 0], vs[:, last], vs[:, to]))
    mine = (slot == full[:, None]) & tail[:, None]
    s["child_tables"].copy_(torch.where(mine, to.int()[:, None], torch.where(shared, rows, -1)))
    s["child_lens"].copy_(lens)


def _move(s, src, dst):
    k, v, ks, vs = (_as_pages(t, s["block"]) for t in s["slabs"])
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    ks[:, dst], vs[:, dst] = ks[:, src], vs[:, src]


def _plain_compact(s):
    refs, tables = s["refs"], s["tables"]
    live, page = refs > 0, torch.arange(len(refs), device=DEV)
    inside = page < live.sum()
    src, dst = (live & ~inside).nonzero()[:, 0], (~live & inside).nonzero()[:, 0]
    _move(s, src, dst)
    page[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    tables.copy_(torch.where(tables >= 0, page[tables.clamp(min=0).long()].int(), -1))


# ---- one pass ------------------------------------------------------------------------

def _codes(s):
    k, v, ks, vs = s["slabs"]
    return {"k": k.view(torch.float8_e4m3fn), "v": v.view(torch.float8_e4m3fn), "k_scale": ks,
            "v_scale": vs}


def _run_pages(s):
    if s["what"] == "copy":
        if own:
            s["cache"].copy_pages(s["src"], s["dst"])
        else:
            _move(s, s["src"].long(), s["dst"].long())
        return _codes(s)
    if s["what"] == "fork":
        if own:
            s["pool"].free(s["child_tables"], s["child_lens"])
            s["pool"].fork(s["cache"], s["child_tables"], s["child_lens"], s["tables"], s["lens"],
                           s["parents"])
        else:
            _plain_fork(s)
        return {"tables": s["child_tables"], "lens": s["child_lens"], "refs": s["refs"],
                **_codes(s)}
    s["tables"].copy_(s["tables0"])
    s["refs"].copy_(s["refs0"])
    if own:
        s["pool"].compact(s["cache"], s["tables"])
    else:
        _plain_compact(s)
    return {"tables": s["tables"], "refs": s["refs"], **_codes(s)}


def run(s):
    if s["op"] == "packed":
        if own:
            s["attn"].run_packed(s["out"], s["q"], s["k"], s["v"], s["cu"])
            return s["out"]
        return _plain_packed(s)
    if s["op"] == "append":
        if own:
            s["cache"].append_batch(0, s["k"], s["v"], s["at_pos"], s["tables"],
                                    None if s["one"] else s["cu"])
        else:
            _plain_append(s)
        return _codes(s)
    if s["op"] == "decode":
        if own:
            s["attn"].run_decode(s["out"], s["q"], s["view"], s["lens"], s["prefix_table"],
                                 s["prefix_len"])
            return s["out"]
        return _plain_decode(s)
    return _run_pages(s)


def _moves(case):
    """Pages (or parts of them, in rows) that a pass of the pages' cases has to move."""
    if case["what"] == "copy":
        return case["count"] * case["block"]
    if case["what"] == "fork":
        lens = _fork_lens(case)
        return sum(lens[p] % case["block"] for p in _fork_parents(case))
    # Expected of a shuffled pool: live pages past the live count.
    live = case["count"]
    return live * (case["pages"] - live) // case["pages"] * case["block"]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "packed":
        lens = _lens(case)
        return {"bytes": 2 * sum(lens) * d * (2 * hq + 2 * hkv),
                "flops": 4 * hq * d * sum(n * (n + 1) // 2 for n in lens)}
    if case["op"] == "append":
        return {"bytes": sum(_lens(case)) * hkv * (6 * d + 8), "flops": 0}
    if case["op"] == "decode":
        lens, prefix = _lens(case), case["prefix"]
        return {"bytes": (prefix + sum(lens)) * hkv * (2 * d + 8) + 4 * len(lens) * hq * d,
                "flops": 4 * hq * d * sum(prefix + n for n in lens)}
    return {"bytes": 2 * _moves(case) * case["layers"] * hkv * (2 * d + 8) + 8 * case["pages"],
            "flops": 0}


# ---- the same in 64 bits, from the definition ------------------------------------------

def _softmax_rows(scores):
    w = torch.exp(scores - scores.max(-1, keepdim=True).values)
    return w / w.sum(-1, keepdim=True)


def _exact_packed(case, s):
    cu, g = _cu(_lens(case)), case["hq"] // case["hkv"]
    out = s["out"].double()
    for a, b in zip(cu, cu[1:]):
        for h in range(case["hq"]):
            kk, vv = s["k"][a:b, h // g].double(), s["v"][a:b, h // g].double()
            for r in range(a, b, 4096):
                e = min(b, r + 4096)
                sc = s["q"][r:e, h].double() @ kk[:e - a].t() / math.sqrt(case["d"])
                late = torch.ones_like(sc, dtype=torch.bool).triu(r - a + 1)
                out[r:e, h] = _softmax_rows(sc.masked_fill_(late, -math.inf)) @ vv[:e - a]
    return out


def _row(table, p, block):
    return int(table[p // block]) * block + p % block


def _quantized(x):
    amax = x.abs().max(-1, keepdim=True).values
    y = torch.where(amax > 0, x * 448.0 / amax, torch.zeros_like(x))
    # Round to E4M3: steps of 2^(e - 3), e the exponent, at least -6.
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step, amax[..., 0] / 448.0


def _exact_append(case, s):
    lens, cached, tables = _lens(case), _cached(case), s["tables"].cpu()
    rows = [_row(tables[b], cached[b] + i, case["block"])
            for b, n in enumerate(lens) for i in range(n)]
    at = torch.tensor(rows, device=DEV)
    k, v, ks, vs = s["slabs"]
    out = {"k": torch.zeros(k.shape, dtype=torch.float64, device=DEV),
           "v": torch.zeros(v.shape, dtype=torch.float64, device=DEV),
           "k_scale": ks.double(), "v_scale": vs.double()}
    for name in ("k", "v"):
        out[name][0, at], out[name + "_scale"][0, at] = _quantized(s[name].double())
    return out


def _exact_decode(case, s):
    tables, block, prefix = s["tables"].cpu(), case["block"], case["prefix"]
    k8, v8, ks, vs = (t[0] for t in s["slabs"])
    g, out = case["hq"] // case["hkv"], s["out"].double()
    pt = s["prefix_table"].cpu()
    for b, n in enumerate(_lens(case)):
        p = torch.arange(prefix + n)
        page = torch.where(p < prefix, pt[(p // block).clamp(max=len(pt) - 1)],
                           tables[b][p // block]).long()
        at = (page * block + p % block).to(DEV)
        kk = k8[at].view(torch.float8_e4m3fn).double() * ks[at].double()[..., None]
        vv = v8[at].view(torch.float8_e4m3fn).double() * vs[at].double()[..., None]
        if not len(at):
            continue
        qb = s["q"][b].double().view(case["hkv"], g, case["d"])
        sc = torch.bmm(qb, kk.permute(1, 2, 0).contiguous()) / math.sqrt(case["d"])
        out[b] = torch.bmm(_softmax_rows(sc), vv.permute(1, 0, 2).contiguous()).view_as(out[b])
    return out


def _exact_pages(case, s):
    block, what = case["block"], case["what"]
    slabs = [t.clone() for t in s["slabs"]]
    moves, more = [], {}   # (page from, page to, rows)
    if what == "copy":
        moves = [(a, b, block) for a, b in zip(s["src"].tolist(), s["dst"].tolist())]
    elif what == "fork":
        refs, tables, lens = s["refs"].tolist(), s["tables"].tolist(), s["lens"].tolist()
        parents, width = s["parents"].tolist(), s["child_tables"].shape[1]
        children = [[-1] * width for _ in parents]
        for i, p in enumerate(parents):
            for j in range(lens[p] // block):
                children[i][j] = tables[p][j]
                refs[tables[p][j]] += 1
        for i, p in enumerate(parents):
            if lens[p] % block:
                page = next(x for x, r in enumerate(refs) if r <= 0)
                refs[page] = 1
                children[i][lens[p] // block] = page
                moves.append((tables[p][lens[p] // block], page, lens[p] % block))
        more = {"tables": _int(children), "lens": _int([lens[p] for p in parents]),
                "refs": _int(refs)}
    else:
        refs, tables = s["refs0"].tolist(), s["tables0"].tolist()
        live = sum(r > 0 for r in refs)
        holes = [x for x in range(live) if refs[x] <= 0]
        name = {x: x for x in range(len(refs))} | {-1: -1}
        for x in range(live, len(refs)):
            if refs[x] > 0:
                to = holes.pop(0)
                name[x], refs[to], refs[x] = to, refs[x], 0
                moves.append((x, to, block))
        more = {"tables": _int([[name[x] for x in row] for row in tables]), "refs": _int(refs)}
    for a, b, n in moves:
        for new, old in zip(slabs, s["slabs"]):
            new[:, b * block:b * block + n] = old[:, a * block:a * block + n]
    return {**more, "k": slabs[0].view(torch.float8_e4m3fn).double(),
            "v": slabs[1].view(torch.float8_e4m3fn).double(), "k_scale": slabs[2].double(),
            "v_scale": slabs[3].double()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"packed": _exact_packed, "append": _exact_append, "decode": _exact_decode,
            "pages": _exact_pages}[case["op"]](case, s)
