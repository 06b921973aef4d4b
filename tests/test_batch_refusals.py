"""What the batch operators refuse, before anything reaches the GPU (CPU only)."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import runtherder_amd as R
from runtherder_amd import _ffi

P = 0x1000   # an aligned address that no refused call looks at
F = ctypes.c_float(0.1)


def refuse(name, args, **change):
    """args: an ordered dict of arguments; each change alone has to be refused."""
    vals = dict(args, **change)
    with pytest.raises(_ffi.RthError) as e:
        _ffi.call(name, *vals.values())
    return str(e.value)


PACKED = dict(out=P, q=P, k=P, v=P, cu=P, seqs=2, rows=64, so=4096, sq=4096, sk=1024, sv=1024, hq=32,
              hkv=8, d=128, scale=F, stream=None)
APPEND = dict(kc=P, vc=P, ks=P, vs=P, k=P, v=P, sk=1024, sv=1024, cu=None, at=P, seqs=2, rows=2, hkv=8, d=128,
              tables=P, width=4, blocks=16, block=64, stream=None)
DECODE = dict(out=P, so=4096, q=P, sq=4096, k=P, v=P, ks=P, vs=P, tables=P, width=4, blocks=16, block=64,
              lens=P, ptable=P, pblocks=2, plen=P, partial=P, seqs=2, hq=32, hkv=8, d=128, scale=F,
              stream=None)
SLABS = dict(k=P, v=P, ks=P, vs=P, layers=2, blocks=16, block=64, hkv=8, d=128)
COPY = dict(SLABS, src=P, dst=P, count=3, stream=None)
RESERVE = dict(refs=P, work=P, status=P, blocks=16, block=64, tables=P, width=4, lens=P, n_new=P, seqs=2,
               stream=None)
FORK = dict(SLABS, refs=P, work=P, status=P, dt=P, dl=P, st=2 * P, sl=2 * P, width=4, src=2, parents=P, kids=2,
            stream=None)
FREE = dict(refs=P, blocks=16, tables=P, width=4, lens=P, drop=None, seqs=2, stream=None)
COMPACT = dict(SLABS, refs=P, work=P, tables=P, width=4, seqs=2, stream=None)


@pytest.mark.parametrize("change,says", [
    (dict(out=None), "null"), (dict(v=None), "null"), (dict(q=P + 8), "16-byte"), (dict(k=P + 2), "16-byte"),
    (dict(cu=None), "cu_seqlens"), (dict(seqs=0), "num_seqs"), (dict(seqs=4097), "num_seqs"),
    (dict(rows=0), "num_rows"), (dict(hq=30), "divisible"), (dict(hq=0), "num_q_heads"), (dict(hkv=0), "num_kv_heads"),
    (dict(d=32), "64, 128, 256"), (dict(d=96), "64, 128, 256"), (dict(sq=4088), "q_stride"), (dict(sq=4100), "q_stride"),
    (dict(sk=1016), "k_stride"), (dict(sv=0), "v_stride"), (dict(so=-4096), "out_stride"),
    (dict(rows=1 << 27), "2^31"),
])
def test_packed(change, says):
    assert says in refuse("rth_attn_packed", PACKED, **change)


@pytest.mark.parametrize("change,says", [
    (dict(kc=None), "null"), (dict(vs=None), "null"), (dict(k=None), "null"), (dict(v=P + 4), "16-byte"),
    (dict(kc=P + 8), "16-byte"), (dict(at=None), "at_pos"), (dict(seqs=0), "num_seqs"), (dict(rows=0), "num_rows"),
    (dict(hkv=0), "num_kv_heads"), (dict(d=12), "multiple of 8"), (dict(d=520), "multiple of 8"),
    (dict(sk=1000), "k_stride"), (dict(sv=1028), "v_stride"), (dict(tables=None), "block_tables"),
    (dict(width=0), "table_blocks"), (dict(blocks=0), "num_blocks"), (dict(block=48), "power of two"),
    (dict(block=16), "power of two"), (dict(blocks=1 << 26), "2^31"), (dict(rows=1 << 29), "2^31"),
])
def test_append(change, says):
    assert says in refuse("rth_kv_append_fp8_batch", APPEND, **change)


@pytest.mark.parametrize("change,says", [
    (dict(out=None), "null"), (dict(q=P + 4), "16-byte"), (dict(k=None), "null"), (dict(v=P + 8), "16-byte"),
    (dict(lens=None), "lens"), (dict(ptable=None), "together"), (dict(plen=None), "together"),
    (dict(pblocks=0), "prefix_blocks"), (dict(partial=None), "partial"), (dict(partial=P + 4), "partial"),
    (dict(seqs=0), "num_seqs"), (dict(seqs=5000), "num_seqs"), (dict(hq=31), "divisible"), (dict(d=512), "64, 128, 256"),
    (dict(so=100), "out_stride"), (dict(sq=4092), "q_stride"), (dict(tables=None), "block_tables"),
    (dict(width=-1), "table_blocks"), (dict(blocks=0), "num_blocks"), (dict(block=100), "power of two"),
    (dict(blocks=1 << 26), "2^31"), (dict(seqs=4096, hq=1 << 13, hkv=1, so=1 << 21, sq=1 << 21), "2^24"),
    (dict(width=(1 << 28) + 1), "2^35"), (dict(seqs=4096, width=1 << 18), "2^35"),
])
def test_decode(change, says):
    assert says in refuse("rth_attn_decode_batch", DECODE, **change)


@pytest.mark.parametrize("change,says", [
    (dict(k=None), "null"), (dict(k=P + 8), "16-byte"), (dict(layers=0), "num_layers"), (dict(blocks=0), "num_blocks"),
    (dict(block=31), "power of two"), (dict(hkv=0), "num_kv_heads"), (dict(d=4), "multiple of 8"),
])
def test_page_slabs(change, says):
    for name, args in (("rth_pages_copy", COPY), ("rth_pages_fork", FORK), ("rth_pages_compact", COMPACT)):
        assert says in refuse(name, args, **change)


@pytest.mark.parametrize("name,args,change,says", [
    ("rth_pages_copy", COPY, dict(src=None), "src"), ("rth_pages_copy", COPY, dict(count=0), "count"),
    ("rth_pages_reserve", RESERVE, dict(refs=None), "refs"), ("rth_pages_reserve", RESERVE, dict(work=None), "work"),
    ("rth_pages_reserve", RESERVE, dict(block=0), "power of two"), ("rth_pages_reserve", RESERVE, dict(n_new=None), "n_new"),
    ("rth_pages_reserve", RESERVE, dict(seqs=4097), "num_seqs"), ("rth_pages_reserve", RESERVE, dict(width=0), "table_blocks"),
    ("rth_pages_fork", FORK, dict(parents=None), "parents"), ("rth_pages_fork", FORK, dict(status=None), "status"),
    ("rth_pages_fork", FORK, dict(dt=2 * P), "of its own"), ("rth_pages_fork", FORK, dict(dl=2 * P), "of its own"),
    ("rth_pages_fork", FORK, dict(kids=0), "num_children"), ("rth_pages_fork", FORK, dict(kids=4097), "num_children"),
    ("rth_pages_fork", FORK, dict(src=0), "num_seqs"),
    ("rth_pages_free", FREE, dict(lens=None), "lens"), ("rth_pages_free", FREE, dict(tables=None), "block_tables"),
    ("rth_pages_free", FREE, dict(blocks=0), "num_blocks"),
    ("rth_pages_compact", COMPACT, dict(work=None), "work"), ("rth_pages_compact", COMPACT, dict(seqs=0), "num_seqs"),
])
def test_pool(name, args, change, says):
    assert says in refuse(name, args, **change)


def test_sizes():
    lib = _ffi.load()
    assert lib.rth_batch_scratch_floats(0, 32, 8, 128) == 0 == lib.rth_batch_scratch_floats(2, 30, 8, 128)
    assert lib.rth_batch_scratch_floats(5000, 32, 8, 128) == 0 == lib.rth_pages_work_ints(0)
    assert R.batch_scratch_floats(4, 32, 8, 128) > 4 * 32 * 130


def test_python_checks():
    """The tensors' own checks: device, type, shape, strides."""
    host = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        R.flash_packed_bf16(host, host, host, host, i, 2, 2, 64, 0.1)
    with pytest.raises(TypeError):
        R.flash_packed_bf16(host.float(), host, host, host, i, 2, 2, 64, 0.1)
    with pytest.raises(TypeError):
        R.flash_decode_batch_bf16(host, host, host, host, host, host, i, 32, i, i, 2, 2, 64, 0.1)
    with pytest.raises(TypeError):
        R.kv_append_fp8_batch(host, host, host, host, host, host, i, i, 32, 2, 64)
    for bad in (0, 16, 33):
        with pytest.raises(ValueError):
            R.PagePool(4, bad, device="cpu")
    pool = R.PagePool(4, 32, device="cpu")
    cache = R.PagedKVCache(1, 5, 32, 1, 8, device="cpu")
    with pytest.raises(ValueError):
        pool.compact(cache, pool.new_tables(1, 2))
    with pytest.raises(TypeError):
        pool.free(pool.new_tables(2, 2), i)
    for layer in (-1, 1):
        with pytest.raises(ValueError):
            cache.append_batch(layer, host, host, i, i)
        with pytest.raises(ValueError):
            cache.batch_view(layer, i)


def test_a_cache_or_pool_elsewhere():
    """Every tensor behind a call lies on the current device: a cache's, a pool's, a view's."""
    rows = torch.zeros((2, 1, 8), dtype=torch.bfloat16)
    i, pages = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 2), dtype=torch.int32)
    cache, pool = R.PagedKVCache(1, 4, 32, 1, 8, device="cpu"), R.PagePool(4, 32, device="cpu")
    for call in (lambda: cache.append_batch(0, rows, rows, i, pages), lambda: cache.copy_pages(i, i),
                 lambda: pool.reserve(pages, i, i), lambda: pool.free(pages, i),
                 lambda: pool.fork(cache, pages, i, pages, i, i), lambda: pool.compact(cache, pages)):
        with pytest.raises(TypeError, match="current device"):
            call()


@pytest.mark.parametrize("header,check", [
    ("runtherder/kernels/batch.h", "static_assert(sizeof(&runtherder::kernels::flash_decode_batch_bf16) > 0);"),
    ("runtherder/attention/batch.h",
     "static_assert(std::is_constructible_v<runtherder::attention::BatchAttention, "
     "const runtherder::attention::AttnConfig&, int>);"),
    ("runtherder/engine/page_pool.h",
     "static_assert(std::is_same_v<decltype(std::declval<const runtherder::engine::PagedKVCache&>()"
     ".batch_view(0, nullptr, 1, 1)), runtherder::attention::KVBatchView>);"),
])
def test_cpp_headers_stand_alone(header, check):
    root = Path(__file__).resolve().parents[1]
    src = f"#include <{header}>\n#include <type_traits>\n#include <utility>\n{check}\nint main() {{ return 0; }}\n"
    res = subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++20", "-fsyntax-only", "-x", "hip",
                          f"-I{root / 'include'}", "--offload-arch=gfx950", "-"],
                         input=src, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
