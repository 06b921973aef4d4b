"""Torch-tensor front end of the C ABI, mirroring the reference's kernel free
functions and its AttentionBackend / KVCache interface (reference
include/runtherder/kernels/*.cuh, include/runtherder/attention/*.h,
include/runtherder/engine/kv_cache.h). Same names, argument order and
meaning; errors raise RthError instead of exiting the process.

torch only provides device memory and the current stream here: every
computation runs in libruntherder_attn.so.

dtypes: bf16 tensors are torch.bfloat16, E4M3 cache bytes torch.uint8, scales
torch.float32, device-resident positions torch.int32 (one element).
"""
from __future__ import annotations

import enum
import math
from dataclasses import dataclass

import torch

from . import _ffi


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# The current stream's handle without a torch.cuda.Stream object around it (2.8
# -> 0.2 us of a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


_ready = False   # the GPU was used (asked of torch once)


def _current_device() -> int:
    """The current device; no tensor's where the GPU was never used."""
    global _ready
    if not _ready:
        _ready = torch.cuda.is_initialized()
        if not _ready:
            return -2
    return _get_device()


def _stream(stream) -> int | None:
    if stream is None:
        if _raw_stream is not None and torch.cuda.is_initialized():
            return _raw_stream(_get_device())
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _need(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor")
    if not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous")


# ---- kernels ---------------------------------------------------------------

def quantize_kv_fp8(q, scale, x, at_pos, rows_per_pos, num_rows, head_dim, stream=None):
    """reference include/runtherder/kernels/quantization.cuh:50-57"""
    _need(q, torch.uint8, "q"); _need(scale, torch.float32, "scale")
    _need(x, torch.bfloat16, "x"); _need(at_pos, torch.int32, "at_pos")
    _ffi.call("rth_kv_quantize_fp8", _p(q), _p(scale), _p(x), _p(at_pos),
              rows_per_pos, num_rows, head_dim, _stream(stream))


def quantize_kv_fp8_scaled(q, scale, x, at_pos, rows_per_pos, num_rows, head_dim, stream=None):
    """Given-scale variant: scale[dst] is an input (no reference counterpart)."""
    _need(q, torch.uint8, "q"); _need(scale, torch.float32, "scale")
    _need(x, torch.bfloat16, "x"); _need(at_pos, torch.int32, "at_pos")
    _ffi.call("rth_kv_quantize_fp8_scaled", _p(q), _p(scale), _p(x), _p(at_pos),
              rows_per_pos, num_rows, head_dim, _stream(stream))


def flash_split_scratch_floats(num_q_heads: int, head_dim: int, max_splits: int) -> int:
    """reference include/runtherder/kernels/flash_decode.cuh:16-24"""
    return int(_ffi.load().rth_split_scratch_floats(num_q_heads, head_dim, max_splits))


def new_flash_split_scratch(num_q_heads, head_dim, max_splits, device="cuda"):
    """Allocates decode scratch (no initialization needed)."""
    n = flash_split_scratch_floats(num_q_heads, head_dim, max_splits)
    return torch.empty(n, dtype=torch.float32, device=device)


def default_num_splits(num_kv_heads: int, device: int = 0) -> int:
    return int(_ffi.load().rth_default_num_splits(num_kv_heads, device))


def flash_decode_split_bf16(out, q, k, v, k_scale, v_scale, partial, num_splits, cache_len,
                            num_q_heads, num_kv_heads, head_dim, scale, stream=None):
    """reference include/runtherder/kernels/flash_decode.cuh:45-59"""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k, torch.uint8, "k"); _need(v, torch.uint8, "v")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(partial, torch.float32, "partial"); _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_decode_split", _p(out), _p(q), _p(k), _p(v), _p(k_scale),
              _p(v_scale), _p(partial), num_splits, _p(cache_len), num_q_heads,
              num_kv_heads, head_dim, float(scale), _stream(stream))


DECODE_MFMA, DECODE_VALU = 1, 2


def decode_path(num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Which split kernel decode runs for the shape: DECODE_MFMA, DECODE_VALU
    or 0 (unsupported). No reference counterpart."""
    return int(_ffi.load().rth_decode_path(num_q_heads, num_kv_heads, head_dim))


def set_decode_kernel(path: int) -> None:
    """Process-wide split-kernel choice for the non-paged decode entries: 0
    (automatic: MFMA where supported) or DECODE_VALU (the VALU kernel for
    every shape), for measurement. No reference counterpart."""
    _ffi.call("rth_set_decode_kernel", int(path))


def flash_decode_split_bf16_noalloc(out, q, k, v, k_scale, v_scale, num_splits, cache_len,
                                    num_q_heads, num_kv_heads, head_dim, scale, stream=None):
    """flash_decode_split_bf16 without caller scratch (no reference
    counterpart): the partials live in the library's fixed per-device array,
    shared by every call on the device (overlapping calls race)."""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k, torch.uint8, "k"); _need(v, torch.uint8, "v")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_decode_split_noalloc", _p(out), _p(q), _p(k), _p(v), _p(k_scale),
              _p(v_scale), num_splits, _p(cache_len), num_q_heads, num_kv_heads, head_dim,
              float(scale), _stream(stream))


def flash_decode_append_split_bf16(out, q, k_cache, v_cache, k_scale, v_scale, k_new, v_new,
                                   partial, num_splits, cache_len, num_q_heads, num_kv_heads,
                                   head_dim, scale, stream=None):
    """Append one token at row *cache_len and decode over *cache_len + 1 keys
    in one call (no reference counterpart: KVCache::append then the decode)."""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k_cache, torch.uint8, "k_cache"); _need(v_cache, torch.uint8, "v_cache")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(k_new, torch.bfloat16, "k_new"); _need(v_new, torch.bfloat16, "v_new")
    _need(partial, torch.float32, "partial"); _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_decode_append_split", _p(out), _p(q), _p(k_cache), _p(v_cache),
              _p(k_scale), _p(v_scale), _p(k_new), _p(v_new), _p(partial), num_splits,
              _p(cache_len), num_q_heads, num_kv_heads, head_dim, float(scale), _stream(stream))


def flash_decode_rope_append_split_bf16(out, q, k_cache, v_cache, k_scale, v_scale, k_new,
                                        v_new, positions, inv_freq, partial, num_splits,
                                        cache_len, num_q_heads, num_kv_heads, head_dim, scale,
                                        stream=None):
    """The per-layer decode step rope_bf16(q, k) -> KVCache::append -> run in
    one call (no reference counterpart; replaces reference
    src/model/supported/llama/llama3.cu:228-234). q and k_new are read only
    (rotated in registers by positions[0]); cache bytes and output equal
    rope_bf16 + flash_decode_append_split_bf16 on the rotated q and k."""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k_cache, torch.uint8, "k_cache"); _need(v_cache, torch.uint8, "v_cache")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(k_new, torch.bfloat16, "k_new"); _need(v_new, torch.bfloat16, "v_new")
    _need(positions, torch.int32, "positions"); _need(inv_freq, torch.float32, "inv_freq")
    _need(partial, torch.float32, "partial"); _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_decode_rope_append_split", _p(out), _p(q), _p(k_cache), _p(v_cache),
              _p(k_scale), _p(v_scale), _p(k_new), _p(v_new), _p(positions), _p(inv_freq),
              _p(partial), num_splits, _p(cache_len), num_q_heads, num_kv_heads, head_dim,
              float(scale), _stream(stream))


def flash_decode_qk_norm_rope_append_split_bf16(out, q, k_cache, v_cache, k_scale, v_scale,
                                                k_new, v_new, q_norm, k_norm, eps, positions,
                                                inv_freq, partial, num_splits, cache_len,
                                                num_q_heads, num_kv_heads, head_dim, scale,
                                                stream=None):
    """The Qwen3 decode step (per-head RMSNorm of q and k, RoPE, append, run)
    in one call (no reference counterpart; replaces reference
    src/model/supported/llama/qwen3.cu:189-202). q and k_new are read only."""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k_cache, torch.uint8, "k_cache"); _need(v_cache, torch.uint8, "v_cache")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(k_new, torch.bfloat16, "k_new"); _need(v_new, torch.bfloat16, "v_new")
    _need(q_norm, torch.bfloat16, "q_norm"); _need(k_norm, torch.bfloat16, "k_norm")
    _need(positions, torch.int32, "positions"); _need(inv_freq, torch.float32, "inv_freq")
    _need(partial, torch.float32, "partial"); _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_decode_qk_norm_rope_append_split", _p(out), _p(q), _p(k_cache),
              _p(v_cache), _p(k_scale), _p(v_scale), _p(k_new), _p(v_new), _p(q_norm),
              _p(k_norm), float(eps), _p(positions), _p(inv_freq), _p(partial), num_splits,
              _p(cache_len), num_q_heads, num_kv_heads, head_dim, float(scale),
              _stream(stream))


def flash_prefill_bf16(out, q, k, v, k_scale, v_scale, n_new, cache_len, num_q_heads,
                       num_kv_heads, head_dim, scale, stream=None):
    """reference include/runtherder/kernels/flash_prefill.cuh:26-39"""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k, torch.uint8, "k"); _need(v, torch.uint8, "v")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_prefill", _p(out), _p(q), _p(k), _p(v), _p(k_scale), _p(v_scale),
              n_new, _p(cache_len), num_q_heads, num_kv_heads, head_dim, float(scale),
              _stream(stream))


PREFILL_SPLIT_MAX_TOKENS = 4096


def flash_prefill_split_bf16(out, q, k, v, k_scale, v_scale, partial, num_splits, n_new,
                             cache_len, num_q_heads, num_kv_heads, head_dim, scale,
                             stream=None):
    """flash_prefill_bf16 split over the keys, for calls after a long cache
    (no reference counterpart; the reference walks every key serially per q
    tile, flash_prefill.cu:34-241): up to 80 tokens (40, where num_splits
    fills the chip at head_dim 128) as split-K decode over (token block, kv
    head) units with the decode's merge, beyond (head_dim 128) the flash prefill
    over num_splits key runs per block of 128 rows with a merge of their own.
    partial: flash_split_scratch_floats(n_new * num_q_heads, head_dim,
    num_splits) floats; 1 <= n_new <= PREFILL_SPLIT_MAX_TOKENS."""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k, torch.uint8, "k"); _need(v, torch.uint8, "v")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(partial, torch.float32, "partial"); _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_prefill_split", _p(out), _p(q), _p(k), _p(v), _p(k_scale),
              _p(v_scale), _p(partial), num_splits, n_new, _p(cache_len), num_q_heads,
              num_kv_heads, head_dim, float(scale), _stream(stream))


def attention_causal_bf16(out, q, k, v, k_scale, v_scale, n_new, cache_len, num_q_heads,
                          num_kv_heads, head_dim, scale, stream=None):
    """reference include/runtherder/kernels/attention.cuh:21-34"""
    _need(out, torch.bfloat16, "out"); _need(q, torch.bfloat16, "q")
    _need(k, torch.uint8, "k"); _need(v, torch.uint8, "v")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(cache_len, torch.int32, "cache_len")
    _ffi.call("rth_attn_naive", _p(out), _p(q), _p(k), _p(v), _p(k_scale), _p(v_scale),
              n_new, _p(cache_len), num_q_heads, num_kv_heads, head_dim, float(scale),
              _stream(stream))


def advance_position(pos, delta=1, stream=None):
    """*pos += delta on device (lets one graph hold several decode steps)."""
    _need(pos, torch.int32, "pos")
    _ffi.call("rth_advance_position", _p(pos), int(delta), _stream(stream))


def rope_bf16(q, k, positions, inv_freq, seq_len, num_q_heads, num_kv_heads, head_dim,
              stream=None):
    """In-place rotate-half RoPE on q and k (reference
    include/runtherder/kernels/rope.cuh:16-25)."""
    _need(q, torch.bfloat16, "q"); _need(k, torch.bfloat16, "k")
    _need(positions, torch.int32, "positions"); _need(inv_freq, torch.float32, "inv_freq")
    _ffi.call("rth_rope_bf16", _p(q), _p(k), _p(positions), _p(inv_freq), seq_len,
              num_q_heads, num_kv_heads, head_dim, _stream(stream))


def rope_append_fp8(q, k_cache, v_cache, k_scale, v_scale, k, v, positions, inv_freq, at_pos,
                    n_new, num_q_heads, num_kv_heads, head_dim, stream=None):
    """rope_bf16(q, k) + KV append in one launch; q rotated in place, k left
    unrotated, cache bytes identical to the two-step sequence (no reference
    counterpart; replaces reference src/model/supported/llama/llama3.cu:228-232)."""
    _need(q, torch.bfloat16, "q"); _need(k, torch.bfloat16, "k"); _need(v, torch.bfloat16, "v")
    _need(k_cache, torch.uint8, "k_cache"); _need(v_cache, torch.uint8, "v_cache")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(positions, torch.int32, "positions"); _need(inv_freq, torch.float32, "inv_freq")
    _need(at_pos, torch.int32, "at_pos")
    _ffi.call("rth_rope_append_fp8", _p(q), _p(k_cache), _p(v_cache), _p(k_scale), _p(v_scale),
              _p(k), _p(v), _p(positions), _p(inv_freq), _p(at_pos), n_new, num_q_heads,
              num_kv_heads, head_dim, _stream(stream))


def qk_norm_rope_append_fp8(q, k_cache, v_cache, k_scale, v_scale, k, v, q_norm, k_norm, eps,
                            positions, inv_freq, at_pos, n_new, num_q_heads, num_kv_heads,
                            head_dim, stream=None):
    """Per-head RMSNorm of q and k, RoPE, then the KV append, in one launch (no
    reference counterpart; replaces reference
    src/model/supported/llama/qwen3.cu:189-200). q updated in place; k read only."""
    _need(q, torch.bfloat16, "q"); _need(k, torch.bfloat16, "k"); _need(v, torch.bfloat16, "v")
    _need(k_cache, torch.uint8, "k_cache"); _need(v_cache, torch.uint8, "v_cache")
    _need(k_scale, torch.float32, "k_scale"); _need(v_scale, torch.float32, "v_scale")
    _need(q_norm, torch.bfloat16, "q_norm"); _need(k_norm, torch.bfloat16, "k_norm")
    _need(positions, torch.int32, "positions"); _need(inv_freq, torch.float32, "inv_freq")
    _need(at_pos, torch.int32, "at_pos")
    _ffi.call("rth_qk_norm_rope_append_fp8", _p(q), _p(k_cache), _p(v_cache), _p(k_scale),
              _p(v_scale), _p(k), _p(v), _p(q_norm), _p(k_norm), float(eps), _p(positions),
              _p(inv_freq), _p(at_pos), n_new, num_q_heads, num_kv_heads, head_dim,
              _stream(stream))


def rmsnorm_bf16(y, x, g, num_tokens, hidden_dim, eps, stream=None):
    """y = bf16((x * rrms) * g) per row (reference
    include/runtherder/kernels/rmsnorm.cuh:14-22); y may alias x."""
    _need(y, torch.bfloat16, "y"); _need(x, torch.bfloat16, "x"); _need(g, torch.bfloat16, "g")
    _ffi.call("rth_rmsnorm_bf16", _p(y), _p(x), _p(g), num_tokens, hidden_dim, float(eps),
              _stream(stream))


def rmsnorm_lanes(hidden_dim: int) -> int:
    """Lane partials of rmsnorm_bf16's sum of squares (its summation order)."""
    return int(_ffi.load().rth_rmsnorm_lanes(hidden_dim))


def _stream_of(stream, device: int) -> int | None:
    """_stream, where the current device is known already."""
    if stream is None and _raw_stream is not None:
        return _raw_stream(device)
    return _stream(stream)


# ---- batches ---------------------------------------------------------------
# No reference counterparts: the reference serves one sequence at a time.

# The tensors of a call lie on the current device, whose streams it runs on.

def _need_on(t: torch.Tensor, dtype: torch.dtype, name: str, device: int) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != device:
        raise TypeError(f"{name} must be a tensor of the current device")
    if not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous")


def _need_rows(t: torch.Tensor, rows: int, heads: int, head_dim: int, name: str,
               device: int) -> int:
    """t: [rows, heads, head_dim] bf16, rows any stride apart; the stride."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be torch.bfloat16, got {t.dtype}")
    if t.get_device() != device:
        raise TypeError(f"{name} must be a tensor of the current device")
    if t.shape != (rows, heads, head_dim):
        raise ValueError(f"{name} must be [{rows}, {heads}, {head_dim}], got {tuple(t.shape)}")
    row, head, one = t.stride()
    if one != 1 or (head != head_dim and heads > 1):
        raise TypeError(f"{name}: a row's heads must be contiguous")
    return row if rows > 1 else heads * head_dim


def _need_here(t: torch.Tensor, name: str, device: int) -> None:
    if t.get_device() != device:
        raise TypeError(f"{name} must be on the current device")


def _need_len(t: torch.Tensor, n: int, name: str, device: int) -> None:
    _need_on(t, torch.int32, name, device)
    if t.numel() != n:
        raise ValueError(f"{name} must hold {n} ints, got {t.numel()}")


def _need_tables(t: torch.Tensor, num_seqs: int, name: str, device: int) -> int:
    """t: [num_seqs, table_blocks] int32; table_blocks."""
    _need_on(t, torch.int32, name, device)
    shape = t.shape
    if len(shape) != 2 or shape[0] != num_seqs:
        raise ValueError(f"{name} must be [{num_seqs}, blocks], got {tuple(shape)}")
    return shape[1]


def _need_slabs_of(k, v, k_scale, v_scale, block_size, num_kv_heads, head_dim, device) -> int:
    """One layer's paged slabs; the number of blocks."""
    _need_on(k, torch.uint8, "k", device); _need_on(v, torch.uint8, "v", device)
    _need_on(k_scale, torch.float32, "k_scale", device)
    _need_on(v_scale, torch.float32, "v_scale", device)
    rows = k.numel() // (num_kv_heads * head_dim)
    if (block_size < 1 or rows % block_size or k.numel() != rows * num_kv_heads * head_dim
            or v.numel() != k.numel() or k_scale.numel() != rows * num_kv_heads
            or v_scale.numel() != k_scale.numel()):
        raise ValueError("slabs must hold whole blocks of [block_size, kv heads, head_dim] codes "
                         "and [block_size, kv heads] scales")
    return rows // block_size


def flash_packed_bf16(out, q, k, v, cu_seqlens, num_q_heads, num_kv_heads, head_dim, scale,
                      stream=None):
    """Causal attention over whole prompts packed one behind the other: rows
    cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of q, out [rows, Hq, D] and k, v
    [rows, Hkv, D] are sequence b. Rows may lie any stride apart (slices of a
    fused projection); rows behind the last sequence stay as they are."""
    dev, n = _current_device(), len(q)
    so = _need_rows(out, n, num_q_heads, head_dim, "out", dev)
    sq = _need_rows(q, n, num_q_heads, head_dim, "q", dev)
    sk = _need_rows(k, n, num_kv_heads, head_dim, "k", dev)
    sv = _need_rows(v, n, num_kv_heads, head_dim, "v", dev)
    _need_on(cu_seqlens, torch.int32, "cu_seqlens", dev)
    _ffi.call("rth_attn_packed", out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, n, so, sq, sk, sv, num_q_heads,
              num_kv_heads, head_dim, scale, _stream_of(stream, dev))


def kv_append_fp8_batch(k_cache, v_cache, k_scale, v_scale, k, v, at_pos, block_tables,
                        block_size, num_kv_heads, head_dim, cu_seqlens=None, stream=None):
    """Appends a batch's rows (k, v [rows, Hkv, D], packed by cu_seqlens, or
    one row per sequence) to the pages of their sequences, sequence b from
    position at_pos[b] on; bytes as PagedKVCache.append's. Rows without a page
    are not stored. Sequences that share a page do not both write to it."""
    dev = _current_device()
    blocks = _need_slabs_of(k_cache, v_cache, k_scale, v_scale, block_size, num_kv_heads,
                            head_dim, dev)
    _append_batch(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                  k, v, at_pos, block_tables, blocks, block_size, num_kv_heads, head_dim,
                  cu_seqlens, dev, stream)


def _append_batch(kc, vc, ks, vs, k, v, at_pos, block_tables, num_blocks, block_size,
                  num_kv_heads, head_dim, cu_seqlens, dev, stream):
    n, seqs = len(k), at_pos.numel()
    sk = _need_rows(k, n, num_kv_heads, head_dim, "k", dev)
    sv = _need_rows(v, n, num_kv_heads, head_dim, "v", dev)
    _need_on(at_pos, torch.int32, "at_pos", dev)
    if cu_seqlens is not None:
        _need_len(cu_seqlens, seqs + 1, "cu_seqlens", dev)
        cu_seqlens = cu_seqlens.data_ptr()
    elif n != seqs:
        raise ValueError("without cu_seqlens, k and v hold one row per sequence")
    width = _need_tables(block_tables, seqs, "block_tables", dev)
    _ffi.call("rth_kv_append_fp8_batch", kc, vc, ks, vs, k.data_ptr(), v.data_ptr(), sk, sv,
              cu_seqlens, at_pos.data_ptr(), seqs, n, num_kv_heads, head_dim,
              block_tables.data_ptr(), width, num_blocks, block_size, _stream_of(stream, dev))


def batch_scratch_floats(num_seqs: int, num_q_heads: int, num_kv_heads: int,
                         head_dim: int) -> int:
    """Floats of flash_decode_batch_bf16's scratch on the current device."""
    return int(_ffi.load().rth_batch_scratch_floats(num_seqs, num_q_heads, num_kv_heads, head_dim))


def flash_decode_batch_bf16(out, q, k, v, k_scale, v_scale, block_tables, block_size, lens,
                            partial, num_q_heads, num_kv_heads, head_dim, scale,
                            prefix_table=None, prefix_len=None, stream=None):
    """One query token of each sequence (q, out [seqs, Hq, D]) over keys
    0 .. lens[b] - 1 of its pages. The first prefix_len[0] keys are shared: they
    lie in the pages of prefix_table and are read once for the whole batch; the
    others in block_tables[b], at their own positions. lens[b] <= 0: an unused
    slot, zeros. partial: batch_scratch_floats floats."""
    dev, seqs = _current_device(), len(q)
    blocks = _need_slabs_of(k, v, k_scale, v_scale, block_size, num_kv_heads, head_dim, dev)
    width = _need_tables(block_tables, seqs, "block_tables", dev)
    _need_on(partial, torch.float32, "partial", dev)
    if partial.numel() < batch_scratch_floats(seqs, num_q_heads, num_kv_heads, head_dim):
        raise ValueError("partial is smaller than batch_scratch_floats")
    _decode_batch(out, q, k, v, k_scale, v_scale, block_tables, width, blocks, block_size, lens,
                  partial, num_q_heads, num_kv_heads, head_dim, scale, prefix_table, prefix_len,
                  seqs, dev, stream)


def _decode_batch(out, q, k, v, k_scale, v_scale, block_tables, width, num_blocks, block_size,
                  lens, partial, num_q_heads, num_kv_heads, head_dim, scale, prefix_table,
                  prefix_len, seqs, dev, stream):
    so = _need_rows(out, seqs, num_q_heads, head_dim, "out", dev)
    sq = _need_rows(q, seqs, num_q_heads, head_dim, "q", dev)
    _need_len(lens, seqs, "lens", dev)
    pt = pn = pl = 0
    if prefix_table is not None and prefix_len is not None:
        _need_on(prefix_table, torch.int32, "prefix_table", dev)
        _need_len(prefix_len, 1, "prefix_len", dev)
        pt, pn, pl = prefix_table.data_ptr(), prefix_table.numel(), prefix_len.data_ptr()
    elif prefix_table is not prefix_len:
        raise ValueError("prefix_table and prefix_len go together")
    _ffi.call("rth_attn_decode_batch", out.data_ptr(), so, q.data_ptr(), sq, k.data_ptr(),
              v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(), width,
              num_blocks, block_size, lens.data_ptr(), pt, pn, pl, partial.data_ptr(), seqs,
              num_q_heads, num_kv_heads, head_dim, scale, _stream_of(stream, dev))


# ---- interface -------------------------------------------------------------

@dataclass(frozen=True)
class AttnConfig:
    """reference include/runtherder/attention/backend.h:14-19"""
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    scale: float

    @staticmethod
    def for_heads(num_q_heads, num_kv_heads, head_dim):
        return AttnConfig(num_q_heads, num_kv_heads, head_dim, 1.0 / math.sqrt(head_dim))


@dataclass(frozen=True)
class KVView:
    """reference include/runtherder/attention/kv_view.h:14-19; block_table /
    block_size (no reference counterpart) describe a paged layout."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    block_table: torch.Tensor | None = None
    block_size: int = 0


@dataclass(frozen=True)
class KVSlabs(KVView):
    """The writable slabs of one layer (KVCache.slabs / PagedKVCache.slabs),
    for the fused decode steps that store the new token into the cache. No
    reference counterpart: the reference appends through KVCache::append and
    reads through KVView only."""

    def view(self) -> KVView:
        return KVView(self.k, self.v, self.k_scale, self.v_scale, self.block_table,
                      self.block_size)


@dataclass(frozen=True)
class KVBatchView:
    """One layer of a paged cache with the block tables of a batch, as
    PagedKVCache.batch_view makes it: block_tables [seqs, table_blocks] int32,
    entries < 0 hold no page. No reference counterpart."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    block_tables: torch.Tensor
    block_size: int
    num_blocks: int
    num_kv_heads: int
    head_dim: int


def _need_slabs(kv):
    if not isinstance(kv, KVSlabs):
        raise TypeError("the fused decode steps write the cache: pass KVCache.slabs(layer) "
                        "(or PagedKVCache.slabs(layer, block_table)), not a read-only view")


class KVCache:
    """reference include/runtherder/engine/kv_cache.h:23-104"""

    def __init__(self, num_layers, max_seq_len, num_kv_heads, head_dim, device="cuda"):
        for name, val in (("num_layers", num_layers), ("max_seq_len", max_seq_len),
                          ("num_kv_heads", num_kv_heads), ("head_dim", head_dim)):
            if val < 1:
                raise ValueError(f"KVCache {name} must be >= 1")
        self.num_layers, self._max_seq_len = num_layers, max_seq_len
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        shape = (num_layers, max_seq_len, num_kv_heads, head_dim)
        self.k = torch.empty(shape, dtype=torch.uint8, device=device)
        self.v = torch.empty(shape, dtype=torch.uint8, device=device)
        self.k_scale = torch.empty(shape[:3], dtype=torch.float32, device=device)
        self.v_scale = torch.empty(shape[:3], dtype=torch.float32, device=device)

    def append(self, layer, k, v, n_new, at_pos, stream=None):
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache append layer out of range")
        if n_new < 1:
            raise ValueError("KVCache append n_new must be >= 1")
        _need(k, torch.bfloat16, "k"); _need(v, torch.bfloat16, "v")
        _need(at_pos, torch.int32, "at_pos")
        _ffi.call("rth_kv_append_fp8", _p(self.k[layer]), _p(self.v[layer]),
                  _p(self.k_scale[layer]), _p(self.v_scale[layer]), _p(k), _p(v),
                  _p(at_pos), n_new, self.num_kv_heads, self.head_dim, _stream(stream))

    def append_rope(self, layer, q, k, v, n_new, positions, inv_freq, at_pos, num_q_heads,
                    stream=None):
        """RoPE on q (in place) and k, then append k, v, in one launch."""
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache append layer out of range")
        if n_new < 1:
            raise ValueError("KVCache append n_new must be >= 1")
        rope_append_fp8(q, self.k[layer], self.v[layer], self.k_scale[layer],
                        self.v_scale[layer], k, v, positions, inv_freq, at_pos, n_new,
                        num_q_heads, self.num_kv_heads, self.head_dim, stream)

    def append_qk_norm_rope(self, layer, q, k, v, n_new, q_norm, k_norm, eps, positions,
                            inv_freq, at_pos, num_q_heads, stream=None):
        """Qwen3 order: RMSNorm of q and k per head, RoPE, then the append."""
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache append layer out of range")
        if n_new < 1:
            raise ValueError("KVCache append n_new must be >= 1")
        qk_norm_rope_append_fp8(q, self.k[layer], self.v[layer], self.k_scale[layer],
                                self.v_scale[layer], k, v, q_norm, k_norm, eps, positions,
                                inv_freq, at_pos, n_new, num_q_heads, self.num_kv_heads,
                                self.head_dim, stream)

    def view(self, layer) -> KVView:
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache view layer out of range")
        return KVView(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])

    def slabs(self, layer) -> KVSlabs:
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache slabs layer out of range")
        return KVSlabs(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])

    def max_seq_len(self) -> int:
        return self._max_seq_len


class PagedKVCache:
    """Paged FP8 KV cache: per layer num_blocks physical blocks of block_size
    positions; the caller's block_table (int32 device tensor, logical block ->
    physical block) goes to append() and view(). No reference counterpart."""

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim,
                 device="cuda"):
        if block_size < 32 or block_size & (block_size - 1):
            raise ValueError("PagedKVCache block_size must be a power of two >= 32")
        self.num_layers, self.num_blocks, self.block_size = num_layers, num_blocks, block_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        shape = (num_layers, num_blocks * block_size, num_kv_heads, head_dim)
        self.k = torch.empty(shape, dtype=torch.uint8, device=device)
        self.v = torch.empty(shape, dtype=torch.uint8, device=device)
        self.k_scale = torch.empty(shape[:3], dtype=torch.float32, device=device)
        self.v_scale = torch.empty(shape[:3], dtype=torch.float32, device=device)

    def append(self, layer, k, v, n_new, at_pos, block_table, stream=None):
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache append layer out of range")
        if n_new < 1:
            raise ValueError("KVCache append n_new must be >= 1")
        _need(k, torch.bfloat16, "k"); _need(v, torch.bfloat16, "v")
        _need(at_pos, torch.int32, "at_pos"); _need(block_table, torch.int32, "block_table")
        _ffi.call("rth_kv_append_fp8_paged", _p(self.k[layer]), _p(self.v[layer]),
                  _p(self.k_scale[layer]), _p(self.v_scale[layer]), _p(k), _p(v), _p(at_pos),
                  n_new, self.num_kv_heads, self.head_dim, _p(block_table), self.block_size,
                  _stream(stream))

    def view(self, layer, block_table) -> KVView:
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache view layer out of range")
        _need(block_table, torch.int32, "block_table")
        return KVView(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                      block_table, self.block_size)

    def slabs(self, layer, block_table) -> KVSlabs:
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache slabs layer out of range")
        _need(block_table, torch.int32, "block_table")
        return KVSlabs(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                       block_table, self.block_size)

    def append_batch(self, layer, k, v, at_pos, block_tables, cu_seqlens=None, stream=None):
        """kv_append_fp8_batch into this layer: the rows of a packed batch
        (cu_seqlens), or one row per sequence, at at_pos[b] of sequence b."""
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache append layer out of range")
        dev = _current_device()
        _need_here(self.k, "the cache", dev)
        rows = layer * self.num_blocks * self.block_size * self.num_kv_heads
        _append_batch(self.k.data_ptr() + rows * self.head_dim,
                      self.v.data_ptr() + rows * self.head_dim,
                      self.k_scale.data_ptr() + 4 * rows, self.v_scale.data_ptr() + 4 * rows, k, v,
                      at_pos, block_tables, self.num_blocks, self.block_size, self.num_kv_heads,
                      self.head_dim, cu_seqlens, dev, stream)

    def batch_view(self, layer, block_tables) -> KVBatchView:
        if not 0 <= layer < self.num_layers:
            raise ValueError("KVCache view layer out of range")
        _need(block_tables, torch.int32, "block_tables")
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be [seqs, blocks]")
        return KVBatchView(self.k[layer], self.v[layer], self.k_scale[layer],
                           self.v_scale[layer], block_tables, self.block_size, self.num_blocks,
                           self.num_kv_heads, self.head_dim)

    def _all(self):
        return (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                self.v_scale.data_ptr(), self.num_layers, self.num_blocks, self.block_size,
                self.num_kv_heads, self.head_dim)

    def copy_pages(self, src, dst, stream=None):
        """Copies page src[i] to page dst[i] in every layer. The dst pages are
        distinct and none of them is a src page."""
        dev = _current_device()
        _need_here(self.k, "the cache", dev)
        _need_on(src, torch.int32, "src", dev)
        n = src.numel()
        _need_len(dst, n, "dst", dev)
        if n:
            _ffi.call("rth_pages_copy", *self._all(), src.data_ptr(), dst.data_ptr(), n,
                      _stream_of(stream, dev))


class PagePool:
    """Which pages of a paged cache are in use, on the device: refs[page]
    counts the block-table entries that hold it, refs <= 0 is free, and the
    lowest free pages are given out first. Block tables are [seqs, blocks]
    int32 with -1 where there is no page (new_tables). Nothing here waits for
    the device: what a call could not do for lack of pages (or of table
    entries) it leaves undone and says in `status`, which stays set until
    the caller clears it. Calls on one pool run one behind the other. No
    reference counterpart."""

    OUT_OF_PAGES, TABLE_TOO_SHORT = 1, 2   # bits of status

    def __init__(self, num_blocks, block_size, device="cuda"):
        if num_blocks < 1:
            raise ValueError("PagePool num_blocks must be >= 1")
        if block_size < 32 or block_size & (block_size - 1):
            raise ValueError("PagePool block_size must be a power of two >= 32")
        self.num_blocks, self.block_size, self.device = num_blocks, block_size, device
        self.refs = torch.zeros(num_blocks, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._work = torch.empty(int(_ffi.load().rth_pages_work_ints(num_blocks)),
                                 dtype=torch.int32, device=device)

    def new_tables(self, num_seqs, table_blocks):
        """Block tables without pages."""
        return torch.full((num_seqs, table_blocks), -1, dtype=torch.int32, device=self.device)

    def _here(self):
        dev = _current_device()
        _need_here(self.refs, "the pool", dev)
        return dev

    def _of(self, cache):
        if cache.num_blocks != self.num_blocks or cache.block_size != self.block_size:
            raise ValueError("the pool and the cache differ in their blocks")
        dev = self._here()
        _need_here(cache.k, "the cache", dev)
        return dev

    def reserve(self, block_tables, lens, n_new, stream=None):
        """Pages for positions lens[b] .. lens[b] + n_new[b] - 1 of sequence b,
        where its table row has none yet."""
        dev, seqs = self._here(), lens.numel()
        _need_on(lens, torch.int32, "lens", dev)
        _need_len(n_new, seqs, "n_new", dev)
        width = _need_tables(block_tables, seqs, "block_tables", dev)
        _ffi.call("rth_pages_reserve", self.refs.data_ptr(), self._work.data_ptr(),
                  self.status.data_ptr(), self.num_blocks, self.block_size,
                  block_tables.data_ptr(), width, lens.data_ptr(), n_new.data_ptr(), seqs,
                  _stream_of(stream, dev))

    def fork(self, cache, dst_tables, dst_lens, src_tables, src_lens, parents, stream=None):
        """Sequence i of dst becomes a copy of sequence parents[i] of src (any
        number of children of one parent; a parent outside src gives an empty
        one): filled pages are shared, a part-filled last page is copied, in all
        layers of `cache`, into a page of the child's own. The dst tables hold no
        pages before (free them first)."""
        dev, n, seqs = self._of(cache), parents.numel(), src_lens.numel()
        _need_on(parents, torch.int32, "parents", dev)
        _need_on(src_lens, torch.int32, "src_lens", dev)
        _need_len(dst_lens, n, "dst_lens", dev)
        width = _need_tables(src_tables, seqs, "src_tables", dev)
        if _need_tables(dst_tables, n, "dst_tables", dev) != width:
            raise ValueError("dst_tables and src_tables must have the same number of blocks")
        _ffi.call("rth_pages_fork", *cache._all(), self.refs.data_ptr(), self._work.data_ptr(),
                  self.status.data_ptr(), dst_tables.data_ptr(), dst_lens.data_ptr(),
                  src_tables.data_ptr(), src_lens.data_ptr(), width, seqs, parents.data_ptr(), n,
                  _stream_of(stream, dev))

    def free(self, block_tables, lens, drop=None, stream=None):
        """Frees the sequences with drop[b] != 0 (None: all): their pages lose
        one reference, their table rows hold none, their lengths are 0."""
        dev, seqs = self._here(), lens.numel()
        _need_on(lens, torch.int32, "lens", dev)
        width = _need_tables(block_tables, seqs, "block_tables", dev)
        if drop is not None:
            _need_len(drop, seqs, "drop", dev)
            drop = drop.data_ptr()
        _ffi.call("rth_pages_free", self.refs.data_ptr(), self.num_blocks,
                  block_tables.data_ptr(), width, lens.data_ptr(), drop, seqs, _stream_of(stream, dev))

    def compact(self, cache, block_tables, stream=None):
        """Moves the pages in use down to the lowest ones, in all layers of
        `cache`, and renames them in block_tables, which are all the tables that
        hold pages of the pool."""
        dev, seqs = self._of(cache), len(block_tables)
        width = _need_tables(block_tables, seqs, "block_tables", dev)
        _ffi.call("rth_pages_compact", *cache._all(), self.refs.data_ptr(),
                  self._work.data_ptr(), block_tables.data_ptr(), width, seqs, _stream_of(stream, dev))


class AttentionBackend:
    """reference include/runtherder/attention/backend.h:24-53"""

    def run(self, out, q, kv: KVView, n_new, cache_len, stream=None):
        raise NotImplementedError


PREFILL_SPLIT_TOKENS = 40        # above (head_dim 128): key runs where they fill the chip
PREFILL_SPLIT_MOST_TOKENS = 80   # the decode route's most
PREFILL_RUNS_TOKENS = 256
PREFILL_RUN_TOKEN_RUNS = 2048


class AdaptiveAttention(AttentionBackend):
    """reference src/attention/adaptive.cu: n_new == 1 -> split decode with
    backend-owned scratch, else flash prefill. Split count defaults to the
    device's (kv head, split) fill count. Calls of 2..PREFILL_SPLIT_TOKENS
    tokens on shapes the MFMA decode kernel serves take the split-K prefill
    (flash_prefill_split_bf16) over the same scratch, with num_splits //
    (2 n_new) splits (no reference counterpart: per call, 16 tokens after 8K
    keys 209 -> 17 us; at an empty cache up to ~2 us slower); at head_dim 128,
    calls of up to PREFILL_RUNS_TOKENS tokens take it as the flash prefill
    over key runs (64 / 128 / 250 tokens after 32K keys, the flash prefill ->
    the runs, 517 / 533 / 538 -> 56 / 88 / 157 us; at an empty cache 2 us
    slower), for which the scratch holds PREFILL_RUN_TOKEN_RUNS token-runs."""

    def __init__(self, config: AttnConfig, num_splits: int | None = None, device="cuda"):
        self.config = config
        self.num_splits = num_splits or default_num_splits(
            config.num_kv_heads, torch.device(device).index or 0)
        dev = torch.device(device)
        self.cus = torch.cuda.get_device_properties(dev).multi_processor_count
        runs = PREFILL_RUN_TOKEN_RUNS if config.head_dim == 128 else 1
        self.partial = new_flash_split_scratch(config.num_q_heads, config.head_dim,
                                               max(self.num_splits, runs), device=device)

    def _split_prefill_splits(self, n_new):
        c = self.config
        if not 2 <= n_new <= PREFILL_RUNS_TOKENS:
            return 0
        few = n_new <= PREFILL_SPLIT_MOST_TOKENS
        if few and decode_path(c.num_q_heads, c.num_kv_heads, c.head_dim) != DECODE_MFMA:
            return 0
        if n_new > PREFILL_SPLIT_TOKENS and c.head_dim == 128:
            # One to two rounds of the key runs' workgroups, within the scratch;
            # past 16 runs only to fill the first.
            blocks = (n_new * (c.num_q_heads // c.num_kv_heads) + 127) // 128 * c.num_kv_heads
            runs = min(2 * self.cus // blocks, max(16, -(-self.cus // blocks)),
                       PREFILL_RUN_TOKEN_RUNS // n_new)
            if not few:
                return runs if runs > 1 else 0
            if runs * blocks >= self.cus:
                return runs
        return max(1, self.num_splits // (2 * n_new)) if few else 0

    def run(self, out, q, kv, n_new, cache_len, stream=None):
        c = self.config
        ps = self._split_prefill_splits(n_new)
        if kv.block_table is not None:
            if ps:
                _ffi.call("rth_attn_prefill_split_paged", _p(out), _p(q), _p(kv.k), _p(kv.v),
                          _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table), kv.block_size,
                          _p(self.partial), ps, n_new, _p(cache_len), c.num_q_heads,
                          c.num_kv_heads, c.head_dim, float(c.scale), _stream(stream))
            elif n_new == 1:
                _ffi.call("rth_attn_decode_split_paged", _p(out), _p(q), _p(kv.k), _p(kv.v),
                          _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table), kv.block_size,
                          _p(self.partial), self.num_splits, _p(cache_len), c.num_q_heads,
                          c.num_kv_heads, c.head_dim, float(c.scale), _stream(stream))
            else:
                _ffi.call("rth_attn_prefill_paged", _p(out), _p(q), _p(kv.k), _p(kv.v),
                          _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table), kv.block_size,
                          n_new, _p(cache_len), c.num_q_heads, c.num_kv_heads, c.head_dim,
                          float(c.scale), _stream(stream))
            return
        if ps:
            flash_prefill_split_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, self.partial,
                                     ps, n_new, cache_len, c.num_q_heads, c.num_kv_heads,
                                     c.head_dim, c.scale, stream)
        elif n_new == 1:
            flash_decode_split_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, self.partial,
                                    self.num_splits, cache_len, c.num_q_heads, c.num_kv_heads,
                                    c.head_dim, c.scale, stream)
        else:
            flash_prefill_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, n_new, cache_len,
                               c.num_q_heads, c.num_kv_heads, c.head_dim, c.scale, stream)

    def run_decode_append(self, out, q, kv, k_new, v_new, cache_len, stream=None):
        """KVCache.append(layer, k_new, v_new, 1, cache_len) + run(..., n_new=1)
        in one call; kv is the layer's KVSlabs (they receive the new token)."""
        _need_slabs(kv)
        c = self.config
        if kv.block_table is not None:
            _ffi.call("rth_attn_decode_append_split_paged", _p(out), _p(q), _p(kv.k), _p(kv.v),
                      _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table), kv.block_size,
                      _p(k_new), _p(v_new), _p(self.partial), self.num_splits, _p(cache_len),
                      c.num_q_heads, c.num_kv_heads, c.head_dim, float(c.scale),
                      _stream(stream))
            return
        flash_decode_append_split_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, k_new, v_new,
                                       self.partial, self.num_splits, cache_len, c.num_q_heads,
                                       c.num_kv_heads, c.head_dim, c.scale, stream)


    def run_decode_rope_append(self, out, q, kv, k_new, v_new, positions, inv_freq, cache_len,
                               stream=None):
        """rope_bf16(q, k_new, positions, inv_freq) + KVCache.append(layer, k_new,
        v_new, 1, cache_len) + run(..., n_new=1) in one call; q and k_new are
        read only (the rotation happens in registers)."""
        _need_slabs(kv)
        c = self.config
        if kv.block_table is not None:
            _ffi.call("rth_attn_decode_rope_append_split_paged", _p(out), _p(q), _p(kv.k),
                      _p(kv.v), _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table),
                      kv.block_size, _p(k_new), _p(v_new), _p(positions), _p(inv_freq),
                      _p(self.partial), self.num_splits, _p(cache_len), c.num_q_heads,
                      c.num_kv_heads, c.head_dim, float(c.scale), _stream(stream))
            return
        flash_decode_rope_append_split_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, k_new,
                                            v_new, positions, inv_freq, self.partial,
                                            self.num_splits, cache_len, c.num_q_heads,
                                            c.num_kv_heads, c.head_dim, c.scale, stream)


    def run_decode_qk_norm_rope_append(self, out, q, kv, k_new, v_new, q_norm, k_norm, eps,
                                       positions, inv_freq, cache_len, stream=None):
        """Qwen3 order: per-head RMSNorm(q, q_norm) and (k_new, k_norm), RoPE,
        KVCache.append and run(..., n_new=1) in one call; q and k_new read only."""
        _need_slabs(kv)
        c = self.config
        if kv.block_table is not None:
            _ffi.call("rth_attn_decode_qk_norm_rope_append_split_paged", _p(out), _p(q),
                      _p(kv.k), _p(kv.v), _p(kv.k_scale), _p(kv.v_scale), _p(kv.block_table),
                      kv.block_size, _p(k_new), _p(v_new), _p(q_norm), _p(k_norm), float(eps),
                      _p(positions), _p(inv_freq), _p(self.partial), self.num_splits,
                      _p(cache_len), c.num_q_heads, c.num_kv_heads, c.head_dim, float(c.scale),
                      _stream(stream))
            return
        flash_decode_qk_norm_rope_append_split_bf16(
            out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, k_new, v_new, q_norm, k_norm, eps,
            positions, inv_freq, self.partial, self.num_splits, cache_len, c.num_q_heads,
            c.num_kv_heads, c.head_dim, c.scale, stream)


class BatchAttention:
    """Attention of a batch of up to max_seqs sequences: whole prompts packed
    one behind the other, and one token of each sequence over a paged cache
    whose first pages all may share. Owns the decode's scratch, so calls of
    one object run one behind the other (one stream, or ordered streams; a
    captured graph counts). No reference counterpart."""

    def __init__(self, config: AttnConfig, max_seqs: int, device="cuda"):
        if max_seqs < 1:
            raise ValueError("BatchAttention max_seqs must be >= 1")
        self.config, self.max_seqs = config, max_seqs
        with torch.cuda.device(device):
            n = max(batch_scratch_floats(b, config.num_q_heads, config.num_kv_heads,
                                         config.head_dim)
                    for b in range(1, max_seqs + 1))
            self.partial = torch.empty(n, dtype=torch.float32, device=device)

    def run_packed(self, out, q, k, v, cu_seqlens, stream=None):
        """flash_packed_bf16 with this configuration (max_seqs does not bind it)."""
        c = self.config
        flash_packed_bf16(out, q, k, v, cu_seqlens, c.num_q_heads, c.num_kv_heads, c.head_dim,
                          c.scale, stream)

    def run_decode(self, out, q, kv: KVBatchView, lens, prefix_table=None, prefix_len=None,
                   stream=None):
        """flash_decode_batch_bf16 over kv with this object's scratch."""
        c, tables = self.config, kv.block_tables
        seqs, width = tables.shape
        if seqs > self.max_seqs:
            raise ValueError(f"{seqs} sequences: this backend was made for {self.max_seqs}")
        if kv.num_kv_heads != c.num_kv_heads or kv.head_dim != c.head_dim:
            raise ValueError("the view and the configuration differ in their kv heads")
        dev = _current_device()
        _need_here(kv.k, "the view", dev); _need_here(self.partial, "the scratch", dev)
        _decode_batch(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, tables, width, kv.num_blocks,
                      kv.block_size, lens, self.partial, c.num_q_heads, c.num_kv_heads, c.head_dim,
                      c.scale, prefix_table, prefix_len, seqs, dev, stream)


class NaiveAttention(AttentionBackend):
    """reference src/attention/naive.cu"""

    def __init__(self, config: AttnConfig):
        self.config = config

    def run(self, out, q, kv, n_new, cache_len, stream=None):
        if kv.block_table is not None:
            raise ValueError("NaiveAttention reads contiguous caches only")
        c = self.config
        attention_causal_bf16(out, q, kv.k, kv.v, kv.k_scale, kv.v_scale, n_new, cache_len,
                              c.num_q_heads, c.num_kv_heads, c.head_dim, c.scale, stream)


class BackendKind(enum.Enum):
    """reference include/runtherder/attention/factory.h:9-12"""
    Naive = 0
    Adaptive = 1


def make_attention_backend(kind: BackendKind, config: AttnConfig) -> AttentionBackend:
    """reference src/attention/factory.cu:11-21"""
    if kind == BackendKind.Naive:
        return NaiveAttention(config)
    if kind == BackendKind.Adaptive:
        return AdaptiveAttention(config)
    raise ValueError("unknown attention BackendKind")
