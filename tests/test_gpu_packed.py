"""Causal attention over packed prompts (no reference counterpart) against the
formula in 64 bits: lengths from none to several tiles and row blocks, head
groups, strides, padding, what masked places may hold, refusals."""
import math

import pytest
import torch

import runtherder_amd as R
from batch_util import assert_attention, attend64, cu_of, ints, normal, score_size
from gpu_util import DEV, step, sync

pytestmark = pytest.mark.gpu


def run(q, k, v, cu, out=None, scale=None, stream=None):
    hq, d = q.shape[1:]
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
    R.flash_packed_bf16(out, q, k, v, cu, hq, k.shape[1], d,
                        d ** -0.5 if scale is None else scale, stream)
    return out


def check(lens, hq, hkv, d, seed, fused=False, pad=0, rows=None, scale=None, size=1.0):
    n = sum(lens) + pad
    if fused:
        x = normal((n, hq + 2 * hkv, d), seed, size)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        xd = x.to(DEV)
        qd, kd, vd = xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:]
    else:
        q, k, v = normal((n, hq, d), seed, size), normal((n, hkv, d), seed + 1), normal((n, hkv, d), seed + 2)
        qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    step(f"packed lens={lens} hq={hq} hkv={hkv} d={d} fused={fused} pad={pad}")
    scale = d ** -0.5 if scale is None else scale
    out = run(qd, kd, vd, ints(cu_of(lens)), scale=scale)
    sync()
    got, cu = out.cpu(), cu_of(lens)
    for b, m in enumerate(lens):
        picked = range(m) if m <= 80 else sorted({0, 1, 31, 32, 63, 64, m - 1, m - 2, m // 2,
                                                  *(rows or ()), *range(7, m, max(1, m // 40))})
        for t in picked:
            if t >= m:
                continue
            at = cu[b]
            want, weight = attend64(q[at + t], k[at:at + t + 1], v[at:at + t + 1], scale)
            assert_attention(got[at + t], want, weight,
                             score_size(q[at + t], k[at:at + t + 1], scale))
    assert (got[cu[-1]:] == 7.0).all()   # rows behind the last sequence stay as they were


@pytest.mark.parametrize("lens", [
    [1], [2], [33], [64], [65], [127, 1, 0, 128], [0, 0, 5], [1] * 70, [300, 0, 17, 513, 64, 1],
])
def test_lengths(lens):
    check(lens, 8, 2, 128, 100 + len(lens) + lens[0])


@pytest.mark.parametrize("hq,hkv,d", [
    (4, 4, 64), (16, 2, 64), (7, 1, 64), (8, 8, 128), (24, 8, 128), (28, 4, 128), (40, 1, 128),
    (5, 1, 128), (4, 2, 256), (16, 4, 256), (9, 3, 256),
])
def test_heads(hq, hkv, d):
    check([130, 3, 77], hq, hkv, d, 200 + hq + d)


@pytest.mark.parametrize("lens,hq,hkv,d", [
    ([1500, 40], 32, 8, 128), ([2049], 16, 8, 64), ([1100, 900], 8, 4, 256), ([4100], 8, 8, 128),
    # The eight-wave workgroups (long sequences, enough of them to fill the chip).
    ([4200], 32, 8, 128), ([3001, 2500, 17], 28, 4, 128), ([4097], 40, 8, 64),
])
def test_long(lens, hq, hkv, d):
    check(lens, hq, hkv, d, 300 + lens[0], rows=[1023, 1024, 1025])


def test_slices_of_a_projection_with_padding():
    check([200, 31, 64], 32, 8, 128, 400, fused=True, pad=9)
    check([70, 1], 6, 2, 256, 401, fused=True, pad=1)
    check([90, 5], 6, 2, 64, 402, fused=True, pad=300)


def test_score_ranges():
    """Scores far apart: the reference maximum moves, or lies far above most keys."""
    check([400, 90], 8, 2, 128, 500, size=30.0)
    check([400], 8, 2, 64, 501, scale=8.0)
    check([130], 4, 1, 256, 502, scale=0.0)
    # Scores that grow along the keys, then fall.
    n, d = 320, 128
    ramp = torch.cat([torch.arange(160.0), torch.arange(160.0, 0, -1)])[:, None, None]
    q = torch.full((n, 2, d), 1.0).to(torch.bfloat16)
    k = (ramp / 4 + torch.zeros(n, 1, d)).to(torch.bfloat16)
    v = normal((n, 1, d), 503)
    out = run(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, n])).cpu()
    for t in range(0, n, 7):
        want, weight = attend64(q[t], k[:t + 1], v[:t + 1], d ** -0.5)
        assert_attention(out[t], want, weight, score_size(q[t], k[:t + 1], d ** -0.5))


def test_a_prompt_is_the_same_in_every_batch():
    """Bit for bit, whatever the batch, its padding and its workgroups' width."""
    for hq, hkv, d in ((32, 8, 128), (6, 2, 64), (4, 4, 256)):
        n = 333
        q, k, v = (normal((4300, h, d), 610 + h, 4.0) for h in (hq, hkv, hkv))
        alone = run(q[:n].to(DEV), k[:n].to(DEV), v[:n].to(DEV), ints([0, n])).cpu()
        front = run(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, 4300])).cpu()
        back = torch.cat([q[-100:], q[:n], q[:7]]), torch.cat([k[-100:], k[:n], k[:7]]), \
            torch.cat([v[-100:], v[:n], v[:7]])
        step(f"packed batch against alone hq={hq} d={d}")
        there = run(*(t.to(DEV) for t in back), ints([0, 100, 100 + n])).cpu()
        sync()
        assert torch.equal(front[:n], alone)
        assert torch.equal(there[100:100 + n], alone)


def test_repeats_bit_for_bit_and_on_a_stream():
    q, k, v = (normal((700, h, 128), 600 + h).to(DEV) for h in (16, 4, 4))
    cu = ints([0, 300, 301, 700])
    a = run(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = torch.empty_like(a)
    run(q, k, v, cu, out=b, stream=s)
    s.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("hq,hkv,d,n", [(8, 2, 128, 200), (4, 4, 64, 150), (4, 2, 256, 90), (32, 8, 128, 4200)])
def test_what_a_row_does_not_see_leaves_no_trace(hq, hkv, d, n):
    """NaN and infinities in K and V: rows in front of them are those of a clean batch, bit
    for bit; the rows that see them have what the formula gives."""
    at = n - 61
    q, k, v = (normal((n + 40, h, d), 700 + h) for h in (hq, hkv, hkv))
    clean = run(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, n, n + 40])).cpu()
    v[at, 0, 5] = math.inf
    v[at + 3, 0, 6] = -math.inf
    v[at + 7, 0, 7] = math.nan
    v[at + 9, 0, 5] = -math.inf            # with the one before: NaN
    v[n - 1, 0, 8] = math.nan              # the last row, which fills up the tile
    k[at + 20, hkv - 1, :] = math.nan
    k[n - 1, 0, 3] = math.inf
    step(f"packed non-finite hq={hq} hkv={hkv} d={d}")
    got = run(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, n, n + 40])).cpu()
    sync()
    assert torch.equal(got[:at], clean[:at]) and torch.equal(got[n:], clean[n:])
    assert torch.isfinite(got[n:].float()).all()
    g = hq // hkv
    f = got.float()
    own = f[:, :g]                          # the heads of kv head 0
    assert (own[at:n - 1, :, 6][:3] == clean.float()[at:at + 3, :g, 6]).all()
    assert (own[at:at + 9, :, 5] == math.inf).all() and torch.isnan(own[at + 9:n - 1, :, 5]).all()
    assert (own[at + 3:n - 1, :, 6] == -math.inf).all()
    assert torch.isfinite(own[at:at + 7, :, 7]).all() and torch.isnan(own[at + 7:n - 1, :, 7]).all()
    if hkv > 1:
        other = f[:, (hkv - 1) * g:]
        assert torch.equal(got[:at + 20, (hkv - 1) * g:], clean[:at + 20, (hkv - 1) * g:])
        assert torch.isnan(other[at + 20:n]).all()


def test_one_row_of_any_stride():
    """The stride of a single row is no part of the call."""
    wide = normal((3, 1001), 5).to(DEV)
    q, k, v = wide[:1, :256].view(1, 2, 128), wide[:1, 256:384].view(1, 1, 128), wide[:1, 384:512].view(1, 1, 128)
    out = torch.zeros((1, 2, 128), dtype=torch.bfloat16, device=DEV)
    step("one row")
    R.flash_packed_bf16(out, q, k, v, ints([0, 1]), 2, 1, 128, 0.1)
    sync()
    assert torch.equal(out, v.expand(1, 2, 128))   # one key: its value
