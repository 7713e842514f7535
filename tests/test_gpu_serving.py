"""Window attention, attention over a paged cache, and the cache's operators, against 64-bit forms.

Tolerances are those of serving_reference.tolerance, derived from the operands' types and sizes.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import seeded
from serving_reference import HALF_STEP, Book, attend, paged_reference, small_weight_tolerance, window_reference, window_seen
from tkmi import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _inside(got, want, tol):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())  # keys that are seen may hold NaN, and say so
    share = ((got - want).abs() / tol).nan_to_num(0.0)
    assert float(share.max()) <= 1, f"worst {float(share.max()):.2f} of the tolerance"


# ------------------------------------------------------------------ window --


def _window_inputs(b, h, hkv, sq, sk, hd, dtype, seed=0):
    return (seeded(b, h, sq, hd, dtype=dtype, seed=seed), seeded(b, hkv, sk, hd, dtype=dtype, seed=seed + 1),
            seeded(b, hkv, sk, hd, dtype=dtype, seed=seed + 2))


def _check_window(q, k, v, window, sinks, valid=None, scale=None):
    scale = 1.5 * q.shape[3] ** -0.5 if scale is None else scale
    want, tol = window_reference(q, k, v, scale, window, sinks, valid)
    both = []
    for invariant in (False, True):  # keys dealt to waves and workgroups where rows are few, and not
        both.append(ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), scale, window, sinks=sinks,
                                         key_valid=None if valid is None else valid.to(DEV),
                                         batch_invariant=invariant))
        _inside(both[-1], want, tol)
    return torch.stack(both)


# lengths around tiles (32 rows, 64 keys) and workgroups (128 rows); windows of one key, around tiles, past the keys
@pytest.mark.parametrize("sq,sk,window,sinks", [
    (1, 1, 1, 0), (1, 700, 100, 4), (2, 65, 64, 0), (31, 31, 8, 1), (33, 64, 33, 2), (64, 64, 1000, 0),
    (129, 129, 1, 0), (128, 300, 63, 64), (200, 200, 65, 65), (257, 640, 128, 3), (300, 300, 17, 200), (77, 77, 16, 2),
])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_window_sizes(sq, sk, window, sinks, hd):
    for dtype in (F16, BF16):
        _check_window(*_window_inputs(1, 2, 1, sq, sk, hd, dtype, seed=sq + hd), window, sinks)


@pytest.mark.parametrize("hd", [8, 24, 40, 72, 80, 96, 136, 200, 248])
def test_window_head_dims_between_tiles(hd):
    for dtype in (F16, BF16):
        _check_window(*_window_inputs(2, 2, 2, 150, 211, hd, dtype, seed=hd), 70, 5)


@pytest.mark.parametrize("h,hkv,b", [(8, 8, 3), (6, 2, 2), (7, 1, 2), (1, 1, 9)])
def test_window_head_layouts(h, hkv, b):
    _check_window(*_window_inputs(b, h, hkv, 140, 140, 64, F16, seed=h), 50, 4)
    _check_window(*_window_inputs(b, h, hkv, 5, 333, 64, BF16, seed=h), 200, 0)


@pytest.mark.parametrize("hd", [40, 64, 128, 256])
@pytest.mark.parametrize("pattern", ["tail", "head", "holes", "nothing"])
def test_window_key_masks_and_what_lies_under_them(hd, pattern):
    """Rows left without a key are zeros; NaN, infinities and the type's lowest value in masked keys and
    values change no bit."""
    b, s = 3, 300
    valid = torch.ones(b, s, dtype=torch.bool)
    if pattern == "tail":
        valid[0, 1:], valid[1, 64:], valid[2, 257:] = False, False, False
    elif pattern == "head":
        valid[:, :130] = False
    elif pattern == "holes":
        valid = torch.rand(b, s, generator=torch.Generator().manual_seed(5)) > 0.6
        valid[1, 100:200] = False
    else:
        valid[1] = False
    for dtype in (F16, BF16):
        q, k, v = _window_inputs(b, 2, 1, s, s, hd, dtype, seed=3)
        clean = _check_window(q, k, v, 40, 2, valid)
        hidden = ~valid[:, None, :, None].expand_as(k)
        for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
            got = _check_window(q, k.masked_fill(hidden, bad), v.masked_fill(hidden, bad), 40, 2, valid)
            assert torch.equal(got, clean)


def test_window_scores_that_rise_and_fall():
    """Scores that grow along the keys (every tile raises the maximum), that shrink, and far below fp16's range."""
    q, k, v = _window_inputs(1, 2, 2, 300, 300, 64, F16, seed=8)
    ramp = torch.linspace(-3, 3, 300)[:, None] * q.float().mean((0, 1, 2)).sign()
    for sign in (1, -1):
        _check_window(q, (k.float() + sign * ramp).half(), v, 100, 4)
        _check_window(q.abs(), (-(k.float().abs()) * 3 + sign * ramp).half(), v, 100, 4)


@pytest.mark.parametrize("low", [2.0 ** -15, 2.0 ** -18, 2.0 ** -22])
def test_window_many_small_weights(low):
    """One key of weight 1 and 3000 of a weight below fp16's normal range that together matter."""
    s, hd = 3001, 64
    q = torch.zeros(1, 1, s, hd, dtype=F16)
    q[..., 0] = 1.0
    k = torch.zeros(1, 1, s, hd, dtype=F16)
    k[:, :, 1:, 0] = math.log(low)
    v = seeded(1, 1, s, hd, dtype=F16, seed=18).abs() + 1
    v[:, :, 0] = 0
    for dtype in (F16, BF16):
        _check_window(q.to(dtype), k.to(dtype), v.to(dtype), s, 0, scale=1.0)
        _check_window(q.to(dtype)[:, :, -2:], k.to(dtype), v.to(dtype), 2000, 1, scale=1.0)


def test_window_views_out_and_neighbours():
    """Views of a fused projection; out in the middle of a larger buffer whose other bytes stay."""
    b, s, h, hkv, hd = 2, 150, 4, 2, 64
    fused = seeded(b, s, h + 2 * hkv, hd, dtype=F16, seed=4).to(DEV)
    q, k, v = (t.transpose(1, 2) for t in (fused[:, :, :h], fused[:, :, h:h + hkv], fused[:, :, h + hkv:]))
    buf = torch.full((b, s + 2, h * hd + 8), 7.0, dtype=F16, device=DEV)
    out = buf[:, 1:-1, 4:-4]
    assert ops.window_attention(q, k, v, 0.125, 33, sinks=1, out=out) is out
    want, tol = window_reference(q.cpu(), k.cpu(), v.cpu(), 0.125, 33, 1)
    _inside(out, want, tol)
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[:, 1:-1, 4:-4] = False
    assert bool((buf[rest] == 7.0).all())
    # shared and broadcast inputs: one batch's keys for all
    k1, v1 = k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)
    want, tol = window_reference(q.cpu(), k1.cpu(), v1.cpu(), 0.125, 33, 1)
    _inside(ops.window_attention(q, k1, v1, 0.125, 33, sinks=1), want, tol)


def test_window_of_every_key_is_flash_attention():
    q, k, v = (t.to(DEV) for t in _window_inputs(2, 4, 4, 500, 500, 64, F16, seed=9))
    want, tol = window_reference(q.cpu(), k.cpu(), v.cpu(), 0.125, 500, 0)
    _inside(ops.flash_attention(q, k, v, 0.125, True), want, tol)
    for window in (500, 10 ** 8):
        _inside(ops.window_attention(q, k, v, 0.125, window), want, tol)


def test_window_bits_do_not_depend_on_the_batch():
    for sq, sk, hd in [(260, 400, 64), (1, 900, 128), (40, 2000, 80)]:
        q, k, v = (t.to(DEV) for t in _window_inputs(40, 2, 1, sq, sk, hd, BF16, seed=sq))
        whole = ops.window_attention(q, k, v, 0.1, 300, sinks=4, batch_invariant=True)
        for n in (0, 17):
            assert torch.equal(ops.window_attention(q[n:n + 1], k[n:n + 1], v[n:n + 1], 0.1, 300, sinks=4,
                                                    batch_invariant=True)[0], whole[n])


@pytest.mark.parametrize("hd", [32, 64, 128, 200])
def test_window_few_rows_and_many_keys(hd):
    """Keys split over workgroups: ends inside tiles, sinks, masks that leave some splits and some rows nothing."""
    for sq, sk, window, sinks in [(1, 9000, 9000, 0), (3, 5000, 4999, 70), (40, 7001, 6000, 1), (2, 4097, 2048, 500)]:
        q, k, v = _window_inputs(1, 2, 1, sq, sk, hd, F16 if sq % 2 else BF16, seed=sq + hd)
        _check_window(q, k, v, window, sinks)
        valid = torch.zeros(1, sk, dtype=torch.bool)
        valid[:, sk // 2:sk // 2 + 300] = True
        valid[:, sk - 1] = sq > 2
        bad = ~valid[:, None, :, None].expand_as(k)
        _check_window(q, k.masked_fill(bad, float("nan")), v.masked_fill(bad, float("inf")), window, sinks, valid)


# fewer than 32 rows a head, groups whose rows end inside, at and past a block of 32; 32 to 96 rows of many heads
@pytest.mark.parametrize("b,h,hkv,sq", [(1, 4, 1, 8), (2, 10, 2, 7), (3, 6, 2, 16), (2, 14, 2, 31), (1, 66, 1, 1),
                                        (40, 8, 8, 3), (40, 8, 2, 32), (24, 12, 4, 33), (33, 8, 4, 64), (33, 8, 4, 65),
                                        (50, 8, 4, 33), (50, 8, 4, 96)])
@pytest.mark.parametrize("hd", [24, 64, 104, 256])
def test_window_short_queries_of_groups(b, h, hkv, sq, hd):
    sk = sq + 170
    q, k, v = _window_inputs(b, h, hkv, sq, sk, hd, F16 if sq % 2 else BF16, seed=sq + h)
    q = q.transpose(1, 2).contiguous().transpose(1, 2)  # heads beside each other, tokens apart
    _check_window(q, k, v, 75, 3)
    valid = torch.rand(b, sk, generator=torch.Generator().manual_seed(sq)) > 0.3
    valid[0, :sk - sq] = False  # rows that see none, some, all of the new keys
    valid[-1] = False
    bad = ~valid[:, None, :, None].expand_as(k)
    out = _check_window(q, k.masked_fill(bad, float("nan")), v.masked_fill(bad, float("inf")), 75, 3, valid)
    assert not out[:, -1].any()


def test_window_short_queries_split_over_workgroups():
    """A group's rows in two blocks, whose keys go to several workgroups: joined per head and row."""
    for dtype, hd in [(F16, 64), (BF16, 128), (F16, 200)]:
        q, k, v = _window_inputs(2, 10, 2, 7, 6000, hd, dtype, seed=hd)
        _check_window(q, k, v, 5000, 9)
        valid = torch.ones(2, 6000, dtype=torch.bool)
        valid[0, 1500:5996] = False
        _check_window(q, k, v, 5000, 9, valid)


def test_window_short_queries_leave_what_lies_around_them():
    q, k, v = (t.to(DEV) for t in _window_inputs(2, 10, 2, 7, 300, 64, F16))
    buf = torch.full((2, 9, 10 * 64 + 8), 7.0, dtype=F16, device=DEV)
    ops.window_attention(q, k, v, 0.1, 100, sinks=2, out=buf[:, 1:-1, 4:-4])
    assert torch.equal(buf[:, 1:-1, 4:-4], ops.window_attention(q, k, v, 0.1, 100, sinks=2))
    buf[:, 1:-1, 4:-4] = 7.0
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("b,h,hkv,sq", [(1, 4, 1, 8), (1, 66, 1, 1), (1, 40, 1, 3), (3, 66, 1, 1)])
@pytest.mark.parametrize("hd", [24, 64, 104, 256])
def test_window_short_queries_of_one_group_partly_masked(b, h, hkv, sq, hd):
    """Groups that span several blocks of 32 rows: rows that see some of the keys, and (last sequence of several) none."""
    sk = sq + 170
    q, k, v = _window_inputs(b, h, hkv, sq, sk, hd, F16 if sq % 2 else BF16, seed=sq + h)
    valid = torch.rand(b, sk, generator=torch.Generator().manual_seed(h)) > 0.3
    valid[0, sk - sq - 40:sk - 2] = False  # all that the window holds but for the last keys
    if b > 1:
        valid[-1] = False
    bad = ~valid[:, None, :, None].expand_as(k)
    out = _check_window(q, k.masked_fill(bad, float("nan")), v.masked_fill(bad, float("inf")), 75, 3, valid)
    assert bool(out[:, 0].any()) and (b == 1 or not out[:, -1].any())


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_window_offsets_past_32_bits(hd):
    """Rows and sequences of q, k, v and out that lie past 2^32 elements."""
    n, far = 2100, 2 ** 21
    buf = torch.empty(n * far, dtype=BF16, device=DEV)

    def rows(count, at):
        return buf.as_strided((1, 2, count, hd), (0, 2 ** 9, far, 1), at)

    for sq, invariant in ((1, False), (40, False), (300, True)):
        q, k, v = _window_inputs(1, 2, 2, sq, n, hd, BF16, seed=hd + sq)
        qd, kd, vd = (rows(t.shape[2], at).copy_(t) for t, at in ((q, 0), (k, 2 ** 18), (v, 2 ** 19)))
        out = buf.as_strided((1, sq, 2 * hd), (0, far, 1), (n - sq) * far + 2 ** 20)
        ops.window_attention(qd, kd, vd, 0.1, 1500, sinks=5, out=out, batch_invariant=invariant)
        want, tol = window_reference(q, k, v, 0.1, 1500, 5)
        _inside(out, want, tol)
    # two sequences that lie so far apart
    q, k, v = _window_inputs(2, 2, 2, 50, 200, hd, BF16, seed=hd)
    qd, kd, vd = (buf.as_strided(t.shape, (2 ** 32 + 8, t.shape[2] * hd, hd, 1), at).copy_(t)
                  for t, at in ((q, 0), (k, 2 ** 18), (v, 2 ** 19)))
    for invariant in (False, True):
        want, tol = window_reference(q, k, v, 0.1, 70, 3)
        _inside(ops.window_attention(qd, kd, vd, 0.1, 70, sinks=3, batch_invariant=invariant), want, tol)


# ------------------------------------------------------------------- paged --


def _cache(lengths, hkv, hd, ps, dtype, seed=0, extra=3, width=None):
    """Pages in scattered order, a table of -1 where a sequence has none, poison in every row that none has."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // ps) for n in lengths]
    pages = sum(counts) + extra
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lengths), width or max(counts + [1])), -1, dtype=torch.int32)
    k = torch.full((pages, hkv, ps, hd), float("nan"), dtype=dtype)
    v = torch.full((pages, hkv, ps, hd), float("inf"), dtype=dtype)
    for b, n in enumerate(lengths):
        for e in range(counts[b]):
            table[b, e] = order.pop()
            rows = min(ps, n - e * ps)
            k[table[b, e], :, :rows] = torch.randn(hkv, rows, hd, generator=gen).to(dtype)
            v[table[b, e], :, :rows] = torch.randn(hkv, rows, hd, generator=gen).to(dtype)
    return k, v, table, torch.tensor(lengths, dtype=torch.int32)


def _check_paged(q, k, v, table, lengths, window=0, sinks=0, **kw):
    scale = 1.5 * q.shape[2] ** -0.5
    got = ops.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lengths.to(DEV), scale, window=window,
                              sinks=sinks, **kw)
    want, tol = paged_reference(q, k, v, table, lengths, scale, window, sinks)
    _inside(got, want, tol)
    return got


# lengths of 0 and 1, around pages and tiles of 32, and long enough for several splits
LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1000]


@pytest.mark.parametrize("ps", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_paged_lengths(hd, ps):
    for dtype in (F16, BF16):
        k, v, table, lengths = _cache(LENGTHS, 2, hd, ps, dtype, seed=hd)
        q = seeded(len(LENGTHS), 4, hd, dtype=dtype, seed=1)
        got = _check_paged(q, k, v, table, lengths)
        assert not bool(got[0].any())
        _check_paged(q, k, v, table, lengths, batch_invariant=True)
        _check_paged(q, k, v, table, lengths, max_length=1)  # a bound that is too low splits, but loses no key


@pytest.mark.parametrize("hd", [8, 24, 40, 72, 80, 96, 136, 248])
def test_paged_head_dims_between_tiles(hd):
    for dtype in (F16, BF16):
        k, v, table, lengths = _cache([200, 77, 3], 1, hd, 32, dtype, seed=hd)
        _check_paged(seeded(3, 3, hd, dtype=dtype, seed=2), k, v, table, lengths)


@pytest.mark.parametrize("h,hkv", [(1, 1), (5, 5), (14, 2), (16, 1), (17, 1), (40, 1), (64, 2)])
def test_paged_head_layouts(h, hkv):
    k, v, table, lengths = _cache([600, 77], hkv, 64, 16, BF16, seed=h)
    _check_paged(seeded(2, h, 64, dtype=BF16, seed=3), k, v, table, lengths)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (31, 33), (32, 0), (100, 64), (5000, 3), (300, 500)])
def test_paged_windows(window, sinks):
    """Windows and sinks at all lengths; entries of pages that neither reaches are -1."""
    lengths = [0, 1, 30, 33, 64, 100, 257, 1000, 2500]
    k, v, table, lens = _cache(lengths, 2, 64, 16, F16, seed=6)
    q = seeded(len(lengths), 4, 64, dtype=F16, seed=7)
    whole = _check_paged(q, k, v, table, lens, window, sinks)
    for b, n in enumerate(lengths):
        for e in range(-(-n // 16)):
            if e * 16 >= sinks and (e + 1) * 16 <= n - window:
                table[b, e] = -1
    assert torch.equal(_check_paged(q, k, v, table, lens, window, sinks), whole)


def test_paged_bad_entries_are_not_followed():
    k, v, table, lengths = _cache([300, 64, 500], 1, 64, 32, F16, seed=8)
    table[0, 3], table[0, 5], table[2, 0], table[2, 7] = -1, k.shape[0], 2 ** 31 - 1, -2 ** 31
    table[1] = -1
    got = _check_paged(seeded(3, 2, 64, dtype=F16, seed=9), k, v, table, lengths)
    assert not bool(got[1].any())
    # lengths past the table (the last page's rows past the sequence, NaN here, now count) and below zero
    lengths[0], lengths[2] = 2 ** 31 - 1, -5
    _check_paged(seeded(3, 2, 64, dtype=F16, seed=9), k, v, table, lengths)


def test_paged_strided_cache_and_out():
    """A token-major cache [pages, page_size, Hkv, hd], a table that is a view, out in a larger buffer."""
    k, v, table, lengths = _cache([200, 130], 2, 64, 16, F16, seed=10)
    q = seeded(2, 6, 64, dtype=F16, seed=11).to(DEV)
    tk, tv = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (k, v))
    wide = torch.full((2, 40), 10 ** 9, dtype=torch.int32, device=DEV)
    wide[:, 5:5 + table.shape[1]] = table.to(DEV)
    buf = torch.full((4, 6 * 64 + 3), 7.0, dtype=F16, device=DEV)
    out = buf[1:3, 1:-2]
    ops.paged_attention(q, tk, tv, wide[:, 5:5 + table.shape[1]], lengths.to(DEV), 0.125, out=out)
    want, tol = paged_reference(q.cpu(), k, v, table, lengths, 0.125)
    _inside(out, want, tol)
    buf[1:3, 1:-2] = 7.0
    assert bool((buf == 7.0).all())


def test_paged_offsets_past_32_bits():
    """Pages whose bytes and elements lie past 2^32 and 2^31."""
    hkv, ps, hd = 8, 256, 256
    pages = 2 ** 32 // (hkv * ps * hd) + 40
    k, v = (torch.empty(pages, hkv, ps, hd, dtype=BF16, device=DEV) for _ in range(2))
    used = torch.tensor([pages - 1, 3, pages - 30, pages // 2 + 1], dtype=torch.int32)
    new_k, new_v = (seeded(1, 4 * ps - 100, hkv, hd, dtype=BF16, seed=i) for i in (12, 13))
    lengths = torch.tensor([4 * ps - 100], dtype=torch.int32)
    ops.cache_append(new_k.to(DEV), new_v.to(DEV), k, v, used[None].to(DEV), lengths.to(DEV))
    q = seeded(1, hkv, hd, dtype=BF16, seed=14)
    got = ops.paged_attention(q.to(DEV), k, v, used[None].to(DEV), lengths.to(DEV), 0.0625)
    ids = used.long().to(DEV)
    want, tol = paged_reference(q, k[ids].cpu(), v[ids].cpu(), torch.arange(4, dtype=torch.int32)[None], lengths, 0.0625)
    _inside(got, want, tol)


def test_paged_long_sequence_splits_and_joins():
    lengths = [40000, 1, 0, 9000]
    k, v, table, lens = _cache(lengths, 1, 64, 64, F16, seed=15)
    q = seeded(4, 8, 64, dtype=F16, seed=16)
    _check_paged(q, k, v, table, lens)
    _check_paged(q, k, v, table, lens, max_length=9000)
    whole = _check_paged(q, k, v, table, lens, batch_invariant=True)
    kd, vd = k.to(DEV), v.to(DEV)
    for n in range(4):
        # alone, under other bounds, in a table of its own pages only and in a wider one
        for width in (table.shape[1], max(-(-lengths[n] // 64), 1), 2 * table.shape[1] + 7):
            own = torch.full((1, width), -1, dtype=torch.int32)
            own[:, :min(width, table.shape[1])] = table[n:n + 1, :width]
            for most in (40000, 100):
                one = ops.paged_attention(q[n:n + 1].to(DEV), kd, vd, own.to(DEV), lens[n:n + 1].to(DEV), 1.5 / 8,
                                          batch_invariant=True, max_length=most)
                assert torch.equal(one[0], whole[n])


@pytest.mark.parametrize("b,hkv,longest", [(130, 1, 9000), (70, 2, 9100), (1030, 1, 300), (300, 1, 8300)])
def test_paged_many_sequences_of_which_some_are_long(b, hkv, longest):
    """Enough sequences for every CU, and among them (first, in the middle, last) some far longer than the others."""
    lengths = [(37 * i) % 61 for i in range(b)]
    lengths[0], lengths[b // 2], lengths[-1] = longest, longest - 333, longest - 1
    k, v, table, lens = _cache(lengths, hkv, 64, 64, BF16, seed=17)
    q = seeded(b, 2 * hkv, 64, dtype=BF16, seed=18)
    _check_paged(q, k, v, table, lens)
    _check_paged(q, k, v, table, lens, window=8200, sinks=3)


# ------------------------------------- weights below fp16's normal range, scores past its integers --


def _sinks_and_small(n, hd, low, seed, every=None):
    """One query; key 0 (and each `every`-th) of score 0 and values 0, the others of score ln(low) and values
    from 1 to 2 (1024 to 2048)."""
    q, k = torch.zeros(hd, dtype=F16), torch.zeros(n, hd, dtype=F16)
    q[0] = 1.0
    k[:, 0] = math.log(low)
    v = 1 + seeded(n, hd, dtype=F16, seed=seed).abs().clamp_max(1)
    k[::every or n, 0] = 0
    v[::every or n] = 0
    return q, k, v * 1024 if every else v


# none is a power of two: a weight lands between two steps of fp16
SMALL = [2.0 ** -13.7, 2.0 ** -24.5, 2.0 ** -25.2, 2.0 ** -27.6]


@pytest.mark.parametrize("low", SMALL)
@pytest.mark.parametrize("form", ["whole", "split", "invariant"])
def test_paged_small_weights(low, form):
    """Weights that only together matter: 3000 tokens in each of 130 sequences, one of them of weight 1; 100000 in one
    sequence with a weight of 1 in every tile, so in every share of its keys."""
    hd, ps, dtype = 64, 64, F16
    n, batch, every = (3000, 130, None) if form == "whole" else (100000, 1, 32)
    q, k, v = _sinks_and_small(n, hd, low, 90, every)
    pages = -(-n // ps)
    kp, vp = (torch.cat([t, t.new_full((-n % ps, hd), float("nan"))]).view(pages, 1, ps, hd) for t in (k, v))
    table = torch.arange(pages, dtype=torch.int32).expand(batch, -1).contiguous()
    got = ops.paged_attention(q.expand(batch, 1, -1).contiguous().to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.full((batch,), n, dtype=torch.int32, device=DEV), 1.0, batch_invariant=form == "invariant")
    o, a, s = attend(q[None], k, v, 1.0, torch.ones(1, n, dtype=torch.bool))
    tol = small_weight_tolerance(o, a, s, dtype, n, hd, float(v.max()), HALF_STEP[dtype], "paged")
    _inside(got, o.expand(batch, -1), tol.expand(batch, -1))


@pytest.mark.parametrize("dtype,p_step", [(F16, 2.0 ** -22), (BF16, 2.0 ** -16)])
def test_paged_weights_are_two_numbers(dtype, p_step):
    """The weights' rounding does not show: few keys and narrow heads, so that the bound is the output's rounding."""
    lengths = [2, 7, 20, 40, 64, 90]
    for hd in (8, 16):
        k, v, table, lens = _cache(lengths, 1, hd, 16, dtype, seed=94)
        q = seeded(len(lengths), 16, hd, dtype=dtype, seed=95)
        got = ops.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens.to(DEV), 0.3)
        for b, n in enumerate(lengths):
            ids = table[b, :-(-n // 16)].long()
            kk, vv = (t[ids, 0].reshape(-1, hd)[:n] for t in (k, v))
            o, a, s = attend(q[b], kk, vv, 0.3, torch.ones(16, n, dtype=torch.bool))
            tol = small_weight_tolerance(o, a, s, dtype, n, hd, float(vv.abs().max()), p_step, "paged")
            _inside(got[b].view(16, hd), o, tol)


@pytest.mark.parametrize("low", SMALL)
@pytest.mark.parametrize("hd", [64, 256])
def test_window_small_weights(low, hd):
    """2 rows (keys over workgroups) and 40 (in workgroups of 128 rows, one after the other) of 20000 such keys."""
    n, dtype = 20000, F16
    q1, k, v = _sinks_and_small(n, hd, low, 91)
    for sq, invariant in ((2, False), (2, True), (40, False), (40, True)):
        q = q1.expand(sq, hd).contiguous()
        got = ops.window_attention(q[None, None].to(DEV), k[None, None].to(DEV), v[None, None].to(DEV), 1.0, n,
                                   batch_invariant=invariant)[0]
        o, a, s = attend(q, k, v, 1.0, window_seen(sq, n, n, 0))
        tol = small_weight_tolerance(o, a, s, dtype, n, hd, 2.0, HALF_STEP[dtype], "window")
        _inside(got, o, tol)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("factor", [2.0 ** 8, 2.0 ** 11, 2.0 ** 12])
def test_scores_of_many_millions(sign, factor):
    """Scores of 2^21 to 2^26, of either sign, the best one ahead by 64 * factor: its key's values are the row."""
    n, hd, ps = 900, 64, 32
    c = torch.randint(129, 255, (n,), generator=torch.Generator().manual_seed(92))
    c[611] = 255 if sign > 0 else 128
    for dtype in (F16, BF16):
        q = torch.full((hd,), 2.0 ** 10, dtype=dtype)
        k = (sign * c * (factor / 2 ** 10))[:, None].expand(n, hd).to(dtype).contiguous()  # 8 bits: exact
        v = seeded(n, hd, dtype=dtype, seed=93)
        want = v[611].double()[None]
        # the weight rounded and its sum not, and the output rounded
        tol = 2.01 * HALF_STEP[dtype] * want.abs() + 2.0 ** -24
        kp, vp = (torch.cat([t, t.new_zeros(-n % ps, hd)]).view(-1, 1, ps, hd).to(DEV) for t in (k, v))
        table = torch.arange(kp.shape[0], dtype=torch.int32, device=DEV)
        for invariant in (False, True):
            for batch in (1, 130):
                got = ops.paged_attention(q.expand(batch, 1, hd).contiguous().to(DEV), kp, vp,
                                          table.expand(batch, -1).contiguous(),
                                          torch.full((batch,), n, dtype=torch.int32, device=DEV), 1.0,
                                          batch_invariant=invariant)
                _inside(got, want.expand(batch, -1), tol.expand(batch, -1))
            for sq in (1, 40):
                got = ops.window_attention(q.expand(1, 1, sq, hd).contiguous().to(DEV), k[None, None].to(DEV),
                                           v[None, None].to(DEV), 1.0, n, batch_invariant=invariant)[0]
                _inside(got[-1:], want, tol)


# ------------------------------------------------------------------- cache --


@pytest.mark.parametrize("hd,hkv,ps", [(64, 2, 16), (8, 1, 32), (128, 4, 64), (80, 3, 16), (256, 1, 1024)])
def test_append(hd, hkv, ps):
    """Ragged counts over page borders; rows without a page, before 0 or past n, and all other bytes stay."""
    lengths, new = [40, 1, 0, 33, 70, 2, 64], [40, 1, 0, 2, 33, 2, 0]
    b, n = len(lengths), 40
    k, v, table, lens = _cache(lengths, hkv, hd, ps, BF16, seed=20)
    new_k, new_v = seeded(b, n, 2, hkv, hd, dtype=BF16, seed=21).unbind(2)
    table[3, 32 // ps] = -1 if 32 // ps else table[3, 0]
    got_k, got_v = k.to(DEV), v.to(DEV)
    fused = torch.stack([new_k, new_v], 2).to(DEV)
    ops.cache_append(fused[:, :, 0], fused[:, :, 1], got_k, got_v, table.to(DEV), lens.to(DEV),
                     new=torch.tensor(new, dtype=torch.int32, device=DEV))
    for i in range(b):
        for r in range(new[i]):
            pos = lengths[i] - new[i] + r
            page = int(table[i, pos // ps])
            if page >= 0:
                k[page, :, pos % ps], v[page, :, pos % ps] = new_k[i, r], new_v[i, r]
    assert torch.equal(got_k.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(got_v.cpu().view(torch.int16), v.view(torch.int16))


def test_append_out_of_place_counts():
    """Counts past n count as n, negative ones as none; positions before 0 and past the table are left out."""
    k, v, table, lens = _cache([3, 20, 50], 1, 64, 16, F16, seed=22)
    new_k, new_v = seeded(3, 4, 1, 64, dtype=F16, seed=23), seeded(3, 4, 1, 64, dtype=F16, seed=24)
    got_k, got_v = k.to(DEV), v.to(DEV)
    lens[2] = 10 ** 6
    ops.cache_append(new_k.to(DEV), new_v.to(DEV), got_k, got_v, table.to(DEV), lens.to(DEV),
                     new=torch.tensor([9, -1, 4], dtype=torch.int32, device=DEV))
    for r in range(1, 4):  # 4 rows for a sequence of 3: the first lies before 0
        k[table[0, 0], :, r - 1], v[table[0, 0], :, r - 1] = new_k[0, r], new_v[0, r]
    assert torch.equal(got_k.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(got_v.cpu().view(torch.int16), v.view(torch.int16))


def test_append_of_a_refused_reservation():
    """The reservation's status, not 0: no byte of the cache changes; 0: as without it."""
    for status in (0, 1, -1):
        k, v, table, lens = _cache([40, 1, 33], 2, 64, 16, F16, seed=25)
        new_k, new_v = seeded(3, 2, 2, 64, dtype=F16, seed=26), seeded(3, 2, 2, 64, dtype=F16, seed=27)
        new = torch.tensor([2, 1, 1], dtype=torch.int32, device=DEV)
        got_k, got_v, want_k, want_v = (t.to(DEV) for t in (k, v, k, v))
        ops.cache_append(new_k.to(DEV), new_v.to(DEV), got_k, got_v, table.to(DEV), lens.to(DEV), new=new,
                         status=torch.tensor([status], dtype=torch.int32, device=DEV))
        if status == 0:
            ops.cache_append(new_k.to(DEV), new_v.to(DEV), want_k, want_v, table.to(DEV), lens.to(DEV), new=new)
        assert torch.equal(got_k.view(torch.int16), want_k.view(torch.int16))
        assert torch.equal(got_v.view(torch.int16), want_v.view(torch.int16))
    with pytest.raises(ValueError, match="status must have 1 entries"):
        ops.cache_append(new_k.to(DEV), new_v.to(DEV), got_k, got_v, table.to(DEV), lens.to(DEV), status=new)


class _State:
    """A cache on the device beside the Book that says what it must hold."""

    def __init__(self, rows, width, pages, layers=2, hkv=2, ps=16, hd=32, dtype=F16):
        self.ps = ps
        self.table = torch.full((rows, width), -7, dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        self.k = seeded(layers, pages, hkv, ps, hd, dtype=dtype, seed=30).to(DEV)
        self.v = seeded(layers, pages, hkv, ps, hd, dtype=dtype, seed=31).to(DEV)
        self.book = Book(self.table.cpu(), self.lengths.cpu(), self.refs.cpu(), ps)
        self.want_k, self.want_v = self.k.cpu(), self.v.cpu()

    def vec(self, values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    def reserve(self, new):
        status = ops.cache_reserve(self.table, self.lengths, self.refs, self.vec(new), self.ps)
        assert int(status) == self.book.reserve(new)
        return self.check()

    def fork(self, parents, children):
        status = ops.cache_fork(self.k, self.v, self.table, self.lengths, self.refs, self.vec(parents),
                                self.vec(children))
        assert int(status) == self.book.fork(parents, children)
        return self.check()

    def free(self, rows):
        ops.cache_free(self.table, self.lengths, self.refs, self.vec(rows), self.ps)
        self.book.free(rows)
        return self.check()

    def compact(self):
        used = ops.cache_compact(self.k, self.v, self.table, self.lengths, self.refs)
        assert int(used) == self.book.compact()
        return self.check()

    def check(self):
        for src, dst, rows in self.book.copies:
            for c in (self.want_k, self.want_v):
                c[:, dst, :, :rows] = c[:, src, :, :rows]
        self.book.copies.clear()
        assert self.table.tolist() == self.book.table
        assert self.lengths.tolist() == self.book.lengths
        assert self.refs.tolist() == self.book.refs
        assert torch.equal(self.k.cpu(), self.want_k) and torch.equal(self.v.cpu(), self.want_v)
        return self


def test_pages_through_their_life():
    s = _State(rows=9, width=6, pages=30)
    s.reserve([0] * 9).reserve([1, 16, 17, 0, 33, 96, 0, 0, 0])
    s.fork([0, 1, 2, 4], [3, 6, 7, 8])          # begun pages are copied, a whole one is shared
    s.reserve([1, 1, 1, 1, 15, 0, 1, 15, 14])
    s.free([2, 2, 50, -1, 5])                    # twice, and rows that are not there
    s.compact().compact()
    s.fork([4, 4, 4], [2, 5, 2])                 # a child twice: refused
    s.fork([4, 9], [2, 5]).fork([4, -1], [2, 5]).fork([4], [9]).fork([4], [0])  # no such row, not empty
    s.fork([4, 4], [2, 5])                       # one parent, two children
    s.fork([], [])
    s.free([4])                                  # its pages live on in the children
    s.free([]).compact()
    s.reserve([0, 0, 96, 0, 0, 0, 0, 0, 0])      # past the table: refused
    s.reserve([0, 0, -1, 0, 0, 0, 0, 0, 0])
    s.free(list(range(9))).compact()
    assert not any(s.book.refs)


def test_pages_run_out():
    s = _State(rows=4, width=8, pages=6)
    s.reserve([90, 0, 0, 0]).reserve([7, 10, 0, 0])     # 6 of 6 pages; then one missing (and one: two)
    s.fork([0, 0], [1, 2])                               # two begun pages, none free
    s.reserve([6, 0, 0, 0])                              # the rest of the last page needs none
    s.fork([0, 0], [1, 2])                               # whole pages need none
    s.reserve([1, 0, 0, 0])
    s.free([0, 1, 2]).reserve([0, 0, 0, 96])
    s = _State(rows=2, width=4, pages=0)
    s.reserve([0, 0]).reserve([1, 0]).compact().free([0]).fork([0], [1])


@pytest.mark.parametrize("pages,rows", [(9000, 1500), (20000, 3)])
def test_pages_in_large_numbers(pages, rows):
    """More rows and pages than one step of a plan takes; rows that need one page and rows that need many."""
    gen = torch.Generator().manual_seed(40)
    s = _State(rows=rows, width=4200, pages=pages, layers=1, hkv=1, hd=8)
    new = torch.randint(0, 60, (rows,), generator=gen).tolist()
    new[0], new[-1] = 40000, 9999
    s.reserve(new)
    s.free([0]).reserve([0] + [17] * (rows - 1)).compact()
    if rows > 1000:
        empty = [b for b, n in enumerate(s.book.lengths) if n == 0]
        s.free(list(range(2, 900, 2))).compact()
        s.fork(list(range(1, 900, 2)), list(range(2, 900, 2)) + [0]).reserve([1] * rows).compact()
        assert empty == [0]


def test_pages_of_token_major_caches_and_views():
    """[layers, pages, page_size, Hkv, hd] storage, a table inside a larger one, one layer's 4-d pages."""
    s = _State(rows=6, width=5, pages=20, hd=40)
    s.k = s.k.transpose(2, 3).contiguous().transpose(2, 3)
    s.v = s.v.transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.full((6, 9), -7, dtype=torch.int32, device=DEV)
    s.table = wide[:, 2:7]
    s.reserve([20, 30, 1, 0, 70, 0]).fork([0, 4], [3, 5]).free([1, 4]).compact()
    assert bool((wide[:, :2] == -7).all()) and bool((wide[:, 7:] == -7).all())
    s.k, s.v, s.want_k, s.want_v = s.k[0], s.v[0], s.want_k[:1], s.want_v[:1]
    used = ops.cache_compact(s.k, s.v, s.table, s.lengths, s.refs)
    assert int(used) == s.book.compact()
    status = ops.cache_fork(s.k, s.v, s.table, s.lengths, s.refs, s.vec([5]), s.vec([1]))
    assert int(status) == s.book.fork([5], [1])
    s.k, s.v = s.k[None], s.v[None]
    s.check()


# ---------------------------------------------------------------- together --


def _stack(layers, d, heads, ffn):
    w = []
    for i in range(layers):
        g = 100 * i
        w.append(dict(
            qkv=seeded(3 * d, d, dtype=F16, seed=g + 1, scale=d ** -0.5).to(DEV),
            o=seeded(d, d, dtype=F16, seed=g + 2, scale=d ** -0.5).to(DEV),
            up=seeded(ffn, d, dtype=F16, seed=g + 3, scale=d ** -0.5).to(DEV),
            down=seeded(d, ffn, dtype=F16, seed=g + 4, scale=ffn ** -0.5).to(DEV)))
    return w


def _layer(x, w, attend):
    """One pre-LN block of this library's operators on rows x [n, d]."""
    d = x.shape[1]
    one, zero = torch.ones(d, device=DEV), torch.zeros(d, device=DEV)
    h = ops.ln_fwd(x, one, zero, 1e-5, out_dtype=F16)
    x = ops.linear_residual(attend(ops.linear(h, w["qkv"])), w["o"], None, x)
    h = ops.ln_fwd(x, one, zero, 1e-5, out_dtype=F16)
    return ops.linear_residual(ops.linear(h, w["up"], gelu=True), w["down"], None, x)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_generation_with_a_cache_matches_whole_sequences(window, sinks):
    """A causal stack token by token over the cache -- prompts of two lengths, a fork, a freed row, a
    compaction on the way, the step captured into a graph -- against the same stack run on the whole
    sequences without a cache."""
    layers, d, heads, ffn, ps = 2, 128, 4, 256, 16
    hd, rows, pages, steps = d // heads, 4, 40, 30
    scale, w = hd ** -0.5, _stack(layers, d, heads, ffn)
    prompts = [37, 16]
    tokens = seeded(rows, 37 + steps, d, seed=50).to(DEV)  # inputs of every position (the fork's differ after it)
    k, v = (torch.full((layers, pages, heads, ps, hd), float("nan"), dtype=F16, device=DEV) for _ in range(2))
    table = torch.full((rows, 8), -1, dtype=torch.int32, device=DEV)
    lengths, refs = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (rows, pages))

    def vec(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    # prompts, padded to one length
    new = vec(prompts + [0, 0])
    assert int(ops.cache_reserve(table, lengths, refs, new, ps)) == 0
    x = tokens[:2, :37].reshape(-1, d).contiguous()
    for i in range(layers):
        def prompt(qkv):
            q, kk, vv = qkv.view(2, 37, 3, heads, hd).unbind(2)
            ops.cache_append(kk, vv, k[i], v[i], table[:2], lengths[:2], new=new[:2])
            valid = torch.arange(37, device=DEV)[None, :] < lengths[:2, None]
            return ops.window_attention(q.transpose(1, 2), kk.transpose(1, 2), vv.transpose(1, 2), scale,
                                        window or 37, sinks=sinks, key_valid=valid).view(-1, d)
        x = _layer(x, w[i], prompt)
    assert int(ops.cache_fork(k, v, table, lengths, refs, vec([0, 0]), vec([2, 3]))) == 0
    ops.cache_free(table, lengths, refs, vec([0]), ps)
    ops.cache_compact(k, v, table, lengths, refs)
    tokens[2:, :37] = tokens[0, :37]

    # steps: row 0 is idle, its length stays 0
    one, status = vec([0, 1, 1, 1]), torch.zeros(1, dtype=torch.int32, device=DEV)
    x_in, x_out = torch.zeros(rows, d, device=DEV), torch.zeros(rows, d, device=DEV)

    def step():
        status.copy_(torch.maximum(status, ops.cache_reserve(table, lengths, refs, one, ps).abs()))
        h = x_in
        for i in range(layers):
            def decode(qkv):
                q, kk, vv = qkv.view(rows, 3, heads, hd).unbind(1)
                ops.cache_append(kk[:, None], vv[:, None], k[i], v[i], table, lengths, new=one)
                return ops.paged_attention(q, k[i], v[i], table, lengths, scale, window=window, sinks=sinks)
            h = _layer(h, w[i], decode)
        x_out.copy_(h)

    starts = [0, 16, 37, 37]
    outs = []
    graph = None
    for t in range(steps):
        x_in.copy_(torch.stack([tokens[b, starts[b] + t] for b in range(rows)]))
        if t == 3:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
                step()
            torch.cuda.current_stream().wait_stream(side)
        if graph is None:
            step()
        else:
            graph.replay()
        if t == 10:  # between two replays: pages move
            torch.cuda.synchronize()
            ops.cache_compact(k, v, table, lengths, refs)
        outs.append(x_out.clone())
    assert int(status) == 0 and lengths.tolist() == [0, 16 + steps, 37 + steps, 37 + steps]

    for b in (1, 2, 3):
        n = starts[b] + steps
        x = tokens[b, :n].contiguous()
        for i in range(layers):
            def whole(qkv):
                q, kk, vv = (t.permute(1, 0, 2)[None] for t in qkv.view(n, 3, heads, hd).unbind(1))
                seen = torch.arange(n, device=DEV)
                seen = (seen[None, :] <= seen[:, None]) & ((seen[None, :] > seen[:, None] - (window or n))
                                                           | (seen[None, :] < sinks))
                p = torch.softmax((q.float() @ kk.float().transpose(2, 3).contiguous() * scale)
                                  .masked_fill(~seen, float("-inf")), -1)
                return (p @ vv.float())[0].permute(1, 0, 2).reshape(n, d).half().contiguous()
            x = _layer(x, w[i], whole)
        got = torch.stack([o[b] for o in outs])
        # both paths round to fp16 at the same places; a last-bit difference in one (2^-11 of values of
        # a few units) passes through two layers of width 128
        assert float((got - x[starts[b]:]).abs().max()) < 2e-2


def test_a_captured_step_that_runs_out_of_pages():
    """A decode step over forked sequences, captured, replayed while pages are missing: every byte of the cache, the
    table, lengths and refs stay; once a sequence has ended, the same graph goes on where it was."""
    layers, heads, hkv, ps, hd, scale = 2, 4, 2, 16, 32, 0.25
    s = _State(rows=4, width=4, pages=6, layers=layers, hkv=hkv, ps=ps, hd=hd)
    s.reserve([32, 20, 0, 0]).fork([0, 1], [2, 3])  # whole pages shared, one begun page copied: one page is free
    one = s.vec([1, 1, 1, 1])
    rows = [seeded(4, (heads + 2 * hkv), hd, dtype=F16, seed=70 + i).to(DEV) for i in range(layers)]
    status, outs = s.vec([0]), [torch.zeros(4, heads * hd, dtype=F16, device=DEV) for _ in range(layers)]

    def step():
        left = ops.cache_reserve(s.table, s.lengths, s.refs, one, ps)
        for i in range(layers):
            q, kk, vv = rows[i][:, :heads], rows[i][:, heads:heads + hkv], rows[i][:, heads + hkv:]
            ops.cache_append(kk[:, None], vv[:, None], s.k[i], s.v[i], s.table, s.lengths, new=one, status=left)
            outs[i].copy_(ops.paged_attention(q, s.k[i], s.v[i], s.table, s.lengths, scale))
        status.copy_(left)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for run in (graph.replay, graph.replay, step):  # rows 0 and 2 need a page each
        run()
        assert int(status) == s.book.reserve([1, 1, 1, 1]) == 1
        s.check()
    s.free([3])  # its copied page is free, the shared one lives on in row 1
    one[3] = 0
    for t in range(2):
        for i in range(layers):
            rows[i].copy_(seeded(4, (heads + 2 * hkv), hd, dtype=F16, seed=80 + 2 * t + i))
        graph.replay()
        assert int(status) == s.book.reserve([1, 1, 1, 0]) == 0
        for i in range(layers):
            for b in range(3):
                page, at = s.book.table[b][(s.book.lengths[b] - 1) // ps], (s.book.lengths[b] - 1) % ps
                s.want_k[i, page, :, at] = rows[i][b, heads:heads + hkv].cpu()
                s.want_v[i, page, :, at] = rows[i][b, heads + hkv:].cpu()
        s.check()
        for i in range(layers):
            want, tol = paged_reference(rows[i][:, :heads].cpu(), s.want_k[i], s.want_v[i], s.table.cpu(),
                                        s.lengths.cpu(), scale)
            _inside(outs[i], want, tol)


def test_empty_calls():
    """No sequences, no heads, no tokens, no pages, no columns."""
    def half(*shape):
        return torch.zeros(*shape, dtype=F16, device=DEV)

    def ints(*shape):
        return torch.zeros(*shape, dtype=torch.int32, device=DEV)

    assert ops.window_attention(half(0, 2, 4, 64), half(0, 1, 4, 64), half(0, 1, 4, 64), 0.1, 4).shape == (0, 4, 128)
    assert ops.window_attention(half(2, 0, 4, 64), half(2, 0, 4, 64), half(2, 0, 4, 64), 0.1, 4).shape == (2, 4, 0)
    assert ops.window_attention(half(2, 2, 0, 64), half(2, 1, 4, 64), half(2, 1, 4, 64), 0.1, 4).shape == (2, 0, 128)
    assert ops.window_attention(half(2, 2, 4, 0), half(2, 1, 4, 0), half(2, 1, 4, 0), 0.1, 4).shape == (2, 4, 0)
    page = half(3, 1, 16, 64)
    assert ops.paged_attention(half(0, 2, 64), page, page, ints(0, 4), ints(0), 0.1).shape == (0, 128)
    assert ops.paged_attention(half(2, 0, 64), half(3, 0, 16, 64), half(3, 0, 16, 64), ints(2, 4), ints(2), 0.1).shape == (2, 0)
    for pages, width in ((page, 0), (half(0, 1, 16, 64), 4)):  # no entries; no pages: nothing is seen
        out = ops.paged_attention(half(2, 2, 64) + 1, pages, pages, ints(2, width), ints(2) + 30, 0.1)
        assert out.shape == (2, 128) and not bool(out.any())
    ops.cache_append(half(2, 0, 1, 64), half(2, 0, 1, 64), page, page, ints(2, 4), ints(2))
    ops.cache_append(half(0, 3, 1, 64), half(0, 3, 1, 64), page, page, ints(0, 4), ints(0))
    assert int(ops.cache_reserve(ints(0, 4), ints(0), ints(5), ints(0), 16)) == 0
    assert int(ops.cache_compact(page, page, ints(0, 4), ints(0), ints(3))) == 0
    ops.cache_free(ints(0, 4), ints(0), ints(5), ints(2), 16)
    assert not bool(page.any())


def test_streams_and_two_graphs():
    """Calls on a side stream, and two captured graphs replayed in turn, each with a workspace of its own."""
    k, v, table, lengths = (t.to(DEV) for t in _cache([5000, 300], 1, 64, 16, F16, seed=60))
    q1, q2 = seeded(2, 4, 64, dtype=F16, seed=61).to(DEV), seeded(2, 4, 64, dtype=F16, seed=62).to(DEV)
    wants = [ops.paged_attention(q, k, v, table, lengths, 0.125) for q in (q1, q2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attention(q1, k, v, table, lengths, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, wants[0])
    graphs = []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.paged_attention(q, k, v, table, lengths, 0.125)
        graphs.append((g, o))
    for _ in range(3):
        for _, o in graphs:
            o.zero_()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, o), want in zip(graphs, wants):
            assert torch.equal(o, want)


def test_window_streams_and_graphs():
    """Keys over workgroups: calls on two streams at once and two graphs replayed in turn, each with a workspace of its
    own, whatever memory held before; the same bits every time."""
    k, v = (seeded(1, 2, 9000, 64, dtype=F16, seed=i).to(DEV) for i in (63, 64))
    qs = [seeded(1, 4, n, 64, dtype=F16, seed=65 + n).to(DEV) for n in (3, 7)]

    def call(q):
        return ops.window_attention(q, k, v, 0.125, 8000, sinks=5)

    wants = [call(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        junk = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(4)]
        del junk  # what the workspaces are made of
        got = []
        for s, q in zip(streams, qs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(call(q))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for g, want in zip(got, wants):
            assert torch.equal(g, want)
    graphs = []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = call(q)
        graphs.append((g, o))
    for _ in range(3):
        for _, o in graphs:
            o.zero_()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, o), q, want in zip(graphs, qs, wants):
            assert torch.equal(o, want) and torch.equal(call(q), want)


def test_wrappers_refuse():
    q = torch.zeros(1, 2, 4, 64, dtype=F16, device=DEV)
    table, vec = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError, match="float16 and bfloat16"):
        ops.window_attention(q.float(), q.float(), q.float(), 0.1, 4)
    with pytest.raises(TypeError, match="k is"):
        ops.window_attention(q, q.bfloat16(), q, 0.1, 4)
    with pytest.raises(ValueError, match="contiguous head_dim"):
        ops.window_attention(q.transpose(2, 3), q, q, 0.1, 4)
    with pytest.raises(ValueError, match="key_valid"):
        ops.window_attention(q, q, q, 0.1, 4, key_valid=torch.ones(1, 5, dtype=torch.bool, device=DEV))
    with pytest.raises(RuntimeError, match="window"):
        ops.window_attention(q, q, q, 0.1, 0)
    with pytest.raises(RuntimeError, match="at most k_len"):
        ops.window_attention(q, q[:, :, :3], q[:, :, :3], 0.1, 4)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.window_attention(torch.zeros(1, 2, 4, 68, dtype=F16, device=DEV)[..., 4:], q, q, 0.1, 4)
    with pytest.raises(RuntimeError, match="page_size"):
        ops.paged_attention(q[:, :, 0], q, q, table, vec, 0.1)
    with pytest.raises(ValueError, match="row per sequence"):
        ops.paged_attention(torch.zeros(2, 2, 64, dtype=F16, device=DEV), q, q, table, vec, 0.1)
    with pytest.raises(ValueError, match="entries"):
        ops.cache_reserve(table, vec, vec, torch.zeros(2, dtype=torch.int32, device=DEV), 16)
    with pytest.raises(TypeError, match="int32"):
        ops.cache_free(table, vec, vec, vec.long(), 16)
    with pytest.raises(ValueError, match="one entry per page"):
        ops.cache_compact(q, q, table, vec, torch.zeros(3, dtype=torch.int32, device=DEV))
