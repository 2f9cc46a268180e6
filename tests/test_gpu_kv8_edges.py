"""The 8-bit paged K/V cache on the GPU at the edges of what its calls allow."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from test_gpu_kv8 import TYPES, Pair, check_attention, dtype_of

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Row offsets that begin behind row 0, as a slice of a batch's has them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("first", [1, 63, 64, 65, 640])
@pytest.mark.parametrize("page", [16, 64])
def test_rows_in_front_of_the_first_sequence(cuda, first, page):
    f = cuda.float32
    p = Pair(cuda, 1, 60, 2, 32, 3, 40, page, seed=first)
    counts = [70, 0, 5]
    cu = (first + np.cumsum([0] + counts)).tolist()
    slots, pos0 = p.ints([0, 2, 1]), p.grow([0, 2, 1], counts)
    k, v = (p.rows(cu[-1] + 9, 2, f) for _ in range(2))
    p.c.append(0, k, v, slots, p.ints(pos0), p.ints(cu))
    p.r.append(0, k.cpu().numpy(), v.cpu().numpy(), [0, 2, 1], pos0, cu)
    p.same()
    out = [cuda.full((cu[-1] + 9, 2, 32), 7.0, device="cuda") for _ in range(2)]
    p.c.read(0, slots, p.ints(pos0), cu[-1] + 9, p.ints(cu), out=out)
    for got, a, b in zip(out, p.r.rows(0, 0, 70), p.r.rows(0, 1, 5)):
        want = np.full((cu[-1] + 9, 2, 32), 7.0, np.float32)
        want[cu[0]:cu[1]], want[cu[2]:cu[3]] = a, b
        assert np.array_equal(got.cpu().numpy(), want)
    p.c.status()


@pytest.mark.parametrize("first", [1, 63, 64, 640])
@pytest.mark.parametrize("n_kv,counts", [(2, [3, 1]), (40, [129, 127])])   # streams of keys; tiles of rows
def test_attention_rows_in_front_of_the_first_sequence(cuda, first, n_kv, counts):
    p = Pair(cuda, 1, 40, n_kv, 32, 2, 20, 16, seed=first)
    p.fill([c + 3 for c in counts], cuda.float32)
    n = sum(counts)
    q = p.rows(first + n + 4, n_kv, cuda.float32)
    at = p.ints([0, 1]), p.ints([3, 3])
    out = cuda.full((first + n + 4, n_kv, 32), 7.0, device="cuda")
    p.c.attention(0, q, *at, p.ints((first + np.cumsum([0] + counts)).tolist()), out=out)
    assert (out[:first] == 7).all() and (out[first + n:] == 7).all()
    want, _ = p.r.attention(0, q[first:first + n].cpu().numpy(), [0, 1], [3, 3], [0, counts[0], n])
    assert np.abs(out[first:first + n].cpu().numpy() - want).max() < 1e-4
    p.c.status()


@pytest.mark.parametrize("cu", [[0, 20, 15, 40], [0, 30, 60, 61], [-3, 10, 20, 40], [0, 40, 10, 39]])
def test_row_offsets_out_of_range_are_reported(cuda, cu):
    """They fall, pass the 40 rows of the call or are negative: every call that takes
    them says so, and touches no row outside."""
    import aion_b200 as A
    for n_kv, group in ((2, 1), (40, 4)):   # streams of keys; tiles of rows
        p = Pair(cuda, 1, 40, n_kv, 32, 4, 8, 16)
        p.fill([60, 60, 60], cuda.float32)
        rows, q, slots, at = p.rows(40, n_kv, cuda.float32), p.rows(40, n_kv * group, cuda.float32), p.ints([0, 1, 2]), p.ints([0, 0, 0])
        k, v, wide = (cuda.full((60, h, 32), 7.0, device="cuda") for h in (n_kv, n_kv, n_kv * group))
        for call in (lambda: p.c.append(0, rows, rows, slots, at, p.ints(cu)),
                     lambda: p.c.read(0, slots, at, 40, p.ints(cu), out=(k[10:50], v[10:50])),
                     lambda: p.c.attention(0, q, slots, at, p.ints(cu), out=wide[10:50])):
            call()
            with pytest.raises(A.AionError) as e:
                p.c.status()
            assert e.value.code == "ARG"
        for t in (k, v, wide):
            assert (t[:10] == 7).all() and (t[50:] == 7).all() and cuda.isfinite(t).all()
        # of skipped sequences there is nothing to say
        p.c.attention(0, q, slots, p.ints([0, -1, -1]), p.ints([0, 40, 39, 100]), out=wide[10:50])
        p.c.status()


# ---------------------------------------------------------------------------
# Lists whose needs add up past 32 bits
# ---------------------------------------------------------------------------
def test_needs_past_32_bits_are_refused(cuda):
    """600 entries of 2^22 pages each: the sum passes 2^31 in the middle of the list."""
    import aion_b200 as A
    n, pages = 600, 1 << 22
    c = A.KV8Cache(1, 40, 1, 16, n + 2, pages, 16)
    seqs = cuda.arange(n + 2, dtype=cuda.int32, device="cuda")
    n_new = cuda.full((n + 2,), pages * 16, dtype=cuda.int32, device="cuda")
    n_new[0], n_new[300], n_new[-1] = 33, 16, 0   # three pages; one page, but behind what is refused; none
    pos0 = c.grow(seqs, n_new).tolist()
    assert pos0 == [0] + [-1] * n + [0]
    with pytest.raises(A.AionError) as e:
        c.status()
    assert e.value.code == "OOM"
    assert c.lens.tolist() == [33] + [0] * (n + 1) and c.refs.tolist() == [1] * 3 + [0] * 37
    assert c.tables[:, :4].tolist() == [[0, 1, 2, -1]] + [[-1] * 4] * (n + 1)


# ---------------------------------------------------------------------------
# Reports that other streams leave
# ---------------------------------------------------------------------------
def test_a_report_that_another_stream_leaves_meanwhile_is_not_lost(cuda):
    """A read of a slot that does not exist runs on one stream while the other
    asks for the status: one of the answers has it."""
    import aion_b200 as A
    p = Pair(cuda, 1, 4, 1, 16, 2, 2, 16)
    slot, at = p.ints([9]), p.ints([0])
    reader, asker = cuda.cuda.Stream(), cuda.cuda.Stream()
    cuda.cuda.synchronize()

    def asked():
        try:
            p.c.status(asker)
        except A.AionError as e:
            assert e.code == "ARG"
            return 1
        return 0

    for i in range(1000):
        with cuda.cuda.stream(reader):
            cuda.cuda._sleep(97 * (i % 500))   # up to 25 us
        p.c.read(0, slot, at, 1, stream=reader)
        got = asked() + asked() + asked()
        reader.synchronize()
        assert got + asked() >= 1, i
    assert asked() == 0


# ---------------------------------------------------------------------------
# Pages whose scales are far apart, or near the end of fp32's range
# ---------------------------------------------------------------------------
def by_terms(p, q, seqs, pos0, counts, scale=None):
    """(out, bound, score bound) of layer 0 in 64 bits.  bound[row][head] = sum of the
    row's weights times 127 V scales, divided by the sum of the weights: what
    relative errors of the terms are relative to, whatever the scales of pages
    that the row does not see or hardly weighs."""
    heads, hd = q.shape[1:]
    group = heads // p.r.k.shape[2]
    scale = 1 / np.sqrt(hd) if scale is None else scale
    out, bound, score = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    at = 0
    for slot, p0, n in zip(seqs, pos0, counts):
        k, v = p.r.rows(0, slot, p0 + n)
        vs = p.r.v_scale[0][p.r.tables[slot, np.arange(p0 + n) // p.r.page]].astype(np.float64)
        for h in range(heads):
            x, g = q[at:at + n, h].astype(np.float64), h // group
            s = x @ k[:, g].T * scale
            s[np.arange(p0 + n)[None, :] > p0 + np.arange(n)[:, None]] = -np.inf
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            out[at:at + n, h], bound[at:at + n, h] = w @ v[:, g], w @ vs[:, g] * 127
            score[at:at + n, h] = abs(scale) * np.abs(x).max(1) * np.abs(k[:, g]).sum(1).max()
        at += n
    return out, bound, score


def check_terms(p, q, seqs, pos0, counts, name, weight, with_cu=True, scale=None, largest=None):
    """Tolerance, relative to `bound`: twice the error of a score (queries to 22
    bits or more, sums of the dot and its two factors in fp32: 2^-21 of the
    largest query times the sum of a key, or, for queries that are held exactly,
    of the `largest` score; and 2^-21 for the exponential), the rounding of the weights (`weight`), fp32 sums of groups of 64 (as in the
    other tests); half a step of the result, infinite where it rounds to that; and, where scales are near the end
    of fp32's range, half of its smallest step for each group's factor, which
    meets up to 64 values of 127."""
    cu = [0] + np.cumsum(counts).tolist()
    got = p.c.attention(0, q, p.ints(seqs), p.ints(pos0), p.ints(cu) if with_cu else None, scale).float().cpu().numpy()
    want, bound, score = by_terms(p, q.float().cpu().numpy(), seqs, pos0, counts, scale)
    score = score if largest is None else largest
    seen = np.concatenate([b + 1 + np.arange(n) for b, n in zip(pos0, counts)])[:, None]
    tol = (2 * (score * 2.0 ** -21 + 2.0 ** -21) + weight + 2.0 ** -22 * (seen / 64 + 4)) * bound + seen * 2.0 ** -143
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
    least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[name]
    tol = tol[..., None] + half * np.abs(want) + least
    top = {"f32": 2.0 ** 128, "f16": 65520, "bf16": 2.0 ** 128}[name]   # rounds to infinity from here on
    big = np.abs(want) > top + tol
    assert (got[big] == np.copysign(np.inf, want[big])).all()
    with np.errstate(invalid="ignore"):
        got = np.where(np.abs(want) > top - tol, np.where(np.isinf(got), want, got), got)
    assert np.isfinite(got).all()
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), f"worst {float((err / tol).max())} of the tolerance"
    p.c.status()


def uneven(p, slot, base, ratio, light, heavy):
    """V scales of a slot's pages: `base`, but 1 / ratio of it on page `heavy`
    (which late rows see alone) and on page `light`, whose keys point away from
    every query of positive channels, so that their weights are about 2^-60."""
    table = p.r.tables[slot]
    p.r.v_scale[0, table[table >= 0]] *= np.float32(base)
    for page in (table[light], table[heavy]):
        p.r.v_scale[0, page] = np.minimum(p.r.v_scale[0, page].astype(np.float64) / ratio, 2.0 ** 100)
    p.r.k[0, table[light]] = -127
    p.r.k_scale[0, table[light]] = 60 * np.log(2) / 127 / np.sqrt(p.r.k.shape[-1]) / 0.8   # 0.8: the mean of |q|
    p.upload()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("base,ratio", [(1e-37, 1.0), (1e-30, 1.0), (1.0, 2.0 ** -10), (1.0, 2.0 ** -20), (1e-20, 2.0 ** -40),
                                        (1e-30, 2.0 ** -70)])
def test_many_rows_over_pages_of_uneven_scales(cuda, name, page, base, ratio):
    """Weights: two fp16 terms for fp32 rows (2^-22 of each), one for the others
    (2^-11), and 2^-32 of the largest term for each key."""
    if name == "f16" and base < 1e-10:
        pytest.skip("results below fp16's range")
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 40, 16, 32, 2, 40, page, seed=page)
    p.fill([320], dt)
    uneven(p, 0, base, ratio, 0 if page == 16 else 1, 320 // page - 1)
    q = p.rows(320, 16, dt).abs()
    check_terms(p, q, [0], [0], [320], name, (2.0 ** -22 if name == "f32" else 2.0 ** -11) + 320 * 2.0 ** -32)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("group,counts,before", [(1, [1, 1], [300, 304]), (4, [1, 1], [319, 100]), (4, [6, 3], [300, 301]),
                                                 (2, [40], [250])])
@pytest.mark.parametrize("base,ratio", [(1.0, 2.0 ** -8), (1.0, 2.0 ** -10), (2.0 ** -10, 2.0 ** -20), (1e-20, 2.0 ** -40)])
def test_few_rows_over_pages_of_uneven_scales(cuda, name, page, group, counts, before, base, ratio):
    """Weights: for each of 64 keys half a step of 24 or 16 bits of a group's largest term."""
    if name == "f16" and base < 1e-10:
        pytest.skip("results below fp16's range")
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 60, 2, 32, 2, 40, page, seed=page)
    p.fill([320] * len(counts), dt)
    for slot in range(len(counts)):
        uneven(p, slot, base, ratio, 0 if page == 16 else 1, 320 // page - 1)
    q = p.rows(sum(counts), 2 * group, dt).abs()
    check_terms(p, q, list(range(len(counts))), before, counts, name, 2.0 ** -19 if name == "f32" else 2.0 ** -11,
                with_cu=max(counts) > 1)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page", [32, 64])
@pytest.mark.parametrize("group,counts,before", [(1, [1, 1], [300, 304]), (4, [1, 1], [319, 100]), (4, [6, 3], [300, 301])])
@pytest.mark.parametrize("base", [1e-30, 1e-37, 1e30])
def test_few_rows_over_scales_near_the_ends_of_the_range(cuda, name, page, group, counts, before, base):
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 60, 2, 32, 2, 40, page, seed=page)
    p.fill([320] * len(counts), dt)
    for slot in range(len(counts)):
        uneven(p, slot, base, 1.0, 1, 320 // page - 1)
    q = p.rows(sum(counts), 2 * group, dt).abs()
    check_terms(p, q, list(range(len(counts))), before, counts, name, 2.0 ** -19 if name == "f32" else 2.0 ** -11,
                with_cu=max(counts) > 1)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n_kv,counts,before", [(2, [1, 1], [300, 9]), (2, [5, 3], [60, 0]), (16, [320], [0])])
def test_pages_of_zeros(cuda, name, page, n_kv, counts, before):
    """K or V of a page all zero: rows that see V of no other are zero, and the page's keys weigh as they are."""
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 60, n_kv, 32, 2, 40, page, seed=page)
    p.fill([a + b for a, b in zip(counts, before)], dt)
    for slot in range(len(counts)):
        t = p.r.tables[slot]
        p.r.v_scale[0, t[0]] = 0
        if t[2] >= 0:
            p.r.k_scale[0, t[2]] = 0
        if t[3] >= 0:
            p.r.v_scale[0, t[3], 1:] = 0
    p.upload()
    q = p.rows(sum(counts), n_kv * 2, dt)
    tiles = n_kv == 16
    weight = {True: 2.0 ** -22 + 320 * 2.0 ** -32, False: 2.0 ** -19}[tiles] if name == "f32" else 2.0 ** -11
    check_terms(p, q, list(range(len(counts))), before, counts, name, weight, with_cu=max(counts) > 1)


# ---------------------------------------------------------------------------
# Queries with one large channel
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,group,counts,before", [
    (2, 1, [1, 1], [299, 130]), (2, 4, [1, 1], [299, 130]), (2, 4, [5, 3], [290, 128]), (16, 1, [320], [0])])   # four kernels
def test_queries_with_one_large_channel(cuda, name, hd, n_kv, group, counts, before):
    """One channel 2^21 times the others, where the keys are 0: the scores come
    from the smallest digits.  508 = 127 2^16 u and 1..3 u (u = 2^-14) are held
    exactly by 24-bit fixed point, by fp16 and by two fp16 terms, so a score is
    off by its fp32 roundings only.  Weights: 64 half steps of 24 or 16 bits of a
    group's largest, or, in tiles, those of the test above."""
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 40, n_kv, hd, 2, 40, 16, seed=hd)
    p.fill([a + b for a, b in zip(counts, before)], dt)
    p.r.k[:] = p.rng.integers(0, 128, p.r.k.shape[:-1])[..., None]
    p.r.k[..., 5] = 0
    p.upload()
    q = cuda.from_numpy(p.rng.integers(1, 4, (sum(counts), n_kv * group, hd)).astype(np.float32) * 2.0 ** -14).to(dt).cuda()
    q[..., 5] = 508
    scale = 10 / (hd * 127 * 2.0 ** -13)
    tiles = n_kv == 16
    weight = {True: 2.0 ** -22 + 320 * 2.0 ** -32, False: 2.0 ** -19}[tiles] if name == "f32" else 2.0 ** -11
    check_terms(p, q, list(range(len(counts))), before, counts, name, weight, with_cu=counts != [1, 1], scale=scale, largest=10 * 1.5 * 1.5)


# ---------------------------------------------------------------------------
# Rows that see nothing
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n_kv,rows", [(2, 3), (16, 320)])   # streams of keys; tiles of rows
def test_rows_that_see_nothing_are_zero_whatever_their_query(cuda, name, n_kv, rows):
    """Slot 0's first 32 positions have no pages; queries that are not finite there and behind."""
    import aion_b200 as A
    p = Pair(cuda, 1, 40, n_kv, 32, 2, 40, 16, seed=rows)
    p.fill([rows + 30], cuda.float32)
    p.c.tables[0, :2] = -1
    q = p.rows(rows, n_kv, dtype_of(cuda, name))
    q[0, 0, 3], q[1, 1, 4], q[-1, 0, 2] = float("nan"), float("inf"), float("nan")
    out = p.c.attention(0, q, p.ints([0]), p.ints([30]), p.ints([0, rows])).float()   # rows 0 and 1: positions 30 and 31
    with pytest.raises(A.AionError) as e:
        p.c.status()
    assert e.value.code == "STATE"
    assert (out[:2] == 0).all()
    assert cuda.isnan(out[-1, 0]).all() and cuda.isfinite(out[-1, 1:]).all() and cuda.isfinite(out[2:-1]).all()


def test_rows_of_a_slot_without_pages_are_zero_and_reported(cuda):
    """Beside rows that have their pages, which come out whole."""
    import aion_b200 as A
    p = Pair(cuda, 1, 20, 1, 16, 4, 3, 16)
    p.fill([20, 20], cuda.float32)
    k, v = p.c.read(0, p.ints([0, 3]), p.ints([19, 0]), 4, p.ints([0, 3, 4]))
    with pytest.raises(A.AionError) as e:
        p.c.status()
    assert e.value.code == "STATE"
    for got, want in zip((k, v), p.r.rows(0, 0, 22)):   # positions 20 and 21: in slot 0's last page, behind its length
        assert np.array_equal(got[:3].cpu().numpy(), want[19:].astype(np.float32)) and (got[3] == 0).all()


@pytest.mark.parametrize("bits,code", [(8, "TIMEOUT"), (15, "TIMEOUT"), (7, "ARG"), (5, "STATE"), (1, "OOM")])
def test_status_reports_the_first_that_applies_once(cuda, bits, code):
    """The word that kernels set, among it what an attention call sets when a
    bounded wait gives up."""
    import aion_b200 as A
    p = Pair(cuda, 1, 4, 1, 16, 2, 2, 16)
    p.c.work[0] = bits
    with pytest.raises(A.AionError) as e:
        p.c.status()
    assert e.value.code == code
    p.c.status()


# ---------------------------------------------------------------------------
# fp32 rows, as close as their bits are
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n_kv,group,hd,page,counts,before", [
    (6, 1, 48, 16, [1, 1, 1], [500, 0, 77]), (2, 4, 128, 64, [1, 1], [300, 17]), (2, 2, 96, 32, [5, 9], [3, 260]),   # streams
    (16, 1, 64, 16, [90, 1, 130, 77], [0, 40, 7, 100]), (8, 4, 48, 32, [37, 64, 129, 1], [0, 3, 70, 11])])           # tiles
def test_fp32_rows_to_their_last_bits(cuda, n_kv, group, hd, page, counts, before):
    p = Pair(cuda, 1, 120, n_kv, hd, 5, 64, page, seed=hd)
    p.fill([a + b for a, b in zip(counts, before)], cuda.float32)
    q = p.rows(sum(counts), n_kv * group, cuda.float32)
    tiles = sum(counts) > 100
    check_terms(p, q, list(range(len(counts))), before, counts, "f32", 2.0 ** -22 + 230 * 2.0 ** -32 if tiles else 2.0 ** -19,
                with_cu=max(counts) > 1)


# ---------------------------------------------------------------------------
# Behind a call that failed
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("over,status", [(dict(n_layers=1000, n_pages=1 << 20, n_kv_heads=8, page_tokens=128, head_size=128), 4),   # 2^47 bytes
                                         (dict(device=99), 5)])
def test_a_failed_create_leaves_nothing_for_the_next_call(cuda, over, status):
    """No memory; no such device.  What runs next, here and in torch, does not see that error."""
    import aion_b200 as A
    shape = dict(device=0, n_layers=1, n_pages=4, n_kv_heads=1, page_tokens=16, head_size=16, max_seqs=2, max_pages=2)
    shape.update(over)
    p = Pair(cuda, 1, 4, 1, 16, 2, 2, 16)
    big, out = A.KV8(**shape), A.KV8()
    cuda.cuda.synchronize()
    assert A.lib().aion_kv8_create(ctypes.byref(big), ctypes.byref(out)) == status and not out.k
    assert p.grow([0], [20]) == [0]
    assert A.lib().aion_kv8_create(ctypes.byref(big), ctypes.byref(out)) == status
    assert (cuda.ones(8, device="cuda") * 2).sum().item() == 16
    p.c.status()


# ---------------------------------------------------------------------------
# Padding
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("counts,with_cu", [([1, 1, 1, 1, 1], False), ([1, 1, 1, 1, 1], True), ([3, 0, 20, 2, 5], True)])
def test_padding_in_front_does_not_hide_a_sequence(cuda, counts, with_cu):
    """Entries that are skipped, or have no rows, name slots that are written behind them."""
    p = Pair(cuda, 1, 20, 2, 32, 4, 4, 16)
    p.fill([17, 33], cuda.float32)
    p.grow([0, 1], [20, 20])
    p.append(0, [0, 1, 0, 1, 9], [-1, -1, 17, 33, -1], counts, cuda.float32, with_cu=with_cu)
    p.same()
    if not with_cu or counts[1]:
        q = p.rows(5, 2, cuda.float32)
        check_attention(p, 0, q, [0, 1, 0, 1, 9], [-1, -1, 17, 33, -1], counts, "f32", with_cu=with_cu)
    p.c.status()
