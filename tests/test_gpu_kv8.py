"""The 8-bit paged K/V cache on the GPU against its plain restatement
(oracle/kv8_ref.py), through the public calls.

Pages, tables and counts are whole numbers and int8 values follow one
definition to the bit, so they are compared for equality.  Attention is
compared with the restatement in 64 bits on the same stored values.  Its
error has these parts, with u the half step of the digits relative to the
largest value (2^-24 for fp32 rows, 2^-17 for 16-bit rows, doubled below):
  scores   scale * 2u max|q| * sum|k|, and fp32 roundings of them;
  weights  exp2 and the digits of the weights: 64 positions * 2u max|v|;
  sums     one fp32 rounding for each 64 positions;
  result   half a step of the row type.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle.kv8_ref import Cache

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Pair:
    """The library's cache and the restatement, given the same calls."""

    def __init__(self, torch, n_layers, n_pages, n_kv, hd, max_seqs, max_pages, page, seed=0):
        import aion_b200 as A
        self.torch = torch
        self.c = A.KV8Cache(n_layers, n_pages, n_kv, hd, max_seqs, max_pages, page)
        self.r = Cache(n_layers, n_pages, n_kv, hd, max_seqs, max_pages, page)
        self.rng = np.random.default_rng(seed)
        # stale bytes and scales in free pages, as after some time of use
        for name in ("k", "v"):
            getattr(self.r, name)[:] = self.rng.integers(-127, 128, self.r.k.shape)
            getattr(self.r, name + "_scale")[:] = self.rng.random(self.r.k_scale.shape) + 0.5
        self.upload()

    def upload(self):
        for name in ("k", "v", "k_scale", "v_scale", "tables", "lens", "refs"):
            getattr(self.c, name).copy_(self.torch.from_numpy(getattr(self.r, name)))

    def ints(self, v):
        return self.torch.tensor(list(v), dtype=self.torch.int32, device="cuda")

    def same(self, values=True):
        for name in ("tables", "lens", "refs") + (("k", "v", "k_scale", "v_scale") if values else ()):
            got, want = getattr(self.c, name).cpu().numpy(), getattr(self.r, name)
            assert np.array_equal(got, want, equal_nan=want.dtype.kind == "f"), name

    def grow(self, seqs, n_new):
        got = self.c.grow(self.ints(seqs), self.ints(n_new)).tolist()
        assert got == self.r.grow(seqs, n_new)
        return got

    def rows(self, n, heads, dt, spread=1.0):
        x = self.rng.standard_normal((n, heads, self.r.k.shape[-1])) * spread
        return self.torch.from_numpy(x.astype(np.float32)).to(dt).cuda()

    def append(self, layer, seqs, pos0, counts, dt, spread=1.0, with_cu=True):
        cu = [0] + np.cumsum(counts).tolist()
        k, v = (self.rows(cu[-1], self.r.k.shape[2], dt, spread) for _ in range(2))
        self.c.append(layer, k, v, self.ints(seqs), self.ints(pos0), self.ints(cu) if with_cu else None)
        self.r.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), seqs, pos0, cu)

    def fill(self, lens, dt, slots=None):
        """Slots of these lengths with rows in every layer."""
        slots = list(range(len(lens))) if slots is None else slots
        pos0 = self.grow(slots, lens)
        for layer in range(self.r.k.shape[0]):
            self.append(layer, slots, pos0, lens, dt)


def check_attention(p, layer, q, seqs, pos0, counts, name, scale=None, with_cu=True, out=None):
    torch = p.torch
    cu = [0] + np.cumsum(counts).tolist()
    got = p.c.attention(layer, q, p.ints(seqs), p.ints(pos0), p.ints(cu) if with_cu else None, scale, out)
    want, info = p.r.attention(layer, q[:cu[-1]].float().cpu().numpy(), seqs, pos0, cu, scale)
    got = got.float().cpu().numpy()[:cu[-1]].astype(np.float64)
    sc = abs(scale) if scale else 1 / np.sqrt(q.shape[2])
    u2 = 2.0 ** -20 if name == "f32" else 2.0 ** -16
    qm, ks, vm, seen = (info[..., i] for i in range(4))
    score = sc * qm * ks * u2 + 2.0 ** -20
    tol = (2 * score + 64 * u2 / 8 + 2.0 ** -22 * (seen / 64 + 4)) * vm
    tol = tol[..., None] + {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name] * np.abs(want) + 2.0 ** -24
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max())} of the tolerance"
    return got


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seed,page,layers,n_kv,hd", [(0, 16, 1, 1, 16), (1, 32, 3, 2, 48), (2, 64, 2, 5, 128), (3, 128, 1, 3, 96)])
def test_page_calls_follow_the_definition(cuda, seed, page, layers, n_kv, hd):
    p = Pair(cuda, layers, 40, n_kv, hd, 9, 8, page, seed)
    rng = np.random.default_rng(seed)
    for step in range(60):
        op = rng.integers(5)
        seqs = rng.permutation(9)[:rng.integers(1, 5)].tolist()
        if op <= 1:
            n_new = (rng.integers(0, 3 * page, len(seqs)) * rng.integers(0, 2, len(seqs))).tolist()
            p.grow(seqs, n_new)
        elif op == 2:
            keep = rng.integers(0, 5 * page, len(seqs)).tolist()
            p.c.trim(p.ints(seqs), p.ints(keep))
            p.r.trim(seqs, keep)
        elif op == 3:
            dst = [s for s in range(9) if s not in seqs][:len(seqs)]
            keep = rng.integers(0, 5 * page, len(dst)).tolist()
            p.c.fork(p.ints(seqs[:len(dst)]), p.ints(dst), p.ints(keep))
            p.r.fork(seqs[:len(dst)], dst, keep)
        else:
            u = p.ints([-1])
            p.c.compact(u)
            assert u.item() == p.r.compact()
        p.same()
    p.c.reset()
    assert p.c.refs.sum().item() == 0 and p.c.lens.sum().item() == 0 and (p.c.tables == -1).all()


@pytest.mark.parametrize("n_pages", [1, 5, 4095, 4096, 4097, 20001])
def test_pages_of_large_and_small_caches(cuda, n_pages):
    """Sweeps over refs that end inside a tile; the last page is the only free one."""
    p = Pair(cuda, 1, n_pages, 1, 16, 4, n_pages, 16)
    p.r.refs[:] = 1
    p.r.refs[-1] = 0
    p.upload()
    assert p.grow([2, 1], [16, 1]) == [0, -1]
    assert p.r.tables[2, 0] == n_pages - 1
    p.same()
    p.r.refs[:] = 0
    p.r.refs[-1] = 1
    p.upload()
    u = p.ints([0])
    p.c.compact(u)
    assert u.item() == p.r.compact() == 1
    p.same()
    assert p.c.tables[2, 0].item() == 0


def test_many_entries_in_one_call(cuda):
    p = Pair(cuda, 1, 5000, 1, 16, 1024, 6, 16)
    rng = np.random.default_rng(5)
    order = rng.permutation(1024).tolist()
    p.grow(order, rng.integers(0, 60, 1024).tolist())
    p.grow(order[::-1], rng.integers(0, 37, 1024).tolist())   # pages run out on the way
    p.c.fork(p.ints(order[:512]), p.ints(order[512:]))
    p.r.fork(order[:512], order[512:])
    p.grow(order, [1] * 1024)
    p.same()
    p.c.trim(p.ints(order))
    p.r.trim(order)
    p.same()


def test_shared_pages_are_copied_before_they_are_written(cuda):
    p = Pair(cuda, 2, 20, 2, 32, 4, 4, 16)
    p.fill([21], cuda.float32)
    p.c.fork(p.ints([0, 0]), p.ints([1, 2]), p.ints([21, 18]))
    p.r.fork([0, 0], [1, 2], [21, 18])
    pos0 = p.grow([1, 2, 0], [3, 3, 0])
    assert pos0 == [21, 18, 21]
    for layer in range(2):
        p.append(layer, [1, 2], pos0[:2], [3, 3], cuda.float32, spread=4.0)
    p.same()
    p.c.status()


def test_grow_serves_what_needs_no_page(cuda):
    """Entry 1 finds no pages; entry 2 needs none and is served; entry 0 got the last."""
    import aion_b200 as A
    p = Pair(cuda, 1, 3, 1, 16, 3, 4, 16)
    p.grow([2], [5])
    assert p.grow([0, 1, 2], [32, 16, 4]) == [0, -1, 5]
    p.same()
    with pytest.raises(A.AionError) as e:
        p.c.status()
    assert e.value.code == "OOM"
    p.c.status()   # reported once


# ---------------------------------------------------------------------------
# Append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page,n_kv,hd", [(16, 6, 48), (32, 1, 16), (64, 4, 128), (128, 2, 80)])
def test_append_and_read(cuda, name, page, n_kv, hd):
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 2, 40, n_kv, hd, 5, 8, page, seed=page)
    for counts, spread in (([page, 1, 3 * page + 5, 0, page - 1], 1.0), ([1, 1, 1, 1, 1], 1.2), ([7, page, 2, 40, 1], 0.1),
                           ([1, 1, 1, 1, 1], 30.0)):
        seqs = [3, 0, 4, 1, 2]
        pos0 = p.grow(seqs, counts)
        p.append(1, seqs, pos0, counts, dt, spread, with_cu=counts != [1] * 5 or spread > 2)
        p.same()
        cu = [0] + np.cumsum(counts).tolist()
        for out in TYPES:
            k, v = p.c.read(1, p.ints(seqs), p.ints(pos0), cu[-1], p.ints(cu), dtype=dtype_of(cuda, out))
            for i, s in enumerate(seqs):
                for got, want in zip((k, v), p.r.rows(1, s, pos0[i] + counts[i])):
                    part = cuda.from_numpy(want[pos0[i]:].astype(np.float32)).to(dtype_of(cuda, out))
                    assert cuda.equal(got[cu[i]:cu[i + 1]].cpu(), part)
    p.c.status()


def test_append_row_strides_and_alignment(cuda):
    """Rows inside a wider matrix, at an offset that forbids 16-byte vectors."""
    p = Pair(cuda, 1, 8, 2, 32, 2, 4, 16)
    pos0 = p.grow([0, 1], [20, 9])
    wide = p.rng.standard_normal((29, 2 * 64 + 7)).astype(np.float32)
    w = cuda.from_numpy(wide).cuda()
    k, v = w[:, 3:67].unflatten(1, (2, 32)), w[:, 67:131].unflatten(1, (2, 32))
    p.c.append(0, k, v, p.ints([0, 1]), p.ints(pos0), p.ints([0, 20, 29]))
    p.r.append(0, k.cpu().numpy(), v.cpu().numpy(), [0, 1], pos0, [0, 20, 29])
    p.same()
    out = cuda.full((29, 2 * 64 + 9), 7.0, device="cuda")
    o = out[:, 5:69].unflatten(1, (2, 32)), out[:, 69:133].unflatten(1, (2, 32))
    p.c.read(0, p.ints([0, 1]), p.ints(pos0), 29, p.ints([0, 20, 29]), out=o)
    want = p.r.rows(0, 0, 20)[0].astype(np.float32)
    assert np.array_equal(o[0][:20].cpu().numpy(), want)
    assert (out[:, :5] == 7).all() and (out[:, 133:] == 7).all()


def test_borders_zeros_and_values_that_are_not_finite(cuda):
    p = Pair(cuda, 1, 8, 3, 16, 3, 2, 16)
    pos0 = p.grow([0, 1, 2], [2, 2, 2])
    x = np.zeros((6, 3, 16), np.float32)
    x[0, 0] = np.linspace(-1, 1, 16)
    x[0, 0, 3] = 0.5 / 127 * 127      # quotients on borders
    x[1, 0] = (np.arange(16) + 0.5) / 127
    x[2, 1, 4], x[3, 2, 5] = np.inf, np.nan
    x[4, 0, 0], x[5, 0, 1] = 1e-44, 3e-45   # denormal scales
    x[4, 1, 0] = 3.4e38
    for part in (x, -x):
        k = cuda.from_numpy(part).cuda()
        p.c.append(0, k, k, p.ints([0, 1, 2]), p.ints(pos0), p.ints([0, 2, 4, 6]))
        p.r.append(0, part, part, [0, 1, 2], pos0, [0, 2, 4, 6])
        p.same()
    # later rows cannot heal a page whose scale is NaN; a page that starts anew can
    pos1 = p.grow([1], [3])
    y = np.ones((3, 3, 16), np.float32)
    p.c.append(0, cuda.from_numpy(y).cuda(), cuda.from_numpy(y).cuda(), p.ints([1]), p.ints(pos1), p.ints([0, 3]))
    p.r.append(0, y, y, [1], pos1, [0, 3])
    p.same()
    q = cuda.ones(1, 3, 16, device="cuda")
    out = p.c.attention(0, q, p.ints([1]), p.ints([4]))
    assert cuda.isfinite(out[0, 0]).all() and cuda.isnan(out[0, 1:]).all()


@pytest.mark.parametrize("seed", range(6))
def test_quotients_next_to_borders(cuda, seed):
    """x = (k + 1/2) s moved by single ulps: the nearest integer of the exact quotient decides."""
    rng = np.random.default_rng(seed)
    p = Pair(cuda, 1, 64, 1, 128, 1, 64, 16)
    pos0 = p.grow([0], [1024])
    x = np.zeros((1024, 1, 128), np.float32)
    for t in range(0, 1024, 16):
        top = np.float32(rng.random() * 10.0 ** rng.integers(-6, 6) + 1e-30)
        s = np.float32(np.float64(top) / 127)
        half = ((rng.integers(-127, 127, (16, 128)) + 0.5) * np.float64(s)).astype(np.float32)
        step = rng.integers(-1, 2, half.shape)
        x[t:t + 16, 0] = np.where(step == 0, half, np.nextafter(half, half + step.astype(np.float32)))
        x[t, 0, 0] = top
        x[t:t + 16, 0] = np.clip(x[t:t + 16, 0], -top, top)
    k = cuda.from_numpy(x).cuda()
    p.c.append(0, k, k, p.ints([0]), p.ints(pos0), p.ints([0, 1024]))
    p.r.append(0, x, x, [0], pos0, [0, 1024])
    p.same()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page,n_kv,group,hd", [(16, 6, 1, 48), (32, 2, 4, 128), (64, 1, 8, 64), (128, 2, 3, 96), (16, 1, 12, 16),
                                                (64, 3, 5, 112)])
def test_attention_of_single_tokens(cuda, name, page, n_kv, group, hd):
    dt = dtype_of(cuda, name)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500]
    p = Pair(cuda, 2, 160, n_kv, hd, 14, 32, page, seed=hd)
    p.fill(lens, dt, slots=list(range(1, 13)))
    order = p.rng.permutation(12)
    q = p.rows(12, n_kv * group, dt, spread=2.0)
    check_attention(p, 1, q, (order + 1).tolist(), [lens[i] - 1 for i in order], [1] * 12, name, with_cu=False)
    p.c.status()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n_kv,group,hd,page,counts,before", [
    (2, 1, 64, 16, [5, 1, 3, 4], [0, 40, 7, 100]),
    (1, 2, 128, 64, [3, 9, 1], [200, 0, 61]),
    (2, 4, 48, 32, [37, 64, 129, 1], [0, 3, 70, 11]),
    (1, 1, 128, 64, [257, 300], [0, 130]),
    (1, 8, 96, 128, [33, 2, 90], [100, 0, 1]),
    (1, 16, 16, 16, [40], [17])])
def test_attention_of_several_tokens(cuda, name, n_kv, group, hd, page, counts, before):
    dt = dtype_of(cuda, name)
    n = len(counts)
    p = Pair(cuda, 1, 200, n_kv, hd, n + 1, 64, page, seed=n)
    p.fill([a + b for a, b in zip(counts, before)], dt)
    q = p.rows(sum(counts), n_kv * group, dt)
    check_attention(p, 0, q, list(range(n)), before, counts, name)
    p.c.status()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_attention_of_one_long_sequence(cuda, name):
    """Few rows, one long axis: the work is cut across the card and joined."""
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 400, 2, 128, 2, 300, 64)
    p.fill([17001], dt)
    q = p.rows(1, 8, dt)
    check_attention(p, 0, q, [0], [17000], [1], name, with_cu=False)
    q = p.rows(3, 8, dt)
    check_attention(p, 0, q, [0], [16998], [3], name)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 30.0, 1e4])
def test_attention_of_flat_and_peaked_scores(cuda, spread):
    p = Pair(cuda, 1, 40, 2, 64, 2, 20, 32)
    p.fill([600], cuda.float32)
    q = p.rows(1, 2, cuda.float32, spread)
    check_attention(p, 0, q, [0], [599], [1], "f32", with_cu=False, scale=None if spread < 100 else 1e-4)
    check_attention(p, 0, q, [0], [599], [1], "f32", with_cu=False, scale=-0.02 if spread < 100 else -1e-5)


def test_attention_rows_that_see_nothing_and_rows_behind_the_last(cuda):
    p = Pair(cuda, 1, 40, 2, 64, 6, 4, 32)
    p.fill([50, 10], cuda.float32)
    q = p.rows(12, 4, cuda.float32)
    out = cuda.full((12, 4, 64), 3.0, device="cuda")
    # sequence 1 was refused, 2 has no rows; rows 9..11 lie behind the last sequence
    p.c.attention(0, q, p.ints([0, 2, 3, 1]), p.ints([46, -1, 5, 5]), p.ints([0, 4, 6, 6, 9]), out=out)
    want, _ = p.r.attention(0, q.cpu().numpy(), [0, 1], [46, 5], [0, 4, 7])
    got = out.cpu().numpy()
    alone = p.c.attention(0, q[:4].contiguous(), p.ints([0]), p.ints([46]), p.ints([0, 4])).cpu().numpy()
    assert np.abs(got[:4] - want[:4]).max() < 1e-4 and np.abs(alone - want[:4]).max() < 1e-4
    assert (got[4:6] == 0).all() and (got[9:] == 3).all()
    p.c.status()


def test_attention_poisoned_query_and_masked_pages(cuda):
    """A NaN query poisons its own row only; what lies behind a row's position is never seen."""
    p = Pair(cuda, 1, 8, 1, 32, 2, 8, 16)
    p.fill([40], cuda.float32)
    p.c.k_scale[0, p.c.tables[0, 2].long()] = float("nan")   # positions 32..39
    p.c.v_scale[0, p.c.tables[0, 2].long()] = float("nan")
    q = p.rows(3, 2, cuda.float32)
    q[1, 0, 7] = float("nan")
    q[1, 1, 3] = float("inf")
    out = p.c.attention(0, q, p.ints([0]), p.ints([30]), p.ints([0, 3])).cpu().numpy()
    assert np.isfinite(out[0]).all() and np.isnan(out[2]).all()
    assert np.isnan(out[1]).all()
    want, _ = p.r.attention(0, q.cpu().numpy(), [0], [30], [0, 1])
    assert np.abs(out[0] - want[0]).max() < 1e-5


def test_attention_strides_and_out(cuda):
    p = Pair(cuda, 1, 20, 2, 32, 2, 8, 16)
    p.fill([70, 33], cuda.float32)
    wide = p.rows(2, 12, cuda.float32)
    q = wide.flatten(1)[:, 33:161].unflatten(1, (4, 32))   # 4-byte aligned only
    out = cuda.zeros(2, 401, device="cuda")[:, 1:129].unflatten(1, (4, 32))
    check_attention(p, 0, q, [0, 1], [69, 32], [1, 1], "f32", with_cu=False, out=out)


# ---------------------------------------------------------------------------
# Many rows a sequence: tiles of 128 rows.  Calls come here from 592 units of 8
# rows on (sequences x K/V heads x rows / 8).  Weights of 16-bit rows are fp16:
# half a step of 2^-11 of each, so 2^-11 of the largest value in all; fp32
# queries and weights have 22 bits, which the digits' bounds hold.
# ---------------------------------------------------------------------------
def check_tiles(p, q, seqs, pos0, counts, name, scale=None, with_cu=True, out=None):
    lines, rows = len(seqs) * p.r.k.shape[2], -(-sum(counts) * (q.shape[1] // p.r.k.shape[2]) // len(seqs))
    assert lines * -(-rows // 8) >= 592 and lines * -(-rows // 256) <= 132   # one wave of blocks
    cu = [0] + np.cumsum(counts).tolist()
    got = p.c.attention(0, q, p.ints(seqs), p.ints(pos0), p.ints(cu) if with_cu else None, scale, out)
    want, info = p.r.attention(0, q[:cu[-1]].float().cpu().numpy(), seqs, pos0, cu, scale)
    got = got.float().cpu().numpy()[:cu[-1]].astype(np.float64)
    sc = abs(scale) if scale else 1 / np.sqrt(q.shape[2])
    u2 = 2.0 ** -20 if name == "f32" else 2.0 ** -16
    qm, ks, vm, seen = (info[..., i] for i in range(4))
    tol = (2 * (sc * qm * ks * u2 + 2.0 ** -20) + 64 * u2 / 8 + 2.0 ** -22 * (seen / 64 + 4)) * vm
    tol += (0 if name == "f32" else 2.0 ** -11) * vm
    tol = tol[..., None] + {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name] * np.abs(want) + 2.0 ** -24
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n_kv,group,hd,page,counts,before", [
    (16, 1, 64, 16, [90, 1, 130, 77], [0, 40, 7, 100]),
    (8, 2, 128, 64, [257, 30, 5, 1], [130, 0, 61, 200]),
    (8, 4, 48, 32, [37, 64, 129, 1], [0, 3, 70, 11]),
    (4, 8, 96, 128, [133, 2, 90], [100, 0, 1]),
    (2, 16, 16, 16, [240], [17]),
    (40, 1, 80, 64, [129, 127], [0, 513]),
    (3, 7, 112, 32, [0, 300, 0, 210], [0, 1, 5, 64])])
def test_attention_of_many_rows(cuda, name, n_kv, group, hd, page, counts, before):
    dt = dtype_of(cuda, name)
    n = len(counts)
    p = Pair(cuda, 1, 120, n_kv, hd, n + 1, 64, page, seed=n + hd)
    p.fill([a + b for a, b in zip(counts, before)], dt)
    check_tiles(p, p.rows(sum(counts), n_kv * group, dt), list(range(n)), before, counts, name)
    p.c.status()


@pytest.mark.parametrize("name", TYPES)
def test_attention_of_single_tokens_with_many_heads(cuda, name):
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 120, 2, 16, 17, 8, 16, seed=3)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 100, 99, 33, 5, 80, 70]
    p.fill(lens, dt)
    check_tiles(p, p.rows(16, 320, dt), list(range(16)), [n - 1 for n in lens], [1] * 16, name, with_cu=False)
    p.c.status()


@pytest.mark.parametrize("spread,scale", [(0.0, None), (1e-3, None), (30.0, None), (1e4, None), (1.0, -0.3), (1.0, 3.0)])
def test_many_rows_of_flat_and_peaked_scores(cuda, spread, scale):
    p = Pair(cuda, 1, 40, 16, 32, 2, 40, 16, seed=1)
    p.fill([320], cuda.float32)
    check_tiles(p, p.rows(320, 16, cuda.float32, spread), [0], [0], [320], "f32", scale)


@pytest.mark.parametrize("name,off", [("f32", 33), ("f16", 1), ("bf16", 3)])
def test_many_rows_with_strides(cuda, name, off):
    dt = dtype_of(cuda, name)
    p = Pair(cuda, 1, 40, 16, 32, 2, 40, 16, seed=2)
    p.fill([330], dt)
    q = p.rows(320, 20, dt).flatten(1)[:, off:off + 512].unflatten(1, (16, 32))
    out = cuda.zeros(320, 521, device="cuda", dtype=dt)[:, 1:513].unflatten(1, (16, 32))
    check_tiles(p, q, [0], [10], [320], name, out=out)


def test_many_rows_that_see_nothing_and_what_poisons_them(cuda):
    import aion_b200 as A
    p = Pair(cuda, 1, 40, 16, 64, 6, 8, 32, seed=4)
    p.fill([186, 95, 0, 5], cuda.float32)
    q = p.rows(320, 16, cuda.float32)
    q[10, 5, 3] = float("nan")
    q[11, 6, 3] = float("-inf")
    clean = p.r.attention(0, q.cpu().numpy(), [0], [46], [0, 140])[0][:140]
    p.c.v_scale[0, p.c.tables[0, 4].long(), 3] = float("nan")   # slot 0, positions 128..159, head 3
    p.c.k_scale[0, p.c.tables[0, 5].long(), 2] = float("nan")   # 160.., head 2
    p.c.tables[1, 1] = -1                                       # slot 1, positions 32..63
    out = cuda.full((320, 16, 64), 3.0, device="cuda")
    # slot 0: 140 rows; 80 of a refused sequence; slot 3: none; slot 1: 90; 10 behind the last sequence
    p.c.attention(0, q, p.ints([0, 2, 3, 1]), p.ints([46, -1, 5, 5]), p.ints([0, 140, 220, 220, 310]), out=out)
    with pytest.raises(A.AionError) as e:
        p.c.status()
    assert e.value.code == "STATE"
    got = out.cpu().numpy()
    assert (got[140:220] == 0).all() and (got[310:] == 3).all()
    nan = np.zeros((140, 16), bool)
    nan[10, 5] = nan[11, 6] = True
    nan[128 - 46:, 3] = True
    nan[160 - 46:, 2] = True
    assert (np.isnan(got[:140]).all(-1) == nan).all() and (np.isnan(got[:140]).any(-1) == nan).all()
    assert np.abs(got[:140] - clean)[~nan].max() < 1e-4
    k, v = p.r.rows(0, 1, 95)
    k, v = (np.delete(x, slice(32, 64), 0) for x in (k, v))
    for r in (0, 20, 31, 57, 58, 59, 89):
        seen = r + 6 if r + 6 <= 32 else 32 + max(r + 6 - 64, 0)
        for h in range(16):
            x = k[:seen, h] @ q[220 + r, h].cpu().numpy().astype(np.float64) / 8
            w = np.exp(x - x.max())
            assert np.abs(got[220 + r, h] - w @ v[:seen, h] / w.sum()).max() < 1e-4


def test_many_rows_captured_and_replayed(cuda):
    p = Pair(cuda, 1, 40, 16, 64, 3, 20, 32, seed=5)
    p.fill([400, 300], cuda.bfloat16)
    q = p.rows(300, 16, cuda.bfloat16)
    seqs, pos0, cu = p.ints([0, 1]), p.ints([0, 0]), p.ints([0, 150, 300])
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        out = p.c.attention(0, q, seqs, pos0, cu)
    for at, rows in (([0, 0], 150), ([200, 100], 200), ([100, -1], 100)):
        pos0.copy_(p.ints(at))
        cu.copy_(p.ints([0, rows, 300]))
        out.fill_(5)
        graph.replay()
        first = out.clone()
        graph.replay()
        eager = p.c.attention(0, q, seqs, pos0, cu)
        assert cuda.equal(first, out) and cuda.equal(eager, out)


def test_many_rows_do_not_change_from_run_to_run_or_beside_another_stream(cuda):
    p = Pair(cuda, 1, 80, 16, 128, 3, 20, 64, seed=6)
    p.fill([700, 500], cuda.float32)
    q = p.rows(400, 16, cuda.float32)
    args = p.ints([0, 1]), p.ints([500, 300]), p.ints([0, 200, 400])
    first = p.c.attention(0, q, *args)
    streams = [cuda.cuda.Stream() for _ in range(3)]
    cuda.cuda.synchronize()
    got = [p.c.attention(0, q, *args, stream=streams[i % 3]) for i in range(9)]
    cuda.cuda.synchronize()
    assert all(cuda.equal(first, g) for g in got)
    p.c.status()


@pytest.mark.parametrize("with_cu", [True, False])
def test_4096_sequences_in_one_call(cuda, with_cu):
    p = Pair(cuda, 1, 9000, 1, 16, 4096, 2, 16, seed=8)
    order = p.rng.permutation(4096)
    for i in range(0, 4096, 1024):   # a page call takes 1024 entries
        s = order[i:i + 1024].tolist()
        p.grow(s, (1 + np.asarray(s) % 20).tolist())
    lens = p.r.lens[order]
    counts = np.where(order % 3 == 0, 0, np.minimum(lens, 2)) if with_cu else np.ones(4096, int)
    pos0 = (lens - counts).tolist()
    p.append(0, order.tolist(), [0] * 4096, lens.tolist(), cuda.float32)
    p.append(0, order.tolist(), pos0, counts.tolist(), cuda.float32, with_cu=with_cu)
    p.same()
    check_attention(p, 0, p.rows(int(counts.sum()), 2, cuda.float32), order.tolist(), pos0, counts.tolist(), "f32", with_cu=with_cu)
    p.c.status()


def test_pages_behind_four_gigabytes(cuda):
    """K and V of 5 GB each, the pages in use at their ends; a layer and a page copy behind 4 GB, too."""
    import aion_b200 as A
    n_pages, nkv, page, hd = 20000, 8, 128, 128
    pool = (2, n_pages, nkv, page, hd)
    k, v = (cuda.empty(pool, dtype=cuda.int8, device="cuda") for _ in range(2))
    ks, vs = (cuda.empty(pool[:3], device="cuda") for _ in range(2))
    refs = cuda.ones(n_pages, dtype=cuda.int32, device="cuda")
    refs[-8:] = 0
    big = A.KV8Cache.wrap(k, v, ks, vs, cuda.full((3, 6), -1, dtype=cuda.int32, device="cuda"),
                          cuda.zeros(3, dtype=cuda.int32, device="cuda"), refs)
    p = Pair(cuda, 2, 8, nkv, hd, 3, 6, page, seed=9)
    x = [p.rows(300, nkv, cuda.float32) for _ in range(2)]
    one, many = p.rows(1, 16, cuda.float32), p.rows(300, 16, cuda.float32)
    got = []
    for c in (p.c, big):
        pos0 = c.grow(p.ints([1]), p.ints([300]))
        c.append(1, x[0], x[1], p.ints([1]), pos0, p.ints([0, 300]))
        c.fork(p.ints([1]), p.ints([2]))
        at = c.grow(p.ints([2]), p.ints([1]))   # copies the last page
        c.append(1, x[0][:1] * 2, x[1][:1] * 2, p.ints([2]), at)
        got.append([c.read(1, p.ints([2]), p.ints([0]), 301, p.ints([0, 301])),
                    c.attention(1, one, p.ints([2]), p.ints([300])),
                    c.attention(1, many, p.ints([1]), p.ints([0]), p.ints([0, 300]))])
        c.status()
    assert big.tables[1, 0].item() == n_pages - 8 and big.tables[2, 2].item() == n_pages - 5
    for a, b in zip(got[0][0], got[1][0]):
        assert cuda.equal(a, b)
    assert cuda.equal(got[0][1], got[1][1]) and cuda.equal(got[0][2], got[1][2])


# ---------------------------------------------------------------------------
# Entries that are refused on the device
# ---------------------------------------------------------------------------
def test_bad_entries_are_skipped_and_reported(cuda):
    import aion_b200 as A
    p = Pair(cuda, 1, 20, 1, 16, 4, 4, 16)
    p.grow([0, 1], [20, 20])
    cases = [lambda: p.grow([0, 0], [1, 1]), lambda: p.grow([4], [1]), lambda: p.grow([-1, 2], [1, 1]),
             lambda: p.grow([0], [-1]), lambda: p.grow([0], [1000]),
             lambda: (p.c.trim(p.ints([1, 1, 9]), p.ints([18, 3, 0])), p.r.trim([1, 1, 9], [18, 3, 0])),
             lambda: (p.c.fork(p.ints([0, 0, 3]), p.ints([0, 3, 2])), p.r.fork([0, 0, 3], [0, 3, 2])),
             lambda: (p.c.fork(p.ints([0, 1]), p.ints([2, 2])), p.r.fork([0, 1], [2, 2]))]
    for call in cases:
        call()
        p.same()
        with pytest.raises(A.AionError) as e:
            p.c.status()
        assert e.value.code == "ARG"
    p.c.status()


def test_rows_without_a_page_are_skipped_and_reported(cuda):
    import aion_b200 as A
    p = Pair(cuda, 1, 20, 1, 16, 4, 3, 16)
    p.grow([0, 1], [20, 20])
    p.c.fork(p.ints([1]), p.ints([2]))
    p.r.fork([1], [2])

    def code(call):
        call()
        p.same()
        with pytest.raises(A.AionError) as e:
            p.c.status()
        return e.value.code

    f = cuda.float32
    assert code(lambda: p.append(0, [0], [30], [5], f)) == "STATE"        # rows 32.. have no page
    assert code(lambda: p.append(0, [0], [47], [9], f)) == "STATE"        # behind the table
    assert code(lambda: p.append(0, [1, 2], [20, 19], [1, 1], f)) == "STATE"   # pages of two slots
    assert code(lambda: p.append(0, [0, 0], [3, 4], [2, 2], f)) == "ARG"
    assert code(lambda: p.append(0, [7, 0], [3, 4], [2, 2], f)) == "ARG"
    q = p.rows(2, 1, f)
    k, _ = p.c.read(0, p.ints([0, 3]), p.ints([19, 0]), 4, p.ints([0, 3, 4]))
    assert code(lambda: None) == "STATE" or True
    k, _ = p.c.read(0, p.ints([0]), p.ints([31]), 2, p.ints([0, 2]))
    with pytest.raises(A.AionError):
        p.c.status()
    assert (k[1] == 0).all()
    out = p.c.attention(0, q, p.ints([9, 0]), p.ints([3, 3]))
    with pytest.raises(A.AionError):
        p.c.status()
    assert (out[0] == 0).all() and cuda.isfinite(out).all()
    p.c.attention(0, q[:1], p.ints([0]), p.ints([1000000]))   # far behind the table
    with pytest.raises(A.AionError):
        p.c.status()
    p.c.tables[0, 0] = 12345   # a damaged table
    p.c.attention(0, q[:1], p.ints([0]), p.ints([18]))
    with pytest.raises(A.AionError):
        p.c.status()


def test_python_checks(cuda):
    import aion_b200 as A
    p = Pair(cuda, 1, 4, 2, 32, 2, 2, 16)
    i = p.ints([0])
    q = cuda.zeros(1, 2, 32, device="cuda")
    for call in (lambda: p.c.attention(0, q.double(), i, i), lambda: p.c.attention(0, q.cpu(), i, i),
                 lambda: p.c.attention(0, q[..., :16], i, i), lambda: p.c.attention(0, q.transpose(1, 2), i, i),
                 lambda: p.c.attention(0, q, i.long(), i), lambda: p.c.attention(0, q, i.cpu(), i),
                 lambda: p.c.attention(0, q, i, i, scale=0.0), lambda: p.c.append(0, q, q.half(), i, i),
                 lambda: p.c.append(0, cuda.cat([q, q]), cuda.cat([q, q]), i, i),
                 lambda: A.KV8Cache.wrap(p.c.k, p.c.v, p.c.k_scale, p.c.v_scale, p.c.tables, p.c.lens, p.c.refs[:3]),
                 lambda: A.KV8Cache.wrap(p.c.k, p.c.v[:, :, :, ::2], p.c.k_scale, p.c.v_scale, p.c.tables, p.c.lens, p.c.refs)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(A.AionError):
        p.c.attention(1, q, i, i)
    with pytest.raises(A.AionError):
        A.KV8Cache(1, 1, 1, 20, 1, 1)


# ---------------------------------------------------------------------------
# As they are used: streams, graphs, a run of calls together
# ---------------------------------------------------------------------------
def test_step_captured_and_replayed(cuda):
    """One decode step (grow, append, attention in two layers) as a CUDA graph,
    replayed while the cache goes on: each replay is the eager step."""
    p = Pair(cuda, 2, 64, 2, 64, 4, 12, 16)
    p.fill([15, 40, 3], cuda.float32)
    seqs, one = p.ints([0, 1, 2]), p.ints([1, 1, 1])
    pos0 = p.ints([0, 0, 0])
    k, v, q = (cuda.zeros(3, n, 64, device="cuda") for n in (2, 2, 4))
    out = cuda.zeros(2, 3, 4, 64, device="cuda")

    def step():
        p.c.grow(seqs, one, pos0)
        for layer in range(2):
            p.c.append(layer, k, v, seqs, pos0)
            p.c.attention(layer, q, seqs, pos0, out=out[layer])

    s = cuda.cuda.Stream()
    s.wait_stream(cuda.cuda.current_stream())
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=s):
        step()
    for i in range(20):
        for t in (k, v, q):
            t.copy_(cuda.from_numpy(p.rng.standard_normal(tuple(t.shape)).astype(np.float32)))
        graph.replay()
        want_pos = p.r.grow([0, 1, 2], [1, 1, 1])
        assert pos0.tolist() == want_pos
        for layer in range(2):
            p.r.append(layer, k.cpu().numpy(), v.cpu().numpy(), [0, 1, 2], want_pos, [0, 1, 2, 3])
            want, _ = p.r.attention(layer, q.cpu().numpy(), [0, 1, 2], want_pos, [0, 1, 2, 3])
            assert np.abs(out[layer].cpu().numpy() - want).max() < 1e-4
    p.same()
    p.c.status()


def test_reads_on_two_streams_at_once(cuda):
    """Attention calls of one cache that overlap have workspaces of their own."""
    p = Pair(cuda, 1, 300, 2, 128, 2, 200, 64)
    p.fill([9000, 3000], cuda.float32)
    q = p.rows(64, 8, cuda.float32)
    want = [p.c.attention(0, q[i:i + 1], p.ints([i % 2]), p.ints([8999 if i % 2 == 0 else 2999])) for i in range(64)]
    streams = [cuda.cuda.Stream() for _ in range(4)]
    slot, at = [p.ints([0]), p.ints([1])], [p.ints([8999]), p.ints([2999])]
    cuda.cuda.synchronize()
    got = [p.c.attention(0, q[i:i + 1], slot[i % 2], at[i % 2], stream=streams[i % 4]) for i in range(64)]
    cuda.cuda.synchronize()
    for g, w in zip(got, want):
        assert cuda.equal(g, w)


def test_results_do_not_change_from_run_to_run(cuda):
    p = Pair(cuda, 1, 400, 4, 128, 8, 100, 64)
    p.fill([3000, 1, 700, 64, 65, 2000], cuda.bfloat16)
    q = p.rows(6, 16, cuda.bfloat16)
    pos0 = [2999, 0, 699, 63, 64, 1999]
    first = p.c.attention(0, q, p.ints(range(6)), p.ints(pos0))
    for _ in range(5):
        assert cuda.equal(first, p.c.attention(0, q, p.ints(range(6)), p.ints(pos0)))


def test_serving_run(cuda):
    """Prompts in chunks, a shared prefix, single tokens, drafts that are taken
    back, sequences that end, a compaction: after each the answers are those of
    the restatement on the same state."""
    p = Pair(cuda, 2, 60, 2, 48, 6, 12, 16, seed=11)
    live = {}

    def feed(slots, counts):
        pos0 = p.grow(slots, counts)
        assert -1 not in pos0
        q = p.rows(sum(counts), 6, cuda.float32)
        for layer in range(2):
            p.append(layer, slots, pos0, counts, cuda.float32)
            check_attention(p, layer, q, slots, pos0, counts, "f32")

    feed([0, 1], [50, 33])
    feed([0, 1], [20, 7])
    p.c.fork(p.ints([0, 0]), p.ints([2, 3]), p.ints([50, 64]))
    p.r.fork([0, 0], [2, 3], [50, 64])
    feed([2, 3, 0], [5, 1, 1])
    for _ in range(4):
        feed([0, 1, 2, 3], [1, 1, 1, 1])
    feed([1, 3], [6, 6])
    keep = [int(p.r.lens[1]) - 4, int(p.r.lens[3]) - 5]
    p.c.trim(p.ints([1, 3]), p.ints(keep))
    p.r.trim([1, 3], keep)
    feed([3, 1], [2, 3])
    p.c.trim(p.ints([0]))
    p.r.trim([0])
    p.c.compact()
    p.r.compact()
    feed([4, 1, 2, 3], [61, 1, 1, 1])
    p.same()
    p.c.status()
