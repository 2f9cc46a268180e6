"""The 8-bit paged K/V cache without a GPU: the plain restatement's own
properties (oracle/kv8_ref.py) and the refusals of the C ABI, all of which
come before any device work."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle.kv8_ref import Cache

ARG, SHAPE = 8, 3


# ---------------------------------------------------------------------------
# The restatement
# ---------------------------------------------------------------------------
def holders(c: Cache) -> np.ndarray:
    n = np.zeros(len(c.refs), np.int32)
    for slot, length in enumerate(c.lens):
        for p in c.tables[slot, :c._pages(length)]:
            n[p] += 1
    return n


@pytest.mark.parametrize("seed", range(4))
def test_pages_are_accounted_for(seed):
    rng = np.random.default_rng(seed)
    c = Cache(1, 24, 1, 16, 6, 8, 16)
    for _ in range(120):
        op = rng.integers(4)
        seqs = rng.permutation(6)[:rng.integers(1, 4)].tolist()
        if op == 0:
            before = c.lens.copy()
            pos0 = c.grow(seqs, rng.integers(0, 40, len(seqs)).tolist())
            assert all(p in (-1, before[s]) for p, s in zip(pos0, seqs))
        elif op == 1:
            c.trim(seqs, rng.integers(0, 60, len(seqs)).tolist())
        elif op == 2:
            c.fork(seqs[:1], [s for s in range(6) if s not in seqs][:1], [int(rng.integers(0, 80))])
        else:
            u = c.compact()
            assert (c.refs[:u] > 0).all() and (c.refs[u:] == 0).all()
        assert (holders(c) == c.refs).all()
        for slot, length in enumerate(c.lens):
            assert (c.tables[slot, c._pages(length):] == -1).all()


@pytest.mark.parametrize("step", [1.0, 1.01, 1.3, 1.9])
def test_repeated_roundings_stay_within_two_and_a_half_scales(step):
    """One value requantized each time the page's scale grows: the bound that
    the rule of 1.25 gives, 0.5 s (1 + 1/1.25 + 1/1.25^2 + ...) = 2.5 s."""
    rng = np.random.default_rng(1)
    c = Cache(1, 1, 1, 16, 1, 1, 128)
    c.grow([0], [128])
    x = (rng.standard_normal((128, 1, 16)) * step ** np.arange(128)[:, None, None]).astype(np.float32)
    for t in range(128):
        c.append(0, x[t:t + 1], x[t:t + 1], [0], [t], [0, 1])
    err = np.abs(c.rows(0, 0, 128)[0] - x)
    assert err.max() <= 2.5001 * c.k_scale[0, 0, 0]


def test_page_that_starts_takes_the_plain_scale():
    x = np.linspace(-3, 3, 32, dtype=np.float32).reshape(2, 1, 16)
    c = Cache(1, 1, 1, 16, 1, 1, 16)
    c.grow([0], [2])
    c.append(0, x, x, [0], [0], [0, 2])
    assert c.k_scale[0, 0, 0] == np.float32(np.float64(np.float32(3)) / 127)
    assert np.abs(c.rows(0, 0, 2)[0] - x).max() <= 0.5001 * c.k_scale[0, 0, 0]
    assert c.k[0, 0, 0, 0, 0] == -127 and c.k[0, 0, 0, 1, 15] == 127


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def view(**over):
    """A cache whose pointers are never followed: the refusals come first."""
    import aion_b200 as A
    f = dict(k=4096, v=8192, k_scale=64, v_scale=128, tables=192, lens=256, refs=320, work=384, device=0, n_layers=2,
             n_pages=8, n_kv_heads=2, page_tokens=16, head_size=64, max_seqs=4, max_pages=4)
    f.update(over)
    return A.KV8(**f)


def append(kv, layer=0, k=1 << 20, v=1 << 21, type_=0, ks=128, vs=128, seqs=64, pos0=64, cu=None, n_seq=2, n_tok=2):
    import aion_b200 as A
    return A.lib().aion_kv8_append(ctypes.addressof(kv), layer, k, v, type_, ks, vs, seqs, pos0, cu, n_seq, n_tok, None)


def attention(kv, layer=0, q=1 << 20, out=1 << 22, type_=0, heads=4, qs=256, os_=256, scale=0.0, seqs=64, pos0=64,
              cu=None, n_seq=2, n_tok=2, ws=1 << 24, wsb=1 << 30):
    import aion_b200 as A
    return A.lib().aion_kv8_attention(ctypes.addressof(kv), layer, q, out, type_, heads, qs, os_, scale, seqs, pos0, cu,
                                      n_seq, n_tok, ws, wsb, None)


@pytest.mark.parametrize("over,status", [
    (dict(page_tokens=24), SHAPE), (dict(page_tokens=8), SHAPE), (dict(page_tokens=256), SHAPE),
    (dict(head_size=24), SHAPE), (dict(head_size=0), SHAPE), (dict(head_size=144), SHAPE),
    (dict(n_layers=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(n_pages=(1 << 24) + 1), SHAPE),
    (dict(n_kv_heads=0), SHAPE), (dict(max_seqs=4097), SHAPE), (dict(max_pages=0), SHAPE),
    (dict(max_pages=(1 << 26) + 1), SHAPE), (dict(k=None), ARG), (dict(work=None), ARG), (dict(k=4097), ARG),
    (dict(v=8200), ARG), (dict(refs=322), ARG)])
def test_cache_is_checked(built, over, status):
    import aion_b200 as A
    kv = view(**over)
    L, p = A.lib(), ctypes.addressof(kv)
    assert append(kv) == status
    assert attention(kv) == status
    assert L.aion_kv8_grow(p, 64, 64, 1, 64, None) == status
    assert L.aion_kv8_compact(p, None, None) == status
    assert L.aion_kv8_status(p, None) == status
    assert L.aion_last_error(None)


def test_null_cache(built):
    import aion_b200 as A
    L = A.lib()
    assert L.aion_kv8_append(None, 0, 64, 64, 0, 128, 128, 64, 64, None, 1, 1, None) == ARG
    assert L.aion_kv8_status(None, None) == ARG
    assert L.aion_kv8_attention_workspace(None, 4, 1, 1) == -1
    assert L.aion_kv8_create(None, None) == ARG
    assert L.aion_kv8_destroy(None) == 0


@pytest.mark.parametrize("over", [
    dict(layer=-1), dict(layer=2), dict(type_=3), dict(type_=-1), dict(k=None), dict(v=None), dict(seqs=None),
    dict(pos0=None), dict(n_seq=1), dict(n_seq=-1), dict(n_tok=-1, n_seq=-1), dict(n_seq=4097, n_tok=4097), dict(ks=127),
    dict(vs=0), dict(ks=-128), dict(k=(1 << 20) + 2), dict(type_=1, v=(1 << 21) + 1)])
def test_append_refuses(built, over):
    assert append(view(), **over) == ARG


@pytest.mark.parametrize("over,status", [
    (dict(heads=3), SHAPE), (dict(heads=0), SHAPE), (dict(layer=2), ARG), (dict(type_=9), ARG), (dict(q=None), ARG),
    (dict(out=None), ARG), (dict(qs=255), ARG), (dict(os_=1), ARG), (dict(scale=float("nan")), ARG),
    (dict(scale=float("inf")), ARG), (dict(out=1 << 20), ARG), (dict(out=(1 << 20) + 2044), ARG), (dict(n_seq=3), ARG),
    (dict(q=(1 << 20) + 1), ARG)])
def test_attention_refuses(built, over, status):
    assert attention(view(), **over) == status


def test_page_calls_refuse(built):
    import aion_b200 as A
    L, kv = A.lib(), view()
    p = ctypes.addressof(kv)
    assert L.aion_kv8_grow(p, 64, 64, 1025, 64, None) == ARG
    assert L.aion_kv8_grow(p, 64, 64, -1, 64, None) == ARG
    assert L.aion_kv8_grow(p, None, 64, 1, 64, None) == ARG
    assert L.aion_kv8_grow(p, 64, 64, 1, None, None) == ARG
    assert L.aion_kv8_fork(p, 64, None, None, 1, None) == ARG
    assert L.aion_kv8_trim(p, None, None, 1, None) == ARG


def test_empty_calls_do_nothing(built):
    """Nothing to do: no launch, so these pass without a GPU."""
    import aion_b200 as A
    L, kv = A.lib(), view()
    p = ctypes.addressof(kv)
    assert append(kv, k=None, v=None, seqs=None, pos0=None, n_seq=0, n_tok=0) == 0
    assert attention(kv, q=None, out=None, seqs=None, pos0=None, n_seq=0, n_tok=0) == 0
    assert L.aion_kv8_grow(p, None, None, 0, None, None) == 0
    assert L.aion_kv8_fork(p, None, None, None, 0, None) == 0
    assert L.aion_kv8_trim(p, None, None, 0, None) == 0


def test_one_workspace_serves_every_call(built):
    """Its size depends on the cache alone, and is 0 where a sequence holds no more than 1024 tokens."""
    import aion_b200 as A
    kv = view(page_tokens=64, max_pages=17)
    sizes = {A.lib().aion_kv8_attention_workspace(ctypes.addressof(kv), heads, n, rows)
             for heads in (4, 64) for n, rows in ((1, 1), (3, 3), (2, 900), (1, 1 << 20), (0, 0))}
    assert len(sizes) == 1 and sizes.pop() > 0
    kv = view(page_tokens=64, max_pages=16)
    assert A.lib().aion_kv8_attention_workspace(ctypes.addressof(kv), 4, 2, 2) == 0


@pytest.mark.parametrize("over,status", [
    (dict(n_layers=65535, n_pages=1 << 24, n_kv_heads=65535, page_tokens=128, head_size=128), SHAPE),   # 2^70 bytes
    (dict(n_layers=1 << 15, n_pages=1 << 24, n_kv_heads=1 << 13, page_tokens=32, head_size=128), SHAPE)])   # 2^64: 0 in 64 bits
def test_sizes_past_64_bits_are_refused(built, over, status):
    import aion_b200 as A
    kv, out = view(**over), A.KV8()
    assert A.lib().aion_kv8_create(ctypes.byref(kv), ctypes.byref(out)) == status
    assert not out.k and append(kv) == status
