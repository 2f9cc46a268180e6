"""The 8-bit paged K/V cache on the GPU at the edges of what its calls allow."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_kv8 import Pair

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
