"""New tokens against the 8-bit paged cache at model level (aion_extend).

The tiny model is restated here in 64 bits from the checkpoint's bytes.  Its
attention reads the K and V values that the library's cache holds after the
call (through oracle/kv8_ref.py), so what is compared is everything but the
rounding to 8 bits; logits agree to 1e-3 of the largest, as for aion_prefill,
whose products these are (about 2^-16 each).  The rounding is checked apart:
every new row is held within half a scale of the restatement's own K and V
row, plus 1e-3 of the page's largest value
for those products.  (Quantizing on both sides instead would let two values
next to a border go apart by a step, and the steps of one layer move the next.)
"""
from __future__ import annotations

import numpy as np
import pytest

import cases
from oracle.kv8_ref import Cache

pytestmark = pytest.mark.gpu
REL = 1e-3


class PlainModel:
    """transformer() (src/kernel_simd.c:1014) over dequantized weights with the cache of oracle/kv8_ref.py."""

    def __init__(self, path):
        raw = path.read_bytes()
        self.dim, self.hid, self.L, self.nh, self.nkv, self.vocab, self.seq = np.frombuffer(raw, np.int32, 7)
        self.hs = self.dim // self.nh
        kv = self.nkv * self.hs
        at = [28]

        def floats(*shape):
            n = int(np.prod(shape))
            x = np.frombuffer(raw, np.float32, n, at[0]).reshape(shape)
            at[0] += 4 * n
            return x.astype(np.float64)

        def quant(*shape):
            n = int(np.prod(shape))
            sc = np.frombuffer(raw, np.float32, n // 32, at[0]).astype(np.float64)
            b = np.frombuffer(raw, np.uint8, n // 2, at[0] + 4 * (n // 32))
            at[0] += 4 * (n // 32) + n // 2
            q = np.stack([(b & 15).astype(np.int32) - 8, (b >> 4).astype(np.int32) - 8], 1).reshape(-1, 32)
            return (q * sc[:, None]).reshape(shape)

        L, d, h = self.L, self.dim, self.hid
        self.emb = quant(self.vocab, d)
        self.rms_att = floats(L, d)
        self.wq, self.wk, self.wv, self.wo = quant(L, d, d), quant(L, kv, d), quant(L, kv, d), quant(L, d, d)
        self.rms_ffn = floats(L, d)
        self.w1, self.w2, self.w3 = quant(L, h, d), quant(L, d, h), quant(L, h, d)
        self.rms_final = floats(d)
        self.re, self.im = floats(self.seq, self.hs // 2), floats(self.seq, self.hs // 2)

    @staticmethod
    def norm(x, w):
        return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * w

    def rope(self, x, pos):
        y = x.reshape(len(x), -1, self.hs // 2, 2)
        re, im = self.re[pos][:, None, :], self.im[pos][:, None, :]
        return np.stack([y[..., 0] * re - y[..., 1] * im, y[..., 0] * im + y[..., 1] * re], -1).reshape(len(x), -1, self.hs)

    def extend(self, cache, lib, seqs, tokens):
        """The logits of the call that the library's cache `lib` has just seen."""
        n = [len(t) for t in tokens]
        pos0 = cache.grow(seqs, n)   # copies shared pages, so it comes before the values are taken over
        for name in ("k", "v", "k_scale", "v_scale"):
            getattr(cache, name)[:] = getattr(lib, name).cpu().numpy()
        assert -1 not in pos0
        cu = [0] + np.cumsum(n).tolist()
        pos = np.concatenate([p + np.arange(k) for p, k in zip(pos0, n)])
        x = self.emb[np.concatenate(tokens)]
        for l in range(self.L):
            a = self.norm(x, self.rms_att[l])
            q, k = self.rope(a @ self.wq[l].T, pos), self.rope(a @ self.wk[l].T, pos)
            v = (a @ self.wv[l].T).reshape(len(x), -1, self.hs)
            for i, slot in enumerate(seqs):
                held = cache.rows(l, slot, pos0[i] + n[i])
                page = cache.tables[slot, np.arange(pos0[i], pos0[i] + n[i]) // cache.page]
                for got, want, sc in zip(held, (k, v), (cache.k_scale, cache.v_scale)):
                    one = sc[l][page][:, :, None]   # a scale; the page's largest value is 127 of it
                    err = np.abs(got[pos0[i]:] - want[cu[i]:cu[i + 1]])
                    assert (err <= (0.5 + 0.127) * one).all(), (err / one).max()
            x = x + cache.attention(l, q, seqs, pos0, cu)[0].reshape(len(x), -1) @ self.wo[l].T
            a = self.norm(x, self.rms_ffn[l])
            g = a @ self.w1[l].T
            x = x + (g / (1 + np.exp(-g)) * (a @ self.w3[l].T)) @ self.w2[l].T
        last = x[np.array(cu[1:]) - 1]
        return self.norm(last, self.rms_final) @ self.emb.T


def check(got, want):
    rel = np.abs(got - want).max(1) / np.abs(want).max(1)
    assert rel.max() <= REL, rel


@pytest.fixture(scope="module")
def plain(tiny_path):
    return PlainModel(tiny_path)


def pair(A, model, page, n_pages, slots=6, per_slot=16):
    c = model.config
    return (A.KV8Cache(c.n_layers, n_pages, c.n_kv_heads, c.head_size, slots, per_slot, page),
            Cache(c.n_layers, n_pages, c.n_kv_heads, c.head_size, slots, per_slot, page))


@pytest.mark.parametrize("page", [16, 32])
def test_serving_run(cuda, tiny_path, plain, golden_tiny, page):
    """Prompts of different lengths, a chunk and single tokens together, a
    shared prefix, a draft taken back, a sequence that ends, a compaction."""
    import aion_b200 as A
    base = np.array(golden_tiny["w4a16_tokens"], np.int32)
    with A.Model(tiny_path) as m:
        c, r = pair(A, m, page, 40)

        def ints(v):
            return cuda.tensor(v, dtype=cuda.int32, device="cuda")

        def step(seqs, tokens):
            check(m.extend(c, seqs, tokens), plain.extend(r, c, seqs, tokens))
            for name in ("tables", "lens", "refs"):
                assert np.array_equal(getattr(c, name).cpu().numpy(), getattr(r, name)), name

        step([0, 1], [base[:50], base[60:79]])
        step([1, 0], [base[79:110], base[50:51]])
        c.fork(ints([0]), ints([2]), ints([40]))
        r.fork([0], [2], [40])
        step([2, 0, 1], [base[100:103], base[51:52], base[110:111]])
        step([0, 1, 2], [base[52:57], base[111:116], base[103:108]])   # drafts
        c.trim(ints([0, 2]), ints([53, 44]))
        r.trim([0, 2], [53, 44])
        step([0, 1, 2], [base[:1], base[1:2], base[2:3]])
        c.trim(ints([0]))
        r.trim([0])
        c.compact()
        r.compact()
        step([3, 2, 1], [base[120:155], base[3:4], base[4:5]])


def test_one_prompt_against_the_fp32_prefill(cuda, tiny_path, golden_tiny):
    """The logits are the fp32 prefill's but for what 8 bits leave out: K and V
    off by 0.3 / 127 of a page's largest value in the mean, about 1 % of a
    typical one, so a tenth of the largest logit is far off."""
    import aion_b200 as A
    prompt = np.array(golden_tiny["w4a16_tokens"][:32], np.int32)
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 8)
        got = m.extend(c, [4], [prompt])
        full = m.prefill(prompt)
        assert np.abs(got - full).max() <= 0.1 * np.abs(full).max()
        assert m.extend(c, [4], [[int(got.argmax())]], want_logits=False) is None
        assert c.lens.tolist()[4] == 33


def test_refusals_leave_the_slots_as_they_were(cuda, tiny_path):
    import aion_b200 as A
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 4)
        m.extend(c, [0], [[1] * 20])
        before = c.tables.clone(), c.lens.clone(), c.refs.clone()

        def code(seqs, tokens, cache=c):
            with pytest.raises(A.AionError) as e:
                m.extend(cache, seqs, tokens)
            for a, b in zip(before, (c.tables, c.lens, c.refs)):
                assert cuda.equal(a, b)
            return e.value.code

        assert code([1, 0], [[1] * 16, [1] * 40]) == "OOM"
        assert code([0, 0], [[1], [1]]) == "ARG"
        assert code([6], [[1]]) == "ARG"
        assert code([1], [[]]) == "ARG"
        assert code([1], [[32000]]) == "ARG"
        assert code([1], [[1]], A.KV8Cache(5, 4, 6, 48, 2, 2, 16)) == "SHAPE"
        wide = A.KV8Cache(6, 40, 6, 48, 2, 40, 16)
        with pytest.raises(A.AionError) as e:
            m.extend(wide, [0], [[1] * 257])
        assert e.value.code == "ARG" and wide.lens.sum().item() == 0 and wide.refs.sum().item() == 0
        m.extend(c, [0], [[1]])
        c.status()


def test_extend_refuses_a_tensor_parallel_or_fp32_context(cuda, tiny_f32_path):
    import aion_b200 as A
    with A.Model(tiny_f32_path) as m:
        with pytest.raises(A.AionError) as e:
            m.extend(pair(A, m, 16, 4)[0], [0], [[1]])
        assert e.value.code == "STATE"


def test_extend_returns_what_earlier_calls_left_to_report(cuda, tiny_path):
    import aion_b200 as A
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 4)
        c.grow(cuda.tensor([0], dtype=cuda.int32, device="cuda"), cuda.tensor([65], dtype=cuda.int32, device="cuda"))
        cuda.cuda.synchronize()
        with pytest.raises(A.AionError) as e:
            m.extend(c, [1], [[1, 2]])
        assert e.value.code == "OOM" and c.lens.sum().item() == 0 and c.refs.sum().item() == 0
        m.extend(c, [1], [[1, 2]])
        assert c.lens[1].item() == 2
        c.status()


def test_a_failure_behind_the_growth_is_undone(cuda, tiny_path):
    """A damaged count of holders: slot 0's last page is not its alone to the append.
    Slot 1, which has grown in the same call, gives its page back."""
    import aion_b200 as A
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 8)
        m.extend(c, [1], [[1] * 20])
        m.extend(c, [0], [[1] * 20])
        c.trim(cuda.tensor([1], dtype=cuda.int32, device="cuda"))
        last = c.tables[0, 1].item()
        c.refs[last] = 0
        cuda.cuda.synchronize()
        before = c.tables.clone(), c.lens.clone(), c.refs.clone()
        with pytest.raises(A.AionError) as e:
            m.extend(c, [1, 0], [[1] * 16, [1]])
        assert e.value.code == "STATE" and "page" in str(e.value)
        for a, b in zip(before, (c.tables, c.lens, c.refs)):
            assert cuda.equal(a, b)
        c.status()
        c.refs[last] = 1
        cuda.cuda.synchronize()
        m.extend(c, [1, 0], [[1] * 16, [1]])
        assert c.lens.tolist()[:2] == [21, 16]


def test_extend_reports_a_wait_that_gave_up_before_it_grows(cuda, tiny_path):
    import aion_b200 as A
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 4)
        c.work[0] = 8   # as an attention call before it would have left it
        cuda.cuda.synchronize()
        with pytest.raises(A.AionError) as e:
            m.extend(c, [1], [[1, 2]])
        assert e.value.code == "TIMEOUT" and c.lens.sum().item() == 0 and c.refs.sum().item() == 0
        m.extend(c, [1], [[1, 2]])
        assert c.lens[1].item() == 2


def test_extend_without_device_memory_for_its_rows(cuda, tiny_path):
    """2^24 tokens: their operands pass the device's memory.  The next call does not see that error."""
    import aion_b200 as A
    with A.Model(tiny_path) as m:
        c, _ = pair(A, m, 16, 4)
        many = np.ones(1 << 24, np.int32)
        with pytest.raises(A.AionError) as e:
            m.extend(c, [0], [many])
        assert e.value.code == "OOM" and c.lens.sum().item() == 0
        m.extend(c, [0], [[1] * 20])
        assert c.lens[0].item() == 20
        c.status()
