"""What is measured of the 8-bit paged K/V cache: its append and read-out, the
attention that reads it, and the calls that share, grow, free and compact its
pages.

A cache holds, for each layer, pages of `page` tokens: int8 K and V values
[layer][page][kv head][token][head_size] and one fp32 scale per (layer, page,
kv head) for K and one for V.  tables[slot] lists a sequence's pages, lens its
tokens, refs counts the sequences that hold a page.

Definitions (fp32 arithmetic, but for x / s, which goes to the nearest integer of
the exact quotient, ties to even; x are the new rows of one page and head):

  append     need = max|x| / 127;  a page that starts with this call takes
             s = need, one that holds earlier rows keeps s where need <= s and
             else takes s' = max(need, 1.25 s), its earlier values becoming
             rint(q * (s / s'));  q = clamp(rint(x / s), -127, 127).
  read       x = q * s.
  attention  token i of a sequence stands at position pos0 + i and sees the
             positions up to its own:
             out = sum_j softmax_j(q . k_j / sqrt(head_size)) v_j.
  grow       makes room for n tokens behind a sequence's last one; the lowest
             free pages go out in list order; a last page that other
             sequences hold too and that is not full is copied first.
  fork       a slot takes over another's pages (one more holder each).
  trim       a sequence gives up its tokens from `keep` on.
  compact    with U pages in use, the i-th used page at or behind U moves to
             the i-th free page before U.

`run` makes one pass: the plain forms below, or the framework's calls.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _append(name, dtype, heads, hd, page, n, t_min, t_max, p_min, p_max, layers=1):
    return {"name": name, "kind": "append", "dtype": dtype, "heads": heads, "hd": hd, "page": page, "n": n,
            "t_min": t_min, "t_max": t_max, "p_min": p_min, "p_max": p_max, "layers": layers}


def _attn(name, dtype, q_heads, heads, hd, page, n, t_min, t_max, p_min, p_max, layers=1):
    return {"name": name, "kind": "attention", "dtype": dtype, "q_heads": q_heads, "heads": heads, "hd": hd,
            "page": page, "n": n, "t_min": t_min, "t_max": t_max, "p_min": p_min, "p_max": p_max, "layers": layers}


def _pages(name, kind, heads, hd, page, layers, n, t_min, t_max, grow, spare):
    return {"name": name, "kind": kind, "heads": heads, "hd": hd, "page": page, "layers": layers, "n": n,
            "t_min": t_min, "t_max": t_max, "grow": grow, "spare": spare}


def listed():
    """t: new tokens a sequence (spread from t_min to t_max over the batch), p: tokens it holds before."""
    return [
        # lock-step decode of 32 sequences at the 7B width, behind 512-token prompts
        _append("append_step_32x7b", "f32", 32, 128, 64, 32, 1, 1, 512, 639),
        # the prompts of that batch: 32 x 512 tokens in one call
        _append("append_prompt_32x512", "f32", 32, 128, 64, 32, 512, 512, 0, 0),
        # ragged chunks of prompts, grouped-query heads, half precision
        _append("append_chunks_bf16", "bf16", 8, 128, 32, 12, 37, 1531, 0, 999, layers=2),
        # one token against the tiny model's cache
        _attn("attn_step_tiny", "f32", 6, 6, 48, 16, 1, 1, 1, 201, 201, layers=6),
        # a lock-step decode step at the 7B width
        _attn("attn_step_32x7b", "f32", 32, 32, 128, 64, 32, 1, 1, 512, 639),
        # a serving batch with long, uneven contexts, grouped-query heads
        _attn("attn_step_16x32k", "bf16", 32, 8, 128, 64, 16, 1, 1, 8193, 32767),
        # one conversation with a very long context: few rows, one long axis
        _attn("attn_step_1x128k", "f16", 32, 8, 128, 128, 1, 1, 1, 131071, 131071),
        # a few drafted tokens a sequence checked at once, the 13B width
        _attn("attn_draft_8x5_13b", "f32", 40, 40, 128, 32, 8, 3, 5, 251, 1777),
        # prompts from their start, the 7B width
        _attn("attn_prompt_8x512_7b", "f32", 32, 32, 128, 64, 8, 512, 512, 0, 0),
        # later chunks of long prompts, grouped-query heads
        _attn("attn_chunk_2x2048", "bf16", 32, 8, 128, 64, 2, 1999, 2048, 4096, 6143),
        # each sequence branches, the branch grows a draft and is dropped
        _pages("pages_branch_64", "branch", 8, 128, 64, 8, 64, 65, 1500, 40, 256),
        # half of the sequences end, the cache is compacted, new ones come in
        _pages("pages_compact_7b", "compact", 32, 128, 64, 32, 16, 250, 512, 0, 8),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["append", "attention", "attention", "attention", "branch", "compact"])
    page = rng.choice([16, 32, 64, 128])
    hd = rng.choice([48, 64, 96, 128, 128])
    heads = rng.choice([1, 2, 4, 6, 8, 16, 32, 40])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "append":
        t_max = rng.choice([1, log(2, 2000)])
        n = log(1, max(1, min(256, 16384 // t_max, 16384 * 32 // (t_max * heads))))
        t_min = rng.randint(1, t_max)
        p_max = log(1, 4000)
        return _append("", dtype, heads, hd, page, n, t_min, t_max, rng.randint(0, p_max), p_max, rng.choice([1, 2]))
    if kind == "attention":
        group = rng.choice([1, 1, 2, 4, 5, 8])
        heads = min(heads, 8 if group > 1 else 40)
        if rng.random() < 0.6:   # a few tokens a sequence
            t_max = rng.choice([1, 1, 1, rng.randint(2, 6)])
            p_max = log(1, 100000)
            n = log(1, max(1, min(256, 16 * 20000 * 8 // (p_max * heads * t_max))))
            p_min = rng.randint(max(0, p_max // 8), p_max)
        else:
            t_max = log(16, 2048)
            p_max = rng.choice([0, log(1, 6000)])
            heads = min(heads, 32 // group if group > 1 else 32)
            n = log(1, max(1, min(32, 2 * 2048 * 7000 * 8 * 4 // (t_max * (t_max + p_max) * heads * group))))
            p_min = rng.randint(0, p_max)
        t_min = rng.randint(max(1, t_max // 2), t_max)
        return _attn("", dtype, heads * group, heads, hd, page, n, t_min, t_max, p_min, p_max, rng.choice([1, 2]))
    layers = rng.choice([1, 2, 8, 32])
    t_max = log(page, 2000)
    room = 1 << 30   # bytes of the pages that may move
    per_tok = 2 * layers * heads * hd
    n = 2 * log(1, max(1, min(64, room // (per_tok * (t_max + page)))))
    return _pages("", kind, heads, hd, page, layers, n, rng.randint(1, t_max), t_max, log(1, 100), rng.randint(0, 64))


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _tokens(case):
    """(new tokens, tokens held before) of each sequence; the two run against each other over the batch."""
    return _spread(case["t_min"], case["t_max"], case["n"]), _spread(case["p_min"], case["p_max"], case["n"])[::-1]


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------
# States
# ---------------------------------------------------------------------------
def _rows(gen, n, heads, hd, dtype):
    """K-like rows: unit variance, every sixteenth channel several times larger, as keys have them."""
    x = torch.randn(n, heads, hd, device="cuda", generator=gen)
    x[..., 5::16] *= 4.0
    return x.to(dtype)


def _pool(gen, shape):
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=gen, dtype=torch.float16).mul_(40).round_()
                   .clamp_(-127, 127))
    return out


def _cache(gen, rnd, case, lens, rooms, n_pages, fill=True):
    """Pages of `rooms` tokens for each slot, handed out in a shuffled order, as after some time of use."""
    layers, heads, hd, page = case["layers"], case["heads"], case["hd"], case["page"]
    max_pages = max(_ceil(r, page) for r in rooms) + 1
    order = list(range(n_pages))
    rnd.shuffle(order)
    tables = np.full((len(lens), max_pages), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    for i, r in enumerate(rooms):
        for j in range(_ceil(r, page)):
            p = order.pop()
            tables[i, j] = p
            refs[p] = 1
    shape = (layers, n_pages, heads, page, hd)
    make = _pool if fill else (lambda g, s: torch.zeros(s, dtype=torch.int8, device="cuda"))
    s = {"k": make(gen, shape), "v": make(gen, shape)}
    for name in ("k_scale", "v_scale"):
        s[name] = 0.02 * torch.exp(0.3 * torch.randn(layers, n_pages, heads, device="cuda", generator=gen))
    s["tables"] = torch.from_numpy(tables).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["refs"] = torch.from_numpy(refs).cuda()
    if own:   # the handle that a program keeps for its cache
        import aion_b200
        s["cache"] = aion_b200.KV8Cache.wrap(s["k"], s["v"], s["k_scale"], s["v_scale"], s["tables"], s["lens"],
                                             s["refs"])
    return s


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    kind, page = case["kind"], case["page"]
    if kind in ("append", "attention"):
        new, old = _tokens(case)
        n_tok = sum(new)
        rooms = [t + p for t, p in zip(new, old)]
        n_pages = sum(_ceil(r, page) for r in rooms) + 3
        s = _cache(gen, rnd, case, rooms, rooms, n_pages)
        s |= {"case": case, "layer": case["layers"] - 1, "pos0": _ints(old), "n_tok": n_tok, "t_max": max(new),
              "l_max": max(rooms), "seqs": torch.arange(case["n"], dtype=torch.int32, device="cuda")}
        s["cu"] = None if max(new) == 1 else _ints(np.concatenate([[0], np.cumsum(new)]))
        dt = DT[case["dtype"]]
        if kind == "append":
            s["new_k"] = _rows(gen, n_tok, case["heads"], case["hd"], dt)
            s["new_v"] = torch.randn(n_tok, case["heads"], case["hd"], device="cuda", generator=gen).to(dt)
        else:
            s["q"] = torch.randn(n_tok, case["q_heads"], case["hd"], device="cuda", generator=gen).to(dt)
        return s
    n, lens = case["n"], _spread(case["t_min"], case["t_max"], case["n"])
    if kind == "branch":   # slots 0..n-1 hold sequences, n..2n-1 are free
        n_pages = sum(_ceil(t, page) + 1 + _ceil(case["grow"], page) for t in lens) + case["spare"]
        s = _cache(gen, rnd, case, lens + [0] * n, [t + case["grow"] for t in lens] + [0] * n, n_pages)
        have = [_ceil(t, page) for t in lens]   # the rooms above only size the tables: keep the pages in use
        tables, refs = s["tables"], s["refs"]
        for i in range(n):
            extra = tables[i, have[i]:].clone()
            refs[extra[extra >= 0].long()] = 0
            tables[i, have[i]:] = -1
        s |= {"src": torch.arange(n, dtype=torch.int32, device="cuda"),
              "dst": torch.arange(n, 2 * n, dtype=torch.int32, device="cuda"), "n_new": _ints([case["grow"]] * n),
              "keep": _ints(lens), "zero": _ints([0] * n)}
    else:   # compact: even slots end first, odd ones next time
        n_pages = sum(_ceil(t, page) for t in lens) + case["spare"]
        s = _cache(gen, rnd, case, lens, lens, n_pages)
        half = [torch.arange(i, n, 2, dtype=torch.int32, device="cuda") for i in range(2)]
        s |= {"ends": half[0], "stays": half[1], "len": s["lens"].clone(), "zero": _ints([0] * ((n + 1) // 2))}
        s["n_ends"], s["n_stays"] = s["len"][0::2].contiguous(), s["len"][1::2].contiguous()
    s["case"] = case
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _places(s):
    """Sequence, position, page and row of each token of a call."""
    n_tok, page = s["n_tok"], s["case"]["page"]
    tok = torch.arange(n_tok, device="cuda")
    if s["cu"] is None:
        seq, off = tok, torch.zeros_like(tok)
    else:
        seq = torch.searchsorted(s["cu"][1:].long(), tok, right=True)
        off = tok - s["cu"].long()[seq]
    pos = s["pos0"].long()[seq] + off
    return seq, pos, s["tables"].long()[s["seqs"].long()[seq], pos // page], pos % page


def _append_one(s, pool, scales, x):
    page = s["case"]["page"]
    pool, scales, x = pool[s["layer"]], scales[s["layer"]], x.float()
    _, _, pages, rows = _places(s)
    heads = x.shape[1]
    amax = x.abs().amax(-1)
    top = torch.full((scales.shape[0], heads), -1.0, device="cuda")
    top.scatter_reduce_(0, pages[:, None].expand(-1, heads), amax, "amax")
    need = (top.double() / 127).float()   # the quotient rounded once: a product with 1 / 127 is not it
    # a sequence's first page may hold rows of earlier calls
    pos0 = s["pos0"].long()
    first = s["tables"].long()[s["seqs"].long(), pos0 // page]
    held = pos0 % page
    fresh = torch.ones(scales.shape[0], dtype=torch.bool, device="cuda")
    fresh[first] = held == 0
    grown = torch.where(need <= scales, scales, torch.maximum(need, scales * 1.25))
    new = torch.where(top < 0, scales, torch.where(fresh[:, None], need, grown))
    ratio = torch.where(new[first] > 0, scales[first] / new[first], torch.zeros_like(new[first]))
    old = pool[first]
    moved = torch.round(old.float() * ratio[:, :, None, None]).to(torch.int8)
    early = torch.arange(page, device="cuda")[None, :] < held[:, None]
    pool[first] = torch.where(early[:, None, :, None], moved, old)
    scales.copy_(new)
    sc = new[pages][:, :, None].double()   # in 64 bits: a quotient may lie next to the border of two values
    x = x.double()
    q = torch.where(sc > 0, torch.round(x / sc), torch.zeros_like(x)).clamp(-127, 127).to(torch.int8)
    pool[pages, :, rows] = q


def _read_one(s, pool, scales):
    _, _, pages, rows = _places(s)
    return pool[s["layer"]][pages, :, rows].float() * scales[s["layer"]][pages][:, :, None]


def _attention(s):
    case, q = s["case"], s["q"]
    n, heads, hd, page = case["n"], case["heads"], case["hd"], case["page"]
    group, t_max, l_max = case["q_heads"] // heads, s["t_max"], s["l_max"]
    at = torch.arange(l_max, device="cuda")
    pages = s["tables"].long()[s["seqs"].long()][:, at // page].clamp_min(0)           # [n][l]

    def held(pool, scales):
        x = pool[s["layer"]][pages, :, (at % page)[None, :]].float()                    # [n][l][heads][hd]
        return (x * scales[s["layer"]][pages][..., None]).transpose(1, 2)               # [n][heads][l][hd]

    tok = torch.arange(t_max, device="cuda")
    if s["cu"] is None:
        rows = torch.arange(n, device="cuda")[:, None]
        live = torch.ones(n, 1, dtype=torch.bool, device="cuda")
    else:
        cu = s["cu"].long()
        rows = (cu[:-1, None] + tok).clamp_max(s["n_tok"] - 1)
        live = tok < (cu[1:] - cu[:-1])[:, None]
    x = q.float()[rows].view(n, t_max, heads, group, hd).permute(0, 2, 3, 1, 4).reshape(n, heads, group * t_max, hd)
    score = x @ held(s["k"], s["k_scale"]).transpose(2, 3) * (1.0 / math.sqrt(hd))      # [n][heads][group t][l]
    limit = s["pos0"].long()[:, None] + tok                                              # the last position seen
    hidden = at[None, None, :] > limit[:, :, None]                                       # [n][t][l]
    score = score.view(n, heads, group, t_max, l_max).masked_fill_(hidden[:, None, None], float("-inf"))
    w = torch.exp(score - score.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).view(n, heads, group * t_max, l_max)
    o = (w @ held(s["v"], s["v_scale"])).view(n, heads, group, t_max, hd).permute(0, 3, 1, 2, 4)
    out = torch.empty(s["n_tok"] + 1, heads * group, hd, device="cuda", dtype=q.dtype)
    to = torch.where(live, rows, torch.full_like(rows, s["n_tok"]))
    out[to] = o.reshape(n, t_max, heads * group, hd).to(q.dtype)
    return out[:-1]


def _grow(s, seqs, n_new):
    page, tables, lens, refs = s["case"]["page"], s["tables"], s["lens"], s["refs"]
    seqs, n_new = seqs.long(), n_new.long()
    old, t = lens[seqs].long(), tables[seqs].long()
    have, want = (old + page - 1) // page, (old + n_new + page - 1) // page
    last = t.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0]
    copy = (n_new > 0) & (old % page > 0) & (refs[last.clamp_min(0)] > 1)
    need = want - have + copy
    upto = torch.cumsum(need, 0)
    free = torch.sort((refs > 0).int(), stable=True).indices
    ok = (upto <= (refs == 0).sum()) | (need == 0)
    col = torch.arange(t.shape[1], device="cuda")[None, :]
    is_new = ok[:, None] & (col >= have[:, None]) & (col < want[:, None])
    is_copy = (ok & copy)[:, None] & (col == have[:, None] - 1)
    rank = (upto - need)[:, None] + torch.where(is_copy, 0, copy[:, None] + col - have[:, None])
    t = torch.where(is_new | is_copy, free[rank.clamp(0, free.numel() - 1)], t)
    tables[seqs] = t.int()
    add = torch.zeros(refs.numel() + 1, dtype=torch.int32, device="cuda")
    add.index_add_(0, torch.where(is_new | is_copy, t, refs.numel()).flatten(),
                   torch.ones(t.numel(), dtype=torch.int32, device="cuda"))
    gone = torch.where(ok & copy, last, refs.numel())
    add.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    refs += add[:-1]
    dst = torch.where(ok & copy, t.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0], last)
    for name in ("k", "v", "k_scale", "v_scale"):
        s[name][:, dst] = s[name][:, last]
    lens[seqs] = torch.where(ok, old + n_new, old).int()
    return torch.where(ok, old, -1).int()


def _hold(s, t, used, by):
    """Adds `by` to the holders of the pages t[:, :used]."""
    refs = s["refs"]
    col = torch.arange(t.shape[1], device="cuda")[None, :]
    add = torch.zeros(refs.numel() + 1, dtype=torch.int32, device="cuda")
    add.index_add_(0, torch.where(used(col), t.long(), refs.numel()).flatten(),
                   torch.full((t.numel(),), by, dtype=torch.int32, device="cuda"))
    refs += add[:-1]


def _trim(s, seqs, keep):
    page, tables, lens = s["case"]["page"], s["tables"], s["lens"]
    seqs = seqs.long()
    old, t = lens[seqs], tables[seqs]
    keep = torch.minimum(old, keep)
    stay, have = ((keep + page - 1) // page)[:, None], ((old + page - 1) // page)[:, None]
    _hold(s, t, lambda col: (col >= stay) & (col < have), -1)
    col = torch.arange(t.shape[1], device="cuda")[None, :]
    tables[seqs] = torch.where((col >= stay) & (col < have), -1, t)
    lens[seqs] = keep


def _fork(s, src, dst, keep):
    page, tables, lens = s["case"]["page"], s["tables"], s["lens"]
    _trim(s, dst, torch.zeros_like(dst))
    src, dst = src.long(), dst.long()
    keep = torch.minimum(lens[src], keep)
    used = ((keep + page - 1) // page)[:, None]
    t = tables[src]
    _hold(s, t, lambda col: col < used, 1)
    col = torch.arange(t.shape[1], device="cuda")[None, :]
    tables[dst] = torch.where(col < used, t, tables[dst])
    lens[dst] = keep


def _compact(s):
    page, tables, lens, refs = s["case"]["page"], s["tables"], s["lens"], s["refs"]
    used = refs > 0
    n_used = int(used.sum())
    src = torch.nonzero(used[n_used:]).flatten() + n_used
    dst = torch.nonzero(~used[:n_used]).flatten()
    for name in ("k", "v", "k_scale", "v_scale"):
        s[name][:, dst] = s[name][:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    to = torch.arange(refs.numel(), device="cuda", dtype=torch.int32)
    to[src] = dst.int()
    col = torch.arange(tables.shape[1], device="cuda")[None, :]
    valid = col < ((lens + page - 1) // page)[:, None]
    tables.copy_(torch.where(valid, to[tables.long().clamp_min(0)], tables))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _held_pages(s):
    """The cache's whole state; its pages are moved as they are, so their bytes are compared, as words."""
    return {"tables": s["tables"], "lens": s["lens"], "refs": s["refs"], "k": s["k"].view(torch.int32),
            "v": s["v"].view(torch.int32), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def run(state):
    s = state
    kind = s["case"]["kind"]
    if kind == "append":   # the rows go into the cache and come back as it holds them
        if own:
            c = s["cache"]
            c.append(s["layer"], s["new_k"], s["new_v"], s["seqs"], s["pos0"], s["cu"])
            k, v = c.read(s["layer"], s["seqs"], s["pos0"], s["n_tok"], s["cu"])
        else:
            _append_one(s, s["k"], s["k_scale"], s["new_k"])
            _append_one(s, s["v"], s["v_scale"], s["new_v"])
            k, v = _read_one(s, s["k"], s["k_scale"]), _read_one(s, s["v"], s["v_scale"])
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "attention":
        if own:
            return s["cache"].attention(s["layer"], s["q"], s["seqs"], s["pos0"], s["cu"])
        return _attention(s)
    if kind == "branch":
        if own:
            c = s["cache"]
            c.fork(s["src"], s["dst"], s["keep"])
            pos0 = c.grow(s["dst"], s["n_new"])
            c.trim(s["dst"], s["zero"])
        else:
            _fork(s, s["src"], s["dst"], s["keep"])
            pos0 = _grow(s, s["dst"], s["n_new"])
            _trim(s, s["dst"], s["zero"])
        return {"pos0": pos0, **_held_pages(s)}
    if own:
        c = s["cache"]
        c.trim(s["ends"], s["zero"][:s["ends"].numel()])
        c.compact()
        pos0 = c.grow(s["ends"], s["n_ends"])
    else:
        _trim(s, s["ends"], s["zero"][:s["ends"].numel()])
        _compact(s)
        pos0 = _grow(s, s["ends"], s["n_ends"])
    s["ends"], s["stays"], s["n_ends"], s["n_stays"] = s["stays"], s["ends"], s["n_stays"], s["n_ends"]
    return {"pos0": pos0, **_held_pages(s)}


def work(case):
    kind, heads, hd, page = case["kind"], case["heads"], case["hd"], case["page"]
    if kind in ("append", "attention"):
        new, old = _tokens(case)
        size = 4 if case["dtype"] == "f32" else 2
        n_tok, tables = sum(new), 4 * sum(_ceil(t + p, page) for t, p in zip(new, old))
        if kind == "append":   # rows in, int8 out; int8 in, fp32 rows out; per value a division and a product
            values = 2 * n_tok * heads * hd
            scales = 8 * heads * sum(_ceil(p % page + t, page) for t, p in zip(new, old))
            return {"bytes": values * (size + 1 + 1 + 4) + 2 * scales + tables, "flops": 3 * values}
        qh = case["q_heads"]
        held = sum(t + p for t, p in zip(new, old))
        pages = sum(_ceil(t + p, page) for t, p in zip(new, old))
        seen = sum(t * p + t * (t + 1) // 2 for t, p in zip(new, old))
        return {"bytes": 2 * held * heads * hd + 8 * pages * heads + tables + 2 * n_tok * qh * hd * size,
                "flops": 4 * seen * qh * hd}
    lens = _spread(case["t_min"], case["t_max"], case["n"])
    pages = [_ceil(t, page) for t in lens]
    size = 2 * case["layers"] * heads * (page * hd + 4)
    if kind == "branch":
        copies = sum(1 for t in lens if t % page)
        made = sum(_ceil(t + case["grow"], page) - p for t, p in zip(lens, pages)) + copies
        return {"bytes": 2 * copies * size + 4 * (4 * sum(pages) + 4 * made), "flops": 0}
    half = min(sum(pages[0::2]), sum(pages[1::2]))   # pages of the half that stays, as far as they have to move
    return {"bytes": 2 * half * size + 4 * 4 * sum(pages), "flops": 0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] not in ("append", "attention"):
        return None
    s = prepare(case, seed)
    new, old = _tokens(case)
    page, layer = case["page"], s["layer"]
    tables = s["tables"].cpu().numpy()
    if case["kind"] == "append":
        out = {}
        for name in ("k", "v"):
            x, scales = s["new_" + name].double(), s[name + "_scale"].double()
            rows, at = torch.empty_like(x), 0
            for i, (t, p) in enumerate(zip(new, old)):
                done = 0
                while done < t:
                    pos = p + done
                    take = min(t - done, page - pos % page)
                    part, pg = x[at + done:at + done + take], int(tables[i, pos // page])
                    need, was = part.abs().amax((0, 2)) / 127, scales[layer, pg]
                    sc = need if pos % page == 0 else torch.where(need <= was, was, torch.maximum(need, 1.25 * was))
                    scales[layer, pg] = sc
                    # the scale is held in 32 bits, and its values are multiples of what is held
                    held = sc.float().double()[None, :, None]
                    rows[at + done:at + done + take] = torch.round(part / held).clamp(-127, 127) * held
                    done += take
                at += t
            out[name], out[name + "_scale"] = rows, scales
        return out
    heads, hd = case["heads"], case["hd"]
    group = case["q_heads"] // heads
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (t, p) in enumerate(zip(new, old)):
        pg = torch.from_numpy(tables[i, :_ceil(p + t, page)].astype(np.int64)).cuda()

        def held(pool, scales, h):
            return (pool[layer][pg, h].double() * scales[layer][pg, h].double()[:, None, None]).reshape(-1, hd)[:p + t]

        for h in range(heads):
            k, v = held(s["k"], s["k_scale"], h), held(s["v"], s["v_scale"], h)
            hidden = torch.arange(p + t, device="cuda")[None, :] > p + torch.arange(t, device="cuda")[:, None]
            for g in range(h * group, (h + 1) * group):
                score = s["q"][at:at + t, g].double() @ k.T / math.sqrt(hd)
                out[at:at + t, g] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
        at += t
    return out
