"""Serving operators: sliding-window attention for prompts, attention of one
new token over a paged key-value cache, and the pages' bookkeeping.

``run`` computes each operator either through this framework (``own`` true:
``kernels.window_attention`` and ``paged_cache.PagedCache``) or in a plain
form of elementary torch operations in 32 bits (``own`` false). Definitions:

* window attention: query i of a prompt sees key j when j <= i, j < kv_len[b]
  and (i - j < window or j < sinks); softmax over the visible keys of
  scale * q.k, times v; a row that sees no key is zero.
* decode attention: the new token of a sequence of len tokens (itself the
  last of them) sees key j when len - 1 - j < window or j < sinks; its own
  key and value are written into the cache first.
* store: len[slot] grows by counts[b] tokens, whose pages are the lowest
  free ones in order of b; token t of row b goes to position len - counts + t.
* pages: children share their parent's full pages and get a copy of its
  partial last page (the lowest free pages, in order); the pages of released
  sequences lose a reference; live pages at or above their own number move,
  lowest first, into the lowest free ones.

A cache is ``pages [layers, pages, 2 (k, v), kv_heads, page_size, head_dim]``
in fp16 with an int32 page table, lengths and reference counts.
"""

from __future__ import annotations

import math
import pathlib
import sys

import numpy as np
import torch

own = False

_PKG = str(pathlib.Path(__file__).resolve().parents[1] / "transformer-kernel_b200")


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import kernels
    import paged_cache

    return kernels, paged_cache


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a first answer's next token on the smallest stack (d 128, 4 heads): pure latency
        dict(name="decode_short", op="decode", seqs=1, heads=4, kv_heads=4, head_dim=32, page=16, lo=97, hi=97,
             window=0, sinks=0),
        # a batch of 256 sequences of up to 256 tokens, d 1024 and 16 heads
        dict(name="decode_batch", op="decode", seqs=256, heads=16, kv_heads=16, head_dim=64, page=16, lo=1, hi=257,
             window=0, sinks=0),
        # four answers over 100,000 tokens of context each: work split over the length
        dict(name="decode_long", op="decode", seqs=4, heads=16, kv_heads=16, head_dim=64, page=64, lo=99001,
             hi=100000, window=0, sinks=0),
        # shared key-value heads, ragged lengths, a window that starts inside a page and a few first tokens
        dict(name="decode_grouped_window", op="decode", seqs=64, heads=32, kv_heads=8, head_dim=128, page=32, lo=129,
             hi=8192, window=2000, sinks=4),
        # a short prompt on the smallest stack
        dict(name="window_short", op="window", batch=1, heads=4, kv_heads=4, seq=100, head_dim=32, window=32, sinks=4,
             padded=False),
        # a padded batch of prompts, d 512 and 8 heads
        dict(name="window_padded", op="window", batch=32, heads=8, kv_heads=8, seq=511, head_dim=64, window=128,
             sinks=4, padded=True),
        # one prompt of 100,000 tokens, d 1024 and 16 heads
        dict(name="window_long", op="window", batch=1, heads=16, kv_heads=16, seq=100000, head_dim=64, window=4096,
             sinks=64, padded=False),
        # shared key-value heads of 128 columns, an odd length
        dict(name="window_grouped", op="window", batch=4, heads=32, kv_heads=8, seq=8191, head_dim=128, window=1024,
             sinks=16, padded=False),
        # admitting one short prompt
        dict(name="store_short", op="store", seqs=1, kv_heads=4, head_dim=32, page=16, lo=77, hi=77),
        # admitting eight prompts of up to 8192 tokens
        dict(name="store_batch", op="store", seqs=8, kv_heads=16, head_dim=64, page=64, lo=2049, hi=8192),
        # one step of a small search: eight sequences forked, the parents dropped, the cache compacted
        dict(name="pages_small", op="pages", layers=4, seqs=8, kv_heads=4, head_dim=32, page=16, lo=20, hi=128,
             keep=0.5),
        # the same with 64 long sequences over four layers
        dict(name="pages_large", op="pages", layers=4, seqs=64, kv_heads=16, head_dim=64, page=32, lo=500, hi=2500,
             keep=0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "window", "window", "store", "pages"])
    hd = rng.choice([16, 32, 64, 64, 128, 128, 256]) if op != "pages" else rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "decode":
        heads = kv * rng.choice([1, 1, 2, 4, 8])
        seqs = _log(rng, 1, 256)
        # no more cached numbers than the long listed case
        most = int(4 * 100000 * 16 * 64 / (seqs * kv * hd))
        hi = _log(rng, 1, max(1, min(100000, most)))
        lo = rng.choice([1, hi, max(1, hi // 2)])
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        return dict(op="decode", seqs=seqs, heads=heads, kv_heads=kv, head_dim=hd, page=rng.choice([16, 32, 64, 128]),
                    lo=lo, hi=hi, window=window, sinks=rng.choice([0, 4, 17, 64]) if window else 0)
    if op == "window":
        heads = kv * rng.choice([1, 1, 2, 4])
        batch = _log(rng, 1, 32)
        window = _log(rng, 1, 4096)
        most = int(16 * 100000 * 64 / (batch * heads * hd))
        seq = max(1, min(most, _log(rng, 1, 100000)))
        return dict(op="window", batch=batch, heads=heads, kv_heads=kv, seq=seq, head_dim=hd, window=window,
                    sinks=rng.choice([0, 1, 4, 64, 130]), padded=rng.random() < 0.4)
    if op == "store":
        seqs = _log(rng, 1, 64)
        hi = max(1, min(8192, _log(rng, 1, 8 * 8192 * 1024 / (seqs * kv * hd))))
        return dict(op="store", seqs=seqs, kv_heads=kv, head_dim=hd, page=rng.choice([16, 32, 64, 128]),
                    lo=rng.choice([1, hi, max(1, hi // 2)]), hi=hi)
    layers, seqs, page = rng.randint(1, 4), _log(rng, 2, 64), rng.choice([16, 32, 64, 128])
    hi = _log(rng, 16, 64 * 2500 * 1024 * 4 / (seqs * kv * hd * layers) / 2 + 16)
    hi = min(hi, 8192)
    return dict(op="pages", layers=layers, seqs=seqs, kv_heads=kv, head_dim=hd, page=page, lo=max(1, hi // 3), hi=hi,
                keep=rng.choice([0.25, 0.5, 0.75]))


def _lengths(n, lo, hi):
    """n lengths spread over [lo, hi], the first one hi: a function of the case alone."""
    return [int(hi - (hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------
# the page layout of a case, by integer arithmetic on the host
# ---------------------------------------------------------------------------
def _scatter(num_pages):
    """A fixed order in which a case's sequences took their pages: neighbours
    of a sequence lie far apart in the pool, as after some time of serving."""
    step = max(1, int(num_pages * 0.6180339887))
    while math.gcd(step, num_pages) != 1:
        step += 1
    return (np.arange(num_pages, dtype=np.int64) * step) % num_pages


def _table(lens, page, num_pages, width, slots):
    table = np.full((slots, width), -1, dtype=np.int32)
    refs = np.zeros(num_pages, dtype=np.int32)
    order, at = _scatter(num_pages), 0
    for s, n in enumerate(lens):
        k = _ceil(n, page)
        table[s, :k] = order[at:at + k]
        refs[order[at:at + k]] = 1
        at += k
    return table, refs


def _pages_case(case):
    """(lengths, pages in the pool, table width, slots that are dropped)."""
    lens = _lengths(case["seqs"], case["lo"], case["hi"])
    used = sum(_ceil(n, case["page"]) for n in lens)
    kept = max(1, int(case["seqs"] * case["keep"]))
    # every parent is forked once, so at most one more page each; the pool is about half full
    return lens, 2 * used + case["seqs"], _ceil(case["hi"], case["page"]), list(range(kept, case["seqs"])), kept


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dev_int(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"decode": _prepare_decode, "window": _prepare_window, "store": _prepare_store,
            "pages": _prepare_pages}[case["op"]](case, seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)


def _cache(state, case, layers):
    """The framework's cache over the same pages, when it is what runs."""
    if not own:
        return
    _, paged_cache = _framework()
    pages, table, refs = state["pages"], state["table"], state["refs"]
    cache = paged_cache.PagedCache(
        num_layers=layers, num_pages=pages.shape[1], page_size=case["page"], kv_heads=case["kv_heads"],
        head_dim=case["head_dim"], max_seqs=table.shape[0], max_pages_per_seq=table.shape[1], pages=pages)
    cache.load(table, state["lens"], refs)
    state["cache"], state["saved"] = cache, cache.snapshot()


def _prepare_decode(case, seed):
    g = _gen(seed)
    H, K, hd, ps, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    lens = _lengths(n, case["lo"], case["hi"])
    width = _ceil(case["hi"], ps)
    num_pages = sum(_ceil(x, ps) for x in lens) + 1
    table, refs = _table(lens, ps, num_pages, width, n)
    # q, k and v of the new tokens are views of one fused projection
    qkv = _randn(g, n, (H + 2 * K) * hd)
    state = dict(case=case, host_lens=lens, pages=_randn(g, 1, num_pages, 2, K, ps, hd), table=_dev_int(table),
                 refs=_dev_int(refs), lens=_dev_int(lens),
                 q=qkv[:, :H * hd].view(n, H, hd), k=qkv[:, H * hd:(H + K) * hd].view(n, K, hd),
                 v=qkv[:, (H + K) * hd:].view(n, K, hd))
    _cache(state, case, 1)
    return state


def _prepare_window(case, seed):
    g = _gen(seed)
    B, H, K, S, hd = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["head_dim"]
    qkv = _randn(g, B, S, H + 2 * K, hd).permute(0, 2, 1, 3)
    kv_len = _dev_int(_lengths(B, max(1, S // 3), S)) if case["padded"] else None
    return dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + K], v=qkv[:, H + K:], kv_len=kv_len)


def _prepare_store(case, seed):
    g = _gen(seed)
    K, hd, ps, n = case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    lens = _lengths(n, case["lo"], case["hi"])
    width, S = _ceil(case["hi"], ps), max(lens)
    num_pages = sum(_ceil(x, ps) for x in lens) + 2
    # the projection of the padded prompts: this layer's keys and values lie behind its queries
    qkv = _randn(g, n, S, 3 * K, hd).permute(0, 2, 1, 3)
    # two pages of other sequences are in the way
    refs = np.zeros(num_pages, dtype=np.int32)
    refs[[0, num_pages // 2]] = 1
    state = dict(case=case, host_lens=lens, pages=_randn(g, 1, num_pages, 2, K, ps, hd),
                 table=torch.full((n, width), -1, dtype=torch.int32, device="cuda"), refs=_dev_int(refs),
                 lens=torch.zeros(n, dtype=torch.int32, device="cuda"), slots=_dev_int(np.arange(n)),
                 counts=_dev_int(lens), k=qkv[:, K:2 * K], v=qkv[:, 2 * K:])
    _cache(state, case, 1)
    return state


def _prepare_pages(case, seed):
    g = _gen(seed)
    lens, num_pages, width, dropped, kept = _pages_case(case)
    n, ps = case["seqs"], case["page"]
    table, refs = _table(lens, ps, num_pages, width, n + kept)
    # the sequences that stay are forked into the empty slots behind the others
    state = dict(case=case, pages=_randn(g, case["layers"], num_pages, 2, case["kv_heads"], ps, case["head_dim"]),
                 table=_dev_int(table), refs=_dev_int(refs), lens=_dev_int(lens + [0] * kept),
                 parents=_dev_int(np.arange(kept)), children=_dev_int(np.arange(n, n + kept)),
                 dropped=_dev_int(np.asarray(dropped, dtype=np.int32)))
    _cache(state, case, case["layers"])
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"decode": _own_decode, "window": _own_window, "store": _own_store,
                "pages": _own_pages}[case["op"]](state, case)
    return {"decode": _plain_decode, "window": _plain_window, "store": _plain_store,
            "pages": _plain_pages}[case["op"]](state, case)


def _own_decode(state, case):
    cache = state["cache"]
    out = cache.attend(0, state["q"], case["head_dim"] ** -0.5, k_new=state["k"], v_new=state["v"],
                       window=case["window"], sinks=case["sinks"])
    return {"out": out, "pages": cache.pages}


def _own_window(state, case):
    kernels, _ = _framework()
    return kernels.window_attention(state["q"], state["k"], state["v"], case["head_dim"] ** -0.5, case["window"],
                                    sinks=case["sinks"], kv_len=state["kv_len"])


def _own_books(cache):
    return {"pages": cache.pages, "table": cache.page_table, "lens": cache.seq_lens, "refs": cache.ref_counts}


def _own_store(state, case):
    cache = state["cache"]
    cache.restore(state["saved"])
    cache.reserve(state["slots"], state["counts"])
    cache.store(0, state["k"], state["v"], state["slots"], state["counts"])
    return _own_books(cache)


def _own_pages(state, case):
    cache = state["cache"]
    cache.restore(state["saved"])
    cache.fork(state["parents"], state["children"])
    cache.release(state["dropped"])
    live = cache.compact()
    return {**_own_books(cache), "live": live}


# -- plain forms --------------------------------------------------------------
def _softmax_times_v(scores, seen, v):
    """softmax over the last axis where ``seen``, times v; rows that see nothing are 0."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(state, case):
    H, K, hd, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pages, table, lens = state["pages"][0], state["table"], state["lens"].long()
    n = lens.shape[0]
    last = lens - 1
    at = table.gather(1, (last // ps)[:, None])[:, 0].long()
    pages[at, 0, :, last % ps] = state["k"]
    pages[at, 1, :, last % ps] = state["v"]
    q = state["q"].float().view(n, K, H // K, hd)
    out = torch.empty(n, K, H // K, hd, device=q.device)
    for b, length in enumerate(state["host_lens"]):
        kv = pages[table[b, :_ceil(length, ps)].long()]              # [n, 2, K, ps, hd]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, K, -1, hd)[:, :, :length].float()
        j = torch.arange(length, device=q.device)
        seen = torch.ones_like(j, dtype=torch.bool)
        if case["window"]:
            seen = (length - 1 - j < case["window"]) | (j < case["sinks"])
        scores = torch.matmul(q[b], kv[0].transpose(1, 2)) * hd ** -0.5
        out[b] = _softmax_times_v(scores, seen, kv[1])
    return {"out": out.view(n, H * hd).to(torch.float16), "pages": state["pages"]}


def _visible(i, j, window, sinks, kv_len):
    """[B or 1, 1, 1, len(i), len(j)]"""
    seen = (j[None, :] <= i[:, None]) & ((i[:, None] - j[None, :] < window) | (j[None, :] < sinks))
    seen = seen[None, None, None]
    if kv_len is not None:
        seen = seen & (j < kv_len.view(-1, 1, 1, 1, 1))
    return seen


def _window_blocks(rows, S, window, sinks, device):
    """(first query, end, indices of the keys that those queries may see), so
    few queries at a time that the scores of ``rows`` heads take about a GB"""
    size = min(1024, max(32, int(3e8 / (rows * min(S, window + 1024)))))
    for i0 in range(0, S, size):
        i1 = min(S, i0 + size)
        lo = max(0, i0 - window + 1)
        yield i0, i1, torch.cat([torch.arange(min(sinks, lo), device=device), torch.arange(lo, i1, device=device)])


def _window_form(state, case, dtype):
    B, H, K, S, hd = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["head_dim"]
    q = state["q"].reshape(B, K, H // K, S, hd)
    out = torch.empty(B, S, K, H // K, hd, device=q.device, dtype=dtype)
    for i0, i1, j in _window_blocks(B * H, S, case["window"], case["sinks"], q.device):
        k, v = state["k"][:, :, j].to(dtype)[:, :, None], state["v"][:, :, j].to(dtype)[:, :, None]
        i = torch.arange(i0, i1, device=q.device)
        scores = torch.matmul(q[:, :, :, i0:i1].to(dtype), k.transpose(-1, -2)) * hd ** -0.5
        seen = _visible(i, j, case["window"], case["sinks"], state["kv_len"])
        out[:, i0:i1] = _softmax_times_v(scores, seen, v).permute(0, 3, 1, 2, 4)
    return out.view(B, S, H * hd)


def _plain_window(state, case):
    return _window_form(state, case, torch.float32).to(torch.float16)


def _plain_reserve(table, lens, refs, slots, counts, ps):
    """Longer sequences and the lowest free pages for them, in order."""
    have, new = (lens[slots] + ps - 1) // ps, lens[slots] + counts
    need = (new + ps - 1) // ps - have
    free = torch.nonzero(refs == 0)[:, 0]
    first = torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    k = col - have[:, None]
    wanted = (k >= 0) & (k < need[:, None])
    page = free[torch.where(wanted, first[:, None] + k, torch.zeros_like(k))]
    table[slots] = torch.where(wanted, page.to(torch.int32), table[slots])
    refs[page[wanted]] = 1
    lens[slots] = new.to(torch.int32)


def _plain_store(state, case):
    ps = case["page"]
    pages, table, lens, refs = state["pages"], state["table"].clone(), state["lens"].clone(), state["refs"].clone()
    slots, counts = state["slots"].long(), state["counts"].long()
    _plain_reserve(table, lens, refs, slots, counts, ps)
    t = torch.arange(state["k"].shape[2], device=table.device)
    pos = (lens[slots] - counts)[:, None] + t[None, :]
    b, t = torch.nonzero(t[None, :] < counts[:, None], as_tuple=True)
    pos = pos[b, t]
    at = table[slots[b], pos // ps].long()
    pages[0][at, 0, :, pos % ps] = state["k"][b, :, t]
    pages[0][at, 1, :, pos % ps] = state["v"][b, :, t]
    return {"pages": pages, "table": table, "lens": lens, "refs": refs}


def _plain_pages(state, case):
    ps = case["page"]
    pages, table, lens, refs = state["pages"], state["table"].clone(), state["lens"].clone(), state["refs"].clone()
    parents, children, dropped = state["parents"].long(), state["children"].long(), state["dropped"].long()
    num_pages = refs.shape[0]
    # fork: the full pages are shared, the partial last one is copied as far as it is used
    n = lens[parents].long()
    rows = table[parents]
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    shared = col < (n // ps)[:, None]
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    partial = n % ps != 0
    free = torch.nonzero(refs == 0)[:, 0]
    rank = torch.cumsum(partial.long(), 0) - 1
    fresh = free[torch.where(partial, rank, torch.zeros_like(rank))]
    refs[fresh[partial]] = 1
    is_last = (col == (n // ps)[:, None]) & partial[:, None]
    old = rows[is_last].long()
    table[children] = torch.where(is_last, fresh[:, None].to(torch.int32), rows)
    lens[children] = lens[parents]
    used = (torch.arange(ps, device=table.device)[None, :] < (n % ps)[partial][:, None])[None, :, None, None, :, None]
    pages[:, fresh[partial]] = torch.where(used, pages[:, old], pages[:, fresh[partial]])
    # release
    gone = table[dropped]
    held = gone[gone >= 0]
    refs.index_add_(0, held.long(), torch.full_like(held, -1))
    table[dropped] = -1
    lens[dropped] = 0
    # compact
    live = refs > 0
    count = live.sum()
    ids = torch.arange(num_pages, device=table.device)
    src, dst = ids[live & (ids >= count)], ids[~live & (ids < count)]
    pages[:, dst] = pages[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    moved = ids.to(torch.int32)
    moved[src] = dst.to(torch.int32)
    table = torch.where(table >= 0, moved[table.clamp(min=0).long()], table)
    return {"pages": pages, "table": table, "lens": lens, "refs": refs, "live": count.to(torch.int32)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op, hd, K = case["op"], case["head_dim"], case["kv_heads"]
    if op == "decode":
        H, w = case["heads"], case["window"]
        seen = [n if not w else min(n, w) + min(case["sinks"], max(0, n - w))
                for n in _lengths(case["seqs"], case["lo"], case["hi"])]
        total, n = sum(seen), case["seqs"]
        # cached keys and values (the new token's come from the projection and go to the cache), q, out
        moved = 2 * (total - n) * K * hd + 2 * 2 * n * K * hd + 2 * n * H * hd
        return {"bytes": 2 * moved, "flops": 4 * total * H * hd}
    if op == "window":
        B, H, S, w, s = case["batch"], case["heads"], case["seq"], case["window"], case["sinks"]
        i = np.arange(S, dtype=np.int64)
        lo = np.maximum(0, i - w + 1)
        lens = _lengths(B, max(1, S // 3), S) if case["padded"] else [S] * B
        pairs = 0
        for n in lens:
            # the band [lo, i] and the first tokens before it, both cut at n
            pairs += int((np.maximum(0, np.minimum(i + 1, n) - lo) + np.minimum(np.minimum(s, lo), n)).sum())
        return {"bytes": 2 * (2 * B * S * H * hd + 2 * sum(lens) * K * hd), "flops": 4 * pairs * H * hd}
    if op == "store":
        tokens = sum(_lengths(case["seqs"], case["lo"], case["hi"]))
        return {"bytes": 2 * 2 * 2 * tokens * K * hd, "flops": 0}
    lens, num_pages, width, dropped, kept = _pages_case(case)
    ps, row = case["page"], 2 * 2 * K * hd * case["layers"]
    table, refs = _table(lens, ps, num_pages, width, case["seqs"])
    copied = 0
    for s in range(kept):
        k, part = lens[s] // ps, lens[s] % ps
        refs[table[s, :k]] += 1
        if part:
            refs[np.flatnonzero(refs == 0)[0]] = 1
            copied += part
    for s in dropped:
        refs[table[s, :_ceil(lens[s], ps)]] -= 1
    count = int((refs > 0).sum())
    copied += ps * int((refs[count:] > 0).sum())
    return {"bytes": 2 * copied * row + 4 * (2 * num_pages + 2 * (case["seqs"] + kept) * width), "flops": 0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """What ``run`` returns, straight from the definitions: one sequence or
    one head at a time, the visible keys picked out by index. Counts and
    tables are whole numbers and have no such value."""
    state = prepare(case, seed)
    hd, K = case["head_dim"], case["kv_heads"]
    if case["op"] == "decode":
        G, ps, outs = case["heads"] // K, case["page"], []
        for b, n in enumerate(state["host_lens"]):
            first = max(0, n - case["window"]) if case["window"] else 0
            j = torch.cat([torch.arange(min(case["sinks"], first)), torch.arange(first, n - 1)]).cuda()
            at, slot = state["table"][b, j // ps].long(), j % ps
            heads = []
            for h in range(K):
                k = torch.cat([state["pages"][0, at, 0, h, slot], state["k"][b, h][None]]).double()
                v = torch.cat([state["pages"][0, at, 1, h, slot], state["v"][b, h][None]]).double()
                x = state["q"][b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(hd)
                w = (x - torch.logsumexp(x, 1, keepdim=True)).exp()
                heads.append(w @ v)
            outs.append(torch.cat(heads).reshape(-1))
        return {"out": torch.stack(outs), "pages": None}
    if case["op"] == "window":
        B, H, S, w, s = case["batch"], case["heads"], case["seq"], case["window"], case["sinks"]
        if B * H * S * (min(w, S) + 1024) > 3e10:
            return None
        out = torch.zeros(B, S, H, hd, device="cuda", dtype=torch.float64)
        size = 2048
        for b in range(B):
            n = S if state["kv_len"] is None else int(state["kv_len"][b])
            for i0 in range(0, S, size):
                i = torch.arange(i0, min(S, i0 + size), device="cuda")[:, None]
                first = min(n, max(0, i0 - w + 1))
                j = torch.cat([torch.arange(min(s, first)), torch.arange(first, min(n, i0 + size))]).cuda()
                if j.numel() == 0:
                    continue
                hidden = (j > i) | ((j <= i - w) & (j >= s))
                empty = hidden.all(1, keepdim=True)
                for h in range(H):
                    x = state["q"][b, h, i[:, 0]].double() @ state["k"][b, h // (H // K), j].double().T / math.sqrt(hd)
                    x = x.masked_fill(hidden & ~empty, -math.inf)
                    y = torch.softmax(x, 1) @ state["v"][b, h // (H // K), j].double()
                    out[b, i[:, 0], h] = y.masked_fill(empty, 0.0)
        return out.view(B, S, H * hd)
    pages, books = state["pages"].double(), dict(table=None, lens=None, refs=None)
    table, refs = state["table"].cpu().numpy().copy(), state["refs"].cpu().numpy().copy()
    ps = case["page"]
    if case["op"] == "store":
        free = iter(np.flatnonzero(refs == 0).tolist())
        for b, n in enumerate(state["host_lens"]):
            for t in range(0, n, ps):
                page, end = next(free), min(n, t + ps)
                pages[0, page, 0, :, :end - t] = state["k"][b, :, t:end].double()
                pages[0, page, 1, :, :end - t] = state["v"][b, :, t:end].double()
        return {"pages": pages, **books}
    lens, _, _, dropped, kept = _pages_case(case)
    holders, fresh = {}, -1
    for s in range(case["seqs"]):
        for page in table[s][table[s] >= 0].tolist():
            holders[page] = s
    for s in range(kept):
        part, k = lens[s] % ps, lens[s] // ps
        if part:
            fresh = next(p for p in range(fresh + 1, refs.size) if p not in holders)
            holders[fresh] = s
            pages[:, fresh, :, :, :part] = pages[:, int(table[s, k]), :, :, :part]
    live = sorted(p for p, s in holders.items() if s not in dropped)
    taken = set(live)
    holes = [p for p in range(len(live)) if p not in taken]
    for src, dst in zip([p for p in live if p >= len(live)], holes):
        pages[:, dst] = pages[:, src]
    return {"pages": pages, **books, "live": None}
