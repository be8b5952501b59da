"""Paged key-value cache: the books against a model in plain Python, the data
against row-by-row copies, decode attention against its definition in 64 bits,
and what is refused.

Decode tolerance, per output element, for weights p_j = exp(s_j - max) and
A = sum p_j |v_j| / sum p_j: rounding each p_j to fp16 costs half a step,
2^-11 p_j (2^-25 below fp16's normal range); the fp32 scores are off by at most
(hd + 2) 2^-24 sum |q_i k_i| scale each, which moves numerator and denominator
by twice that; 2^x and the merge of the parts add a few 2^-22; the output is
rounded to fp16, 2^-11 |out| (2^-25 below its normal range)."""

from __future__ import annotations

import math

import pytest
import torch

import _tklib as tk
import paged_cache
from paged_cache import PagedCache

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# a model of the books
# ---------------------------------------------------------------------------
class Model:
    """What the calls do, one entry after the other."""

    def __init__(self, num_pages, page_size, max_seqs, width):
        self.ps, self.width = page_size, width
        self.seqs = [[] for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.refs = [0] * num_pages

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, counts):
        for s, c in zip(slots, counts):
            if s == -1:
                continue
            self.lens[s] += c
            while len(self.seqs[s]) * self.ps < self.lens[s]:
                self.seqs[s].append(self.take())

    def fork(self, parents, children):
        copies = []
        for p, c in zip(parents, children):
            if p == -1 or c == -1:
                continue
            full = self.lens[p] // self.ps
            pages = self.seqs[p][:full]
            if self.lens[p] % self.ps:
                pages = pages + [self.take()]
                copies.append((self.seqs[p][full], pages[-1], self.lens[p] % self.ps))
            self.seqs[c], self.lens[c] = list(pages), self.lens[p]
        for p, c in zip(parents, children):
            if p != -1 and c != -1:
                for page in self.seqs[c][:self.lens[c] // self.ps]:
                    self.refs[page] += 1
        return copies

    def release(self, slots):
        for s in slots:
            if s == -1:
                continue
            for page in self.seqs[s]:
                self.refs[page] -= 1
            self.seqs[s], self.lens[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        for s, d in zip(src, dst):
            self.refs[d], self.refs[s] = self.refs[s], 0
        new = dict(zip(src, dst))
        self.seqs = [[new.get(p, p) for p in pages] for pages in self.seqs]
        return live, list(zip(src, dst))

    def table(self):
        return [pages + [-1] * (self.width - len(pages)) for pages in self.seqs]


def same_books(cache, model):
    n = [-(-x // model.ps) for x in model.lens]
    table = cache.page_table.tolist()
    assert cache.seq_lens.tolist() == model.lens
    for s, pages in enumerate(model.table()):
        assert table[s][:n[s]] == pages[:n[s]], f"slot {s}"
    assert cache.ref_counts.tolist() == model.refs


def make(num_pages=64, page_size=16, max_seqs=8, width=12, layers=2, kv_heads=2, head_dim=32, **kw):
    cache = PagedCache(num_layers=layers, num_pages=num_pages, page_size=page_size, kv_heads=kv_heads,
                       head_dim=head_dim, max_seqs=max_seqs, max_pages_per_seq=width, **kw)
    return cache, Model(num_pages, page_size, max_seqs, width)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# refusals that need no device
# ---------------------------------------------------------------------------
def test_status_names_every_bit_of_the_header():
    assert sorted(paged_cache.STATUS) == [1, 2, 4, 8, 16, 32]


@pytest.mark.parametrize("change, error", [
    (dict(page_size=24), tk.TKError), (dict(page_size=8), tk.TKError), (dict(page_size=512), tk.TKError),
    (dict(head_dim=96), tk.TKError), (dict(num_pages=0), ValueError), (dict(max_seqs=8193), ValueError),
    (dict(num_pages=(1 << 20) + 1), ValueError), (dict(max_pages_per_seq=0), ValueError),
    (dict(device="cpu"), tk.TKError), (dict(pages=torch.zeros(1)), tk.TKError)])
def test_cache_refuses_on_host(change, error):
    sizes = dict(num_layers=1, num_pages=4, page_size=16, kv_heads=1, head_dim=32, max_seqs=2, max_pages_per_seq=2)
    with pytest.raises(error):
        PagedCache(**{**sizes, **change})


def c_cache(**change):
    fields = dict(page_table=16, seq_lens=16, ref_counts=16, free_mask=16, status=16, live=16, scratch=16, pool=16,
                  max_seqs=8, table_width=4, num_pages=32, page_size=16, layers=2, kv_heads=2, hd=64)
    return tk.Cache(**{**fields, **change})


def test_c_entries_refuse_on_host():
    """Refused before any device call, so this needs no GPU."""
    lib = tk.lib()
    ok = c_cache()
    for bad, status in ((c_cache(pool=None), -1), (c_cache(page_size=48), -2), (c_cache(hd=96), -2),
                        (c_cache(max_seqs=0), -1), (c_cache(num_pages=1 << 21), -1), (c_cache(free_mask=4), -1)):
        assert lib.tk_cache_reserve(bad, 16, 16, 1, 0, None) == status
        assert lib.tk_cache_compact(bad, None) == status
        assert lib.tk_last_error() != b""
    assert lib.tk_cache_reserve(ok, 16, 16, 8193, 0, None) == -1
    assert lib.tk_cache_reserve(ok, None, 16, 1, 0, None) == -1
    assert lib.tk_cache_reserve(ok, None, None, 0, 0, None) == 0   # nothing to do
    assert lib.tk_cache_fork(ok, 16, None, 1, None) == -1
    assert lib.tk_cache_release(ok, None, 1, None) == -1
    # store: layer, strides, alignment, null
    assert lib.tk_cache_store(ok, 2, 16, 16, 64, 64, 64, 16, None, 1, 4, None) == -1
    assert lib.tk_cache_store(ok, 0, 16, 16, 64, 60, 64, 16, None, 1, 4, None) == -1
    assert lib.tk_cache_store(ok, 0, 8, 16, 64, 64, 64, 16, None, 1, 4, None) == -1
    assert lib.tk_cache_store(ok, 0, None, 16, 64, 64, 64, 16, None, 1, 4, None) == -1
    # decode: layer, heads, lone k_new, rows without slots, scale, window, strides, out
    def dec(layer=0, qs=64, k=16, v=16, kvs=64, slots=16, ld=256, B=1, H=4, scale=1.0, w=0, s=0, m=0):
        return lib.tk_attn_decode(ok, layer, 16, 4 * qs, qs, k, v, 2 * kvs, kvs, slots, 16, ld, B, H, scale, w, s,
                                  m, None, 0, None)
    for kw in (dict(layer=-1), dict(H=3), dict(H=0), dict(v=None), dict(slots=None, B=9), dict(scale=0.0),
               dict(scale=float("nan")), dict(scale=-1.0), dict(w=-1), dict(s=-1), dict(m=-1), dict(qs=63), dict(kvs=60),
               dict(ld=255), dict(ld=128)):
        assert dec(**kw) == -1, kw


# ---------------------------------------------------------------------------
# books and data
# ---------------------------------------------------------------------------
@gpu
def test_books_follow_the_model(cuda_device):
    """A long run of calls leaves exactly the model's books; padding entries
    are skipped, pages come lowest first."""
    g = torch.Generator().manual_seed(0)
    cache, model = make(num_pages=150, max_seqs=8, width=12)
    rand = lambda n: int(torch.randint(n, (1,), generator=g))  # noqa: E731
    for step in range(120):
        empty = [s for s in range(8) if model.lens[s] == 0]
        held = [s for s in range(8) if model.lens[s] > 0]
        kind = rand(4)
        if kind == 0 or not held:
            slots = [s for s in range(8) if rand(2)] + [-1]
            counts = [min(rand(40), 12 * 16 - model.lens[s]) if s >= 0 else 5 for s in slots]
            cache.reserve(ints(*slots), ints(*counts))
            model.reserve(slots, counts)
        elif kind == 1 and empty:
            children = empty[:1 + rand(len(empty))]
            parents = [held[rand(len(held))] for _ in children]
            if rand(2):
                parents[0] = -1
            cache.fork(ints(*parents), ints(*children))
            model.fork(parents, children)
        elif kind == 2:
            slots = held[:1 + rand(len(held))] + [-1]
            cache.release(slots)
            model.release(slots)
        else:
            live = cache.compact()
            assert int(live) == model.compact()[0]
        same_books(cache, model)
    cache.check()


@gpu
@pytest.mark.parametrize("page_size, head_dim, kv_heads", [(16, 8, 3), (32, 64, 1), (256, 16, 2), (64, 256, 2)])
def test_store_fork_compact_move_the_data(cuda_device, page_size, head_dim, kv_heads):
    """Rows land at their positions, forks read the same rows, and everything
    else in the pool stays as it was."""
    lens, layers, width = [page_size * 2 + 5, 1, page_size, 3 * page_size - 1], 2, 4
    cache, model = make(num_pages=40, page_size=page_size, max_seqs=8, width=width, layers=layers, kv_heads=kv_heads,
                        head_dim=head_dim)
    g = torch.Generator(device="cuda").manual_seed(1)
    cache.pages.copy_(torch.randn(cache.pages.shape, generator=g, device="cuda").half())
    want = cache.pages.clone()
    cache.reserve([6], [page_size * 3])
    model.reserve([6], [page_size * 3])
    slots, S = [2, 0, 5, 3], max(lens)
    cache.reserve(slots, lens)
    model.reserve(slots, lens)
    for layer in range(layers):
        # keys and values as views of one fused projection
        qkv = torch.randn(4, S, 3, kv_heads, head_dim, generator=g, device="cuda").half()
        k, v = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
        cache.store(layer, k, v, ints(*slots), ints(*lens))
        for b, s in enumerate(slots):
            for t in range(lens[b]):
                want[layer, model.seqs[s][t // page_size], 0, :, t % page_size] = k[b, :, t]
                want[layer, model.seqs[s][t // page_size], 1, :, t % page_size] = v[b, :, t]
    torch.testing.assert_close(cache.pages, want, rtol=0, atol=0)
    parents, children = [2, 2, 5, 3], [1, 4, 7, -1]
    cache.fork(parents, children)
    for src, dst, rows in model.fork(parents, children):
        want[:, dst, :, :, :rows] = want[:, src, :, :, :rows]
    torch.testing.assert_close(cache.pages, want, rtol=0, atol=0)
    cache.release([6, 2])
    model.release([6, 2])
    live = cache.compact()
    count, moves = model.compact()
    for src, dst in moves:
        want[:, dst] = want[:, src]
    assert int(live) == count and len(moves) > 0
    same_books(cache, model)
    torch.testing.assert_close(cache.pages, want, rtol=0, atol=0)
    cache.copy_pages([0, 3], [39, 38])
    want[:, [39, 38]] = want[:, [0, 3]]
    torch.testing.assert_close(cache.pages, want, rtol=0, atol=0)
    cache.check()


@gpu
def test_store_continues_a_sequence(cuda_device):
    """Two stores in a row: the second one's tokens follow the first one's,
    across a page boundary; rows with a count of zero store nothing."""
    cache, _ = make(layers=1, kv_heads=1, head_dim=16)
    cache.pages.zero_()
    k = torch.arange(1, 31, device="cuda").half().view(1, 1, 30, 1).expand(1, 1, 30, 16).contiguous()
    cache.reserve([3], [11])
    cache.store(0, k[:, :, :11], -k[:, :, :11], [3])
    cache.reserve([3], [19])
    cache.store(0, k[:, :, 11:], -k[:, :, 11:], [3], [19])
    cache.reserve([3], [0])
    cache.store(0, k[:, :, :5], k[:, :, :5], [3], [0])
    pages = cache.page_table[3, :2].long()
    rows = cache.pages[0, pages, :, 0].transpose(0, 1).reshape(2, 32, 16)
    torch.testing.assert_close(rows[0, :30], k[0, 0], rtol=0, atol=0)
    torch.testing.assert_close(rows[1, :30], -k[0, 0], rtol=0, atol=0)
    assert not rows[:, 30:].any()
    cache.check()


@gpu
def test_snapshot_undoes_appended_tokens(cuda_device):
    cache, model = make()
    cache.reserve([0, 1], [20, 16])
    model.reserve([0, 1], [20, 16])
    saved = cache.snapshot()
    cache.reserve([0, 1], [30, 1])
    cache.fork([0], [2])
    cache.restore(saved)
    same_books(cache, model)
    cache.reserve([1], [1])
    model.reserve([1], [1])
    same_books(cache, model)
    other, _ = make()
    other.load(cache.page_table, cache.seq_lens, cache.ref_counts)
    same_books(other, model)
    other.reserve([4], [50])
    model.reserve([4], [50])
    same_books(other, model)


@gpu
def test_many_pages_and_sequences(cuda_device):
    """Books larger than one pass of the single-CTA kernels: 300,000 pages
    (the free bits are scanned in several rounds), 3,000 entries a call."""
    cache, _ = make(num_pages=300_000, max_seqs=4000, width=100, layers=1, kv_heads=1, head_dim=8)
    n = 3000
    slots = torch.randperm(4000, generator=torch.Generator().manual_seed(3))[:n].int().cuda()
    counts = (torch.arange(n, dtype=torch.int32) * 37 % 1500 + 1).cuda()
    cache.reserve(slots, counts)
    need = (counts + 15) // 16
    first = torch.cumsum(need, 0) - need
    k = torch.arange(100, device="cuda")[None, :]
    want = torch.where(k < need[:, None], first[:, None] + k, -1)
    torch.testing.assert_close(cache.page_table[slots.long()].long(), want, rtol=0, atol=0)
    used = int(need.sum())
    assert used > 100_000
    assert bool((cache.ref_counts[:used] == 1).all()) and not bool(cache.ref_counts[used:].any())
    cache.release(slots[: n // 2])
    live = int(cache.compact())
    assert live == int(need[n // 2:].sum())
    table = cache.page_table[slots[n // 2:].long()]
    assert sorted(table[table >= 0].tolist()) == list(range(live))
    assert bool((cache.ref_counts[:live] == 1).all()) and not bool(cache.ref_counts[live:].any())
    cache.check()


@gpu
@pytest.mark.parametrize("call, bit", [
    (lambda c: c.reserve([2], [64 * 16]), 4),                       # longer than the row
    (lambda c: c.reserve(ints(1, 1), ints(1, 1)), 2),               # the same slot twice
    (lambda c: c.reserve(ints(8), ints(1)), 2),
    (lambda c: c.reserve(ints(-2), ints(1)), 2),
    (lambda c: c.reserve(ints(2), ints(-1)), 2),
    (lambda c: c.reserve([0], [1], require_empty=True), 16),
    (lambda c: c.reserve([2, 3, 4, 5, 6], [190] * 5), 1),           # 60 pages wanted, 59 left
    (lambda c: c.fork([0], [1]), 16),                               # the child holds a sequence
    (lambda c: c.fork(ints(0, 0), ints(2, 2)), 2),
    (lambda c: c.fork(ints(9), ints(2)), 2),
    (lambda c: c.release(ints(0, 0)), 2),
    (lambda c: c.release(ints(77)), 2),
    (lambda c: c.store(0, *[torch.zeros(1, 2, 40, 32, device="cuda").half()] * 2, [0], [40]), 4),
    (lambda c: c.store(0, *[torch.zeros(1, 2, 4, 32, device="cuda").half()] * 2, ints(9), [4]), 2),
], ids=lambda x: None if isinstance(x, int) else "")
def test_refused_calls_change_nothing(cuda_device, call, bit):
    cache, _ = make(num_pages=62 if bit == 1 else 64)
    cache.reserve([0, 1], [30, 3])
    cache.pages.fill_(1.0)
    books, saved = cache._books[4 * -(-cache.num_pages // 128) + 8:].clone(), cache.snapshot()
    call(cache)
    assert int(cache.status) & bit
    with pytest.raises(tk.TKError, match="PagedCache"):
        cache.check()
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)
    # and neither do the calls that follow
    cache.reserve([2], [5])
    cache.release([0])
    cache.fork([0], [3])
    cache.compact()
    q = torch.ones(2, 2, 32, device="cuda").half()
    out = torch.full((2, 64), 7.0, device="cuda").half()
    cache.attend(0, q, 1.0, k_new=q, v_new=q, out=out)
    torch.testing.assert_close(cache._books[4 * -(-cache.num_pages // 128) + 8:], books, rtol=0, atol=0)
    assert bool((cache.pages == 1).all()) and bool((out == 7).all())
    cache.restore(saved)
    cache.reserve([2], [5])
    cache.check()
    tk.check_device_errors(cuda_device)


@gpu
def test_wrong_arguments_raise(cuda_device):
    cache, _ = make()
    kv = torch.zeros(2, 2, 4, 32, device="cuda").half()
    q = torch.zeros(2, 4, 32, device="cuda").half()
    for call in (
        lambda: cache.reserve([0, 0], [1, 1]), lambda: cache.reserve([8], [1]), lambda: cache.reserve([0], [1, 2]),
        lambda: cache.reserve(torch.tensor([0], device="cuda"), ints(1)), lambda: cache.fork([0, 1], [2]),
        lambda: cache.copy_pages([0, 1], [2, 2]), lambda: cache.copy_pages([0, 1], [1, 2]),
        lambda: cache.copy_pages([0], [64]), lambda: cache.store(0, kv, kv[:, :, :3], [0, 1]),
        lambda: cache.store(0, kv, kv, [0]), lambda: cache.store(0, kv[:, :1], kv[:, :1], [0, 1]),
        lambda: cache.attend(0, q[:, :3], 1.0), lambda: cache.attend(0, q, 1.0, k_new=q[:, :2]),
        lambda: cache.attend(0, q, 1.0, slots=[0]), lambda: cache.attend(0, q, 1.0, out=torch.zeros(2, 128)),
        lambda: cache.restore(ints(1)), lambda: cache.load(ints(1), ints(1), ints(1)),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: cache.store(2, kv, kv, [0, 1]), lambda: cache.store(0, kv.float(), kv.float(), [0, 1]),
        lambda: cache.store(0, kv, kv.transpose(1, 2).contiguous().transpose(1, 2), [0, 1]),
        lambda: cache.attend(-1, q, 1.0), lambda: cache.attend(0, q.float(), 1.0), lambda: cache.attend(0, q, 0.0),
        lambda: cache.attend(0, q.cpu(), 1.0), lambda: cache.attend(0, q, 1.0, window=-1),
        lambda: cache.reserve(torch.tensor([0], dtype=torch.int32), ints(1)),
    ):
        with pytest.raises(tk.TKError):
            call()
    cache.check()


@gpu
def test_alignment_is_checked(cuda_device):
    """Rows that 16-byte loads cannot take are refused before a launch; a
    dimension of one entry may have any stride."""
    cache, _ = make()
    cache.reserve([0, 1], [4, 4])
    flat = torch.zeros(4096, device="cuda").half()
    q = flat[:256].view(2, 4, 32)
    off = flat[4:4 + 2 * 2 * 32].view(2, 2, 32)                      # 8 bytes off
    odd = torch.as_strided(flat, (2, 2, 32), (100, 36, 1))           # rows 72 bytes apart
    for k in (off, odd):
        with pytest.raises(tk.TKError, match="16-byte"):
            cache.attend(0, q, 1.0, k_new=k, v_new=k)
    with pytest.raises(tk.TKError, match="even strides"):
        cache.attend(0, torch.as_strided(flat, (2, 4, 32), (129, 32, 1)), 1.0)
    with pytest.raises(tk.TKError, match="4-byte aligned rows"):
        cache.attend(0, q, 1.0, out=torch.as_strided(flat, (2, 128), (131, 1)))
    with pytest.raises(tk.TKError, match="16-byte"):
        kv = torch.as_strided(flat, (2, 2, 4, 32), (1001, 128, 32, 1))
        cache.store(0, kv, kv, [0, 1])
    one = torch.as_strided(flat, (1, 2, 32), (7, 32, 1))
    cache.attend(0, torch.as_strided(flat, (1, 4, 32), (3, 32, 1)), 1.0, k_new=one, v_new=one, slots=[1])
    token = torch.as_strided(flat, (1, 2, 1, 32), (5, 32, 3, 1))
    cache.store(0, token, token, [0])
    cache.check()
    tk.check_device_errors(cuda_device)


@gpu
@pytest.mark.parametrize("slots, bit", [((0, 5, 1), 4), ((0, 1, 1), 2), ((0, 1, 8), 2)])
def test_store_applies_whole_or_not_at_all(cuda_device, slots, bit):
    """One row that cannot be (an empty slot, a slot twice, a slot that does
    not exist): the other rows are not stored either."""
    cache, _ = make(layers=1, kv_heads=1, head_dim=16)
    cache.pages.zero_()
    cache.reserve([0, 1], [4, 4])
    k = torch.ones(3, 1, 4, 16, device="cuda").half()
    cache.store(0, k, k, ints(*slots))
    assert int(cache.status) == bit and not cache.pages.any()
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
def attend_reference(q, k, v, scale, window=0, sinks=0):
    """One sequence in 64 bits: q [H, hd], k, v [Hkv, n, hd]. Returns the
    context [H, hd] and the tolerance of each element."""
    H, hd = q.shape
    G, n = H // k.shape[0], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(n, device=q.device)
    seen = (n - 1 - j < window) | (j < sinks) if window else torch.ones_like(j, dtype=torch.bool)
    k, v = k[:, seen].repeat_interleave(G, 0), v[:, seen].repeat_interleave(G, 0)
    s = torch.einsum("hd,hjd->hj", q, k) * scale
    s_err = (hd + 2) * 2.0 ** -24 * scale * torch.einsum("hd,hjd->hj", q.abs(), k.abs()).amax(1)[:, None]
    p = torch.exp(s - s.amax(1, keepdim=True))
    total = p.sum(1, keepdim=True)
    out = torch.einsum("hj,hjd->hd", p, v) / total
    A = torch.einsum("hj,hjd->hd", p, v.abs()) / total
    tiny = torch.einsum("hj,hjd->hd", (p < 2.0 ** -14).double(), v.abs()) / total * 2.0 ** -25
    tol = (2.0 ** -11 + 2 * s_err + 8 * 2.0 ** -22) * A + tiny + 2.0 ** -11 * out.abs() + 2.0 ** -25
    return out, tol


def filled(lens, page_size, kv_heads, head_dim, seed=0, width=None, layers=1, extra=3, garbage=float("nan"),
           shuffle=True):
    """A cache whose slot s holds lens[s] random tokens in shuffled pages;
    rows that hold no token are NaN. Returns it with the keys and values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, max(-(-n // page_size) for n in lens)) if width is None else width
    used = sum(-(-n // page_size) for n in lens)
    cache, _ = make(num_pages=used + extra, page_size=page_size, max_seqs=len(lens), width=width, layers=layers,
                    kv_heads=kv_heads, head_dim=head_dim)
    cache.pages.fill_(garbage)
    order = torch.randperm(used + extra, generator=torch.Generator().manual_seed(seed))[:used].tolist() if shuffle \
        else list(range(used))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    refs = torch.zeros(used + extra, dtype=torch.int32)
    kv, at = [], 0
    for s, n in enumerate(lens):
        pages = order[at:at + -(-n // page_size)]
        at += len(pages)
        table[s, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        refs[pages] = 1
        x = torch.randn(2, kv_heads, n, head_dim, generator=g, device="cuda").half()
        kv.append(x)
        for i, page in enumerate(pages):
            rows = x[:, :, i * page_size:(i + 1) * page_size]
            cache.pages[layers - 1, page, :, :, :rows.shape[2]] = rows
    cache.load(table, torch.tensor(lens, dtype=torch.int32), refs)
    return cache, kv, g


def check_decode(cache, kv, g, heads, layer=0, window=0, sinks=0, new=True, rows=None):
    """attend over every slot in ``rows`` (default all, by position) against
    the definition; with ``new`` the last token comes as k_new / v_new and its
    place in the pages holds something else."""
    hd, K, ps = cache.head_dim, cache.kv_heads, cache.page_size
    rows = list(range(len(kv))) if rows is None else rows
    q = torch.randn(len(rows), heads, hd, generator=g, device="cuda").half()
    scale = hd ** -0.5
    k_new = v_new = None
    before = cache.pages.clone()
    if new:
        fused = torch.zeros(len(rows), 2, K, hd, device="cuda").half()
        for b, s in enumerate(rows):
            if s >= 0 and kv[s].shape[2] > 0:
                n = kv[s].shape[2]
                fused[b] = kv[s][:, :, n - 1]
                cache.pages[layer, cache.page_table[s, (n - 1) // ps].long(), :, :, (n - 1) % ps] = float("inf")
        k_new, v_new = fused[:, 0], fused[:, 1]
    out = torch.full((len(rows), heads * hd), 9.0, device="cuda").half()
    slots = None if rows == list(range(len(kv))) else ints(*rows)
    got = cache.attend(layer, q, scale, k_new=k_new, v_new=v_new, slots=slots, window=window, sinks=sinks, out=out)
    tk.check_device_errors(torch.device("cuda:0"))
    cache.check()
    assert got.data_ptr() == out.data_ptr()
    for b, s in enumerate(rows):
        row = got[b].view(heads, hd)
        if s < 0:
            assert bool((row == 9).all())
            continue
        if kv[s].shape[2] == 0:
            assert not row.any()
            continue
        ref, tol = attend_reference(q[b], kv[s][0], kv[s][1], scale, window, sinks)
        err = (row.double() - ref).abs()
        assert bool((err <= tol).all()), f"row {b} (len {kv[s].shape[2]}): worst {float((err / tol).max()):.2f} x tol"
    # the new token's rows are the only ones that changed, to its key and value
    assert torch.equal(cache.pages.view(torch.int16), before.view(torch.int16))


@gpu
@pytest.mark.parametrize("head_dim", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv_heads, heads", [(2, 2), (1, 5), (2, 24)])
def test_decode_head_layouts(cuda_device, head_dim, kv_heads, heads):
    cache, kv, g = filled([1, 16, 17, 33, 0, 150, 64], 16, kv_heads, head_dim)
    check_decode(cache, kv, g, heads)
    check_decode(cache, kv, g, heads, new=False)


@gpu
@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("head_dim", [32, 64])
def test_decode_page_sizes(cuda_device, page_size, head_dim):
    cache, kv, g = filled([page_size, page_size + 1, 2 * page_size - 1, 700, 1], page_size, 2, head_dim)
    check_decode(cache, kv, g, 4)


@gpu
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 3), (16, 0), (40, 16), (100, 33), (64, 70), (300, 5),
                                           (10000, 4)])
@pytest.mark.parametrize("head_dim", [32, 128])
def test_decode_window_and_sinks(cuda_device, window, sinks, head_dim):
    cache, kv, g = filled([1, 2, 40, 41, 100, 116, 133, 256, 400], 16, 2, head_dim)
    check_decode(cache, kv, g, 4, window=window, sinks=sinks)


@gpu
def test_decode_hidden_keys_may_hold_anything(cuda_device):
    """Keys outside the window are NaN; so is every row past the lengths."""
    cache, kv, g = filled([300, 90], 32, 2, 64)
    for s in range(2):
        n = kv[s].shape[2]
        for t in list(range(4, n - 50)):
            cache.pages[0, cache.page_table[s, t // 32].long(), :, :, t % 32] = float("nan")
    check_decode(cache, kv, g, 2, window=50, sinks=4)


@gpu
def test_decode_long_and_ragged(cuda_device):
    cache, kv, g = filled([5000, 1, 20011, 777], 64, 2, 64)
    check_decode(cache, kv, g, 8)
    check_decode(cache, kv, g, 8, window=4096, sinks=17)


def run_each_way(cache, call):
    """The output of ``call(max_len)`` for bounds that make the library give a
    segment a warp or a CTA, and for none (wide tables: split over the GPU)."""
    return [call(m).clone() for m in (1, 2047, 4096, 0)]


@gpu
@pytest.mark.parametrize("head_dim", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv_heads, heads", [(16, 16), (3, 36)])
def test_decode_every_division_of_the_work(cuda_device, head_dim, kv_heads, heads):
    """Tables wide enough that the calls are split; with bounds on the
    lengths the same rows run by a warp or a CTA each. Sequences shorter than
    a step, empty ones, one that spans many CTAs, padding between them."""
    lens = [3, 0, 1500, 1, 40, 33, 0, 700, 64, 16, 2500] + [17] * 21
    cache, kv, g = filled(lens, 16, kv_heads, head_dim, width=300)
    for window, sinks in ((0, 0), (600, 20)):
        check_decode(cache, kv, g, heads, window=window, sinks=sinks)
        check_decode(cache, kv, g, heads, window=window, sinks=sinks, rows=[10, -1, 0, 1, 2, -1, 7])
    q = torch.randn(len(lens), heads, head_dim, generator=g, device="cuda").half()
    scale = head_dim ** -0.5
    outs = run_each_way(cache, lambda m: cache.attend(0, q, scale, max_len=m))
    for b, n in enumerate(lens):
        if n == 0:
            assert not any(o[b].any() for o in outs)
            continue
        ref, tol = attend_reference(q[b], kv[b][0], kv[b][1], scale)
        for o in outs:
            assert bool(((o[b].view(heads, head_dim).double() - ref).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("max_len", [0, 300])
def test_decode_more_rows_than_the_split_takes(cuda_device, max_len):
    """700 rows read three sequences (without new tokens that is allowed): too
    many rows to be split, in a wide table a CTA and below a bound a warp each."""
    cache, kv, g = filled([290, 1, 77], 16, 2, 64, width=400)
    q = torch.randn(700, 4, 64, generator=g, device="cuda").half()
    slots = (torch.arange(700, device="cuda") % 3).int()
    out = cache.attend(0, q, 0.125, slots=slots, max_len=max_len).view(700, 4, 64)
    for s in range(3):
        rows = torch.arange(s, 700, 3, device="cuda")
        for b in rows[::29].tolist():
            ref, tol = attend_reference(q[b], kv[s][0], kv[s][1], 0.125)
            assert bool(((out[b].double() - ref).abs() <= tol).all())
    assert bool(torch.isfinite(out).all())
    cache.check()


@gpu
def test_decode_one_long_sequence_over_the_whole_gpu(cuda_device):
    """One key-value head, 50,000 keys: hundreds of parts joined in order."""
    cache, kv, g = filled([50000], 64, 1, 64)
    check_decode(cache, kv, g, 8)
    cache, kv, g = filled([1, 30000, 2], 128, 1, 256)
    check_decode(cache, kv, g, 20)


@gpu
def test_decode_rows_slots_and_layers(cuda_device):
    """Rows in any order, padding rows untouched, the last of three layers."""
    cache, kv, g = filled([50, 0, 20, 99, 16], 16, 2, 32, layers=3)
    check_decode(cache, kv, g, 6, layer=2, rows=[3, -1, 0, 4, -1, 1])


@gpu
def test_decode_strides_and_default_out(cuda_device):
    """q, k and v as views of a fused projection, and of one laid out head by head."""
    cache, kv, g = filled([70, 31], 16, 2, 64)
    K, hd, H = 2, 64, 4
    fused = torch.randn(2, (H + 2 * K) * hd, generator=g, device="cuda").half()
    q = fused[:, :H * hd].view(2, H, hd)
    for b in range(2):
        fused[b, H * hd:] = kv[b][:, :, -1].reshape(-1)
    k, v = fused[:, H * hd:(H + K) * hd].view(2, K, hd), fused[:, (H + K) * hd:].view(2, K, hd)
    a = cache.attend(0, q, 0.125, k_new=k, v_new=v)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(2, 500, device="cuda").half()
    b = cache.attend(0, by_head, 0.125, out=wide[:, :H * hd])
    assert torch.equal(a, b) and not wide[:, H * hd:].any()
    for r in range(2):
        ref, tol = attend_reference(q[r], kv[r][0], kv[r][1], 0.125)
        assert bool(((a[r].view(H, hd).double() - ref).abs() <= tol).all())


@gpu
def test_decode_large_scores(cuda_device):
    """Scores of several hundred: the running maximum grows and shrinks what came before."""
    cache, kv, g = filled([400], 16, 1, 64, garbage=0.0)
    for t in range(400):
        kv[0][0, 0, t] *= 1 + t % 7
        cache.pages[0, cache.page_table[0, t // 16].long(), 0, 0, t % 16] = kv[0][0, 0, t]
    check_decode(cache, kv, g, 4)


@gpu
def test_decode_repeats_bit_for_bit(cuda_device):
    cache, kv, g = filled([3000, 5, 1234], 16, 2, 128)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").half()
    first = cache.attend(0, q, 0.1)
    for _ in range(5):
        assert torch.equal(cache.attend(0, q, 0.1), first)


@gpu
def test_decode_reports_bad_books(cuda_device):
    """A page outside the pool reads as zeros and is reported; so are a slot
    and a length that cannot be."""
    for change, bit in ((lambda c: c.page_table[0].fill_(10 ** 6), 8), (lambda c: c.page_table[0].fill_(-7), 8),
                        (lambda c: c.seq_lens[0].fill_(10 ** 6), 4), (lambda c: c.seq_lens[0].fill_(-3), 4)):
        cache, kv, g = filled([40, 20], 16, 2, 64)
        q = torch.randn(2, 2, 64, generator=g, device="cuda").half()
        change(cache)
        cache.attend(0, q, 0.1, k_new=q, v_new=q)
        assert int(cache.status) == bit
        with pytest.raises(tk.TKError):
            tk.check_device_errors(cuda_device)
    cache, kv, g = filled([40, 20], 16, 2, 64)
    cache.attend(0, q, 0.1, slots=ints(0, 5))
    assert int(cache.status) == 2
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)


@gpu
@pytest.mark.parametrize("rows, kv_heads, width", [(2, 2, 3), (40, 16, 3), (5, 2, 400)])
def test_decode_refuses_two_new_tokens_for_one_sequence(cuda_device, rows, kv_heads, width):
    """In every division of the work (a CTA or a warp per segment, split);
    without new tokens a sequence may be read by several rows."""
    cache, kv, g = filled([40] * rows, 16, kv_heads, 64, width=width)
    before = cache.pages.clone()
    q = torch.randn(rows, kv_heads, 64, generator=g, device="cuda").half()
    slots = torch.arange(rows, dtype=torch.int32, device="cuda")
    slots[rows - 1] = 0
    out = cache.attend(0, q, 0.125, slots=slots)
    for b, s in ((0, 0), (rows - 1, 0)):
        ref, tol = attend_reference(q[b], kv[s][0], kv[s][1], 0.125)
        assert bool(((out[b].view(kv_heads, 64).double() - ref).abs() <= tol).all())
    cache.check()
    cache.attend(0, q, 0.125, k_new=q, v_new=q, slots=slots)
    assert int(cache.status) == 2
    page = cache.page_table[0, 2].long()
    assert torch.equal(cache.pages[0, page].view(torch.int16), before[0, page].view(torch.int16))
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)


@gpu
def test_pool_beyond_32_bit_offsets(cuda_device):
    """A pool of 2.4e9 numbers (4.8 GB): pages at its end are stored, forked,
    attended and compacted like those at its start."""
    ps, K, hd, P = 256, 16, 256, 1150
    cache, _ = make(num_pages=P, page_size=ps, max_seqs=4, width=8, layers=1, kv_heads=K, head_dim=hd)
    assert cache.pages.numel() > 2 ** 31
    table = torch.full((4, 8), -1, dtype=torch.int32)
    refs = torch.zeros(P, dtype=torch.int32)
    table[0, :2] = torch.tensor([P - 2, P - 1], dtype=torch.int32)
    refs[P - 2:] = 1
    cache.load(table, torch.tensor([300, 0, 0, 0], dtype=torch.int32), refs)
    g = torch.Generator(device="cuda").manual_seed(4)
    kv = torch.randn(2, K, 300, hd, generator=g, device="cuda").half()
    cache.store(0, kv[0][None], kv[1][None], [0])
    q = torch.randn(1, K, hd, generator=g, device="cuda").half()
    ref, tol = attend_reference(q[0], kv[0], kv[1], hd ** -0.5)
    for _ in range(2):
        got = cache.attend(0, q, hd ** -0.5, slots=[0]).view(K, hd)
        assert bool(((got.double() - ref).abs() <= tol).all())
        cache.fork([0], [1])
        assert torch.equal(cache.attend(0, q, hd ** -0.5, slots=[1]).view(K, hd), got)
        cache.release([1])
        assert int(cache.compact()) == 2
        assert cache.page_table[0, :2].tolist() == [0, 1]
    cache.check()


@gpu
def test_calls_replay_from_a_graph(cuda_device):
    """A captured step (one more token per sequence, then attention) replays
    on changing books; two graphs of one cache, replayed in turn."""
    lens = [30, 64, 0, 15]
    cache, kv, g = filled(lens, 16, 2, 64, width=8, extra=20, garbage=0.0)
    eager, _, _ = filled(lens, 16, 2, 64, width=8, extra=20, garbage=0.0)
    slots, one = ints(0, 1, 3, -1), ints(1, 1, 1, 1)
    q = torch.randn(4, 4, 64, generator=g, device="cuda").half()
    x = torch.randn(2, 4, 2, 64, generator=g, device="cuda").half()
    outs = [torch.zeros(4, 256, device="cuda").half() for _ in range(2)]

    def step(c, out, w):
        c.reserve(slots, one)
        return c.attend(0, q, 0.125, k_new=x[0], v_new=x[1], slots=slots, window=w, sinks=2, out=out)

    graphs = []
    saved = cache.snapshot()
    for out, w in zip(outs, (0, 20)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(cache, out, w)
        graphs.append(graph)
    cache.restore(saved)
    want = torch.zeros(4, 256, device="cuda").half()
    for i in range(40):
        x.add_(0.01)
        graphs[i % 2].replay()
        step(eager, want, (0, 20)[i % 2])
        assert torch.equal(outs[i % 2], want), i
    assert torch.equal(cache.page_table, eager.page_table) and torch.equal(cache.seq_lens, eager.seq_lens)
    cache.check()


@gpu
def test_another_stream_and_two_devices_worth_of_handles(cuda_device):
    """Calls follow the current stream; two caches on one device do not touch each other."""
    cache, kv, g = filled([500, 77], 16, 2, 64)
    other, kv2, g2 = filled([33, 410], 16, 2, 64, seed=9)
    q = torch.randn(2, 2, 64, generator=g, device="cuda").half()
    want = [c.attend(0, q, 0.125) for c in (cache, other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(want[0]) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, o in zip((cache, other), streams, outs):
            with torch.cuda.stream(s):
                c.attend(0, q, 0.125, out=o)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@gpu
@pytest.mark.parametrize("pairs, ps", [(33, 16), (64, 32), (513, 16), (1000, 16), (4000, 16)])
def test_many_forks_follow_the_model(cuda_device, pairs, ps):
    """More pairs than a warp, and than the planning CTA, has threads. Parents
    end inside or at the end of a page or are empty, some entries are padding,
    and pages handed out are far fewer than pairs in half of the rounds: the
    whole table, lengths, references and every copied row are the model's."""
    g = torch.Generator().manual_seed(pairs)
    for round_ in range(4):
        parents_n = max(1, pairs // 3)
        if round_ == 0:    # whole pages first, then partial ones
            lens = [ps * 2] * (parents_n // 2) + [ps + 1 + i % (ps - 1) for i in range(parents_n - parents_n // 2)]
        elif round_ == 1:  # one partial page in sixteen
            lens = [ps * (1 + i % 3) - (i % 16 == 5) for i in range(parents_n)]
        else:
            lens = torch.randint(0, 3 * ps + 1, (parents_n,), generator=g).tolist()
        used = sum(-(-n // ps) for n in lens)
        cache, model = make(num_pages=used + pairs + 5, page_size=ps, max_seqs=parents_n + pairs, width=3, layers=2,
                            kv_heads=1, head_dim=8)
        dev_g = torch.Generator(device="cuda").manual_seed(round_)
        cache.pages.copy_(torch.randn(cache.pages.shape, generator=dev_g, device="cuda").half())
        slots = list(range(parents_n))
        cache.reserve(slots, lens)
        model.reserve(slots, lens)
        parents = sorted(int(x) for x in torch.randint(0, parents_n, (pairs,), generator=g))
        children = (torch.randperm(pairs, generator=g) + parents_n).tolist()
        for i in range(0, pairs, 7):
            if i % 2:
                parents[i] = -1
            else:
                children[i] = -1
        want = cache.pages.clone()
        copies = model.fork(parents, children)
        cache.fork(ints(*parents), ints(*children))
        cache.check()
        same_books(cache, model)
        if copies:
            src, dst, rows = (torch.tensor(x, device="cuda") for x in zip(*copies))
            for n in range(1, ps):
                at = rows == n
                want[:, dst[at], :, :, :n] = want[:, src[at], :, :, :n]
        torch.testing.assert_close(cache.pages, want, rtol=0, atol=0)


@gpu
@pytest.mark.parametrize("rows, kv_heads, width", [(64, 2, 3), (80, 16, 3), (9, 2, 400)])
@pytest.mark.parametrize("fault, bit", [("twice", 2), ("slot", 2), ("too long", 4), ("negative", 4)])
@pytest.mark.parametrize("at", [0, -1])
def test_decode_with_new_tokens_applies_whole_or_not_at_all(cuda_device, rows, kv_heads, width, fault, bit, at):
    """One row that cannot be, first or last in the list, in every division of
    the work: no row's token is stored; the same call without the fault
    applies to all rows."""
    cache, kv, g = filled([40] * rows, 16, kv_heads, 64, width=width)
    before = cache.pages.clone()
    q = torch.randn(rows, kv_heads, 64, generator=g, device="cuda").half()
    new = torch.randn(2, rows, kv_heads, 64, generator=g, device="cuda").half()
    slots = torch.arange(rows, dtype=torch.int32, device="cuda")
    out = torch.full((rows, kv_heads * 64), 7.0, device="cuda").half()
    saved = cache.snapshot()
    if fault == "twice":
        slots[at] = rows // 2
    elif fault == "slot":
        slots[at] = rows
    else:
        cache.seq_lens[at] = 10 ** 6 if fault == "too long" else -3
    cache.attend(0, q, 0.125, k_new=new[0], v_new=new[1], slots=slots, out=out)
    assert int(cache.status) == bit
    assert torch.equal(cache.pages.view(torch.int16), before.view(torch.int16))
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)
    cache.restore(saved)
    slots.copy_(torch.arange(rows))
    cache.attend(0, q, 0.125, k_new=new[0], v_new=new[1], slots=slots, out=out)
    cache.check()
    page = cache.page_table[:, 2].long()
    assert torch.equal(cache.pages[0, page, 0, :, 7], new[0]) and torch.equal(cache.pages[0, page, 1, :, 7], new[1])
    for b in (0, rows // 2, rows - 1):
        k = torch.cat([kv[b][0][:, :-1], new[0][b][:, None]], 1)
        v = torch.cat([kv[b][1][:, :-1], new[1][b][:, None]], 1)
        ref, tol = attend_reference(q[b], k, v, 0.125)
        assert bool(((out[b].view(kv_heads, 64).double() - ref).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("rows, kv_heads, width", [(64, 2, 3), (80, 16, 3), (9, 2, 400)])
def test_decode_reports_a_wait_that_gave_up(cuda_device, rows, kv_heads, width):
    """With no time to wait, in every division of the work: the status word
    says so, no output is made from the keys that came, later calls do nothing,
    and the context goes on."""
    cache, kv, g = filled([40] * rows, 16, kv_heads, 64, width=width)
    q = torch.randn(rows, kv_heads, 64, generator=g, device="cuda").half()
    out = torch.full((rows, kv_heads * 64), 7.0, device="cuda").half()
    saved = cache.snapshot()
    old = tk.set_wait_limit_ns(0)
    try:
        cache.attend(0, q, 0.125, out=out)
        assert int(cache.status) == 32
    finally:
        tk.set_wait_limit_ns(old)
    assert bool((out == 7).all())
    cache.attend(0, q, 0.125, out=out)
    assert bool((out == 7).all())
    with pytest.raises(tk.TKError, match="gave up"):
        cache.check()
    with pytest.raises(tk.TKError, match="timed out"):
        tk.check_device_errors(cuda_device)
    cache.restore(saved)
    cache.attend(0, q, 0.125, out=out)
    cache.check()
    for b in (0, rows - 1):
        ref, tol = attend_reference(q[b], kv[b][0], kv[b][1], 0.125)
        assert bool(((out[b].view(kv_heads, 64).double() - ref).abs() <= tol).all())


@gpu
def test_copy_pages_applies_whole_or_not_at_all(cuda_device):
    """A page outside the pool in the list: no page is copied; and a cache that
    has refused a call copies nothing."""
    cache, _ = make(num_pages=300, layers=2)
    cache.pages.copy_(torch.arange(300, device="cuda").view(1, -1, 1, 1, 1, 1).expand(cache.pages.shape).half())
    before, saved = cache.pages.clone(), cache.snapshot()
    src, dst = list(range(100)), list(range(150, 250))
    for at, pages, bad in ((99, "dst", 300), (0, "src", -1), (50, "dst", -5), (99, "src", 2 ** 30)):
        s, d = ints(*src), ints(*dst)
        (s if pages == "src" else d)[at] = bad
        cache._call("tk_cache_copy_pages", s.data_ptr(), d.data_ptr(), 100)
        assert int(cache.status) == 8 and torch.equal(cache.pages, before)
        with pytest.raises(tk.TKError):
            tk.check_device_errors(cuda_device)
        cache.copy_pages(src, dst)  # refused before
        assert int(cache.status) == 8 and torch.equal(cache.pages, before)
        cache.restore(saved)
    cache.copy_pages(src, dst)
    before[:, dst] = before[:, src]
    assert torch.equal(cache.pages, before)
    cache.check()
    tk.check_device_errors(cuda_device)


@gpu
@pytest.mark.parametrize("page", [64, 10 ** 6, -7])
def test_fork_and_store_report_pages_outside_the_pool(cuda_device, page):
    """Books from elsewhere with such a page: the calls are reported, and write
    nothing but what is theirs."""
    cache, _ = make(layers=1, kv_heads=1, head_dim=16)
    cache.reserve([0, 1, 2], [40, 40, 40])
    cache.pages.fill_(1.0)
    saved = cache.snapshot()
    k = torch.full((2, 1, 40, 16), 2.0, device="cuda").half()
    for call in (lambda: cache.store(0, k, k, [0, 1]), lambda: cache.fork([0, 1], [3, 4])):
        cache.page_table[0, 1] = page
        others = cache.page_table[2, :3].long()
        call()
        assert int(cache.status) == 8
        assert bool((cache.pages[0, others] == 1).all())
        with pytest.raises(tk.TKError, match="outside the pool"):
            cache.check()
        with pytest.raises(tk.TKError):
            tk.check_device_errors(cuda_device)
        cache.restore(saved)
    cache.check()
