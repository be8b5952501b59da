"""Paged key-value cache on the device, and the attention that reads it.

``PagedCache`` keeps the keys and values of many sequences in fixed-size
pages of one fp16 pool ``[layers, num_pages, 2 (k, v), kv_heads, page_size,
head_dim]`` and its books (page table, lengths, reference counts) in int32
tensors on the same device, so a serving loop need not wait for the device:

    cache = PagedCache(num_layers=4, num_pages=4096, page_size=64, kv_heads=16, head_dim=64,
                       max_seqs=64, max_pages_per_seq=128)
    cache.reserve(slots, counts)                 # pages for the prompts' tokens
    cache.store(layer, k, v, slots, counts)      # per layer
    ...
    cache.reserve(slots, ones)                   # one more token per sequence
    ctx = cache.attend(layer, q, scale, k_new=k, v_new=v, slots=slots)   # per layer

``fork`` lets a sequence continue in several ways (full pages are shared, a
partial last one is copied), ``release`` frees, ``compact`` moves the pages in
use to the lowest numbers. Every call is one or two launches on the current
stream. Slot lists are int32 tensors on the cache's device (slot -1 is
padding) or Python ints, each slot at most once (a fork's parents any number
of times). With tensors nothing waits for the device and a call can be
captured into a CUDA graph; lists of ints are uploaded by a copy that waits
for the stream and cannot be captured, and so it is with ``copy_pages``, which
takes nothing else, ``load`` from host tensors and ``check``.

A call applies whole or not at all: one that the device refuses (out of pages,
a slot named twice, a sequence longer than its row) changes nothing in the
cache and sets the status word, after which the cache's calls do nothing --
``attend`` leaves its output unwritten -- until ``check()`` has raised the
reason and ``restore`` / ``load`` / ``reset`` has put the books in order. The
output of an ``attend`` that is itself refused is unspecified. A page table
that names pages outside the pool (books from elsewhere) and a wait that gives
up are only found while a call runs: it is reported too, but may have applied
in part. Calls on one cache must be ordered on the GPU (one stream, or streams
that wait for each other). The reference recomputes all keys and values in every
forward (src/optimized.py:488-554), so nothing here has a counterpart in it.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

import _tklib as tk

__all__ = ["PagedCache", "STATUS"]

# bits of the status word (tk_cache_status)
STATUS = {
    1: "out of pages",
    2: "a slot is out of range or named twice, or a count is negative",
    4: "a sequence is longer than its row of the page table, or has fewer tokens than the call stores",
    8: "the page table or a list of pages names a page outside the pool",
    16: "a slot that has to be empty holds a sequence",
    32: "a device wait gave up",
}

Slots = Union[torch.Tensor, Sequence[int]]


def _words(num_pages: int) -> int:
    return -(-num_pages // 128) * 4


def _strides(t: torch.Tensor) -> tuple:
    """Strides in elements; 0 where a dimension has one entry and its stride means nothing."""
    return tuple(st if n > 1 else 0 for n, st in zip(t.shape, t.stride()))


class PagedCache:
    """Keys and values of up to ``max_seqs`` sequences of up to
    ``max_pages_per_seq * page_size`` tokens each. ``pages`` hands in the pool
    (contiguous fp16, the shape above); else it is allocated, uninitialised:
    rows that hold no token are never used."""

    def __init__(
        self,
        num_layers: int,
        num_pages: int,
        page_size: int,
        kv_heads: int,
        head_dim: int,
        max_seqs: int,
        max_pages_per_seq: int,
        pages: Optional[torch.Tensor] = None,
        device: Optional[torch.device] = None,
    ) -> None:
        sizes = dict(num_layers=num_layers, num_pages=num_pages, kv_heads=kv_heads, max_seqs=max_seqs,
                     max_pages_per_seq=max_pages_per_seq)
        for name, value in sizes.items():
            if int(value) < 1:
                raise ValueError(f"{name} must be at least 1, got {value}")
        if max_seqs > 8192 or num_pages > 1 << 20 or max_pages_per_seq > 1 << 20:
            raise ValueError("max_seqs goes up to 8192, num_pages and max_pages_per_seq up to 2**20")
        if page_size not in (16, 32, 64, 128, 256):
            raise tk.TKError("PagedCache", -2, f"page_size {page_size} is not a power of two in 16..256")
        if not tk.lib().tk_attn_supported(int(head_dim)):
            raise tk.TKError("PagedCache", -2, f"head_dim {head_dim} not in {{8,16,32,64,128,256}}")
        shape = (num_layers, num_pages, 2, kv_heads, page_size, head_dim)
        if pages is None:
            dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
            if dev.type != "cuda":
                raise tk.TKError("PagedCache", -1, "the cache lives on a CUDA device (no CPU fallback)")
            pages = torch.empty(shape, dtype=torch.float16, device=dev)
        tk.require_cuda(pages)
        if tuple(pages.shape) != shape or pages.dtype != torch.float16 or not pages.is_contiguous():
            raise ValueError(f"pages must be a contiguous fp16 tensor {shape}, got {tuple(pages.shape)} {pages.dtype}")
        if device is not None and torch.device(device).index not in (None, pages.device.index):
            raise ValueError(f"pages live on {pages.device}, not on {device}")
        self.num_layers, self.num_pages, self.page_size = int(num_layers), int(num_pages), int(page_size)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.max_seqs, self.max_pages_per_seq = int(max_seqs), int(max_pages_per_seq)
        self.pages = pages
        self.device = pages.device
        # one buffer holds all the books, so that a snapshot is one copy
        words, table = _words(num_pages), max_seqs * max_pages_per_seq
        sizes = [words, 4, 4, table, max_seqs, num_pages]
        self._books = torch.zeros(sum(sizes), dtype=torch.int32, device=self.device)
        mask, status, live, page_table, self.seq_lens, self.ref_counts = self._books.split(sizes)
        self.page_table = page_table.view(max_seqs, max_pages_per_seq)
        self.status, self.live_pages = status[0], live[0]
        self._scratch = torch.empty(3 * num_pages + 1, dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            need = tk.lib().tk_attn_decode_workspace_bytes(self.head_dim)
        if need < 0:
            raise tk.TKError("PagedCache", need, tk.lib().tk_last_error().decode(errors="replace"))
        self._workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        self._c = tk.Cache(
            page_table.data_ptr(), self.seq_lens.data_ptr(), self.ref_counts.data_ptr(), mask.data_ptr(),
            status.data_ptr(), live.data_ptr(), self._scratch.data_ptr(), pages.data_ptr(), max_seqs,
            max_pages_per_seq, num_pages, page_size, num_layers, kv_heads, head_dim)
        self._handle, self._lib, self._index = ctypes.byref(self._c), tk.lib(), self.device.index
        self._workspace_ptr, self._workspace_bytes = self._workspace.data_ptr(), need
        self.reset()

    # -- the books as a whole ---------------------------------------------------
    def reset(self) -> None:
        """Every slot empty, every page free."""
        self._books.zero_()
        self.page_table.fill_(-1)
        self._call("tk_cache_rebuild")

    def load(self, page_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor) -> None:
        """Takes over books made elsewhere (a checkpoint): whole tables of
        this cache's sizes. Pages without references become free."""
        for name, new, mine in (("page_table", page_table, self.page_table), ("seq_lens", seq_lens, self.seq_lens),
                                ("ref_counts", ref_counts, self.ref_counts)):
            if new.shape != mine.shape:
                raise ValueError(f"{name} must have shape {tuple(mine.shape)}, got {tuple(new.shape)}")
        self._books.zero_()
        self.page_table.copy_(page_table)
        self.seq_lens.copy_(seq_lens)
        self.ref_counts.copy_(ref_counts)
        self._call("tk_cache_rebuild")

    def snapshot(self) -> torch.Tensor:
        """The books as one tensor, for ``restore``. The pages' data is not in
        it: going back is exact while no page that was in use has been
        released and written since (dropping tokens that were only appended,
        forks that were only added)."""
        return self._books.clone()

    def restore(self, saved: torch.Tensor) -> None:
        if saved.shape != self._books.shape or saved.dtype != torch.int32 or saved.device != self.device:
            raise ValueError("not a snapshot of a cache of these sizes on this device")
        self._books.copy_(saved)

    def check(self) -> None:
        """Waits for the device and raises if a call was refused."""
        code = int(self.status.item())
        if code:
            reasons = "; ".join(text for bit, text in STATUS.items() if code & bit)
            raise tk.TKError("PagedCache", -6, reasons or f"status {code}")

    # -- sequences -----------------------------------------------------------------
    def reserve(self, slots: Slots, counts: Slots, require_empty: bool = False) -> None:
        """Sequence ``slots[i]`` grows by ``counts[i]`` tokens; the pages they
        reach into are the lowest free ones, in the order of the entries."""
        s, c = self._slots(slots), self._ints(counts, "counts")
        self._same_length(s, c)
        self._call("tk_cache_reserve", s.data_ptr(), c.data_ptr(), s.numel(), int(bool(require_empty)))

    def fork(self, parents: Slots, children: Slots) -> None:
        """Empty slot ``children[i]`` becomes a copy of ``parents[i]``: full
        pages are shared, the used rows of a partial last page are copied.
        Store the parents' reserved tokens first: what is stored in a shared
        page later is the other holders' as well."""
        p, c = self._ints(parents, "parents"), self._slots(children)
        self._same_length(p, c)
        self._call("tk_cache_fork", p.data_ptr(), c.data_ptr(), p.numel())

    def release(self, slots: Slots) -> None:
        """Empties the slots; pages that no other sequence holds become free."""
        s = self._slots(slots)
        self._call("tk_cache_release", s.data_ptr(), s.numel())

    def compact(self) -> torch.Tensor:
        """Moves the n pages in use to ids 0..n-1 (the k-th one at or above n
        into the k-th free one below it) in every layer, and returns n as a
        one-element tensor that the next ``compact`` overwrites."""
        self._call("tk_cache_compact")
        return self.live_pages

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copies the data of whole pages, in every layer; the books stay as
        they are. Page ids are Python ints."""
        src, dst = [int(x) for x in src], [int(x) for x in dst]
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} source pages, {len(dst)} destinations")
        if any(not 0 <= x < self.num_pages for x in src + dst):
            raise ValueError(f"page ids go from 0 to {self.num_pages - 1}")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            raise ValueError("a destination page is named twice or is also a source")
        for i in range(0, len(src), 8192):
            s, d = self._upload(src[i:i + 8192]), self._upload(dst[i:i + 8192])
            self._call("tk_cache_copy_pages", s.data_ptr(), d.data_ptr(), s.numel())

    # -- keys and values -----------------------------------------------------------
    def store(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: Slots,
              counts: Optional[Slots] = None) -> None:
        """Writes the last ``counts[b]`` tokens of sequence ``slots[b]`` (all
        S of them without ``counts``), which ``reserve`` has made room for.
        ``k`` and ``v`` are logically ``[B, kv_heads, S, head_dim]`` fp16 with
        the same strides and a contiguous last dimension, e.g. views of the
        fused QKV projection; token t >= counts[b] is padding."""
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or shape[1] != self.kv_heads or shape[3] != self.head_dim:
            raise ValueError(f"k/v must be [B, {self.kv_heads}, S, {self.head_dim}], got {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
        B, _, S, _ = shape
        k_b, k_h, k_s, k_1 = strides = k.stride()
        if (not (k.dtype == v.dtype == torch.float16) or not (k.device == v.device == self.device) or k_1 != 1
                or v.stride() != strides):
            self._check_data("store", k, v)
        slots = self._slots(slots)
        if slots.numel() != B:
            raise ValueError(f"{B} rows, but {slots.numel()} slots")
        counts_ptr = None
        if counts is not None:
            counts = self._ints(counts, "counts")
            if counts.numel() != B:
                raise ValueError(f"{B} rows, but {counts.numel()} counts")
            counts_ptr = counts.data_ptr()
        self._call("tk_cache_store", layer, k.data_ptr(), v.data_ptr(), k_b, k_h, k_s, slots.data_ptr(), counts_ptr,
                   B, S)

    def attend(
        self,
        layer: int,
        q: torch.Tensor,
        scale: float,
        k_new: Optional[torch.Tensor] = None,
        v_new: Optional[torch.Tensor] = None,
        slots: Optional[Slots] = None,
        window: int = 0,
        sinks: int = 0,
        max_len: int = 0,
        out: Optional[torch.Tensor] = None,
    ) -> torch.Tensor:
        """Attention of one new token per row, the last of its sequence;
        returns the context ``[B, H * head_dim]`` fp16.

        ``q`` is ``[B, H, head_dim]`` fp16 (any strides, contiguous last
        dimension); query head h reads key-value head ``h // (H // kv_heads)``.
        With ``k_new`` / ``v_new`` ``[B, kv_heads, head_dim]`` the token's key
        and value are written into the cache as well, for all rows or none. ``window`` > 0 hides the
        keys that lie ``window`` or more tokens back, except the first
        ``sinks``. Without ``slots`` row b is sequence b; rows with slot -1
        are left as they are, an empty sequence gives zeros. ``max_len`` > 0
        bounds the rows' lengths where the caller knows better than the
        table's width; it only helps to choose how the work is divided."""
        K, hd = self.kv_heads, self.head_dim
        shape = q.shape
        if len(shape) != 3 or shape[2] != hd or shape[1] == 0 or shape[1] % K:
            raise ValueError(f"q must be [B, a multiple of {K} heads, {hd}], got {tuple(shape)}")
        B, H, _ = shape
        q_b, q_h, q_1 = q.stride()
        if q.dtype != torch.float16 or q.device != self.device or q_1 != 1:
            self._check_data("attend", q)
        if k_new is None and v_new is None:
            k_ptr, v_ptr, k_b, k_h = None, None, 0, 0
        elif k_new is None or v_new is None:
            raise ValueError("k_new and v_new come together")
        else:
            if not (k_new.shape == v_new.shape == (B, K, hd)):
                raise ValueError(f"k_new/v_new must be {(B, K, hd)}, got {tuple(k_new.shape)} and "
                                 f"{tuple(v_new.shape)}")
            k_b, k_h, k_1 = strides = k_new.stride()
            if (not (k_new.dtype == v_new.dtype == torch.float16) or not (k_new.device == v_new.device == self.device)
                    or k_1 != 1 or v_new.stride() != strides):
                self._check_data("attend", k_new, v_new)
            k_ptr, v_ptr = k_new.data_ptr(), v_new.data_ptr()
        ld = H * hd
        if out is None:
            out = q.new_empty((B, ld))
        else:
            if out.shape != (B, ld) or out.dtype != torch.float16 or (out.stride(1) != 1 and out.numel() > 0):
                raise ValueError(f"out must be fp16 {(B, ld)} with a contiguous last dimension")
            if out.device != self.device:
                tk.require_cuda(self.pages, out)
            if B > 1:
                ld = out.stride(0)
        slots_ptr = None
        if slots is not None:
            slots = self._slots(slots)
            if slots.numel() != B:
                raise ValueError(f"{B} rows, but {slots.numel()} slots")
            slots_ptr = slots.data_ptr()
        self._call("tk_attn_decode", layer, q.data_ptr(), q_b, q_h, k_ptr, v_ptr, k_b, k_h, slots_ptr, out.data_ptr(),
                   ld, B, H, scale, window, sinks, max_len, self._workspace_ptr, self._workspace_bytes)
        return out

    # -- helpers ---------------------------------------------------------------------
    def _call(self, name: str, *args) -> None:
        index = self._index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return self._call(name, *args)
        status = getattr(self._lib, name)(self._handle, *args, tk.stream_handle(self.device))
        if status != tk.TK_OK:
            raise tk.TKError(name, status, self._lib.tk_last_error().decode(errors="replace"))

    def _check_data(self, what: str, *tensors: torch.Tensor) -> None:
        for t in tensors:
            if t.device != self.device:
                tk.require_cuda(self.pages, *tensors)
            if t.dtype != torch.float16:
                raise tk.TKError(what, -2, "the cache and its inputs are float16")
            if t.stride(-1) != 1 and t.numel():
                raise tk.TKError(what, -1, "inputs need a contiguous last dimension")
        if len(tensors) == 2 and tensors[0].stride() != tensors[1].stride() \
                and _strides(tensors[0]) != _strides(tensors[1]):
            raise tk.TKError(what, -1, "keys and values need identical strides")

    def _upload(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def _ints(self, values: Slots, name: str) -> torch.Tensor:
        if not isinstance(values, torch.Tensor):
            return self._upload([int(x) for x in values])
        if values.dim() != 1 or values.dtype != torch.int32:
            raise ValueError(f"{name} must be a one-dimensional int32 tensor or a list of ints")
        if values.device != self.device:
            tk.require_cuda(self.pages, values)
        return values.contiguous()

    def _slots(self, slots: Slots) -> torch.Tensor:
        if not isinstance(slots, torch.Tensor):
            slots = [int(x) for x in slots]
            real = [x for x in slots if x != -1]
            if any(not 0 <= x < self.max_seqs for x in real) or len(set(real)) != len(real):
                raise ValueError(f"slots are distinct numbers from 0 to {self.max_seqs - 1}, or -1")
        return self._ints(slots, "slots")

    @staticmethod
    def _same_length(a: torch.Tensor, b: torch.Tensor) -> None:
        if a.numel() != b.numel():
            raise ValueError(f"lists of different lengths: {a.numel()} and {b.numel()}")
