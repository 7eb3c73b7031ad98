"""Paged KV cache of several sequences, its whole state in device memory.

FixedKVBuffer (kv_buffer.py) gives one sequence one buffer; here sequences share a
pool of pages, so samples of one prompt, or frames with a common prefix, hold its
K / V once. One tensor holds every layer,

    store[layer, 0 | 1, page, kv_head, slot, dim]      (0 = K, 1 = V)

and position t of sequence s lies in slot t % page_size of page
table[s, t // page_size]. Page numbers, lengths and reference counts are device
tensors and every operation is one or a few asynchronous launches (rb_kv_pages_*),
so a decoding loop needs no host round trip and can be captured into a CUDA graph.

A round of decoding:

    cache.reserve(seqs, counts)            # room for the round's tokens
    per layer: cache.write(k, v, seqs, layer=l); cache.attend(q, seqs, l, ahead=1)
    cache.commit(seqs, counts)             # or compact(seqs, paths, counts): an accepted path

Operations take sequence numbers and counts as int32 tensors on the cache's device
(lists are copied there). A call that cannot be served (no free page, a sequence
named twice, a count outside the room) changes nothing and raises the cache's status
word; ``check()`` reads it and raises. Only ``write`` works token by token: it leaves out
those that have no place of their own, and ``commit`` refuses them. Calls on one cache must
be ordered: one stream, or events between streams.
"""
from __future__ import annotations

import ctypes
import torch

from respect_b200 import _lib
from respect_b200.kernels.attention import _rows as rows
from respect_b200.kernels.attention import paged_attention

STATUS = {1: "a sequence that does not exist, is named twice, or is a fork's target in use",
          2: "not enough free pages",
          3: "a count, length, path or position outside the sequence's room",
          4: "a write or commit into a page that is missing or that another sequence holds (reserve again after a fork)"}


class PagedCacheError(RuntimeError):
    """An operation on a PagedKVCache was refused on the device."""


class PagedKVCache:
    """A pool of ``pages`` pages of ``page_size`` tokens for up to ``max_seqs`` sequences of
    up to ``max_pages`` pages each (default: the whole pool)."""

    def __init__(self, layers: int, kv_heads: int, pages: int, page_size: int, max_seqs: int,
                 max_pages: int | None = None, head_dim: int = 128, dtype: torch.dtype = torch.bfloat16,
                 device="cuda") -> None:
        if min(layers, kv_heads, pages, page_size, max_seqs, head_dim) < 1:
            raise ValueError("PagedKVCache: every size must be positive")
        i32 = dict(dtype=torch.int32, device=device)
        max_pages = pages if max_pages is None else max_pages
        self._adopt(torch.zeros(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device),
                    torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(max_seqs, **i32),
                    torch.zeros(max_seqs, **i32), torch.zeros(pages, **i32))

    @classmethod
    def from_state(cls, store: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, held: torch.Tensor,
                   refs: torch.Tensor) -> "PagedKVCache":
        """A cache on existing state tensors (contiguous; used in place): store [layers, 2, pages,
        kv_heads, page_size, head_dim], and int32 table [max_seqs, max_pages] (-1 = no page), lengths
        and held [max_seqs] (tokens and pages of each sequence), refs [pages] (its holders)."""
        self = cls.__new__(cls)
        self._adopt(store, table, lengths, held, refs)
        return self

    def _adopt(self, store, table, lengths, held, refs) -> None:
        if store.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"PagedKVCache holds bf16 or fp32, not {store.dtype}")
        if not store.is_cuda:
            raise ValueError("respect_b200 operators take CUDA tensors (no CPU path)")
        if store.dim() != 6 or store.shape[1] != 2 or min(store.shape) < 1:
            raise ValueError(f"store must be [layers, 2, pages, kv_heads, page_size, head_dim], got {tuple(store.shape)}")
        n = table.shape[0] if table.dim() == 2 else 0
        for name, t, shape in (("table", table, (n, table.shape[-1])), ("lengths", lengths, (n,)), ("held", held, (n,)),
                               ("refs", refs, (store.shape[2],))):
            if t.dtype != torch.int32 or t.device != store.device or tuple(t.shape) != shape or t.numel() == 0:
                raise ValueError(f"{name} must be a non-empty int32 tensor {shape} on {store.device}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if not store.is_contiguous():
            raise ValueError("store must be contiguous")
        self.store, self.table, self.lengths, self.held, self.refs = store, table, lengths, held, refs
        self.device, self.dtype, self._dev = store.device, store.dtype, store.get_device()
        self.layers, _, self.pages, self.kv_heads, self.page_size, self.head_dim = store.shape
        self.max_seqs, self.max_pages = table.shape
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = _lib.KVPages(store.data_ptr(), self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim,
                               store.element_size(), self.max_seqs, self.max_pages, table.data_ptr(),
                               lengths.data_ptr(), held.data_ptr(), refs.data_ptr(), self.status.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._ws_bytes = _lib.lib().rb_kv_pages_workspace(self._ref)
        if self._ws_bytes == 0:
            raise ValueError("PagedKVCache: a shape the native library does not take (rows of whole 16-byte "
                             "pieces, at most 2^30 tokens per sequence)")
        self._ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device)

    # ---------------------------------------------------------------- arguments
    def _list(self, x, name: str, n: int | None = None) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(list(x), dtype=torch.int32, device=self.device)
        if x.dtype is not torch.int32 or x.get_device() != self._dev or x.dim() != 1:
            raise TypeError(f"{name} must be a list or an int32 tensor of one dimension on {self.device}")
        m = x.numel()
        if n is not None and m != n:
            raise ValueError(f"{name} holds {m} entries, expected {n}")
        if m > _lib.PAGES_MAX_LIST:
            raise ValueError(f"{name}: at most {_lib.PAGES_MAX_LIST} sequences per call")
        return x if x.is_contiguous() else x.contiguous()

    def _call(self, name: str, *args) -> None:
        _lib.launch(name, self.store, self._ref, *args)

    # ---------------------------------------------------------------- operations
    def reserve(self, seqs, counts) -> None:
        """Room for counts[i] more tokens after the committed ones of seqs[i]: the lowest free
        pages, in list order. A partly filled last page that other sequences hold is copied
        first (the last of the list's holders keeps it when nobody else does)."""
        s = self._list(seqs, "seqs")
        c = self._list(counts, "counts", s.numel())
        self._call("rb_kv_pages_reserve", s.data_ptr(), c.data_ptr(), s.numel(), self._ws.data_ptr(), self._ws_bytes)

    def write(self, k: torch.Tensor, v: torch.Tensor, seqs, offsets=None, layer: int | None = None) -> None:
        """K and V of new tokens to the positions after the committed ones, inside reserved room
        (tokens outside it, or on a page that another sequence holds, are left out and raise the status):
        tokens [offsets[i], offsets[i + 1]) belong to seqs[i] (default: one token each). k, v
        [tokens, kv_heads, head_dim] for one ``layer``, [layers, tokens, kv_heads, head_dim] for all."""
        s = self._list(seqs, "seqs")
        n, ks = s.numel(), k.shape
        want = (self.layers,) if layer is None else ()
        if len(ks) != 3 + len(want) or ks != v.shape or ks[:-3] != want or ks[-2:] != (self.kv_heads, self.head_dim):
            raise ValueError(f"k {tuple(ks)}, v {tuple(v.shape)} do not fit: expected "
                             f"[{'layers, ' if layer is None else ''}tokens, {self.kv_heads}, {self.head_dim}]")
        if layer is not None and not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} of {self.layers}")
        T = ks[-3]
        if offsets is None:
            if T != n:
                raise ValueError(f"{T} tokens for {n} sequences: pass offsets")
        else:
            if not isinstance(offsets, torch.Tensor):
                offsets = torch.tensor(list(offsets), dtype=torch.int32, device=self.device)
            if offsets.dtype is not torch.int32 or offsets.get_device() != self._dev or offsets.shape != (n + 1,):
                raise ValueError(f"offsets must be int32 [{n + 1}] on {self.device}")
            offsets = offsets.contiguous()
        k, v = rows(k, "k", self.store), rows(v, "v", self.store)
        sk, sv = k.stride(), v.stride()
        x = _lib.KVTokens(k.data_ptr(), v.data_ptr(), sk[0] if layer is None else 0, sk[-3], sk[-2],
                          sv[0] if layer is None else 0, sv[-3], sv[-2], layer or 0, self.layers if layer is None else 1, T)
        self._call("rb_kv_pages_write", ctypes.byref(x), s.data_ptr(), None if offsets is None else offsets.data_ptr(), n)

    def commit(self, seqs, counts) -> None:
        """The next counts[i] written tokens of seqs[i] belong to it. Refused where a write would be:
        past the reserved room, or on a page that another sequence holds (commit before a fork)."""
        s = self._list(seqs, "seqs")
        c = self._list(counts, "counts", s.numel())
        self._call("rb_kv_pages_commit", s.data_ptr(), c.data_ptr(), s.numel())

    def fork(self, src, dst) -> None:
        """The empty sequences dst[i] take the committed tokens of src[i]; pages are shared."""
        a = self._list(src, "src")
        d = self._list(dst, "dst", a.numel())
        self._call("rb_kv_pages_fork", a.data_ptr(), d.data_ptr(), a.numel(), self._ws.data_ptr(), self._ws_bytes)

    def compact(self, seqs, paths, counts) -> None:
        """Commit an accepted path (kv_buffer.compact on pages): of the tokens written after the
        committed ones, numbers paths[i, :counts[i]] (strictly increasing) move to the front, in
        every layer, and are committed; the pages past them are given back."""
        s = self._list(seqs, "seqs")
        c = self._list(counts, "counts", s.numel())
        if not isinstance(paths, torch.Tensor):
            wide = max((len(p) for p in paths), default=0)
            paths = torch.tensor([list(p) + [0] * (wide - len(p)) for p in paths], dtype=torch.int32,
                                 device=self.device).reshape(len(paths), wide)
        if paths.dtype != torch.int32 or paths.device != self.device or paths.dim() != 2 or paths.shape[0] != s.numel():
            raise ValueError(f"paths must be lists or an int32 tensor [{s.numel()}, width] on {self.device}")
        width = paths.shape[1]
        if (paths.stride(1) != 1 and width > 1) or paths.stride(0) < width:
            paths = paths.contiguous()       # rows that overlap, as of an expanded list
        self._call("rb_kv_pages_compact", s.data_ptr(), paths.data_ptr(), max(paths.stride(0), width), width,
                   c.data_ptr(), s.numel(), self._ws.data_ptr(), self._ws_bytes)

    def truncate(self, seqs, lengths) -> None:
        """Keep lengths[i] tokens of seqs[i]; its other pages, reserved ones too, are given back."""
        s = self._list(seqs, "seqs")
        n = self._list(lengths, "lengths", s.numel())
        self._call("rb_kv_pages_truncate", s.data_ptr(), n.data_ptr(), s.numel())

    def free(self, seqs) -> None:
        """Give back every page of the sequences; they are empty afterwards."""
        s = self._list(seqs, "seqs")
        self._call("rb_kv_pages_truncate", s.data_ptr(), None, s.numel())

    # ---------------------------------------------------------------- views
    def layer_kv(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(K, V) pages of one layer, [pages, kv_heads, page_size, head_dim]."""
        return self.store[layer, 0], self.store[layer, 1]

    def attend(self, q: torch.Tensor, seqs, layer: int, ahead: int = 0, sm_scale: float | None = None,
               max_length: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """paged_attention of q [n, H, head_dim] over the tokens of seqs in one layer: the
        committed ones and ``ahead`` written after them. Without a ``max_length`` scratch and launch
        are sized for max_pages * page_size tokens a sequence: 64 sequences of 512 tokens, 28 / 4
        heads, in a cache of 4,096 pages of 16 take 67 us and 239 MB of scratch, with max_length=1024
        32 us and 15 MB."""
        k, v = self.layer_kv(layer)
        return paged_attention(q, k, v, self.table, self.lengths, sm_scale, self._list(seqs, "seqs"), ahead, max_length,
                               out)

    def check(self, clear: bool = True) -> None:
        """Raise PagedCacheError if an operation since the last check was refused (synchronises)."""
        code = int(self.status.item())
        if code:
            if clear:
                self.status.zero_()
            raise PagedCacheError(f"PagedKVCache: {STATUS.get(code, code)}")
