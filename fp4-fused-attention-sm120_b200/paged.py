"""The paged FP4 key / FP16 value cache, attention of new tokens over it, and
the pages' bookkeeping.

A cache is three tensors (PagedCache); sequences name their pages in an int32
block table [sequences, pages].  A serving step appends each sequence's new
token (cache_append: rotate, quantise, store) and attends over all of them
(paged_attention).  A prompt is appended the same way; its own attention is
fused_fp4_attention, over a cached prefix by way of cache_gather.  PagePool
deals the pages out on the host: allocate, fork with copy on write, compact,
free; copy_pages does the copying.
"""
from __future__ import annotations

import ctypes
import operator

from . import _serving as sv

__all__ = ["PagedCache", "cache_append", "cache_gather", "paged_attention_workspace_size", "paged_attention",
           "paged_attention_lse", "copy_pages", "PagePool"]

PAGE_SIZES = (16, 32, 64, 128)


class PagedCache:
    """One layer's cache over three CUDA tensors:

    k_codes  uint8   [pages, kv_heads, page_size, head_dim / 2]
    k_scales uint8   [pages, kv_heads, page_size, head_dim / 32]
    v        float16 [pages, kv_heads, page_size, head_dim]

    Each page is contiguous; pages may be apart (a view of one layer of a
    larger tensor).  The tensors need not be initialised.  The calls go by the
    addresses that the tensors had here, so the cache keeps that memory, and its
    attributes are read-only: another tensor is another PagedCache."""

    def __init__(self, k_codes, k_scales, v):
        torch = sv.torch()
        if v.dim() != 4 or not v.is_cuda or v.dtype != torch.float16:
            raise ValueError("v must be a float16 CUDA tensor [pages, kv_heads, page_size, head_dim]")
        P, H, S, D = v.shape
        if D not in (32, 64, 96, 128, 160, 256) or S not in PAGE_SIZES:
            raise ValueError(f"head_dim {D} must be 32/64/96/128/160/256 and page_size {S} one of {PAGE_SIZES}")
        if P < 1 or H < 1:
            raise ValueError("a cache needs a page and a head")
        for name, t, width in (("k_codes", k_codes, D // 2), ("k_scales", k_scales, D // 32), ("v", v, D)):
            if t.shape != (P, H, S, width) or t.device != v.device or (name != "v" and t.dtype != torch.uint8):
                raise ValueError(f"{name} must be [{P}, {H}, {S}, {width}] on {v.device}")
            if not t[0].is_contiguous():
                raise ValueError(f"a page of {name} must be contiguous")
            if t.data_ptr() % 16 or (t.stride(0) * t.element_size()) % 16:
                raise ValueError(f"{name} and its page stride must be 16-byte aligned")
            if P > 1 and t.stride(0) < t[0].numel():
                raise ValueError(f"pages of {name} overlap")
        # (Aliases, which hold the memory whatever becomes of the caller's tensors.)
        self._k_codes, self._k_scales, self._v = k_codes.detach(), k_scales.detach(), v.detach()
        self._pages, self._kv_heads, self._page_size, self._head_dim = P, H, S, D
        self._device, self._index = v.device, v.device.index
        self._struct = sv.CacheStruct(k_codes.data_ptr(), k_scales.data_ptr(), v.data_ptr(),
                                      max(k_codes.stride(0), k_codes[0].numel()),
                                      max(k_scales.stride(0), k_scales[0].numel()),
                                      2 * max(v.stride(0), v[0].numel()), P, S, H, D)
        self._at = ctypes.addressof(self._struct)

    k_codes, k_scales, v, pages, kv_heads, page_size, head_dim, device, struct = (
        property(operator.attrgetter("_" + name)) for name in
        ("k_codes", "k_scales", "v", "pages", "kv_heads", "page_size", "head_dim", "device", "struct"))

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, device="cuda"):
        """A new cache (its memory as it comes)."""
        torch = sv.torch()
        shape = (pages, kv_heads, page_size)
        return cls(torch.empty(shape + (head_dim // 2,), dtype=torch.uint8, device=device),
                   torch.empty(shape + (head_dim // 32,), dtype=torch.uint8, device=device),
                   torch.empty(shape + (head_dim,), dtype=torch.float16, device=device))


def cache_append(cache, K, V, block_table, positions, seq_ids=None, Q=None, table=None, interleaved=False,
                 scale_mode="reference", stream=None):
    """Puts tokens into the cache (fp4attn_cache_append): K and V [tokens,
    kv_heads, head_dim], float16 or float32, any token and head strides.  Token
    i is token positions[i] of sequence seq_ids[i] (default: sequence i); a
    negative position marks padding.  With a rotary ``table`` the keys are
    rotated by their positions first.  With Q [tokens, heads, head_dim] returns
    the queries rotated the same way, contiguous.  No two tokens of a call may
    have the same place in the cache."""
    args = (cache._at, cache._index, K, V, block_table, positions, seq_ids, Q, table, interleaved,
            sv.scale_mode(scale_mode))
    if stream is None:
        return sv.native().cache_append(*args)
    with sv.on(cache._device, stream):
        return sv.native().cache_append(*args)


def cache_gather(cache, block_table, starts, lengths, max_length, heads=None, dtype=None, stream=None):
    """K and V [sequences, heads, max_length, head_dim] (float16 by default) of
    tokens starts[s] .. starts[s] + lengths[s] - 1 of every sequence, zeros
    behind them (fp4attn_cache_gather).  starts=None reads from token 0; heads
    (default: the cache's) repeats each key/value head for its query heads, as
    fused_fp4_attention wants them."""
    args = (cache._at, cache._index, block_table, starts, lengths, max_length, heads, dtype)
    if stream is None:
        return sv.native().cache_gather(*args)
    with sv.on(cache._device, stream):
        return sv.native().cache_gather(*args)


def paged_attention_workspace_size(cache, batch, heads):
    """Bytes of device workspace paged_attention needs for this many sequences
    and query heads, whatever their lengths."""
    return int(sv.lib().fp4attn_paged_attention_workspace_size(batch, heads, cache.kv_heads, cache.head_dim))


def _attend(Q, cache, block_table, seq_lens, softmax_scale, scale_mode, out_dtype, out, with_lse, workspace, stream):
    args = (Q, cache._at, cache._index, block_table, seq_lens, softmax_scale, sv.scale_mode(scale_mode),
            out_dtype, out, with_lse, workspace)
    if stream is None:
        return sv.native().attend(*args)
    with sv.on(cache._device, stream):
        return sv.native().attend(*args)


def paged_attention(Q, cache, block_table, seq_lens, softmax_scale=None, scale_mode="reference", out_dtype=None,
                    out=None, workspace=None, stream=None):
    """Attention of one new token per sequence over the cache
    (fp4attn_paged_attention): Q [batch, heads, head_dim], already rotated;
    block_table [batch, pages]; seq_lens int32 [batch], the new token counted.
    Returns [batch, heads, head_dim] of out_dtype (default Q's).  Query head h
    reads key/value head h // (heads / kv_heads); a sequence of length 0 gives
    zeros.  Give ``out`` and ``workspace`` (uint8, of at least
    paged_attention_workspace_size bytes, not shared by calls in flight at once)
    to allocate nothing."""
    return _attend(Q, cache, block_table, seq_lens, softmax_scale, scale_mode, out_dtype, out, False, workspace,
                   stream)


def paged_attention_lse(Q, cache, block_table, seq_lens, softmax_scale=None, scale_mode="reference", out_dtype=None,
                        out=None, workspace=None, stream=None):
    """paged_attention that also returns the natural log-sum-exp of the scaled
    scores, float32 [batch, heads] (+inf for a sequence of length 0), by which
    attentions over parts of a context are joined."""
    return _attend(Q, cache, block_table, seq_lens, softmax_scale, scale_mode, out_dtype, out, True, workspace, stream)


def copy_pages(caches, src, dst, stream=None):
    """Copies pages src[i] to dst[i] within every cache of ``caches`` (the
    layers of a model, one page numbering), in one launch for up to eight
    layers and 64 pages (fp4attn_copy_pages).  src and dst: sequences of ints or
    CPU integer tensors.  No page may be written twice, or both read and
    written."""
    caches = list(caches)
    if not caches:
        return
    device = caches[0]._device
    if any(c._device != device for c in caches):
        raise ValueError("the caches must be on one device")
    args = ([c._at for c in caches], device.index, _page_numbers(src, "src"), _page_numbers(dst, "dst"))
    if stream is None:
        return sv.native().copy_pages(*args)
    with sv.on(device, stream):
        sv.native().copy_pages(*args)


def _page_numbers(pages, name):
    """A contiguous int32 CPU tensor of page numbers (their range is checked by the library)."""
    torch = sv.torch()
    if not isinstance(pages, torch.Tensor):
        pages = torch.tensor(pages) if len(pages) else torch.empty(0, dtype=torch.int64)
    if pages.dtype is not torch.int32 and not pages.is_cuda:
        if pages.is_floating_point() or pages.is_complex() or pages.dtype is torch.bool:
            raise TypeError(f"{name}: page numbers must be integers, not {pages.dtype}")
        narrow = pages.to(torch.int32)
        if not torch.equal(narrow.to(torch.int64), pages.to(torch.int64)):
            raise ValueError(f"{name}: page number out of range")
        pages = narrow
    return pages.contiguous()


class PagePool:
    """Which sequence owns which pages of a cache, on the host.

    Pages are counted: a forked sequence shares its parent's pages, and the
    page that the next token of either falls into is copied first, if it is
    shared.  Methods that move contents return (src, dst) page lists, to be
    given to copy_pages before the next kernel that reads or writes the cache."""

    def __init__(self, pages, page_size):
        if pages < 1 or page_size not in PAGE_SIZES:
            raise ValueError(f"pages >= 1 and page_size one of {PAGE_SIZES}")
        self.pages, self.page_size = pages, page_size
        self._free = list(range(pages - 1, -1, -1))  # the lowest page is dealt first
        self._uses = [0] * pages
        self._tables: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self) -> int:
        page = self._free.pop()
        self._uses[page] = 1
        return page

    def _drop(self, page) -> None:
        self._uses[page] -= 1
        if self._uses[page] == 0:
            self._free.append(page)

    def new(self) -> int:
        """A new, empty sequence's number."""
        seq = self._next
        self._next += 1
        self._tables[seq], self._lengths[seq] = [], 0
        return seq

    def length(self, seq) -> int:
        return self._lengths[seq]

    def table(self, seq) -> list[int]:
        """The sequence's pages, in order."""
        return list(self._tables[seq])

    def extend(self, seq, tokens):
        """Makes room for `tokens` more tokens of a sequence, whose length grows
        by them, and returns the (src, dst) copies they need first: its last page,
        if that is partly filled and shared.  MemoryError, with nothing changed,
        when the pages do not suffice."""
        if tokens < 0:
            raise ValueError("tokens must be >= 0")
        table, length = self._tables[seq], self._lengths[seq]
        want = -(-(length + tokens) // self.page_size)
        own = tokens > 0 and length % self.page_size != 0 and self._uses[table[-1]] > 1
        if want - len(table) + own > len(self._free):
            raise MemoryError(f"{want - len(table) + own} pages wanted, {len(self._free)} free")
        src, dst = [], []
        if own:
            src.append(table[-1])
            dst.append(self._take())
            self._drop(table[-1])
            table[-1] = dst[0]
        while len(table) < want:
            table.append(self._take())
        self._lengths[seq] = length + tokens
        return src, dst

    def fork(self, seq) -> int:
        """A new sequence with the same tokens, in the same pages."""
        child = self.new()
        self._tables[child], self._lengths[child] = list(self._tables[seq]), self._lengths[seq]
        for page in self._tables[child]:
            self._uses[page] += 1
        return child

    def truncate(self, seq, length) -> None:
        """Gives up a sequence's tokens behind `length`, and the pages that held only them."""
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f"length {length} outside [0, {self._lengths[seq]}]")
        table = self._tables[seq]
        while len(table) > -(-length // self.page_size):
            self._drop(table.pop())
        self._lengths[seq] = length

    def free(self, seq) -> None:
        """Gives up a sequence; pages that no other shares are free again."""
        for page in reversed(self._tables.pop(seq)):
            self._drop(page)
        del self._lengths[seq]

    def compact(self):
        """Moves the used pages to the lowest numbers and returns the (src, dst)
        copies; every table changes with them."""
        used = self.pages - len(self._free)
        holes = [p for p in range(used) if self._uses[p] == 0]
        moved = [p for p in range(used, self.pages) if self._uses[p]]
        to = dict(zip(moved, holes))
        for p, q in to.items():
            self._uses[q], self._uses[p] = self._uses[p], 0
        for table in self._tables.values():
            table[:] = [to.get(p, p) for p in table]
        self._free = list(range(self.pages - 1, used - 1, -1))
        return moved, holes

    def block_table(self, seqs, device=None, pages=None):
        """int32 [len(seqs), pages] for the kernels (as many pages as the longest
        sequence has, by default; unused entries are 0)."""
        torch = sv.torch()
        seqs = list(seqs)
        longest = max((len(self._tables[s]) for s in seqs), default=0)
        pages = max(1, longest) if pages is None else pages
        if pages < longest:
            raise ValueError(f"a sequence has {longest} pages, more than {pages}")
        rows = [self._tables[s] + [0] * (pages - len(self._tables[s])) for s in seqs]
        return torch.tensor(rows, dtype=torch.int32).reshape(len(seqs), pages).to("cpu" if device is None else device)
