"""A paged cache of rows in HBM and its page operations, over svsx_cache_* (include/svsx.h): the keys and values that a model stores token by token, in
pages that sequences take, share and give back.

Every call is enqueued on torch's current stream of the cache's device, never waits for the GPU, and may be captured into a graph.  Calls
that change a cache must be ordered among each other and with its readers, as one stream does; calls of one PagedCache from several threads on one
stream are (a call is up to two launches, which follow one another)."""
from __future__ import annotations

import ctypes as C
import threading

from . import _lib
from .attention import _dtypes, _elsewhere, _invalid, _no_gradient, _on_device, _stream, paged_attention

_MOST = 4096  # entries of one call (include/svsx.h)


class PagedCache:
    """``keys`` [layers, pages, heads, page_size, key_dim] and ``values`` [..., value_dim] (None: the rows are keys and values at once), ``table``
    [sequences, max_pages] and ``lengths`` [sequences] int32, ``refs`` [pages] int32 (how many sequences hold the page).  float32, float16 or bfloat16 rows.

    Pages are taken lowest first, in the order of a call's entries.  An entry that names no sequence, a sequence that the call named before, or more
    rows than there is room for is refused on the device: it changes nothing and counts in ``failures`` (an int32 tensor of one element; reading it waits)."""

    def __init__(self, n_pages: int, page_size: int, n_heads: int, key_dim: int, value_dim: int | None = None, n_layers: int = 1, dtype=None, n_sequences: int = 256,
                 max_pages: int | None = None, device: int = 0):
        import torch

        value_dim = key_dim if value_dim is None else value_dim
        dtype = torch.float16 if dtype is None else dtype
        if min(n_pages, page_size, n_heads, key_dim, n_layers, n_sequences) < 1 or value_dim < 0:
            raise _invalid("sizes of a cache are positive (value_dim may be 0)")
        max_pages = n_pages if max_pages is None else max_pages
        dev = torch.device("cuda", device)
        shape = (n_layers, n_pages, n_heads, page_size)
        self._adopt(torch.zeros(*shape, key_dim, dtype=dtype, device=dev), torch.zeros(*shape, value_dim, dtype=dtype, device=dev) if value_dim else None,
                    torch.full((n_sequences, max_pages), -1, dtype=torch.int32, device=dev), torch.zeros(n_sequences, dtype=torch.int32, device=dev),
                    torch.zeros(n_pages, dtype=torch.int32, device=dev))

    @classmethod
    def from_device(cls, keys, values, table, lengths, refs) -> "PagedCache":
        """Adopt torch tensors that hold a cache already; they are changed in place and kept alive by the cache."""
        self = cls.__new__(cls)
        self._adopt(keys, values, table, lengths, refs)
        return self

    def _adopt(self, keys, values, table, lengths, refs):
        import torch

        if keys.dim() != 5 or (values is not None and (values.dim() != 5 or values.shape[:4] != keys.shape[:4] or values.dtype != keys.dtype)):
            raise _invalid("keys and values are [layers, pages, heads, page_size, dim] of one type")
        if keys.dtype not in _dtypes():
            raise _invalid(f"unsupported row type {keys.dtype} (float32, float16, bfloat16)")
        layers, pages, heads, page_size, key_dim = keys.shape
        if table.dim() != 2 or lengths.shape != table.shape[:1] or refs.shape != (pages,) or any(x.dtype != torch.int32 for x in (table, lengths, refs)):
            raise _invalid("table [sequences, max_pages], lengths [sequences] and refs [pages] are int32")
        for name, x in (("keys", keys), ("values", values), ("table", table), ("lengths", lengths), ("refs", refs)):
            if x is not None:
                _on_device(name, x, keys.device)
                if not x.is_contiguous():
                    raise _invalid(f"{name} must be contiguous")
        self.keys, self.values, self.table, self.lengths, self.refs = keys, values, table, lengths, refs
        self.failures = torch.zeros(1, dtype=torch.int32, device=keys.device)
        self.device, self._index = keys.device, keys.get_device()
        self.n_sequences, self.page_size = table.shape[0], page_size
        self._int32, self._int64 = torch.int32, torch.int64
        self._rows = ((heads, key_dim), (heads, values.shape[4]) if values is not None else None)
        self._desc = _lib.CacheDesc(C.sizeof(_lib.CacheDesc), self._index, _dtypes()[keys.dtype], layers, pages, heads, page_size, key_dim,
                                    values.shape[4] if values is not None else 0, table.shape[0], table.shape[1], keys.data_ptr(),
                                    values.data_ptr() if values is not None else None, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), self.failures.data_ptr())
        self._at = C.addressof(self._desc)
        size = C.c_size_t()
        _lib.check(_lib.lib().svsx_cache_workspace(self._at, _MOST, C.byref(size)))  # checks the description, too
        # calls that change a cache follow one another, so one workspace serves them all.  A call is two launches and the interpreter lets other threads run meanwhile: the lock
        # keeps their launches from coming between
        self._lock = threading.Lock()
        self._space, self._space_bytes = torch.empty(size.value, dtype=torch.uint8, device=keys.device), size.value
        self._space_at = self._space.data_ptr()

    def _list(self, x, name):
        """A vector of int32 on the cache's device; a list on the host is copied there first (and the host waits for that)."""
        import torch

        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x, dtype=torch.int32).to(self.device)
        if x.dtype != self._int32 or x.dim() != 1 or not x.is_contiguous():
            raise _invalid(f"{name} must be a contiguous vector of int32")
        if x.get_device() != self._index:
            raise _elsewhere(name, x)
        return x

    def extend(self, sequences, offsets, n_tokens: int):
        """Sequence ``sequences[i]`` grows by ``offsets[i + 1] - offsets[i]`` rows; returns the slot of each of the ``n_tokens`` new rows (int64, for
        ``write``; -1 where an entry was refused or no entry has the row)."""
        sequences, offsets = self._list(sequences, "sequences"), self._list(offsets, "offsets")
        n = sequences.shape[0]
        if offsets.shape[0] != n + 1:
            raise _invalid(f"{n} sequences need {n + 1} offsets, got {offsets.shape[0]}")
        if n_tokens < 0:
            raise _invalid("n_tokens must not be negative")
        slots = sequences.new_empty(n_tokens, dtype=self._int64)
        with self._lock:
            rc = _lib.lib().svsx_cache_extend_device(self._at, sequences.data_ptr(), offsets.data_ptr(), n, n_tokens, slots.data_ptr(), self._space_at, self._space_bytes,
                                                     _stream(self._index))
        if rc:
            _lib.check(rc)
        return slots

    def write(self, slots, keys, values=None, layer: int = 0) -> None:
        """Rows ``keys`` [tokens, heads, key_dim] (and ``values``) of one layer to their slots.  Slots of one call differ; those outside the cache (-1) are skipped.
        No gradient flows into the cache: rows that require one are refused outside torch.no_grad()."""
        if slots.dtype != self._int64 or slots.dim() != 1 or not slots.is_contiguous():
            raise _invalid("slots must be a contiguous vector of int64")
        if slots.get_device() != self._index:
            raise _elsewhere("slots", slots)
        if (values is None) != (self.values is None):
            raise _invalid("values are given exactly where the cache holds values")
        if not 0 <= layer < self.keys.shape[0]:
            raise _invalid(f"layer {layer} of a cache of {self.keys.shape[0]} layers")
        n = slots.shape[0]
        ks = self._check_rows("keys", keys, n, self._rows[0])
        vs = self._check_rows("values", values, n, self._rows[1]) if values is not None else (0, 0)
        _no_gradient(keys, values)
        with self._lock:
            rc = _lib.lib().svsx_cache_write_device(self._at, layer, slots.data_ptr(), n, keys.data_ptr(), ks[0], ks[1], values.data_ptr() if values is not None else 0, vs[0], vs[1],
                                                    _stream(self._index))
        if rc:
            _lib.check(rc)

    def _check_rows(self, name, x, n, row):
        if x.dtype != self.keys.dtype or x.shape != (n, *row):
            raise _invalid(f"{name} must be {self.keys.dtype} {[n, *row]}, got {x.dtype} {list(x.shape)}")
        strides = x.stride()
        if strides[2] != 1 and row[1] > 1:
            raise _invalid(f"rows of {name} must be contiguous")
        if x.get_device() != self._index:
            raise _elsewhere(name, x)
        return strides

    def _copy(self, sources, targets, share):
        sources, targets = self._list(sources, "sources"), self._list(targets, "targets")
        n = sources.shape[0]
        if targets.shape[0] != n:
            raise _invalid(f"{n} sources and {targets.shape[0]} targets")
        with self._lock:
            rc = _lib.lib().svsx_cache_copy_device(self._at, sources.data_ptr(), targets.data_ptr(), n, share, self._space_at, self._space_bytes, _stream(self._index))
        if rc:
            _lib.check(rc)

    def copy(self, sources, targets) -> None:
        """Each target, an empty sequence, becomes a copy of its source, in pages of its own."""
        self._copy(sources, targets, 0)

    def fork(self, sources, targets) -> None:
        """Each target, an empty sequence, becomes its source: full pages are held by both, a partly filled last page is copied."""
        self._copy(sources, targets, 1)

    def free(self, sequences) -> None:
        """The sequences become empty; pages nobody holds any more are free."""
        sequences = self._list(sequences, "sequences")
        with self._lock:
            rc = _lib.lib().svsx_cache_free_device(self._at, sequences.data_ptr(), sequences.shape[0], _stream(self._index))
        if rc:
            _lib.check(rc)

    def compact(self):
        """Used pages move to the front of the pool; returns each page's new place (int32 [pages], -1 for a page that was free)."""
        moved = self.refs.new_empty(self.refs.shape[0])
        with self._lock:
            rc = _lib.lib().svsx_cache_compact_device(self._at, moved.data_ptr(), self._space_at, self._space_bytes, _stream(self._index))
        if rc:
            _lib.check(rc)
        return moved

    def attend(self, queries, sequences=None, layer: int = 0, value_dim: int | None = None, scale: float | None = None, return_lse: bool = False):
        """``paged_attention`` of ``queries`` [n, heads, key_dim] over one layer; row i belongs to ``sequences[i]`` (default: sequence i)."""
        if not 0 <= layer < self.keys.shape[0]:
            raise _invalid(f"layer {layer} of a cache of {self.keys.shape[0]} layers")
        with self._lock:
            return paged_attention(queries, self.keys[layer], self.values[layer] if self.values is not None else None, self.table, self.lengths, sequences=sequences,
                                   value_dim=value_dim, scale=scale, return_lse=return_lse)
