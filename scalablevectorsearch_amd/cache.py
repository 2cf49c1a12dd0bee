"""A paged cache of rows in HBM and its page operations, over svsx_cache_* (include/svsx.h): the keys and values that a model stores token by token, in
pages that sequences take, share and give back.

Every call is enqueued on torch's current stream of the cache's device, never waits for the GPU, and may be captured into a graph.  Calls
that change a cache must be ordered among each other and with its readers, as one stream does."""
from __future__ import annotations

import ctypes as C

from . import _lib
from .attention import _dtypes, _invalid, _on_device, _stream, paged_attention


def _list(x, device, name):
    import torch

    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x, dtype=torch.int32).to(device)
    if x.dtype != torch.int32 or x.dim() != 1 or not x.is_contiguous():
        raise _invalid(f"{name} must be a contiguous vector of int32")
    _on_device(name, x, device)
    return x


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
        self.device = keys.device
        self.n_sequences, self.page_size = table.shape[0], page_size
        self._desc = _lib.CacheDesc(C.sizeof(_lib.CacheDesc), keys.device.index, _dtypes()[keys.dtype], layers, pages, heads, page_size, key_dim,
                                    values.shape[4] if values is not None else 0, table.shape[0], table.shape[1], keys.data_ptr(),
                                    values.data_ptr() if values is not None else None, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), self.failures.data_ptr())
        self._ref = C.byref(self._desc)
        size = C.c_size_t()
        _lib.check(_lib.lib().svsx_cache_workspace(self._ref, 0, C.byref(size)))  # checks the description, too
        self._space = size.value

    def _workspace(self, n):
        import torch

        return torch.empty(self._space + 4 * n, dtype=torch.uint8, device=self.device)

    def extend(self, sequences, offsets, n_tokens: int):
        """Sequence ``sequences[i]`` grows by ``offsets[i + 1] - offsets[i]`` rows; returns the slot of each of the ``n_tokens`` new rows (int64, for
        ``write``; -1 where an entry was refused or no entry has the row)."""
        import torch

        sequences, offsets = _list(sequences, self.device, "sequences"), _list(offsets, self.device, "offsets")
        n = sequences.shape[0]
        if offsets.shape[0] != n + 1:
            raise _invalid(f"{n} sequences need {n + 1} offsets, got {offsets.shape[0]}")
        if n_tokens < 0:
            raise _invalid("n_tokens must not be negative")
        slots = torch.empty(n_tokens, dtype=torch.int64, device=self.device)
        ws = self._workspace(n)
        _lib.check(_lib.lib().svsx_cache_extend_device(self._ref, sequences.data_ptr(), offsets.data_ptr(), n, n_tokens, slots.data_ptr(), ws.data_ptr(), ws.shape[0],
                                                       _stream(self.device)))
        return slots

    def write(self, slots, keys, values=None, layer: int = 0) -> None:
        """Rows ``keys`` [tokens, heads, key_dim] (and ``values``) of one layer to their slots.  Slots of one call differ; those outside the cache (-1) are skipped."""
        import torch

        if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
            raise _invalid("slots must be a contiguous vector of int64")
        _on_device("slots", slots, self.device)
        if (values is None) != (self.values is None):
            raise _invalid("values are given exactly where the cache holds values")
        if not 0 <= layer < self.keys.shape[0]:
            raise _invalid(f"layer {layer} of a cache of {self.keys.shape[0]} layers")
        n, heads = slots.shape[0], self.keys.shape[2]
        for name, x, pool in (("keys", keys, self.keys), ("values", values, self.values)):
            if x is None:
                continue
            if x.dtype != pool.dtype or x.shape != (n, heads, pool.shape[4]):
                raise _invalid(f"{name} must be {pool.dtype} [{n}, {heads}, {pool.shape[4]}], got {x.dtype} {list(x.shape)}")
            if x.stride(2) != 1 and x.shape[2] > 1:
                raise _invalid(f"rows of {name} must be contiguous")
            _on_device(name, x, self.device)
        _lib.check(_lib.lib().svsx_cache_write_device(self._ref, layer, slots.data_ptr(), n, keys.data_ptr(), keys.stride(0), keys.stride(1),
                                                      values.data_ptr() if values is not None else None, values.stride(0) if values is not None else 0,
                                                      values.stride(1) if values is not None else 0, _stream(self.device)))

    def _copy(self, sources, targets, share):
        sources, targets = _list(sources, self.device, "sources"), _list(targets, self.device, "targets")
        n = sources.shape[0]
        if targets.shape[0] != n:
            raise _invalid(f"{n} sources and {targets.shape[0]} targets")
        ws = self._workspace(n)
        _lib.check(_lib.lib().svsx_cache_copy_device(self._ref, sources.data_ptr(), targets.data_ptr(), n, share, ws.data_ptr(), ws.shape[0], _stream(self.device)))

    def copy(self, sources, targets) -> None:
        """Each target, an empty sequence, becomes a copy of its source, in pages of its own."""
        self._copy(sources, targets, 0)

    def fork(self, sources, targets) -> None:
        """Each target, an empty sequence, becomes its source: full pages are held by both, a partly filled last page is copied."""
        self._copy(sources, targets, 1)

    def free(self, sequences) -> None:
        """The sequences become empty; pages nobody holds any more are free."""
        sequences = _list(sequences, self.device, "sequences")
        _lib.check(_lib.lib().svsx_cache_free_device(self._ref, sequences.data_ptr(), sequences.shape[0], _stream(self.device)))

    def compact(self):
        """Used pages move to the front of the pool; returns each page's new place (int32 [pages], -1 for a page that was free)."""
        import torch

        moved = torch.empty(self.refs.shape[0], dtype=torch.int32, device=self.device)
        ws = self._workspace(0)
        _lib.check(_lib.lib().svsx_cache_compact_device(self._ref, moved.data_ptr(), ws.data_ptr(), ws.shape[0], _stream(self.device)))
        return moved

    def attend(self, queries, sequences=None, layer: int = 0, value_dim: int | None = None, scale: float | None = None, return_lse: bool = False):
        """``paged_attention`` of ``queries`` [n, heads, key_dim] over one layer; row i belongs to ``sequences[i]`` (default: sequence i)."""
        if not 0 <= layer < self.keys.shape[0]:
            raise _invalid(f"layer {layer} of a cache of {self.keys.shape[0]} layers")
        return paged_attention(queries, self.keys[layer], self.values[layer] if self.values is not None else None, self.table, self.lengths, sequences=sequences,
                               value_dim=value_dim, scale=scale, return_lse=return_lse)
