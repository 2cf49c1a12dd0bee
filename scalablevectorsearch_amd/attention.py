"""Attention over rows that live in HBM, over svsx_paged_attention_device and svsx_latent_expanded_device (include/svsx.h): the exhaustive inner
products of ``FlatIndex`` with a softmax over them in the place of the k best.

Calls are enqueued on torch's current stream of the queries' device, never wait for the GPU, and may be captured into a graph."""
from __future__ import annotations

import ctypes as C
import functools

from . import _lib


@functools.lru_cache(maxsize=None)
def _dtypes() -> dict:
    """torch dtype -> svsx_dtype of the row types that attention and the paged cache take."""
    import torch

    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 4}


def _invalid(message: str) -> _lib.SvsxError:
    return _lib.SvsxError(_lib.INVALID_ARGUMENT, message)


def _on_device(name, x, device) -> None:
    if x.device != device or device.type != "cuda":
        raise _invalid(f"{name} must be on one GPU with the other arrays, is on {x.device}")


def _stream(device) -> int:
    import torch

    return torch.cuda.current_stream(device).cuda_stream


def _rows(name, x, dims):
    if x.dim() != dims:
        raise _invalid(f"{name} must have {dims} dimensions, has {x.dim()}")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise _invalid(f"rows of {name} must be contiguous")


def paged_attention(queries, keys, values, table, lengths, sequences=None, value_dim: int | None = None, scale: float | None = None, return_lse: bool = False):
    """One new token's attention per row of ``queries`` [n, heads, dim] over paged rows.

    ``keys`` [pages, key_heads, page_size, dim] and ``values`` [pages, key_heads, page_size, value_dim] of the queries' type (float32, float16,
    bfloat16; any strides, rows contiguous); ``values`` = None: the first ``value_dim`` columns of a key row are its value.  ``heads`` is a multiple of
    ``key_heads``; consecutive heads share a key head.  Query i attends to the first ``lengths[s]`` rows of sequence s = ``sequences[i]`` (default: i): row r is row
    r % page_size of page ``table[s, r // page_size]``.  A table entry that is no page is a hole whose rows are left out -- with page_size 1,
    ``table`` may be the int32 ids of a search over these rows, missing neighbours included.

    Returns softmax(scale * queries . keys) . values [n, heads, value_dim] (scale: default dim ** -0.5) and with ``return_lse`` the
    logarithm of each softmax's denominator [n, heads] float32, which joins results over parts of the rows.  A query with no rows gives zeros and -inf."""
    import torch

    _rows("queries", queries, 3)
    _rows("keys", keys, 4)
    n, heads, dim = queries.shape
    pages, key_heads, page_size, key_dim = keys.shape
    dtype, device = queries.dtype, queries.device
    if dtype not in _dtypes():
        raise _invalid(f"unsupported row type {dtype} (float32, float16, bfloat16)")
    if keys.dtype != dtype or key_dim != dim:
        raise _invalid(f"keys must be {dtype} rows of {dim}, are {keys.dtype} rows of {key_dim}")
    if values is not None:
        _rows("values", values, 4)
        if values.dtype != dtype or values.shape[:3] != keys.shape[:3]:
            raise _invalid(f"values must be {dtype} {list(keys.shape[:3])} rows, are {values.dtype} {list(values.shape[:3])}")
        if value_dim is None:
            value_dim = values.shape[3]
        if value_dim != values.shape[3]:
            raise _invalid(f"value_dim {value_dim} of values with {values.shape[3]} columns")
        _on_device("values", values, device)
    elif value_dim is None:
        value_dim = dim
    if table.dim() != 2 or table.dtype != torch.int32 or (table.stride(1) != 1 and table.shape[1] > 1):
        raise _invalid("table must be int32 [sequences, pages], rows contiguous")
    if lengths.dtype != torch.int32 or lengths.shape != table.shape[:1] or not lengths.is_contiguous():
        raise _invalid("lengths must be int32, one for each row of table")
    if sequences is not None:
        if sequences.dtype != torch.int32 or sequences.shape != (n,) or not sequences.is_contiguous():
            raise _invalid("sequences must be int32, one for each query")
        _on_device("sequences", sequences, device)
    elif table.shape[0] != n:
        raise _invalid(f"{n} queries and {table.shape[0]} sequences: say which with `sequences`")
    for name, x in (("queries", queries), ("keys", keys), ("table", table), ("lengths", lengths)):
        _on_device(name, x, device)
    out = torch.empty((n, heads, value_dim), dtype=dtype, device=device)
    lse = torch.empty((n, heads), dtype=torch.float32, device=device) if return_lse else None
    qs, ks = queries.stride(), keys.stride()
    vs = values.stride() if values is not None else (0, 0, 0)
    desc = _lib.AttentionDesc(
        C.sizeof(_lib.AttentionDesc), device.index, _dtypes()[dtype], n, heads, key_heads, dim, value_dim, pages, page_size, table.shape[0], table.shape[1],
        table.stride(0), queries.data_ptr(), qs[0], qs[1], keys.data_ptr(), ks[0], ks[1], ks[2],
        values.data_ptr() if values is not None else None, vs[0], vs[1], vs[2],
        table.data_ptr(), lengths.data_ptr(), sequences.data_ptr() if sequences is not None else None, dim**-0.5 if scale is None else scale,
        out.data_ptr(), lse.data_ptr() if return_lse else None)
    ref = C.byref(desc)
    size = C.c_size_t()
    L = _lib.lib()
    _lib.check(L.svsx_paged_attention_workspace(ref, C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    _lib.check(L.svsx_paged_attention_device(ref, ws.data_ptr() if ws is not None else None, size.value, _stream(device)))
    return (out, lse) if return_lse else out


def latent_attention(queries, rows, table, lengths, value_dim: int, sequences=None, scale: float | None = None, return_lse: bool = False):
    """Latent attention in its absorbed form: ONE row a token, ``rows`` [pages, 1, page_size, dim], is the key of every head and its first
    ``value_dim`` columns (the latent vector) are the value.  ``queries`` [n, heads, dim] are in the rows' space: a head's key projection applied to
    its query, then the query's rotary part; the result [n, heads, value_dim] is what the head's value projection takes.  Otherwise as ``paged_attention``
    (``scale`` is that of the projected head, dim ** -0.5 only by default)."""
    return paged_attention(queries, rows, None, table, lengths, sequences=sequences, value_dim=value_dim, scale=scale, return_lse=return_lse)


def latent_attention_expanded(queries, rows, w_key, w_value, query_offsets, row_offsets, scale: float | None = None, causal: bool = True, out=None):
    """Latent attention in its expanded form, for prompts: every row's keys and values are made from its latent vector, head by head.

    ``rows`` [n_rows, rank + rope]: a token's latent vector and its rotary key, which all heads share.  ``w_key`` [heads, nope, rank] and ``w_value``
    [heads, value_dim, rank]: head h's key is (w_key[h] latent, rotary key), its value w_value[h] latent.  ``queries`` [n_tokens, heads, nope + rope].
    Sequence i has queries ``query_offsets[i]:query_offsets[i + 1]`` and rows ``row_offsets[i]:row_offsets[i + 1]`` (int32, on the GPU, rising); its last query
    is aligned with its last row, and with ``causal`` a query sees the rows up to its own.  A query that sees no row gives zeros.  Queries behind
    the last sequence give zeros, or with ``out`` [n_tokens, heads, value_dim] (contiguous) leave their rows as they were."""
    import torch

    _rows("queries", queries, 3)
    _rows("rows", rows, 2)
    _rows("w_key", w_key, 3)
    _rows("w_value", w_value, 3)
    t, heads, dim = queries.shape
    n_rows, width = rows.shape
    nope, rank, value_dim = w_key.shape[1], w_key.shape[2], w_value.shape[1]
    dtype, device = queries.dtype, queries.device
    if dtype not in _dtypes():
        raise _invalid(f"unsupported row type {dtype} (float32, float16, bfloat16)")
    if any(x.dtype != dtype for x in (rows, w_key, w_value)):
        raise _invalid(f"rows, w_key and w_value must be {dtype} like the queries")
    rope = dim - nope
    if w_key.shape[0] != heads or w_value.shape[0] != heads or w_value.shape[2] != rank or rope < 0 or width != rank + rope:
        raise _invalid(f"queries {list(queries.shape)}, rows {list(rows.shape)}, w_key {list(w_key.shape)} and w_value {list(w_value.shape)} do not fit together")
    if query_offsets.dim() != 1 or query_offsets.shape != row_offsets.shape or query_offsets.shape[0] < 1:
        raise _invalid("query_offsets and row_offsets must be vectors of sequences + 1 elements")
    for name, x in (("query_offsets", query_offsets), ("row_offsets", row_offsets)):
        if x.dtype != torch.int32 or not x.is_contiguous():
            raise _invalid(f"{name} must be contiguous int32")
        _on_device(name, x, device)
    for name, x in (("queries", queries), ("rows", rows), ("w_key", w_key), ("w_value", w_value)):
        _on_device(name, x, device)
    w_key, w_value = w_key.contiguous(), w_value.contiguous()
    keep = out is not None
    if keep:
        if out.dtype != dtype or out.shape != (t, heads, value_dim) or not out.is_contiguous():
            raise _invalid(f"out must be contiguous {dtype} [{t}, {heads}, {value_dim}]")
        _on_device("out", out, device)
    else:
        out = torch.empty((t, heads, value_dim), dtype=dtype, device=device)
    desc = _lib.ExpandedDesc(
        C.sizeof(_lib.ExpandedDesc), device.index, _dtypes()[dtype], query_offsets.shape[0] - 1, t, n_rows, heads, nope, rope, rank, value_dim, queries.data_ptr(),
        queries.stride(0), queries.stride(1), rows.data_ptr(), rows.stride(0), w_key.data_ptr(), w_value.data_ptr(), query_offsets.data_ptr(), row_offsets.data_ptr(),
        dim**-0.5 if scale is None else scale, int(causal), int(keep), out.data_ptr())
    ref = C.byref(desc)
    size = C.c_size_t()
    L = _lib.lib()
    _lib.check(L.svsx_latent_expanded_workspace(ref, C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    _lib.check(L.svsx_latent_expanded_device(ref, ws.data_ptr() if ws is not None else None, size.value, _stream(device)))
    return out
