"""Attention over rows that live in HBM, over svsx_paged_attention_device and svsx_latent_expanded_device (include/svsx.h): the exhaustive inner
products of ``FlatIndex`` with a softmax over them in the place of the k best.

Calls are enqueued on torch's current stream of the queries' device, never wait for the GPU, and may be captured into a graph.  They are for serving:
no gradient flows through them, and where torch would record one (an input that requires it, outside torch.no_grad()) they refuse."""
from __future__ import annotations

import ctypes as C
import functools
import struct

from . import _lib


@functools.lru_cache(maxsize=None)
def _dtypes() -> dict:
    """torch dtype -> svsx_dtype of the row types that attention and the paged cache take."""
    import torch

    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 4}


def _invalid(message: str) -> _lib.SvsxError:
    return _lib.SvsxError(_lib.INVALID_ARGUMENT, message)


def _elsewhere(name, x) -> _lib.SvsxError:
    return _invalid(f"{name} must be on one GPU with the other arrays, is on {x.device}")


def _on_device(name, x, device) -> None:
    if x.device != device or device.type != "cuda":
        raise _elsewhere(name, x)


def _no_gradient(*arrays) -> None:
    """A result that is cut off from its inputs' gradients, without a word, would be a wrong one."""
    for x in arrays:
        if x is not None and x.requires_grad:
            import torch

            if torch.is_grad_enabled():
                raise _invalid("no gradient flows through this call: use torch.no_grad(), or detach the inputs")


def _stream(index: int) -> int:
    """torch's current stream of a device, as the library takes it."""
    import torch

    return torch._C._cuda_getCurrentRawStream(index)


def _rows(name, x, dims):
    if x.dim() != dims:
        raise _invalid(f"{name} must have {dims} dimensions, has {x.dim()}")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise _invalid(f"rows of {name} must be contiguous")


# svsx_attention_desc, laid out by struct: a third of the time that filling a ctypes structure takes
_ATTENTION = struct.Struct("@Nii10NP2NP3NP3N3PfPP")


def paged_attention(queries, keys, values, table, lengths, sequences=None, value_dim: int | None = None, scale: float | None = None, return_lse: bool = False):
    """One new token's attention per row of ``queries`` [n, heads, dim] over paged rows.

    ``keys`` [pages, key_heads, page_size, dim] and ``values`` [pages, key_heads, page_size, value_dim] of the queries' type (float32, float16,
    bfloat16; any strides, rows contiguous); ``values`` = None: the first ``value_dim`` columns of a key row are its value.  ``heads`` is a multiple of
    ``key_heads``; consecutive heads share a key head.  Query i attends to the first ``lengths[s]`` rows of sequence s = ``sequences[i]`` (default: i): row r is row
    r % page_size of page ``table[s, r // page_size]``.  A table entry that is no page is a hole whose rows are left out -- with page_size 1,
    ``table`` may be the int32 ids of a search over these rows, missing neighbours included.

    Returns softmax(scale * queries . keys) . values [n, heads, value_dim] (scale: default dim ** -0.5) and with ``return_lse`` the
    logarithm of each softmax's denominator [n, heads] float32, which joins results over parts of the rows.  A query with no rows gives zeros and -inf.
    Sums are float32; 16-bit rows round the softmax's weights to their type before these meet the values (float32 rows: 32 bits throughout)."""
    import torch

    if queries.dim() != 3 or keys.dim() != 4:
        raise _invalid(f"queries must have 3 dimensions and keys 4, have {queries.dim()} and {keys.dim()}")
    n, heads, dim = queries.shape
    pages, key_heads, page_size, key_dim = key_shape = keys.shape
    qs, ks = queries.stride(), keys.stride()
    dtype, device = queries.dtype, queries.get_device()
    code = _dtypes().get(dtype)
    if code is None:
        raise _invalid(f"unsupported row type {dtype} (float32, float16, bfloat16)")
    if dim < 1:
        raise _invalid("queries have no columns")
    if keys.dtype != dtype or key_dim != dim:
        raise _invalid(f"keys must be {dtype} rows of {dim}, are {keys.dtype} rows of {key_dim}")
    if (qs[2] != 1 or ks[3] != 1) and dim > 1:
        raise _invalid("rows of queries and keys must be contiguous")
    if values is not None:
        if values.dim() != 4 or values.dtype != dtype or values.shape[:3] != key_shape[:3]:
            raise _invalid(f"values must be {dtype} {list(key_shape[:3])} rows, are {values.dtype} {list(values.shape)}")
        columns, vs = values.shape[3], values.stride()
        if vs[3] != 1 and columns > 1:
            raise _invalid("rows of values must be contiguous")
        if value_dim is None:
            value_dim = columns
        elif value_dim != columns:
            raise _invalid(f"value_dim {value_dim} of values with {columns} columns")
        if values.get_device() != device:
            raise _elsewhere("values", values)
        value_ptr = values.data_ptr()
    else:
        vs, value_ptr = (0, 0, 0), 0
        if value_dim is None:
            value_dim = dim
    if table.dim() != 2 or table.dtype != torch.int32:
        raise _invalid("table must be int32 [sequences, pages], rows contiguous")
    table_sequences, max_pages = table.shape
    ts = table.stride()
    if ts[1] != 1 and max_pages > 1:
        raise _invalid("table must be int32 [sequences, pages], rows contiguous")
    if lengths.dtype != torch.int32 or lengths.shape != (table_sequences,) or not lengths.is_contiguous():
        raise _invalid("lengths must be int32, one for each row of table")
    sequence_ptr = 0
    if sequences is not None:
        if sequences.dtype != torch.int32 or sequences.shape != (n,) or not sequences.is_contiguous():
            raise _invalid("sequences must be int32, one for each query")
        if sequences.get_device() != device:
            raise _elsewhere("sequences", sequences)
        sequence_ptr = sequences.data_ptr()
    elif table_sequences != n:
        raise _invalid(f"{n} queries and {table_sequences} sequences: say which with `sequences`")
    if device < 0 or keys.get_device() != device or table.get_device() != device or lengths.get_device() != device:
        for name, x in (("queries", queries), ("keys", keys), ("table", table), ("lengths", lengths)):
            _on_device(name, x, queries.device)
    if value_dim < 0:
        raise _invalid("value_dim must be positive")
    _no_gradient(queries, keys, values)
    out = queries.new_empty((n, heads, value_dim))
    lse = queries.new_empty((n, heads), dtype=torch.float32) if return_lse else None
    try:
        desc = _ATTENTION.pack(
            _ATTENTION.size, device, code, n, heads, key_heads, dim, value_dim, pages, page_size, table_sequences, max_pages, ts[0], queries.data_ptr(), qs[0], qs[1],
            keys.data_ptr(), ks[0], ks[1], ks[2], value_ptr, vs[0], vs[1], vs[2], table.data_ptr(), lengths.data_ptr(), sequence_ptr, dim**-0.5 if scale is None else scale,
            out.data_ptr(), lse.data_ptr() if return_lse else 0)
    except OverflowError:
        raise _invalid("scale must be finite") from None
    L = _lib.lib()
    size = C.c_size_t()
    rc = L.svsx_paged_attention_workspace(desc, C.byref(size))
    if rc == 0:
        bytes_ = size.value
        ws = queries.new_empty(bytes_, dtype=torch.uint8) if bytes_ else None
        rc = L.svsx_paged_attention_device(desc, ws.data_ptr() if bytes_ else 0, bytes_, _stream(device))
    if rc:
        _lib.check(rc)
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
    the last sequence give zeros, or with ``out`` [n_tokens, heads, value_dim] (contiguous) leave their rows as they were.
    Sums are float32; 16-bit rows round the expanded keys and values, and the softmax's weights, to their type (float32 rows: 32 bits throughout), and where a float16 key or value
    would exceed 65504, the queries of its head that see it are answered row by row in the latent space, which is right and slow."""
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
    if dim < 1:
        raise _invalid("queries have no columns")
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
    _no_gradient(queries, rows, w_key, w_value, out)
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
    _lib.check(L.svsx_latent_expanded_device(ref, ws.data_ptr() if ws is not None else None, size.value, _stream(device.index)))
    return out
