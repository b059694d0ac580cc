"""Paged caches: the append of several tokens of several sequences, attention
over them with a window and first tokens that stay visible, and the dense rows
they hold, as HIP kernels (``nibble_paged_append``, ``nibble_attention_paged``
and ``nibble_paged_values`` of the C ABI).

The step around a layer's attention of :mod:`nibblegemm_amd.glue` where the
sequences share one pool of memory: a server gives a sequence pages as it
grows and takes back those that it no longer sees.

Layout
------
``k_pages`` and ``v_pages`` are ``[n_pages, n_kv, page, D]``, ``page`` 16, 32,
64, 128 or 256 rows, D 64 or 128, of any strides that are multiples of 16 bytes
with a row's elements adjacent: a pool with a row's heads side by side is the
view ``pool.transpose(1, 2)`` of ``[n_pages, page, n_kv, D]``.  ``table`` int32
``[B, width]`` names the pages of each sequence: its rows ``m page ..`` are page
``table[b, m]``, and an entry that is no page of the cache (-1, say) is none.
Sequence b holds ``lengths[b]`` rows before a call; its ``sizes[b]`` new tokens
(all ``T`` where sizes is None) are the rows behind them.

The elements are fp16 or bf16, as the queries are, or 8-bit floats
(``torch.float8_e4m3fn``) with ``scales``, the pair (k_scales, v_scales) of uint8
``[n_pages, n_kv]`` tensors: a value is ``code 2^(scale - 127)``, one power of two
for a page and head (255 is none: the values under it are NaN).  The append takes
the least one from -15 to 8, in bf16 from -117 to 120, under which a page's rows
fit (448, the largest code, times it).  Under these all codes are values of the
queries' type, but for the last: there codes end at 240, and larger ones, which the
append does not write, are infinite.

Tables, lengths, sizes and scales are read on the GPU, so a captured call
follows their contents.  No operator here has a backward.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _native
from .glue import _HALF_DTYPES, _check_gpu, _check_half, _check_index, _in_order
from .ops import _call, _check_no_backward, _stream, _workspace, _ws_plan

#: Rows that a page may have.
PAGE_ROWS = (16, 32, 64, 128, 256)

Scales = Tuple[torch.Tensor, torch.Tensor]

_FLOAT8 = torch.float8_e4m3fn


def paged_cache(n_pages: int, n_kv: int, page: int, head_dim: int = 128,
                dtype: torch.dtype = torch.float16,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor, Optional[Scales]]:
    """An empty cache: ``(k_pages, v_pages, scales)`` of ``dtype`` fp16, bf16 or
    ``torch.float8_e4m3fn``; scales is None but for the last."""
    if page not in PAGE_ROWS:
        raise ValueError(f"a page must have one of {PAGE_ROWS} rows, got {page}")
    if dtype not in _HALF_DTYPES and dtype != _FLOAT8:
        raise RuntimeError(f"dtype must be fp16, bf16 or float8_e4m3fn, got {dtype}")
    k, v = (torch.zeros((n_pages, n_kv, page, head_dim), dtype=dtype, device=device)
            for _ in range(2))
    if dtype != _FLOAT8:
        return k, v, None
    ks, vs = (torch.full((n_pages, n_kv), 127, dtype=torch.uint8, device=device) for _ in range(2))
    return k, v, (ks, vs)


def _check_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 scales: Optional[Scales], index: int, written: bool):
    """Checks a cache on GPU ``index`` (its 16-bit type is the caller's to check):
    the batch and the arguments that name it to the library."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"the pages must both be [n_pages, n_kv, page, D], got {tuple(shape)} and "
                         f"{tuple(v_pages.shape)}")
    n_pages, n_kv, page, D = shape
    if page not in PAGE_ROWS:
        raise ValueError(f"a page must have one of {PAGE_ROWS} rows, got {page}")
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise RuntimeError("the elements of a cache row must be adjacent")
    k_scales = v_scales = None
    if scales is not None:
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if t.dtype is not _FLOAT8:
                raise RuntimeError(f"{name} must be float8_e4m3fn beside scales, got {t.dtype}")
            if t.get_device() != index:
                raise RuntimeError(f"{name} must live on GPU {index}, got {t.device}")
            _check_no_backward(name, t)
        for name, t in zip(("k_scales", "v_scales"), scales):
            if t.get_device() != index:
                _check_gpu(name, t, k_pages)
            if t.dtype is not torch.uint8 or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous uint8 tensor")
            if t.shape != (n_pages, n_kv):
                raise ValueError(f"{name} must be [{n_pages}, {n_kv}], got {list(t.shape)}")
        k_scales, v_scales = scales[0].data_ptr(), scales[1].data_ptr()
    elif k_pages.dtype is _FLOAT8:
        raise RuntimeError("8-bit pages need scales")
    if table.dim() != 2:
        raise ValueError(f"table must be [B, width], got {list(table.shape)}")
    _check_index("table", table, table.shape, k_pages)
    if written:
        for n, k, v in zip(shape, ks, vs):
            if n > 1 and (k == 0 or v == 0):
                raise RuntimeError("the pages are written and must not be expanded views")
    return table.shape[0], (k_pages.data_ptr(), v_pages.data_ptr(), k_scales, v_scales,
                            table.data_ptr(), n_pages, n_kv, page, D, table.shape[1],
                            ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])


def _check_types(x: torch.Tensor, name: str, **others: Optional[torch.Tensor]) -> None:
    """``x`` and the others are of one 16-bit type, on one GPU, and nothing
    follows them."""
    if _in_order(x.dtype, x.get_device(), x, *others.values()):
        return
    _check_half(name, x, x)
    for other, t in others.items():
        if t is not None:
            _check_half(other, t, x)


def paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 table: torch.Tensor, lengths: torch.Tensor, sizes: Optional[torch.Tensor] = None,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5, rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 interleaved: bool = False, positions: Optional[torch.Tensor] = None,
                 scales: Optional[Scales] = None) -> torch.Tensor:
    """Norms of the query and key heads, their rotary embedding and the append
    of ``T`` tokens of ``B`` sequences to a paged cache, in one pass.

    qkv fp16 or bf16 [B, T, (n_heads + 2 n_kv) * D], the q|k|v projection's
    output; the cache as the module says.  Each q and k head is normalised, ``x /
    sqrt(mean(x^2) + eps) * weight`` (weights [D] of qkv's dtype; None: no norm
    of those heads), then rotated by the (cos, sin) of
    :func:`nibblegemm_amd.glue.rope_tables` (None: no rotation), whose ``R / 2``
    columns turn the first R elements of a head, a multiple of 16: element i with
    ``i + R / 2``, or, ``interleaved``, 2 i with 2 i + 1.  ``positions`` int32 [B,
    T] are the tokens' rotary positions (None: their rows).  All in fp32 with one
    rounding.  k and v go to the rows behind ``lengths``; q is returned as [B, T,
    n_heads * D].  The pages' and scales' version counters rise.

    A token whose row has no page or whose position is no row of the tables is
    padding, as those behind ``sizes`` are: it writes no row and its q is zero.
    Pages that one call writes must belong to one sequence each, once.

    In 8 bits a page that begins with a new row takes the scale of its new rows; in
    one that holds earlier rows the scale may rise, and the codes of the earlier
    rows are halved as often (under a scale of 255 they are NaN, stay so, and the
    page takes the new rows' scale).  Rows behind the new ones are left as they
    are.  Magnitudes that qkv's type does not reach count as its largest value;
    infinities and NaN are stored as NaN and have no part in a scale."""
    _check_types(qkv, "qkv", q_weight=q_weight, k_weight=k_weight,
                 **({} if scales is not None else {"k_pages": k_pages, "v_pages": v_pages}))
    if qkv.dim() != 3 or not qkv.is_contiguous():
        raise RuntimeError("qkv must be a contiguous [B, T, ..] tensor")
    dtype, dev = qkv.dtype, qkv.device
    batch, cache = _check_cache(k_pages, v_pages, table, scales, dev.index, True)
    n_kv, D = cache[6], cache[8]
    B, T, width = qkv.shape
    n_heads = width // D - 2 * n_kv if D else 0
    if batch != B:
        raise ValueError(f"a table of {batch} sequences beside tokens of {B}")
    if n_heads < 1 or width % D:
        raise ValueError(f"qkv must be [B, T, (n_heads + 2 * {n_kv}) * {D}], got {tuple(qkv.shape)}")
    _check_index("lengths", lengths, (B,), qkv)
    if sizes is not None:
        _check_index("sizes", sizes, (B,), qkv)
    if positions is not None:
        _check_index("positions", positions, (B, T), qkv)
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and (t.shape != (D,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [{D}] tensor, got {tuple(t.shape)}")
    cos_p = sin_p = None
    rope_rows = rope_dim = 0
    if rope is not None:
        cos, sin = rope
        for name, t in (("rope cos", cos), ("rope sin", sin)):
            if t.get_device() != dev.index:
                _check_gpu(name, t, qkv)
            _check_no_backward(name, t)
            if t.dtype is not torch.float32 or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous fp32 GPU tensor")
            if t.dim() != 2 or t.shape != cos.shape or t.shape[0] < 1 or t.shape[1] % 8 or \
                    not 8 <= t.shape[1] <= D // 2:
                raise ValueError(f"{name} must be [rows, R / 2], R a multiple of 16 up to {D}, got "
                                 f"{tuple(t.shape)}")
        cos_p, sin_p, rope_rows, rope_dim = cos.data_ptr(), sin.data_ptr(), cos.shape[0], \
            2 * cos.shape[1]
    out = torch.empty((B, T, n_heads * D), dtype=dtype, device=dev)
    _call(_native.binding().paged_append, dev, qkv.data_ptr(), _HALF_DTYPES[dtype], B, T, n_heads,
          *cache, lengths.data_ptr(), sizes.data_ptr() if sizes is not None else None,
          positions.data_ptr() if positions is not None else None,
          q_weight.data_ptr() if q_weight is not None else None,
          k_weight.data_ptr() if k_weight is not None else None, float(eps), cos_p, sin_p,
          rope_rows, rope_dim, 1 if interleaved else 0, out.data_ptr())
    increment_version((k_pages, v_pages) if scales is None else (k_pages, v_pages, *scales))
    return out


def attention_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, lengths: torch.Tensor,
                    sizes: Optional[torch.Tensor] = None, window: Optional[int] = None,
                    sinks: int = 0, scale: Optional[float] = None,
                    scales: Optional[Scales] = None) -> torch.Tensor:
    """Attention of the newest tokens of every sequence over its paged cache.

    q fp16 or bf16 [B, T, n_heads * D], as :func:`paged_append` returns it; the
    cache, which holds the tokens' own rows already, as the module says.  Token i
    of sequence b is row ``r = lengths[b] + i`` and sees the rows up to its own
    that have a page; with a ``window`` those of the last ``window`` rows (its own
    among them) and the first ``sinks`` of the sequence alone, so that the pages
    between may be taken back (-1 in the table).  Returns [B, T, n_heads * D]: per
    query head ``softmax(scale q k^T) v`` over what the token sees, head i reading
    kv head ``i // (n_heads // n_kv)``, scale ``1 / sqrt(D)`` by default, in fp32
    with the probabilities rounded to q's dtype (in fp16 those below 2^-21 of the
    largest in steps of 2^-31 of it).  Scores are below 2^28 log(2) in magnitude,
    2^31 log(2) in bf16.

    Tokens behind a sequence's last, and tokens that see nothing, give zeros. Rows
    that a token does not see have no part in its output, whatever they hold, and
    whatever their page's scale is.  An infinity in the values of a row that it
    sees comes out as it is, or as NaN where the row's weight rounds to zero; a
    NaN as NaN.  ``lengths`` count from zero to the rows of the table, ``sizes``
    to T.  A token whose own row is behind the table, as one whose row has no
    page, sees the rows before it all the same.

    How the rows are split over the GPU goes by T, not by ``sizes``: where ``T *
    n_heads // n_kv`` is large, a sequence of one token is one workgroup a kv head
    however long it is.  Single tokens over long sequences beside a prompt's part
    are faster as a call of their own (512 tokens and seven single ones over 8000
    to 65000 rows: 1.2 ms together, 0.24 apart)."""
    _check_types(q, "q", **({} if scales is not None else {"k_pages": k_pages, "v_pages": v_pages}))
    if q.dim() != 3 or not q.is_contiguous():
        raise RuntimeError("q must be a contiguous [B, T, ..] tensor")
    dtype, dev = q.dtype, q.device
    batch, cache = _check_cache(k_pages, v_pages, table, scales, dev.index, False)
    n_kv, D = cache[6], cache[8]
    B, T, width = q.shape
    if batch != B:
        raise ValueError(f"a table of {batch} sequences beside tokens of {B}")
    if not D or width % D:
        raise ValueError(f"q must be [B, T, n_heads * {D}], got {tuple(q.shape)}")
    n_heads = width // D
    _check_index("lengths", lengths, (B,), q)
    if sizes is not None:
        _check_index("sizes", sizes, (B,), q)
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    ext = _native.binding()
    key = ("paged", B, T, n_heads, n_kv, D, cache[7] * cache[9])
    plan = _ws_plan.get(key)
    if plan is None:
        need, counters = ext.attention_paged_workspace_bytes(*key[1:])
        plan = (need, counters if counters else -1)
        _ws_plan[key] = plan
    ws, ws_bytes = _workspace(plan, dev, _stream(dev))
    out = torch.empty_like(q)
    _call(ext.attention_paged, dev, q.data_ptr(), _HALF_DTYPES[dtype], B, T, n_heads, *cache,
          lengths.data_ptr(), sizes.data_ptr() if sizes is not None else None,
          0 if window is None else min(int(window), 1 << 30), min(int(sinks), 1 << 30),
          float(D ** -0.5 if scale is None else scale), out.data_ptr(),
          ws.data_ptr() if ws is not None else None, ws_bytes)
    return out


def paged_values(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, scales: Optional[Scales] = None,
                 dtype: Optional[torch.dtype] = None,
                 rows: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows that the sequences' pages hold, as dense caches of
    :mod:`nibblegemm_amd.glue`: keys and values [B, n_kv, rows, D], the first
    ``rows`` rows of every sequence (all that the table has room for by default),
    zeros from ``lengths[b]`` on and where there is no page.  ``dtype`` is that of
    16-bit pages; of 8-bit ones fp16 (the default) or bf16, and the values are
    exact where the append for that type wrote them."""
    if scales is None:
        _check_types(k_pages, "k_pages", v_pages=v_pages)
        if dtype is not None and dtype != k_pages.dtype:
            raise RuntimeError(f"the values of {k_pages.dtype} pages are {k_pages.dtype}, not {dtype}")
        dtype = k_pages.dtype
    else:
        _check_gpu("k_pages", k_pages, k_pages)
        dtype = torch.float16 if dtype is None else dtype
        if dtype not in _HALF_DTYPES:
            raise RuntimeError(f"dtype must be fp16 or bf16, got {dtype}")
    dev = k_pages.device
    B, cache = _check_cache(k_pages, v_pages, table, scales, dev.index, False)
    n_kv, D = cache[6], cache[8]
    _check_index("lengths", lengths, (B,), k_pages)
    rows = cache[7] * cache[9] if rows is None else int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative, got {rows}")
    k, v = (torch.empty((B, n_kv, rows, D), dtype=dtype, device=dev) for _ in range(2))
    _call(_native.binding().paged_values, dev, *cache, _HALF_DTYPES[dtype], B, lengths.data_ptr(),
          rows, k.data_ptr(), v.data_ptr())
    return k, v


__all__ = ["PAGE_ROWS", "attention_paged", "paged_append", "paged_cache", "paged_values"]
