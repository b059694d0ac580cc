"""Decode-step glue around the projections: RMSNorm and grouped-query attention
over a KV cache, as HIP kernels (``nibble_rmsnorm_f16`` and
``nibble_attention_decode_f16`` of the C ABI), and the same step for several
tokens of several sequences at once: head norms, rotary embedding and the cache
append in one pass (``nibble_qk_norm_rope``) and attention of a tree of drafted
tokens over the cache (``nibble_attention_tree``).

The reference runs these as PyTorch / transformers ops of the model it
decodes with QuantLinear layers swapped in (bench/bench_model.py:131-154,
:177-188).  Here they let a whole Llama-shaped token step -- norms,
projections, attention, residual adds -- run as kernels in one HIP graph
(:class:`nibblegemm_amd.decode_step.GlueDecodeStep`).

Like every kernel entry point of this package, these raise RuntimeError when
the native library is missing; there is no PyTorch fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native
from .ops import _call, _check_no_backward, _raise, _stream, _workspace, _ws_plan

HEAD_DIM = 128
LLAMA3_ROPE_THETA = 500000.0


def _check_f16(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU")
    if t.dtype != torch.float16:
        raise RuntimeError(f"{name} must be fp16, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """``fp16(x * r * weight)`` per row, ``r = 1 / sqrt(mean(x^2) + eps)``,
    computed in fp32 with one rounding (transformers' LlamaRMSNorm rounds
    ``x * r`` to fp16 before the weight).  x fp16 [rows, cols], weight fp16
    [cols]; cols a multiple of 8 up to 16384."""
    _check_f16("x", x)
    _check_f16("weight", weight)
    if x.dim() != 2 or weight.dim() != 1 or weight.numel() != x.size(1):
        raise ValueError(f"expected x [rows, cols] and weight [cols], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if weight.device != x.device:
        raise RuntimeError("x and weight must be on the same device")
    ext = _native.binding()
    y = torch.empty_like(x)
    rc = ext.rmsnorm(x.data_ptr(), x.size(0), x.size(1), weight.data_ptr(), float(eps),
                     y.data_ptr(), _stream(x.device))
    if rc:
        _raise(rc, ext)
    return y


def rope_tables(max_seq: int, head_dim: int = HEAD_DIM, theta: float = LLAMA3_ROPE_THETA,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, fp32 [max_seq, head_dim / 2], of the rotary embedding
    ``angle(p, i) = p * theta^(-2 i / head_dim)`` (computed in float64)."""
    inv = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    ang = torch.outer(torch.arange(max_seq, dtype=torch.float64), inv)
    return (ang.cos().float().to(device).contiguous(), ang.sin().float().to(device).contiguous())


def attention_decode(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: int,
                     rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """Attention of the token at position ``pos`` over the cache, which
    holds tokens ``0 .. pos - 1``.

    qkv fp16 [1, (n_heads + 2 n_kv) * 128]: the token's q | k | v (the q|k|v
    projection's output).  k_cache, v_cache fp16 [n_kv, max_seq, 128]; the
    call writes the token's k (rotated) and v at row ``pos`` (and raises the
    caches' version counters, as a tensor operation would).  Returns fp16
    [1, n_heads * 128] = ``softmax(q k^T / sqrt(128)) v`` per query head,
    head i reading kv head ``i // (n_heads // n_kv)``.  ``rope`` is the
    (cos, sin) pair of :func:`rope_tables` or None."""
    for name, t in (("qkv", qkv), ("k_cache", k_cache), ("v_cache", v_cache)):
        _check_f16(name, t)
    if k_cache.dim() != 3 or k_cache.shape != v_cache.shape or k_cache.size(2) != HEAD_DIM:
        raise ValueError(f"caches must both be [n_kv, max_seq, {HEAD_DIM}], got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    n_kv, max_seq = k_cache.size(0), k_cache.size(1)
    if qkv.dim() != 2 or qkv.size(0) != 1 or qkv.size(1) % HEAD_DIM:
        raise ValueError(f"qkv must be [1, (n_heads + 2 n_kv) * {HEAD_DIM}], got {tuple(qkv.shape)}")
    n_heads = qkv.size(1) // HEAD_DIM - 2 * n_kv
    if rope is not None:
        cos, sin = rope
        for name, t in (("rope cos", cos), ("rope sin", sin)):
            if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous fp32 GPU tensor")
            if t.shape != (max_seq, HEAD_DIM // 2):
                raise ValueError(f"{name} must be [{max_seq}, {HEAD_DIM // 2}], got {tuple(t.shape)}")
        cos_p, sin_p = cos.data_ptr(), sin.data_ptr()
    else:
        cos_p = sin_p = None
    ext = _native.binding()
    dev = qkv.device
    stream = _stream(dev)
    key = ("attention", n_heads, n_kv, max_seq, pos)
    plan = _ws_plan.get(key)
    if plan is None:
        plan = ext.attention_workspace_bytes(n_heads, n_kv, HEAD_DIM, max_seq, pos, stream)
        _ws_plan[key] = plan
    ws, ws_bytes = _workspace(plan, dev, stream)
    out = torch.empty((1, max(n_heads, 0) * HEAD_DIM), dtype=torch.float16, device=dev)
    rc = ext.attention(qkv.data_ptr(), n_heads, n_kv, HEAD_DIM, k_cache.data_ptr(),
                       v_cache.data_ptr(), max_seq, int(pos), cos_p, sin_p, out.data_ptr(),
                       ws.data_ptr() if ws is not None else None, ws_bytes, stream)
    if rc:
        _raise(rc, ext)
    increment_version((k_cache, v_cache))
    return out


def attention_bytes(n_kv: int, pos: int) -> int:
    """Cache bytes one call reads and writes: k and v rows 0 .. pos."""
    return 2 * n_kv * (pos + 1) * HEAD_DIM * 2


_HALF_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def _check_half(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.dtype not in _HALF_DTYPES:
        raise RuntimeError(f"{name} must be fp16 or bf16, got {t.dtype}")
    if t.dtype != like.dtype:
        raise RuntimeError(f"{name} must be {like.dtype}, got {t.dtype}")
    _check_gpu(name, t, like)
    _check_no_backward(name, t)
    if t.is_neg():
        raise RuntimeError(f"{name} must hold its values as they are (resolve_neg)")


def _in_order(dtype: torch.dtype, index: int, *tensors: Optional[torch.Tensor]) -> bool:
    """Whether every tensor passes :func:`_check_half` beside one of this dtype
    on this GPU, at a glance: the checks that name what is wrong take longer
    than a small call's kernel."""
    if index < 0 or dtype not in _HALF_DTYPES or getattr(forward_ad, "_current_level", -1) >= 0:
        return False
    for t in tensors:
        if t is not None and (t.dtype is not dtype or t.get_device() != index or t.requires_grad
                              or t.is_neg()):
            return False
    return True


def _check_gpu(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU")
    if t.device != like.device:
        raise RuntimeError(f"{name} must live on {like.device}, got {t.device}")


def _check_index(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> None:
    if (t.dtype is torch.int32 and t.get_device() == like.get_device() and t.shape == shape
            and t.is_contiguous()):
        return
    _check_gpu(name, t, like)
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 tensor")
    raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def _cache_strides(x: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor):
    """Checks the caches' shapes beside the tokens ``x`` ``[B, T, ..]`` or
    ``[T, ..]``: their batched shape, and the batch, head and row strides of
    both."""
    shape = k_cache.shape
    if v_cache.shape != shape:
        raise ValueError(f"caches must have one shape, got {tuple(shape)} and {tuple(v_cache.shape)}")
    if len(shape) != x.dim() + 1:
        raise ValueError(f"caches must have {x.dim() + 1} dimensions beside {x.dim()} of the tokens, "
                         f"got {tuple(shape)}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if len(shape) == 3:
        shape, ks, vs = (1, *shape), (0, *ks), (0, *vs)
    elif shape[0] != x.shape[0]:
        raise ValueError(f"caches of {shape[0]} sequences beside tokens of {x.shape[0]}")
    if 0 in shape[1:]:
        raise ValueError(f"the caches are empty: {tuple(shape)}")
    if ks[3] != 1 or vs[3] != 1:
        raise RuntimeError("the elements of a cache row must be adjacent")
    return shape, ks, vs


def qk_norm_rope(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 positions: torch.Tensor, slots: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5,
                 rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """Norms of the query and key heads, their rotary embedding and the cache
    append of ``T`` tokens of ``B`` sequences, in one pass.

    qkv fp16 or bf16 [B, T, (n_heads + 2 n_kv) * D], the q|k|v projection's
    output, D 64 or 128.  k_cache, v_cache [B, n_kv, max_seq, D] of its dtype,
    of any strides that are multiples of 8 with a row's elements adjacent.
    ``positions`` and ``slots`` int32 [B, T]: a token's rotary position and its
    cache row.  Each q and k head is normalised, ``x / sqrt(mean(x^2) + eps) *
    weight`` (weights [D] of qkv's dtype; None: no norm of those heads), then
    rotated by the (cos, sin) of :func:`rope_tables` (None: no rotation), in
    fp32 with one rounding.  k and v go to row ``slots`` of their sequence's
    caches, whose version counters rise; q is returned as [B, T, n_heads * D].

    A token whose slot is no row of the cache (-1, say) or whose position is
    no row of the tables is padding: it writes no cache row and its q is zero.
    The slots of one sequence's tokens must differ: of two tokens in one row
    either may remain, in parts of 16 bytes.  One sequence may come without
    its batch dimension: qkv [T, ..] (and q so), caches [n_kv, max_seq, D],
    positions and slots [T].  Positions, slots and caches are read on the GPU,
    so a captured call follows their contents.  There is no backward."""
    dtype, dev = qkv.dtype, qkv.device
    if not _in_order(dtype, qkv.get_device(), qkv, k_cache, v_cache, q_weight, k_weight):
        for name, t in (("qkv", qkv), ("k_cache", k_cache), ("v_cache", v_cache),
                        ("q_weight", q_weight), ("k_weight", k_weight)):
            if t is not None:
                _check_half(name, t, qkv)
    if qkv.dim() not in (2, 3) or not qkv.is_contiguous():
        raise RuntimeError("qkv must be a contiguous [B, T, ..] or [T, ..] tensor")
    (B, n_kv, max_seq, D), ks, vs = _cache_strides(qkv, k_cache, v_cache)
    for n, k, v in zip((B, n_kv, max_seq), ks, vs):
        if n > 1 and (k == 0 or v == 0):
            raise RuntimeError("the caches are written and must not be expanded views")
    lead = qkv.shape[:-1]
    T, width = qkv.shape[-2:]
    n_heads = width // D - 2 * n_kv
    if width % D or n_heads < 1:
        raise ValueError(f"qkv must be [.., (n_heads + 2 * {n_kv}) * {D}], got {tuple(qkv.shape)}")
    _check_index("positions", positions, lead, qkv)
    _check_index("slots", slots, lead, qkv)
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and (t.shape != (D,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [{D}] tensor, got {tuple(t.shape)}")
    cos_p = sin_p = None
    rope_rows = 0
    if rope is not None:
        cos, sin = rope
        for name, t in (("rope cos", cos), ("rope sin", sin)):
            if t.get_device() != dev.index:
                _check_gpu(name, t, qkv)
            _check_no_backward(name, t)
            if t.dtype is not torch.float32 or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous fp32 GPU tensor")
            if t.dim() != 2 or t.shape != (cos.shape[0], D // 2) or t.shape[0] < 1:
                raise ValueError(f"{name} must be [rows, {D // 2}], got {tuple(t.shape)}")
        cos_p, sin_p, rope_rows = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    out = torch.empty((*lead, n_heads * D), dtype=dtype, device=dev)
    _call(_native.binding().qk_norm_rope, dev, qkv.data_ptr(), _HALF_DTYPES[dtype], B, T, n_heads,
          n_kv, D, k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
          max_seq, positions.data_ptr(), slots.data_ptr(),
          q_weight.data_ptr() if q_weight is not None else None,
          k_weight.data_ptr() if k_weight is not None else None, float(eps), cos_p, sin_p,
          rope_rows, out.data_ptr())
    increment_version((k_cache, v_cache))  # (autograd may have saved one before)
    return out


def attention_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   lengths: torch.Tensor, mask: Optional[torch.Tensor] = None,
                   sizes: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of trees of drafted tokens over their sequences' caches.

    q fp16 or bf16 [B, T, n_heads * D], as :func:`qk_norm_rope` returns it, D
    64 or 128; k_cache, v_cache [B, n_kv, max_seq, D] as there.  ``lengths``
    int32 [B]: the rows a sequence's cache held before its tree; the tree's
    tokens lie in the rows behind them, in order.  ``mask`` bool [T, T] or
    [B, T, T]: ``mask[i, j]`` is whether token i sees token j (:func:`tree_mask`
    makes one from parents); None: the tokens up to itself, a run of tokens
    such as a prompt's next part.  ``sizes`` int32 [B]: the tokens of each
    sequence's tree, T where it is None.  Every token sees all ``lengths`` rows
    before the tree.  Returns [B, T, n_heads * D]: per query head
    ``softmax(scale q k^T) v`` over what the token sees, head i reading kv head
    ``i // (n_heads // n_kv)``, scale ``1 / sqrt(D)`` by default, in fp32 with
    the probabilities rounded to q's dtype (in fp16 those below 2^-21 of the
    largest in steps of 2^-31 of it).  Scores are below 2^28 log(2) in magnitude,
    2^31 log(2) in bf16: their rounding in fp32 would overflow beyond.

    Tokens behind a sequence's last, and tokens that see nothing, give zeros.
    Rows that a token does not see have no part in its output, whatever they
    hold; rows behind the tree are not read.  An infinity in the values of a row
    that it sees comes out as it is, or as NaN where the row's weight rounds to
    zero; a NaN as NaN.  ``lengths`` and ``sizes`` count
    as far as the cache goes.  One sequence may come without its batch
    dimension: q [T, ..], caches [n_kv, max_seq, D], lengths [1], sizes [1].
    Lengths, sizes and mask are read on the GPU, so a captured call follows
    their contents.  There is no backward."""
    dtype, dev = q.dtype, q.device
    if not _in_order(dtype, q.get_device(), q, k_cache, v_cache):
        for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
            _check_half(name, t, q)
    if q.dim() not in (2, 3) or not q.is_contiguous():
        raise RuntimeError("q must be a contiguous [B, T, ..] or [T, ..] tensor")
    (B, n_kv, max_seq, D), ks, vs = _cache_strides(q, k_cache, v_cache)
    T, width = q.shape[-2:]
    n_heads = width // D
    if width % D:
        raise ValueError(f"q must be [.., n_heads * {D}], got {tuple(q.shape)}")
    _check_index("lengths", lengths, (B,), q)
    if sizes is not None:
        _check_index("sizes", sizes, (B,), q)
    mask_p, mask_batches = None, 1
    if mask is not None:
        if mask.get_device() != dev.index:
            _check_gpu("mask", mask, q)
        if mask.dtype is not torch.bool or not mask.is_contiguous():
            raise RuntimeError("mask must be a contiguous bool tensor")
        if mask.shape not in ((T, T), (B, T, T)):
            raise ValueError(f"mask must be [{T}, {T}] or [{B}, {T}, {T}], got {list(mask.shape)}")
        mask_p, mask_batches = mask.data_ptr(), B if mask.dim() == 3 else 1
    ext = _native.binding()
    key = ("tree", B, T, n_heads, n_kv, D, max_seq)
    plan = _ws_plan.get(key)
    if plan is None:
        plan = (ext.attention_tree_workspace_bytes(B, T, n_heads, n_kv, D, max_seq), -1)
        _ws_plan[key] = plan
    ws, ws_bytes = _workspace(plan, dev, _stream(dev))
    out = torch.empty_like(q)
    _call(ext.attention_tree, dev, q.data_ptr(), _HALF_DTYPES[dtype], B, T, n_heads, n_kv, D,
          k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2], max_seq,
          lengths.data_ptr(), mask_p, mask_batches, sizes.data_ptr() if sizes is not None else None,
          float(D ** -0.5 if scale is None else scale), out.data_ptr(),
          ws.data_ptr() if ws is not None else None, ws_bytes)
    return out


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """The mask of :func:`attention_tree` for trees given by ``parents``, int
    [T] or [B, T]: the index of a token's parent, which comes before it, or -1
    for a token that follows the cached ones.  bool [T, T] or [B, T, T]: a
    token sees itself and its ancestors.  Tensor operations on the parents' device,
    a few for each level of the deepest tree, which wait for their results: masks
    are made outside a captured step, and on the CPU where the parents are there."""
    if parents.dim() not in (1, 2) or parents.is_floating_point():
        raise ValueError(f"parents must be an integer [T] or [B, T] tensor, got {parents.dtype} "
                         f"{tuple(parents.shape)}")
    p = (parents if parents.dim() == 2 else parents[None]).long()
    T = p.shape[-1]
    i = torch.arange(T, device=p.device)
    if bool((p >= i).any()) or bool((p < -1).any()):
        raise ValueError("a parent must come before its token, or be -1")
    seen = torch.eye(T, dtype=torch.bool, device=p.device).expand(p.shape[0], T, T).clone()
    at = p  # the ancestor each token has reached
    while bool((at >= 0).any()):
        b, t = (at >= 0).nonzero(as_tuple=True)
        seen[b, t, at[b, t]] = True
        at = torch.where(at >= 0, p.gather(1, at.clamp(min=0)), -1)
    return seen.reshape(*parents.shape, T)


__all__ = ["HEAD_DIM", "LLAMA3_ROPE_THETA", "rmsnorm", "rope_tables", "attention_decode",
           "attention_bytes", "qk_norm_rope", "attention_tree", "tree_mask"]
