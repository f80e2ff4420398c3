"""Attention of packed, paged and shared-prefix batches.

The operator of this package picks keys for a sparse attention; next to it a
serving step attends densely: to prompts that are shorter than the selection, in
layers without an indexer, and to long prefixes that a batch has in common.  The
layouts are those of ``batched`` and ``paged``: queries packed as ``[sum Q_b, Hq, D]``
with int32 prefix sums, the queries of a request being its LAST ``Q_b`` tokens, keys
and values packed as ``[sum N_b, H, D]`` or in pools of pages (``page_size`` a multiple
of 128) behind a block table.  ``Hq`` is a multiple of ``H``; query head ``h`` reads key
head ``h // (Hq // H)``.  The reference selects keys only and attends nowhere.

* ``attention_varlen``: whole prompts, chunks at the end of a context, single tokens;
* ``attention_paged``: the same with keys behind a block table;
* ``shared_prefix_attention``, ``shared_prefix_attention_paged``: a prefix that the
  whole batch shares, read once for all requests, in front of every request's own keys.

All of them take bf16 or fp16 with head dimension 64 or 128, keep scores, softmax
statistics and sums in fp32, round the softmax weights to the element type once, for the
product with the values, and never read lengths back to the host, so a call can be
captured into a CUDA graph and replayed with other lengths in the same buffers.  A row
that sees no key, or whose scores are all ``-inf``, gets zeros and a log-sum-exp of
``-inf``.  There is no backward pass: the framework serves, and tensors that ask for
gradients or carry forward-mode tangents are refused.

A call takes its workspace from the caching allocator, and a captured graph keeps its
own: 4 MB for a single token, up to 175 MB for the partial results of long entries that
are cut (64 tokens of 64/8 heads: 135 MB), and about 1 KB per row and query head more
with a prefix (8192 rows of 64 heads: 674 MB).  The first call with given shapes and types
takes about 45 us of host time for its checks, later ones 18.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any

from . import _lib
from .operator import _require

TILE_KEYS = 128
check_status = _lib.check_serving_status


def _rows_ok(tensor: Any) -> bool:
    """Contiguous heads whose strides keep them on 16-byte boundaries."""

    *outer, inner = tensor.stride()
    return inner == 1 and all(s % 8 == 0 for s in outer)


def _check_kv(q: Any, k: Any, v: Any, what: str, rank: int) -> None:
    _require(k.dim() == rank and k.shape == v.shape,
             f"{what} keys and values must both have shape {'[N, H, D]' if rank == 3 else '[P, page_size, H, D]'}")
    _require(k.dtype == q.dtype and v.dtype == q.dtype, f"{what} keys and values must have the type of q")
    _require(k.device == q.device and v.device == q.device, f"{what} keys and values must live on the same device as q")
    _require(k.shape[-1] == q.shape[-1], f"{what} keys must have the head dimension of q")
    heads = k.shape[-2]
    _require(heads > 0 and q.shape[1] > 0 and q.shape[1] % heads == 0 and q.shape[1] // heads <= 128,
             f"the query heads must be a multiple of the {what} key heads, at most 128 times as many")
    _require(k.numel() == 0 or (_rows_ok(k) and _rows_ok(v)),
             f"{what} keys and values must be contiguous in their last dimension and 16-byte aligned in every row")
    _require(rank == 4 or k.shape[0] <= _lib.MAX_ATTENTION_KEYS, f"need less than 2^31 {what} keys, at most {_lib.MAX_ATTENTION_KEYS}")
    if rank == 4:
        pages, page_size = k.shape[:2]
        _require(pages > 0 and page_size > 0 and page_size % TILE_KEYS == 0, "page_size must be a positive multiple of 128")
        _require(pages * page_size < 1 << 31, "pages * page_size must stay below 2^31")


def _check_ints(torch: Any, tensor: Any, name: str, device: Any, count: int | None) -> None:
    _require(tensor.dtype == torch.int32 and tensor.dim() == 1 and tensor.is_contiguous(), f"{name} must be contiguous int32")
    _require(count is None or tensor.shape[0] == count, f"{name} must have {count} entries")
    _require(tensor.device == device, f"{name} must live on the same device as q")


def _segment(k: Any, v: Any, table: Any = None) -> Any:
    """Strides and sizes of packed (``table`` is None) or paged keys, without their addresses."""

    if table is None:
        return _lib.KvSegment(0, 0, k.stride(0), k.stride(1), 0, v.stride(0), v.stride(1), 1, k.shape[0], 0)
    return _lib.KvSegment(table.stride(0) if table.dim() == 2 else 0, *k.stride()[:3], *v.stride()[:3],
                          k.shape[0], k.shape[1], table.shape[-1])


def _check_call(torch: Any, q: Any, own: tuple, prefix: tuple | None, prefix_keys: int, cu_seqlens_q: Any, lengths: Any, out: Any,
                causal: bool, scale: float | None) -> _lib.CallTemplate:
    """``own`` and ``prefix`` are ``(k, v)`` packed or ``(k_pool, v_pool, table)``; ``lengths`` are cumulative for packed keys."""

    _require(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    _require(q.dim() == 3, "q must have shape [T, Hq, D]")
    _require(q.dtype in (torch.bfloat16, torch.float16), "q must be bfloat16 or float16")
    tokens, heads, dim = q.shape
    device = q.device
    _require(dim in (64, 128), "the head dimension must be 64 or 128")
    _require(q.numel() == 0 or _rows_ok(q), "q must be contiguous in its last dimension and 16-byte aligned in every row")
    _require(tokens * heads < 1 << 31, "rows * heads must stay below 2^31")
    paged = len(own) == 3
    _check_kv(q, own[0], own[1], "own", 4 if paged else 3)
    _check_ints(torch, cu_seqlens_q, "cu_seqlens_q", device, None)
    requests = cu_seqlens_q.shape[0] - 1
    _require(requests >= 1, "cu_seqlens_q must be [B+1] with B >= 1")
    if paged:
        table = own[2]
        _require(table.dtype == torch.int32 and table.dim() == 2, "block_table must be int32 [B, table_pages]")
        _require(table.shape[0] == requests, "block_table must have one row per request")
        _require(table.shape[1] > 0, "block_table must have at least one column")
        _require(table.device == device, "block_table must live on the same device as q")
        _require((table.stride(1) == 1 or table.shape[1] == 1) and table.stride(0) >= 0, "block_table rows must be contiguous")
        _check_ints(torch, lengths, "seqlens_k", device, requests)
    else:
        _check_ints(torch, lengths, "cu_seqlens_k", device, requests + 1)
    if prefix is not None:
        _check_kv(q, prefix[0], prefix[1], "prefix", 4 if paged else 3)
        _require(prefix[0].shape[-2] == own[0].shape[-2], "prefix and own keys must have the same heads")
        if paged:
            _check_ints(torch, prefix[2], "prefix_table", device, None)
            _require(0 <= prefix_keys <= prefix[2].shape[0] * own[0].shape[1], "prefix_table does not cover the prefix keys")
            _require(prefix_keys <= _lib.MAX_ATTENTION_KEYS, f"need at most {_lib.MAX_ATTENTION_KEYS} prefix keys")
    if out is not None:
        _require(out.shape == q.shape and out.dtype == q.dtype and out.device == device and (out.numel() == 0 or _rows_ok(out)),
                 "out must have the shape, type and device of q and 16-byte aligned rows")
        strides = sorted((s, n) for s, n in zip(out.stride()[:2], out.shape[:2]) if n > 1)
        _require(all(s >= dim for s, _ in strides) and (len(strides) < 2 or strides[1][0] >= strides[0][0] * strides[0][1]),
                 "out must not overlap itself")
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    _require(0.0 < scale < 1e38, "scale must be positive and finite")
    strides = out.stride() if out is not None else (heads * dim, dim)
    args = _lib.AttentionArgs(
        None, None, None, None, None, None, None, 0, None, None, None, None, None, None, q.stride(0), q.stride(1), strides[0], strides[1], 0, _segment(*own),
        _segment(*prefix) if prefix_keys else _lib.KvSegment(), scale,
        _lib.ELEMENT_BF16 if q.dtype == torch.bfloat16 else _lib.ELEMENT_FP16, tokens, heads, own[0].shape[-2], dim, requests,
        prefix_keys, int(causal), 3 if out is None else 2, 0)
    needed = ctypes.c_size_t(0)
    if tokens:
        _lib.check(_lib.load_library().itk_attention_workspace_bytes(ctypes.byref(args), ctypes.byref(needed)))
    return _lib.CallTemplate(args, workspace_bytes=needed.value, device=device, tokens=tokens, paged=paged)


_TEMPLATES: dict = {}


def _attend(q: Any, own: tuple, prefix: tuple | None, prefix_keys: int, cu_seqlens_q: Any, lengths: Any, causal: bool,
            scale: float | None, out: Any, return_lse: bool) -> Any:
    import torch

    tensors = (q, cu_seqlens_q, lengths, *own)
    if prefix is not None:
        tensors += prefix
    if out is not None:
        tensors += (out,)
    if scale is not None:
        scale = float(scale)
    _lib.refuse_gradients(torch, *tensors)
    key = (_lib.metadata(torch, tensors), len(own), prefix is not None, prefix_keys, bool(causal), scale)
    template = _TEMPLATES.get(key)
    if template is None:
        template = _lib.CallTemplate.keep(_TEMPLATES, key, _check_call(
            torch, q, own, prefix, prefix_keys, cu_seqlens_q, lengths, out, causal, scale))
    written = () if out is None else (out,)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)      # (new_empty takes 0.8 us longer)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    if template.tokens:
        # of the caching allocator, on the call's stream: two calls, streams or captured graphs never share it
        workspace = q.new_empty(template.workspace_bytes, dtype=torch.uint8)
        # in the order of the argument block: rows, lengths, workspace, own keys, prefix
        k, v = own[0].data_ptr(), own[1].data_ptr()
        rows, result, ends = q.data_ptr(), out.data_ptr(), lengths.data_ptr()
        words = [rows, result, 0 if lse is None else lse.data_ptr(), cu_seqlens_q.data_ptr(), 0 if template.paged else ends,
                 ends if template.paged else 0, workspace.data_ptr(), template.workspace_bytes, k, v,
                 own[2].data_ptr() if template.paged else 0]
        aligned = rows | result | k | v
        if prefix_keys:
            k, v = prefix[0].data_ptr(), prefix[1].data_ptr()
            words += [k, v, prefix[2].data_ptr() if template.paged else 0]
            aligned |= k | v
        _require(aligned & 15 == 0, "q, out, keys and values must be 16-byte aligned")
        _lib.launch(torch, _lib.load_library().itk_attention, template.fill(words), template.device, written)
    return (out, lse) if return_lse else out


def attention_varlen(q: Any, kv: tuple[Any, Any], cu_seqlens_q: Any, cu_seqlens_k: Any, *, causal: bool = True,
                     scale: float | None = None, out: Any = None, return_lse: bool = False) -> Any:
    """Attention of a packed batch; ``[T, Hq, D]`` like ``q``, with ``return_lse`` also fp32 ``[T, Hq]``.

    ``q`` is ``[T, Hq, D]``, ``kv = (k, v)`` both ``[N, H, D]``; request ``b`` owns rows
    ``cu_seqlens_q[b]:cu_seqlens_q[b+1]`` and keys ``cu_seqlens_k[b]:cu_seqlens_k[b+1]`` (int32 ``[B+1]`` each, lengths of
    zero allowed).  With ``causal`` row i of its Q sees its first ``N - Q + i + 1`` keys, else all N.  ``scale`` (positive)
    defaults to ``D ** -0.5``.  Rows of no request are zero, or left as they were in a given ``out``; their
    log-sum-exp is ``-inf``.  ``out`` may be ``q`` itself and shares no other memory with the inputs.
    """

    return _attend(q, tuple(kv), None, 0, cu_seqlens_q, cu_seqlens_k, causal, scale, out, return_lse)


def attention_paged(q: Any, pools: tuple[Any, Any], block_table: Any, cu_seqlens_q: Any, seqlens_k: Any, *, causal: bool = True,
                    scale: float | None = None, out: Any = None, return_lse: bool = False) -> Any:
    """``attention_varlen`` with the keys in ``pools = (k_pool, v_pool)``, both ``[P, page_size, H, D]``.

    Key j of request b lies on page ``block_table[b, j // page_size]`` (int32 ``[B, table_pages]``); ``seqlens_k`` int32 ``[B]``
    counts the request's keys (``PagePlan.lengths``).  Page ids outside the pool are clamped and reported by
    ``check_status``.
    """

    return _attend(q, (*pools, block_table), None, 0, cu_seqlens_q, seqlens_k, causal, scale, out, return_lse)


def shared_prefix_attention(q: Any, prefix_kv: tuple[Any, Any], kv: tuple[Any, Any], cu_seqlens_q: Any, cu_seqlens_k: Any, *,
                            scale: float | None = None, out: Any = None, return_lse: bool = False) -> Any:
    """Causal attention of a packed batch whose requests all continue the same prefix.

    ``prefix_kv`` ``[P, H, D]`` each: every row sees all P prefix keys, then its own keys as in ``attention_varlen``.  The
    prefix is attended by the rows of all requests together, so its keys and values are read once for the batch.
    """

    return _attend(q, tuple(kv), tuple(prefix_kv), prefix_kv[0].shape[0], cu_seqlens_q, cu_seqlens_k, True, scale, out, return_lse)


def shared_prefix_attention_paged(q: Any, pools: tuple[Any, Any], prefix_table: Any, prefix_keys: int, block_table: Any,
                                  cu_seqlens_q: Any, seqlens_k: Any, *, scale: float | None = None, out: Any = None,
                                  return_lse: bool = False) -> Any:
    """``shared_prefix_attention`` with prefix and own keys in the same pools.

    ``prefix_table`` int32 lists the pages of the ``prefix_keys`` prefix keys; ``block_table`` and ``seqlens_k`` describe every
    request's own keys, which start on a page of their own.
    """

    return _attend(q, (*pools, block_table), (*pools, prefix_table), int(prefix_keys), cu_seqlens_q, seqlens_k, True, scale, out,
                   return_lse)


__all__ = ["attention_paged", "attention_varlen", "check_status", "shared_prefix_attention", "shared_prefix_attention_paged"]
