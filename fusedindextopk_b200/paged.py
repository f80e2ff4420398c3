"""Index keys in a paged cache.

Serving stacks keep keys in fixed-size pages handed out by an allocator, so a
sequence's keys are not contiguous.  The reference supports contiguous keys only
(``src/fused_index_topk/inputs.py:31-32``).  Here the pool is
``kv_pool [pages, page_size, 128]`` e4m3 with ``scale_pool [pages, page_size]``
fp32, and ``block_table`` (int32) lists the pages of the logical key sequence in
order.  ``page_size`` must be a multiple of 128, the kernel's key tile: the TMA
producer, the epilogue's scale load and the sample gather then only swap the
tile's row offset (``tile_table[t] * 128``), and everything a caller sees (ids,
``[k_start, k_end)``, the number of keys) stays in logical positions.

Together with ``batched.varlen_ranges`` one block table serves a whole batch: the
logical key space is the concatenation of the sequences, each starting on a page
boundary.

The bookkeeping of such a cache runs on the device as well, without a host read:
``plan_pages`` turns request lengths and a list of free pages into block tables,
slots, the flat block table and the key ranges that ``fused_index_topk_paged``
takes; ``append_tokens`` writes a step's keys, values and (quantised) index keys
to those slots; ``attention.attention_paged`` reads them.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Any

from . import _lib
from .operator import _WORKSPACES, Workspace, _require, make_workspace, replay_or_run

TILE_KEYS = 128


def expand_block_table(block_table: Any, page_size: int) -> Any:
    """int32 ``[pages_used]`` pages -> int32 ``[pages_used * page_size / 128]`` physical 128-key tiles."""

    import torch

    _require(page_size >= TILE_KEYS and page_size % TILE_KEYS == 0, "page_size must be a positive multiple of 128")
    _require(block_table.dtype == torch.int32 and block_table.dim() == 1, "block_table must be int32 [pages]")
    per_page = page_size // TILE_KEYS
    within = torch.arange(per_page, device=block_table.device, dtype=torch.int32)
    return (block_table.unsqueeze(1) * per_page + within.unsqueeze(0)).reshape(-1).contiguous()


def _tile_table_buffers(workspace: Workspace, pages_used: int, per_page: int, device: Any) -> dict[str, Any]:
    """Workspace-owned buffers of the per-call block-table expansion (allocated once per table length)."""

    import torch

    key = f"paged_{pages_used}_{per_page}"
    buffers = workspace.buffers.get(key)
    if buffers is None:
        buffers = {
            "pages": torch.empty(pages_used, device=device, dtype=torch.int32),
            "tiles": torch.empty(pages_used * per_page, device=device, dtype=torch.int32),
            "within": torch.arange(per_page, device=device, dtype=torch.int32),
            "bad": torch.zeros(pages_used, device=device, dtype=torch.bool),
            "bad_any": torch.zeros(1, device=device, dtype=torch.bool),
        }
        workspace.buffers[key] = buffers
    return buffers


def _expand_on_device(buffers: dict[str, Any], block_table: Any, pages: int) -> None:
    """Physical 128-key tiles of the block table as it is NOW, into the workspace's buffer.

    Enqueued on every call (and part of the replayed CUDA graph), because a serving engine updates its
    block table in place, often from its own kernels, without any host-visible version change.  An
    entry outside the pool is clamped, so that the kernels never read outside the pool, and recorded:
    ``block_table_was_valid`` reports it.
    """

    import torch

    per_page = int(buffers["within"].numel())
    torch.clamp(block_table, 0, pages - 1, out=buffers["pages"])
    torch.ne(block_table, buffers["pages"], out=buffers["bad"])
    torch.any(buffers["bad"], dim=0, keepdim=True, out=buffers["bad_any"])
    torch.mul(buffers["pages"], per_page, out=buffers["pages"])
    torch.add(buffers["pages"].unsqueeze(1), buffers["within"].unsqueeze(0), out=buffers["tiles"].view(-1, per_page))


def block_table_was_valid(workspace: Workspace) -> bool:
    """Whether every block-table entry of the paged calls made through this workspace named a pool page.

    Synchronises; meant for tests and for debugging a serving integration, not for the hot path.
    """

    for name, buffers in workspace.buffers.items():
        if name.startswith("paged_") and bool(buffers["bad_any"].item()):
            return False
    return True


def scatter_to_pages(kv: Any, kv_scales: Any, page_size: int, *, pool_pages: int | None = None,
                     generator: Any = None) -> tuple[Any, Any, Any]:
    """Place contiguous keys into randomly chosen pages of a fresh pool.

    Returns ``(kv_pool [P, page_size, 128], scale_pool [P, page_size], block_table int32)``; unused
    pool rows are filled with a byte pattern and NaN scales so that a wrong page shows up in results.
    For tests and for callers migrating a contiguous cache.
    """

    import torch

    keys = int(kv.shape[0])
    used = (keys + page_size - 1) // page_size
    pool_pages = max(used, pool_pages or used + 3)
    order = torch.randperm(pool_pages, generator=generator)[:used].to(torch.int32)
    kv_pool = torch.full((pool_pages * page_size, _lib.HEAD_DIM), 0x3C, dtype=torch.uint8, device=kv.device)
    scale_pool = torch.full((pool_pages * page_size,), float("nan"), dtype=torch.float32, device=kv.device)
    rows = torch.arange(keys, device=kv.device)
    target = order.to(kv.device).long()[rows // page_size] * page_size + rows % page_size
    kv_pool[target] = kv.view(torch.uint8)
    scale_pool[target] = kv_scales
    return (kv_pool.view(torch.float8_e4m3fn).view(pool_pages, page_size, _lib.HEAD_DIM),
            scale_pool.view(pool_pages, page_size), order.to(kv.device))


def fused_index_topk_paged(q: Any, kv_pool_pair: tuple[Any, Any], block_table: Any, keys: int, weights: Any,
                           k_start: Any, k_end: Any, top_k: int = _lib.TOP_K, *, workspace: Workspace | None = None,
                           seed: int = 0, use_graph: bool = True) -> Any:
    """Exact Top-K ids (logical key positions) with the keys read through a block table.

    ``kv_pool_pair = (kv_pool [P, page_size, 128] e4m3, scale_pool [P, page_size] fp32)``;
    ``block_table`` int32 ``[ceil(keys / page_size)]`` on the same device; ``keys`` is the logical
    number of keys.  Returns int32 ``[Q, K]`` like ``fused_index_topk`` (the workspace's output buffer; from the
    second call with the same tensors and block table on, one CUDA-graph replay).
    """

    import torch

    kv_pool, scale_pool = kv_pool_pair
    _require(top_k == _lib.TOP_K, f"top_k must be {_lib.TOP_K}")
    _require(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    _require(kv_pool.dim() == 3 and kv_pool.shape[2] == _lib.HEAD_DIM, "kv_pool must have shape [P, page_size, 128]")
    pages, page_size = int(kv_pool.shape[0]), int(kv_pool.shape[1])
    _require(page_size % TILE_KEYS == 0, "page_size must be a positive multiple of 128")
    _require(tuple(scale_pool.shape) == (pages, page_size) and scale_pool.dtype == torch.float32,
             "scale_pool must be float32 [P, page_size]")
    _require(q.dtype == torch.float8_e4m3fn and kv_pool.dtype == torch.float8_e4m3fn, "q and kv_pool must be float8_e4m3fn")
    _require(q.dim() == 3 and q.shape[1] == _lib.HEADS and q.shape[2] == _lib.HEAD_DIM, "q must have shape [Q, 64, 128]")
    rows = int(q.shape[0])
    _require(rows > 0 and 0 < keys <= _lib.MAX_KEYS, f"need Q > 0 and 0 < keys <= {_lib.MAX_KEYS}")
    _require(weights.dtype == torch.float32 and tuple(weights.shape) == (rows, _lib.HEADS), "weights must be float32 [Q, 64]")
    _require(k_start.dtype == torch.int32 and k_end.dtype == torch.int32 and tuple(k_start.shape) == (rows,)
             and tuple(k_end.shape) == (rows,), "k_start and k_end must be int32 [Q]")
    for name, tensor in (("q", q), ("kv_pool", kv_pool), ("scale_pool", scale_pool), ("weights", weights),
                         ("k_start", k_start), ("k_end", k_end), ("block_table", block_table)):
        _require(tensor.is_contiguous(), f"{name} must be contiguous")
        _require(tensor.device == q.device, f"{name} must live on the same device as q")
    _require(block_table.dtype == torch.int32 and block_table.dim() == 1, "block_table must be int32 [pages]")
    _require(int(block_table.numel()) * page_size >= keys, "block_table does not cover the keys")

    if workspace is None:
        key = (rows, keys, str(q.device), int(seed))
        workspace = _WORKSPACES.get(key)
        if workspace is None:
            workspace = make_workspace(rows, keys, q.device, seed=seed)
            _WORKSPACES[key] = workspace
    _require(workspace.rows == rows and workspace.keys == keys, "workspace was made for a different problem size")
    flat_kv = kv_pool.view(pages * page_size, _lib.HEAD_DIM)
    flat_scales = scale_pool.view(pages * page_size)
    buffers = _tile_table_buffers(workspace, int(block_table.numel()), page_size // TILE_KEYS, q.device)
    return replay_or_run(workspace, (q, flat_kv, flat_scales, weights, k_start, k_end), tile_table=buffers["tiles"],
                         use_graph=use_graph, prologue=lambda: _expand_on_device(buffers, block_table, pages),
                         key_extra=(int(block_table.data_ptr()),))


@dataclass
class PagePlan:
    """Buffers of one step's page plan (``make_page_plan``); ``plan_pages`` fills them in place.

    ``block_table``  the caller's int32 ``[B, table_pages]`` table, updated in place, -1 behind a request's pages
    ``slots``        int64 ``[rows]`` position of every new token in the pools (page * page_size + offset), -1 = padding
    ``cu_seqlens_q`` int32 ``[B+1]`` prefix sums of the new tokens
    ``lengths``      int32 ``[B]`` keys of every request after the step
    ``flat_table``   int32 ``[B * table_pages]`` the requests' pages one after another, 0 behind them
    ``k_start, k_end`` int32 ``[rows]`` causal key range of every new token in the key space of ``flat_table``
    ``pages_needed`` int32 ``[1]`` pages taken from the free list
    """

    requests: int
    table_pages: int
    rows: int
    page_size: int
    slots: Any
    cu_seqlens_q: Any
    lengths: Any
    flat_table: Any
    k_start: Any
    k_end: Any
    pages_needed: Any
    block_table: Any = None
    # checked argument blocks of this plan's sizes and buffers, without addresses
    templates: dict = field(default_factory=dict, init=False, repr=False, compare=False)

    def __setattr__(self, name: str, value: Any) -> None:
        self.__dict__[name] = value
        self.__dict__["templates"] = {}         # another size or buffer: checked again (a copy keeps the blocks that it has)


def make_page_plan(requests: int, table_pages: int, rows: int, *, page_size: int, device: Any) -> PagePlan:
    """Buffers for the page plans of steps with ``requests`` requests and at most ``rows`` new tokens.

    ``table_pages`` is the width of the block table.  ``page_size`` must be a multiple of 128.
    """

    import torch

    _require(0 < requests <= _lib.MAX_PLAN_REQUESTS, f"need 0 < requests <= {_lib.MAX_PLAN_REQUESTS}")
    _require(table_pages > 0 and 0 <= rows < 1 << 31, "need table_pages > 0 and 0 <= rows < 2^31")
    _require(page_size >= TILE_KEYS and page_size % TILE_KEYS == 0, "page_size must be a positive multiple of 128")
    _require(requests * table_pages * page_size < 1 << 31, "requests * table_pages * page_size must stay below 2^31")
    device = torch.device(device)
    _require(device.type == "cuda", "a page plan lives on a CUDA device (there is no CPU path)")

    def buffer(count, dtype=torch.int32):
        return torch.empty(count, dtype=dtype, device=device)

    return PagePlan(requests, table_pages, rows, page_size, buffer(rows, torch.int64), buffer(requests + 1), buffer(requests),
                    buffer(requests * table_pages), buffer(rows), buffer(rows), buffer(1))


def plan_pages(plan: PagePlan, block_table: Any, lengths: Any, new_tokens: Any, free_pages: Any) -> PagePlan:
    """Pages, slots and key ranges of one step, in one launch and without a host read.

    Request ``b`` holds ``lengths[b]`` tokens (int32 ``[B]``) on the first ``ceil(lengths[b] / page_size)`` pages of its
    row of ``block_table`` (int32 ``[B, table_pages]``) and gets ``new_tokens[b]`` more; the pages it lacks are taken from
    ``free_pages`` (int32 ``[F]``) in request order, the first ``pages_needed[0]`` of them.  Everything lands in the
    plan's buffers and in ``block_table`` itself; calling it again with the same arguments gives the same result.  The
    inputs must not share memory with those: ``plan.lengths`` serves as another plan's ``lengths`` (two plans in turn), not
    as its own's.

    A request that outgrows its table row, a free list that is too short (negative entries are no pages: padding) and more
    new tokens than ``rows`` are reported by ``check_serving_status``; their tokens get slot -1 (or no row), their cells -1, and
    nothing is written out of range.  A cell that an earlier plan left without a page is not reported again.

    The key space of ``flat_table``, ``k_start`` and ``k_end`` has ``requests * table_pages * page_size`` keys;
    ``fused_index_topk_paged`` takes 262144 of them at most.  A larger plan serves appends and attention; its keys cannot be
    selected from in one call.
    """

    import torch

    tensors = (block_table, lengths, new_tokens, free_pages)
    key = _lib.metadata(torch, tensors)
    template = plan.templates.get(key)
    if template is None:
        template = _lib.CallTemplate.keep(plan.templates, key, _check_plan(torch, plan, *tensors))
    block = template.fill((
        block_table.data_ptr(), lengths.data_ptr(), new_tokens.data_ptr(), free_pages.data_ptr(), plan.slots.data_ptr(),
        plan.cu_seqlens_q.data_ptr(), plan.lengths.data_ptr(), plan.flat_table.data_ptr(), plan.k_start.data_ptr(),
        plan.k_end.data_ptr(), plan.pages_needed.data_ptr()))
    _lib.launch(torch, _lib.load_library().itk_plan_pages, block, template.device, (
        block_table, plan.slots, plan.cu_seqlens_q, plan.lengths, plan.flat_table, plan.k_start, plan.k_end, plan.pages_needed))
    plan.__dict__["block_table"] = block_table
    return plan


def _check_plan(torch: Any, plan: PagePlan, block_table: Any, lengths: Any, new_tokens: Any, free_pages: Any) -> _lib.CallTemplate:
    rows, requests = plan.rows, plan.requests
    device = plan.slots.device
    for name, count, dtype in (("slots", rows, torch.int64), ("cu_seqlens_q", requests + 1, torch.int32),
                               ("lengths", requests, torch.int32), ("flat_table", requests * plan.table_pages, torch.int32),
                               ("k_start", rows, torch.int32), ("k_end", rows, torch.int32), ("pages_needed", 1, torch.int32)):
        buffer = getattr(plan, name)
        _require(buffer.is_cuda and buffer.device == device and buffer.dtype == dtype and buffer.dim() == 1
                 and buffer.shape[0] >= count and buffer.is_contiguous(),
                 f"the plan's {name} must be contiguous {dtype} with {count} entries on one CUDA device")
    for name, tensor, count in (("lengths", lengths, requests), ("new_tokens", new_tokens, requests),
                                ("free_pages", free_pages, None)):
        _require(tensor.dtype == torch.int32 and tensor.dim() == 1 and tensor.is_contiguous(), f"{name} must be contiguous int32")
        _require(tensor.device == device, f"{name} must live on the plan's device")
        _require(count is None or tensor.shape[0] == count, f"{name} must have one entry per request")
    _require(block_table.dtype == torch.int32 and tuple(block_table.shape) == (requests, plan.table_pages),
             "block_table must be int32 [requests, table_pages]")
    _require(block_table.device == device, "block_table must live on the plan's device")
    _require((block_table.stride(1) == 1 or plan.table_pages == 1) and (block_table.stride(0) >= plan.table_pages or requests == 1),
             "block_table rows must be contiguous and must not overlap")
    return _lib.CallTemplate(_lib.PagePlanArgs(
        *[None] * 11, max(block_table.stride(0), plan.table_pages), requests, plan.table_pages, plan.page_size,
        free_pages.shape[0], rows), device=device)


def append_tokens(slots: Any, kv: tuple[Any, Any], pools: tuple[Any, Any], *, index_keys: Any = None,
                  index_pools: tuple[Any, Any] | None = None) -> None:
    """Write a step's tokens to their slots of the pools, in one launch.

    ``slots`` int64 ``[T]`` (``PagePlan.slots``; tokens with a negative slot are skipped); ``kv = (k, v)`` bf16 or fp16
    ``[T, H, D]`` (D 64 or 128, any token and head strides that are multiples of 8); ``pools = (k_pool, v_pool)`` of the same
    type ``[P, page_size, H, D]``.  ``index_keys`` ``[T, 128]`` fp32 or bf16 are quantised like
    ``quantize.quantize_contiguous_index_kv`` does into ``index_pools = (kv_pool e4m3 [P, page_size, 128], scale_pool fp32
    [P, page_size])``, the pools ``fused_index_topk_paged`` reads.

    Slots must differ from one another: of two tokens with the same slot either may be kept, in parts too.  The pools share no
    memory with one another or with the tokens.  A slot behind the pool is skipped and reported by
    ``check_serving_status``.  Tensors that ask for gradients or carry forward-mode tangents are refused.
    """

    import torch

    k, v = kv
    k_pool, v_pool = pools
    tensors = (slots, k, v, k_pool, v_pool)
    if index_keys is not None or index_pools is not None:
        _require(index_keys is not None and index_pools is not None, "index_keys and index_pools go together")
        tensors += (index_keys, *index_pools)
    _lib.refuse_gradients(torch, *tensors)
    key = _lib.metadata(torch, tensors)
    template = _APPEND_TEMPLATES.get(key)
    if template is None:
        template = _lib.CallTemplate.keep(_APPEND_TEMPLATES, key, _check_append(torch, *tensors))
    addresses = [t.data_ptr() for t in tensors]
    aligned = 0
    for address in addresses[1:7]:
        aligned |= address
    _require(aligned & 15 == 0, "keys, values, index keys and their pools must be 16-byte aligned")
    _lib.launch(torch, _lib.load_library().itk_append_tokens, template.fill(addresses), template.device,
                (k_pool, v_pool) if index_pools is None else (k_pool, v_pool, *index_pools))


_APPEND_TEMPLATES: dict = {}


def _check_append(torch: Any, slots: Any, k: Any, v: Any, k_pool: Any, v_pool: Any, index_keys: Any = None, index_pool: Any = None,
                  index_scales: Any = None) -> _lib.CallTemplate:
    _require(k.is_cuda, "k must be a CUDA tensor (there is no CPU path)")
    device = k.device
    _require(k.dim() == 3 and k.shape == v.shape, "k and v must both have shape [T, H, D]")
    tokens, heads, dim = k.shape
    _require(dim in (64, 128), "the head dimension must be 64 or 128")
    _require(heads > 0 and tokens < 1 << 31, "need at least one head and less than 2^31 tokens")
    _require(k.dtype in (torch.bfloat16, torch.float16), "k and v must be bfloat16 or float16")
    _require(k_pool.dim() == 4 and k_pool.shape == v_pool.shape and tuple(k_pool.shape[2:]) == (heads, dim),
             "the pools must both have shape [P, page_size, H, D]")
    pages, page_size = k_pool.shape[0], k_pool.shape[1]
    _require(0 < pages * page_size < 1 << 31, "need 0 < pages * page_size < 2^31")
    _require(slots.dtype == torch.int64 and tuple(slots.shape) == (tokens,) and slots.is_contiguous(), "slots must be contiguous int64 [T]")
    for name, tensor in (("k", k), ("v", v), ("k_pool", k_pool), ("v_pool", v_pool)):
        _require(tensor.dtype == k.dtype, f"{name} must have the type of k")
        _require(tensor.device == device, f"{name} must live on the same device as k")
        _require(tensor.stride(-1) == 1 and all(s % 8 == 0 for s in tensor.stride()[:-1]),
                 f"{name} must be contiguous in its last dimension and 16-byte aligned in every row")
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        _require(all(s > 0 for s, n in zip(pool.stride(), pool.shape) if n > 1), f"{name} must not overlap itself")
    _require(slots.device == device, "slots must live on the same device as k")
    index_stride = index_dtype = 0
    if index_keys is not None:
        _require(index_keys.dtype in (torch.float32, torch.bfloat16) and tuple(index_keys.shape) == (tokens, _lib.HEAD_DIM),
                 "index_keys must be float32 or bfloat16 [T, 128]")
        _require((index_keys.stride(1) == 1) and index_keys.stride(0) % 8 == 0,
                 "index_keys must be contiguous in the last dimension and 16-byte aligned in every row")
        _require(index_pool.dtype == torch.float8_e4m3fn and tuple(index_pool.shape) == (pages, page_size, _lib.HEAD_DIM)
                 and index_pool.is_contiguous(), "the index pool must be contiguous float8_e4m3fn [P, page_size, 128]")
        _require(index_scales.dtype == torch.float32 and tuple(index_scales.shape) == (pages, page_size)
                 and index_scales.is_contiguous(), "the index scales must be contiguous float32 [P, page_size]")
        _require(index_keys.device == device and index_pool.device == device and index_scales.device == device,
                 "index keys and pools must live on the same device as k")
        index_stride, index_dtype = index_keys.stride(0), 1 if index_keys.dtype == torch.bfloat16 else 0
    return _lib.CallTemplate(_lib.AppendArgs(
        None, None, None, None, None, None, None, None, *k.stride()[:2], *v.stride()[:2], *k_pool.stride()[:3],
        *v_pool.stride()[:3], index_stride, index_dtype, tokens, heads, dim, pages, page_size), device=device)


check_serving_status = _lib.check_serving_status

__all__ = ["PagePlan", "append_tokens", "block_table_was_valid", "check_serving_status", "expand_block_table",
           "fused_index_topk_paged", "make_page_plan", "plan_pages", "scatter_to_pages"]
